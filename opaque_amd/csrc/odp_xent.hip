// Softmax cross entropy of x W^T over a large vocabulary, a piece of it at a time.
//
//   u = x W^T,  z = u or c tanh(u / c)
//   m_t = max_v z_tv,  s_t = sum_v exp(z_tv - m_t),  loss_t = (m_t - z_t,y(t)) + log s_t
//   p_tv = exp(z_tv - m_t) / s_t,  d_tv = g_t (p_tv - [v = y(t)]) (1 - (z_tv / c)^2)
//   dx = d W,  dW = d^T x
//
// The tokens that bear a loss are first gathered (k_xent_pick, k_xent_pack),
// so that prompts and padding cost nothing in the products.  The forward's
// tiles of logits leave the registers as their rows' maximum and sum of
// exponentials (k_xent_stats), which k_xent_losses joins, and in float32 where
// a backward pass follows and they are few enough to keep.  The backward takes
// a piece of the vocabulary at a time: d in the inputs' type, from the kept
// logits (k_xent_dkept) or from their product formed again (k_xent_dlogits),
// multiplied by W (k_xent_dx) and by x (k_xent_dw).
//
// Bounds: the products, at the matrix cores' rate from a few hundred tokens
// on; below, W's bytes.  n tokens, V x D head: 2 n V D flops for the loss, 4
// more for dx and dW (2 again where the logits are formed twice).  4096 tokens,
// 128256 x 4096 bfloat16, loss and gradients: 10.7 ms, 12.9 TFLOP at 1211
// TFLOP/s (a library product of 8192^3 runs at 1216).  One token's loss: 180 us,
// W at 5.8 TB/s.
//
// Sums, statistics and losses are float32; d is rounded to the inputs' type
// because the matrix cores take it so (a relative 2^-8 of an entry at most in
// bfloat16, of the order of the rounding of the gradients themselves).  What
// rounding takes off the target's entry, often the row's only large one, is added
// to dx in float32 (k_xent_dx_rows): alone it would leave a row of dx as far off as
// that entry.  dW takes d as it is rounded: a row of dW that is the target of one
// token is that entry times x, off by the entry's rounding beside its own, and
// rows of many tokens by about as much of their size (against 64 bits 0.0021 of
// the values for 700 tokens, 0.0017 with nothing rounded but the results).  Giving
// it back in dW's tiles, tokens found by their targets and added sixteen a step
// of the matrix cores, was right and cost more than it gives: loss and gradients
// of 777 x 32003 x 1000 297 us against 257, one token of 128256 x 4096 696 against
// 595, 4096 of them 12.2 ms against 10.8 (targets as frequent as in text).
#include <cfloat>

#include "odp_internal.h"

namespace {

#include "odp_tile.h"

constexpr float LOG2E = 1.44269504088896340736f;

// The tiles a workgroup walks, of tm x tn: XCD j (blockIdx % 8) takes the j-th
// eighth, its workgroups one tile each in turn, in groups of 8 tile rows
// walked column by column, so that the tiles one L2 serves at a time share
// operands.
struct Walk {
  int tm, tn, each, at, step;
  __device__ __forceinline__ Walk(int tm_, int tn_) : tm(tm_), tn(tn_) {
    each = (tm * tn + 7) / 8;
    at = blockIdx.x >> 3;
    step = gridDim.x >> 3;
  }
  // The tile at the walk's place; false past the end.
  __device__ __forceinline__ bool tile(int& ti, int& tj) const {
    const int p = (blockIdx.x & 7) * each + at;
    if (at >= each || p >= tm * tn) return false;
    const int per = 8 * tn, g = p / per, gm = min(tm - 8 * g, 8), r = p - g * per;
    ti = 8 * g + r % gm;
    tj = r / gm;
    return true;
  }
  __device__ __forceinline__ void next() { at += step; }
};

// Of a difference: x log2(e) formed before the subtraction would be off by the
// last place of the larger operand.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// c tanh(u / c), within 16 2^-24 of itself however large c is (c - 2 c / (1 +
// exp(2 u / c)) alone would be off by a share of c).  y = u / c below 0.8: tanh y =
// y (945 + 105 y^2 + y^4) / (945 + 420 y^2 + 15 y^4), five terms of its continued
// fraction (off by a relative 8e-9 at most), times c as u itself.  Above: (e - 1)
// / (e + 1) with e = exp(2 |y|), which is 5 or more there; tanh is 1 in float32
// from |y| = 10 on.
constexpr float CAP_NEAR = 0.8f;
__device__ __forceinline__ float softcap_near(float u, float inv_cap) {
  const float y = u * inv_cap, q = y * y;
  const float num = __builtin_fmaf(q, 105.f + q, 945.f);
  const float den = __builtin_fmaf(q, __builtin_fmaf(q, 15.f, 420.f), 945.f);
  return u * (num * __builtin_amdgcn_rcpf(den));
}
__device__ __forceinline__ float softcap_any(float u, float cap, float inv_cap) {
  const float y = __builtin_fabsf(u) * inv_cap;
  const float e = fast_exp(y > 10.f ? 20.f : 2.f * y);  // NaN stays
  const float far = __builtin_copysignf(cap * ((e - 1.f) * __builtin_amdgcn_rcpf(e + 1.f)), u);
  return y < CAP_NEAR ? softcap_near(u, inv_cap) : far;
}

// Softcaps N logits of a lane.  Most lie near (logits of up to 24 under a cap
// of 30), and where a wave's all do, the exponentials are jumped over: losses of
// 4096 x 128256 x 4096 bfloat16 take 3.61 ms (3.49 uncapped), without the jump
// 3.66 (3.43); of 4096 x 32000 x 256 156 us (116), without it 181 (106).
template <int N>
__device__ __forceinline__ void softcap_all(float (&v)[N], float cap, float inv_cap) {
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) top = fmaxf(top, __builtin_fabsf(v[k]));  // NaN is dropped, and stays in both branches
  if (__builtin_amdgcn_ballot_w64(!(top * inv_cap < CAP_NEAR)) == 0) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = softcap_near(v[k], inv_cap);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = softcap_any(v[k], cap, inv_cap);
  }
}

// ---------------------------------------------------------------------------
// Rows that bear a loss.
// ---------------------------------------------------------------------------

// What the forward leaves of a row for the backward (ODP_XENT_STAT floats): the
// maximum of its logits, the sum of exponentials below it and p(target) - 1.
// One rounded log-sum-exp would take its last place off every d, more than all
// of a nearly certain target's.
constexpr int STAT = ODP_XENT_STAT;
__device__ __forceinline__ void no_stat(float* stat, int64_t i) {
  if (stat == nullptr) return;
#pragma unroll
  for (int k = 0; k < STAT; ++k) stat[STAT * i + k] = 0.f;
}

// where[i] = the place of row i among the packed rows, -1 for a row without a
// loss, -2 for one whose target lies outside the vocabulary (loss NaN).
// keep: every row is packed, with target -1 where it bears no loss.  count[0]:
// the packed rows, count[1] (float32): the targets that are not `ignore`.
__global__ __launch_bounds__(1024) void k_xent_pick(const void* __restrict__ target, int wide, int64_t n,
                                                    int64_t vocab, int64_t ignore, int keep, int32_t* __restrict__ act,
                                                    int32_t* __restrict__ tgt, int32_t* __restrict__ where,
                                                    int32_t* __restrict__ count, float* __restrict__ losses,
                                                    float* __restrict__ stat) {
  __shared__ int32_t sums[16], other[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t base = 0, counted = 0;
  for (int64_t i0 = 0; i0 < n; i0 += 1024) {
    const int64_t i = i0 + threadIdx.x;
    int64_t t = -1;
    bool live = false;
    if (i < n) {
      t = wide ? ((const int64_t*)target)[i] : (int64_t)((const int32_t*)target)[i];
      live = t != ignore && t >= 0 && t < vocab;
      if (!live) {
        if (losses != nullptr) losses[i] = t == ignore ? 0.f : __uint_as_float(0x7fc00000u);
        no_stat(stat, i);
      }
    }
    const bool taken = keep ? i < n : live;
    const uint64_t m = __builtin_amdgcn_ballot_w64(taken);
    const uint64_t some = __builtin_amdgcn_ballot_w64(i < n && t != ignore);
    __syncthreads();
    if (lane == 0) {
      sums[wave] = __popcll(m);
      other[wave] = __popcll(some);
    }
    __syncthreads();
    int32_t before = base, all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += sums[w];
      all += sums[w];
      counted += other[w];
    }
    const int32_t k = before + __popcll(m & ((1ull << lane) - 1));
    if (taken) {
      act[k] = (int32_t)i;
      tgt[k] = live ? (int32_t)t : -1;
    }
    if (i < n) where[i] = live ? k : t == ignore ? -1 : -2;
    base += all;
  }
  if (threadIdx.x == 0) {
    count[0] = base;
    ((float*)count)[1] = (float)counted;
  }
}

// Packed rows xc [count][width] from x's rows `act`, columns past `cols` zero.
// FEW: of up to XENT_FEW tokens, which every workgroup picks from by itself
// (the first one writes k_xent_pick's results), one launch instead of two.
struct Pick {
  const void* target;
  int wide, keep;
  int64_t n, vocab, ignore;
  int32_t *act, *tgt, *where, *count;
  float *losses, *stat;
};
constexpr int XENT_FEW = 1024;
template <int DT, bool FEW>
__global__ __launch_bounds__(256) void k_xent_pack(const char* __restrict__ x, int64_t ldx, int64_t cols,
                                                   int64_t width, Pick p, int vec, char* __restrict__ xc) {
  constexpr int ES = Tile<DT, 0>::ES, V = 16 / ES;
  __shared__ int32_t picked[FEW ? XENT_FEW : 1], sums[4], other[4];
  int total = 0;
  if (FEW) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int counted = 0;
    for (int i0 = 0; i0 < (int)p.n; i0 += 256) {
      const int i = i0 + threadIdx.x;
      const bool in = i < (int)p.n;
      const int64_t t = !in ? -1 : p.wide ? ((const int64_t*)p.target)[i] : (int64_t)((const int32_t*)p.target)[i];
      const bool live = in && t != p.ignore && t >= 0 && t < p.vocab, taken = p.keep ? in : live;
      const uint64_t m = __builtin_amdgcn_ballot_w64(taken);
      const uint64_t some = __builtin_amdgcn_ballot_w64(in && t != p.ignore);
      __syncthreads();
      if (lane == 0) {
        sums[wave] = __popcll(m);
        other[wave] = __popcll(some);
      }
      __syncthreads();
      int k = total + __popcll(m & ((1ull << lane) - 1));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (w < wave) k += sums[w];
        total += sums[w];
        counted += other[w];
      }
      if (taken) picked[k] = i;
      if (blockIdx.x == 0 && in) {
        if (!live) {
          if (p.losses != nullptr) p.losses[i] = t == p.ignore ? 0.f : __uint_as_float(0x7fc00000u);
          no_stat(p.stat, i);
        }
        if (taken) {
          p.act[k] = i;
          p.tgt[k] = live ? (int32_t)t : -1;
        }
        p.where[i] = live ? k : t == p.ignore ? -1 : -2;
      }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      p.count[0] = total;
      ((float*)p.count)[1] = (float)counted;
    }
    __syncthreads();
  } else {
    total = *p.count;
  }
  const int64_t pieces = width / V;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t k = i / pieces, c = (i - k * pieces) * V;
  if (k >= total) return;
  const char* src = x + ((int64_t)(FEW ? picked[k] : p.act[k]) * ldx + c) * ES;
  u32x4_t v = {0, 0, 0, 0};
  if (vec) {
    v = *(const u32x4_t*)src;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (c + e >= cols) continue;
      if constexpr (DT == ODP_DTYPE_F32) v[e] = ((const uint32_t*)src)[e];
      else v[e / 2] |= (uint32_t)((const uint16_t*)src)[e] << (16 * (e & 1));
    }
  }
  odp_gstore((u32x4_t*)(xc + (k * width + c) * ES), v);
}

struct Xent {
  const void* xc;  // [count][width]
  const void* w;   // [vocab][ldw]
  int64_t ldw, vocab, width, n;
  const int32_t* count;
  const int32_t* act;
  const int32_t* tgt;
  float cap, inv_cap;  // softcap and 1 / softcap (cap 0: none)
};

// ---------------------------------------------------------------------------
// Forward: per (row, tile of the vocabulary) the maximum and the sum of
// exponentials below it, and each row's target logit.
//
// A softmax in one pass over the logits: m = max(m1, m2), s = s1 exp(m1 - m) +
// s2 exp(m2 - m) joins lanes, waves and, in k_xent_losses, tiles.  Workgroups
// stay on their CU and walk tiles, so that the next tile's first loads pass
// beside the exponentials of the last (4096 x 128256 x 4096 bfloat16: 3.46 ms,
// 1240 TFLOP/s, against 3.60 with a workgroup a tile; matrix cores busy 70 % of
// the time, no LDS conflicts; 3.7 ms and 63 % with 2.1 GB of logits stored).  47
// tokens: 22 us for 32000 x 2048 (6.0 TB/s); one: 175 us for 128256 x 4096 (6.0
// TB/s).  float32, 1024 x 50257 x 768: 663 us, 119 TFLOP/s.
// ---------------------------------------------------------------------------
template <int DT, int S, bool CAP, bool WHOLE>
__device__ __forceinline__ void stats_tile(const Xent& p, const typename Tile<DT, S>::Acc& acc, int cnt, int64_t o0,
                                           int64_t n0, const int32_t (&tgt)[Tile<DT, S>::BI], float* red,
                                           float* __restrict__ ztgt, float* __restrict__ logits, int64_t ldl) {
  using T = Tile<DT, S>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = T::wm(wave), wn = T::wn(wave);
  // Columns of this lane are c0 + 16 j + e of the tile; `edge` columns of it exist.
  const int c0 = wn + t_col(0), edge = (int)min((int64_t)T::NT, p.vocab - n0);
  static_for<T::BI>([&](auto ii) __attribute__((always_inline)) {
    constexpr int i = decltype(ii)::value;
    // The row's target, counted from c0 (no column of the lane for none here).
    const int at = tgt[i] - (int)n0 - c0;
    float z[T::BJ][4], m = -INFINITY, zt = 0.f;
    bool here = false;
#pragma unroll
    for (int j = 0; j < T::BJ; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) z[j][e] = acc[i][j][e];
      if (CAP) softcap_all(z[j], p.cap, p.inv_cap);
    }
#pragma unroll
    for (int j = 0; j < T::BJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = z[j][e];
        const bool hit = at == 16 * j + e;
        zt = hit ? v : zt;
        here |= hit;
        z[j][e] = WHOLE || c0 + 16 * j + e < edge ? v : -INFINITY;
        m = fmaxf(m, z[j][e]);
      }
    if (here) ztgt[o0 + wm + t_row(i)] = zt;
    if (logits != nullptr && o0 + wm + t_row(i) < cnt) {
      float* to = logits + (o0 + wm + t_row(i)) * ldl + n0 + c0;
#pragma unroll
      for (int j = 0; j < T::BJ; ++j) odp_gstore((f32x4_t*)(to + 16 * j), f32x4_t{z[j][0], z[j][1], z[j][2], z[j][3]});
    }
    const float ms = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < T::BJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s += fast_exp(z[j][e] - ms);
    // The row's other columns of this wave: lanes 16, 32 and 48 further on.
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) {
      const float m2 = __shfl_xor(m, off), s2 = __shfl_xor(s, off);
      const float mm = fmaxf(m, m2), ref = mm == -INFINITY ? 0.f : mm;
      s = s * fast_exp(m - ref) + s2 * fast_exp(m2 - ref);
      m = mm;
    }
    if (lane < 16) {
      float* r = red + 2 * (wave / T::WR * T::OT + wm + t_row(i));
      r[0] = m;
      r[1] = s;
    }
    __builtin_amdgcn_sched_barrier(0);
  });
}

template <int DT, int S, bool CAP>
__global__ __launch_bounds__((Tile<DT, S>::THREADS), 2) void k_xent_stats(Xent p, float* __restrict__ pmax,
                                                                     float* __restrict__ psum,
                                                                     float* __restrict__ ztgt,
                                                                     float* __restrict__ logits, int64_t ldl) {
  using T = Tile<DT, S>;
  __shared__ float red[T::WC * T::OT * 2];  // [waves across n][rows][maximum, sum]
  const int cnt = *(const ODP_CONST int32_t*)p.count;
  Walk walk((cnt + T::OT - 1) / T::OT, (int)((p.vocab + T::NT - 1) / T::NT));
  const int wm = T::wm(threadIdx.x >> 6);
  Product<DT, S, true, true> prod;
  int ti, tj;
  auto begin = [&]() {
    prod.begin(Operand{p.xc, p.width, (int64_t)ti * T::OT, cnt}, Operand{p.w, p.ldw, (int64_t)tj * T::NT, p.vocab},
               (int32_t)p.width);
  };
  bool more = walk.tile(ti, tj);
  if (more) begin();
  while (more) {
    const int64_t o0 = (int64_t)ti * T::OT, n0 = (int64_t)tj * T::NT;
    typename T::Acc acc;
    prod.run(acc);
    int32_t tgt[T::BI];
#pragma unroll
    for (int i = 0; i < T::BI; ++i) tgt[i] = o0 + wm + t_row(i) < cnt ? p.tgt[o0 + wm + t_row(i)] : -1;
    const int column = tj;
    walk.next();
    more = walk.tile(ti, tj);
    if (more) begin();
    if (n0 + T::NT <= p.vocab) stats_tile<DT, S, CAP, true>(p, acc, cnt, o0, n0, tgt, red, ztgt, logits, ldl);
    else stats_tile<DT, S, CAP, false>(p, acc, cnt, o0, n0, tgt, red, ztgt, logits, ldl);
    __syncthreads();
    for (int r = threadIdx.x; r < T::OT; r += T::THREADS) {
      if (o0 + r >= cnt) break;
      float m = -INFINITY, s = 0.f;
#pragma unroll
      for (int w = 0; w < T::WC; ++w) m = fmaxf(m, red[2 * (w * T::OT + r)]);
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int w = 0; w < T::WC; ++w)
        s += red[2 * (w * T::OT + r) + 1] * fast_exp(red[2 * (w * T::OT + r)] - ref);
      pmax[(int64_t)column * p.n + o0 + r] = m;
      psum[(int64_t)column * p.n + o0 + r] = s;
    }
  }
}

// Joins the tiles' statistics: R rows a workgroup, 256 / R threads each.  Bound
// by latency: 4 us for one row of 1002 tiles, 11 us for 4096 of 501.
template <int R>
__global__ __launch_bounds__(256) void k_xent_losses(const float* __restrict__ pmax, const float* __restrict__ psum,
                                                     const float* __restrict__ ztgt, int tiles, int64_t n,
                                                     const int32_t* __restrict__ count,
                                                     const int32_t* __restrict__ act, const int32_t* __restrict__ tgt,
                                                     float* __restrict__ losses, float* __restrict__ stat) {
  constexpr int Q = 256 / R;
  __shared__ float rm[Q][R + 1], rs[Q][R + 1];
  const int r = threadIdx.x % R, q = threadIdx.x / R;
  const int64_t row = (int64_t)blockIdx.x * R + r;
  const bool on = row < *count;
  float m = -INFINITY, s = 0.f;
  if (on) {
#pragma unroll 4
    for (int t = q; t < tiles; t += Q) {
      const float m2 = pmax[(int64_t)t * n + row], s2 = psum[(int64_t)t * n + row];
      const float mm = fmaxf(m, m2), ref = mm == -INFINITY ? 0.f : mm;
      s = s * fast_exp(m - ref) + s2 * fast_exp(m2 - ref);
      m = mm;
    }
  }
  rm[q][r] = m;
  rs[q][r] = s;
  __syncthreads();
  // Halves joined in one order.
  for (int h = Q / 2; h > 0; h /= 2) {
    if (q < h) {
      const float m2 = rm[q + h][r], s2 = rs[q + h][r];
      const float mm = fmaxf(m, m2), ref = mm == -INFINITY ? 0.f : mm;
      rs[q][r] = s = s * fast_exp(m - ref) + s2 * fast_exp(m2 - ref);
      rm[q][r] = m = mm;
    }
    __syncthreads();
  }
  if (q != 0 || !on) return;
  const float ref = m == -INFINITY ? 0.f : m;
  // Not the log-sum-exp less the target's logit: a small loss would keep little of its bits.
  const float loss = tgt[row] >= 0 ? (ref - ztgt[row]) + logf(s) : 0.f;
  const int64_t at = act[row];
  float* to = stat + STAT * at;
  to[0] = ref;
  to[1] = s;
  to[2] = expm1f(-loss);
  if (tgt[row] >= 0) losses[at] = loss;
}

// The sum of the losses (in fp64, in one order), over *over where it is given.
__global__ __launch_bounds__(1024) void k_xent_reduce(const float* __restrict__ losses, int64_t n,
                                                      const float* __restrict__ over, float* __restrict__ out) {
  __shared__ double red[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += (double)losses[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) s += red[w];
  *out = over != nullptr ? (float)s / *over : (float)s;
}

// ---------------------------------------------------------------------------
// Stores of a tile in the operands' type: rows o (of `rows`) of pitch ld from
// row o0, columns n0 + .. below `cols`, val(i, j) the blocks' entries.  16-bit
// tiles go through LDS beside the ring, 32 rows of a wave at a time, so that
// rows leave in 16-byte pieces.
// ---------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ uint16_t* t_staged() {
  __shared__ __attribute__((aligned(16))) uint16_t s[N];
  return s;
}
template <int DT, int S, typename Val>
__device__ __forceinline__ void t_store(void* out, int64_t ld, int64_t o0, int64_t rows, int64_t n0, int64_t cols,
                                        Val val) {
  using T = Tile<DT, S>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = T::wm(wave), wn = T::wn(wave);
  if constexpr (DT == ODP_DTYPE_F32) {
    static_for<T::BI * T::BJ>([&](auto q) __attribute__((always_inline)) {
      constexpr int i = decltype(q)::value / T::BJ, j = decltype(q)::value % T::BJ;
      const int64_t o = o0 + wm + t_row(i), n = n0 + wn + t_col(j);
      const f32x4_t v = val(Idx<i>{}, Idx<j>{});
      if (o < rows && n < cols) odp_gstore((f32x4_t*)((float*)out + o * ld + n), v);
      __builtin_amdgcn_sched_barrier(0);
    });
  } else {
    constexpr int PART = 32 * T::WN;  // elements of a wave's 32 rows
    uint16_t* stg = t_staged<T::WAVES * PART>() + wave * PART;
    static_for<T::BI / 2>([&](auto hh) __attribute__((always_inline)) {
      constexpr int h = decltype(hh)::value;
      static_for<2 * T::BJ>([&](auto q) __attribute__((always_inline)) {
        constexpr int ib = decltype(q)::value / T::BJ, j = decltype(q)::value % T::BJ;
        const f32x4_t v = val(Idx<2 * h + ib>{}, Idx<j>{});
        const int r = t_row(ib), c = t_col(j);
        *(u32x2_alias_t*)&stg[r * T::WN + 8 * ((c >> 3) ^ (r & 7)) + (c & 7)] =
            u32x2_t{odp_f2bf2(v[0], v[1]), odp_f2bf2(v[2], v[3])};
        __builtin_amdgcn_sched_barrier(0);
      });
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = 8 * k + (lane >> 3), c = lane & 7;
        const u32x4_t v = *(const u32x4_alias_t*)&stg[r * T::WN + 8 * (c ^ (r & 7))];
        const int64_t o = o0 + wm + 32 * h + r, n = n0 + wn + 8 * c;
        if (o < rows && n < cols) odp_gstore((u32x4_t*)((uint16_t*)out + o * ld + n), v);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  }
}

// ---------------------------------------------------------------------------
// Backward: d of the vocabulary's columns [v0, v0 + vc), [count][ldd], with
// zeros up to ldd (a multiple of the tile).  The forward's product again:
// 4096 x 64256 x 4096 bfloat16 1.80 ms, 1195 TFLOP/s.
// ---------------------------------------------------------------------------
template <int DT, int S>
struct DRows {  // of a lane's rows of a tile
  float m[Tile<DT, S>::BI];   // maximum of the logits
  float gs[Tile<DT, S>::BI];  // gradient over the sum of exponentials below it: g p = gs exp(z - m)
  float gt[Tile<DT, S>::BI];  // gradient times p(target) - 1
  int32_t tgt[Tile<DT, S>::BI];  // target less the piece's first column
};
constexpr int32_t NO_LOSS = INT32_MIN;  // a target may lie anywhere beside the piece

template <int DT, int S, bool CAP, bool WHOLE>
__device__ __forceinline__ void dlogits_tile(const Xent& p, const typename Tile<DT, S>::Acc& acc, const DRows<DT, S>& rows,
                                             int cnt, int64_t o0, int64_t n0, int64_t vc, void* dl, int64_t ldd,
                                             float* __restrict__ rest) {
  using T = Tile<DT, S>;
  const int wm = T::wm(threadIdx.x >> 6), wn = T::wn(threadIdx.x >> 6);
  // Columns of this lane are c0 + 16 j + e of the tile; `edge` columns of it exist.
  const int c0 = wn + t_col(0), edge = (int)min((int64_t)T::NT, vc - n0);
  t_store<DT, S>(dl, ldd, o0, cnt, n0, ldd, [&](auto ii, auto jj) __attribute__((always_inline)) {
    constexpr int i = decltype(ii)::value, j = decltype(jj)::value;
    const int at = (int)((uint32_t)rows.tgt[i] - (uint32_t)n0 - (uint32_t)c0);
    const bool live = rows.tgt[i] != NO_LOSS;
    f32x4_t d;
    float over = 0.f, zs[4];
    bool here = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) zs[e] = acc[i][j][e];
    if (CAP) softcap_all(zs, p.cap, p.inv_cap);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float z = zs[e];
      const bool hit = at == 16 * j + e;
      here |= hit;
      float q = hit ? rows.gt[i] : fast_exp(z - rows.m[i]) * rows.gs[i];
      if (CAP) {
        const float y = z * p.inv_cap;
        q *= 1.f - y * y;
      }
      d[e] = live && (WHOLE || c0 + 16 * j + e < edge) ? q : 0.f;
      if (DT == ODP_DTYPE_BF16) over = hit ? q - odp_round_bf16(q) : over;
    }
    if (DT == ODP_DTYPE_BF16 && here && live) rest[o0 + wm + t_row(i)] = over;
    return d;
  });
}

template <int DT, int S, bool CAP>
__global__ __launch_bounds__((Tile<DT, S>::THREADS), (DT == ODP_DTYPE_BF16 && S == 1 ? 1 : 2)) void k_xent_dlogits(Xent p, int64_t v0, int64_t vc,
                                                                       const float* __restrict__ stat,
                                                                       const float* __restrict__ g, int g_stride,
                                                                       const float* __restrict__ over, void* dl,
                                                                       int64_t ldd, float* __restrict__ rest) {
  using T = Tile<DT, S>;
  const int cnt = *(const ODP_CONST int32_t*)p.count;
  Walk walk((cnt + T::OT - 1) / T::OT, (int)(ldd / T::NT));
  const int wm = T::wm(threadIdx.x >> 6);
  const void* w = (const char*)p.w + v0 * p.ldw * T::ES;
  const float part = over != nullptr ? *over : 1.f;
  Product<DT, S, true, true> prod;
  int ti, tj;
  auto begin = [&]() {
    prod.begin(Operand{p.xc, p.width, (int64_t)ti * T::OT, cnt}, Operand{w, p.ldw, (int64_t)tj * T::NT, vc},
               (int32_t)p.width);
  };
  bool more = walk.tile(ti, tj);
  if (more) begin();
  while (more) {
    const int64_t o0 = (int64_t)ti * T::OT, n0 = (int64_t)tj * T::NT;
    typename T::Acc acc;
    prod.run(acc);
    DRows<DT, S> rows;
#pragma unroll
    for (int i = 0; i < T::BI; ++i) {
      const int64_t o = o0 + wm + t_row(i);
      const int32_t t = o < cnt ? p.tgt[o] : -1;
      const int64_t row = o < cnt ? p.act[o] : 0;
      const float gr = t >= 0 ? g[row * g_stride] / part : 0.f;
      rows.m[i] = t >= 0 ? stat[STAT * row] : 0.f;
      rows.gs[i] = t >= 0 ? gr / stat[STAT * row + 1] : 0.f;
      rows.gt[i] = t >= 0 ? gr * stat[STAT * row + 2] : 0.f;
      rows.tgt[i] = t >= 0 ? t - (int32_t)v0 : NO_LOSS;
    }
    walk.next();
    more = walk.tile(ti, tj);
    if (more) begin();
    if (n0 + T::NT <= vc) dlogits_tile<DT, S, CAP, true>(p, acc, rows, cnt, o0, n0, vc, dl, ldd, rest);
    else dlogits_tile<DT, S, CAP, false>(p, acc, rows, cnt, o0, n0, vc, dl, ldd, rest);
  }
}

// The same from kept logits (pitch ldl): a workgroup takes KEPT_COLS columns of
// a row, a thread 16 bytes of d at a time, all of its loads in flight.  Bound
// by HBM: 4096 x 64256 to bfloat16 277 us, 5.7 TB/s; 1024 x 50257 in float32 61
// us, 6.7 TB/s (part of it still in the cache).
constexpr int KEPT_COLS = 4096;
template <int DT, bool CAP>
__global__ __launch_bounds__(256) void k_xent_dkept(Xent p, const float* __restrict__ logits, int64_t ldl, int64_t v0,
                                                    int64_t vc, int parts, const float* __restrict__ stat,
                                                    const float* __restrict__ g, int g_stride,
                                                    const float* __restrict__ over, char* __restrict__ dl, int64_t ldd,
                                                    float* __restrict__ rest) {
  constexpr int ES = Tile<DT, 0>::ES, V = 16 / ES, ROUNDS = KEPT_COLS / 256 / V;
  const int64_t k = blockIdx.x / (uint32_t)parts;
  const int c0 = (int)(blockIdx.x - (uint32_t)k * (uint32_t)parts) * KEPT_COLS;
  if (k >= *(const ODP_CONST int32_t*)p.count) return;
  const float* from = logits + k * ldl + v0;
  f32x4_t z[ROUNDS][V / 4];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int c = c0 + (r * 256 + (int)threadIdx.x) * V;
#pragma unroll
    for (int h = 0; h < V / 4; ++h)
      if (c < ldd) z[r][h] = __builtin_nontemporal_load((const ODP_GMEM f32x4_t*)(const ODP_GMEM void*)(from + c + 4 * h));
  }
  const int32_t t = p.tgt[k];
  const int64_t row = p.act[k];
  const int at = t - (int)v0;
  const float part = over != nullptr ? *over : 1.f, gr = t >= 0 ? g[row * g_stride] / part : 0.f;
  const float m = t >= 0 ? stat[STAT * row] : 0.f, gs = t >= 0 ? gr / stat[STAT * row + 1] : 0.f;
  const float gt = t >= 0 ? gr * stat[STAT * row + 2] : 0.f;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int c = c0 + (r * 256 + (int)threadIdx.x) * V;
    if (c >= ldd) return;
    float d[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float y = z[r][e / 4][e % 4];
      const bool hit = at == c + e;
      float q = hit ? gt : fast_exp(y - m) * gs;
      if (CAP) q *= 1.f - y * p.inv_cap * (y * p.inv_cap);
      d[e] = t >= 0 && c + e < vc ? q : 0.f;
      if (DT == ODP_DTYPE_BF16 && hit && t >= 0) rest[k] = q - odp_round_bf16(q);
    }
    char* to = dl + (k * ldd + c) * ES;
    if constexpr (DT == ODP_DTYPE_F32) {
      odp_gstore((f32x4_t*)to, f32x4_t{d[0], d[1], d[2], d[3]});
    } else {
      odp_gstore((u32x4_t*)to, u32x4_t{odp_f2bf2(d[0], d[1]), odp_f2bf2(d[2], d[3]), odp_f2bf2(d[4], d[5]),
                                       odp_f2bf2(d[6], d[7])});
    }
  }
}

// How many slices of the contraction each tile of dx is split into: the
// fewest of 1 .. DX_SPLIT with which the workgroups fill the 256 CUs' rounds
// best, as far as the slots (`cap` tiles) and slices of 16 steps go.  32 is where
// no measured head loses; 64 would gain on heads of few columns and cost on
// 32000 x 2048.  dx, us, in up to 16, 32 and 64 slices: bfloat16, 128 tokens, 128256 x 512 139, 78 and 48,
// 32000 x 2048 44, 31 and 43; 777 tokens, 32000 x 2048 103, 102 and 101; float32,
// one token, 50257 x 768 103, 56 and 48 (64 slices cost dx_rows 4 us more).
constexpr int DX_SPLIT = 32;
__host__ __device__ inline int dx_split(int tiles, int cap, int64_t steps) {
  int best = 1, rounds = (tiles + 255) / 256;
  for (int s = 2; s <= DX_SPLIT && s * tiles <= cap && steps >= 16 * s; ++s) {
    const int r = (s * tiles + 255) / 256;
    if (r * best < rounds * s) best = s, rounds = r;
  }
  return best;
}

// Slot s of dx [slices][count][width] (float32) (+)= d[:, slice s] W[slice s].
// W's rows are the contraction: they are staged as they lie and transposed by
// the LDS reads.  4096 x 4096 over 64256: 1.56-1.59 ms, 1360-1380 TFLOP/s;
// float32, 1024 x 768 over 50257 in 5 slices: 693 us, 114 TFLOP/s.
template <int DT, int S>
__global__ __launch_bounds__((Tile<DT, S>::THREADS), 2) void k_xent_dx(Xent p, int64_t v0, int64_t vc, int64_t piece,
                                                                     const void* dl, int64_t ldd, int cap, int first,
                                                                     float* __restrict__ slots) {
  using T = Tile<DT, S>;
  const int cnt = *(const ODP_CONST int32_t*)p.count;
  const int tm = (cnt + T::OT - 1) / T::OT, tn = (int)((p.width + T::NT - 1) / T::NT);
  if (tm == 0) return;
  const int split = dx_split(tm * tn, cap, piece / T::EK);
  int ti, tj;
  if (!Walk(tm, tn * split).tile(ti, tj)) return;  // a workgroup per tile
  const int s = tj / tn;
  tj -= s * tn;
  const int64_t o0 = (int64_t)ti * T::OT, n0 = (int64_t)tj * T::NT;
  // Slices of whole steps, the same for every piece.
  const int64_t per = (piece / T::EK + split - 1) / split * T::EK, k0 = s * per;
  const int32_t kn = (int32_t)max((int64_t)0, min(per, vc - k0));
  if (kn == 0 && !first) return;
  typename T::Acc acc;
  Product<DT, S, true, false> prod;
  prod.begin(Operand{(const char*)dl + k0 * T::ES, ldd, o0, cnt},
             Operand{(const char*)p.w + (v0 + k0) * p.ldw * T::ES, p.ldw, n0, p.width}, kn);
  prod.run(acc);
  const int wave = threadIdx.x >> 6;
  const int wm = T::wm(wave), wn = T::wn(wave);
  float* out = slots + (int64_t)s * cnt * p.width;
  static_for<T::BI * T::BJ>([&](auto q) __attribute__((always_inline)) {
    constexpr int i = decltype(q)::value / T::BJ, j = decltype(q)::value % T::BJ;
    const int64_t o = o0 + wm + t_row(i), n = n0 + wn + t_col(j);
    if (o < cnt && n < p.width) {
      f32x4_t* at = (f32x4_t*)(out + o * p.width + n);
      f32x4_t v = acc[i][j];
      if (!first) v = v + *(const ODP_GMEM f32x4_t*)(const ODP_GMEM void*)at;
      odp_gstore(at, v);
    }
    __builtin_amdgcn_sched_barrier(0);
  });
}

// dx [n][cols] in the inputs' type from the slots; rows without a loss are
// zero, rows with a target outside the vocabulary NaN.
template <int DT>
__global__ __launch_bounds__(256) void k_xent_dx_rows(const float* __restrict__ slots, int64_t width, int64_t cols,
                                                      int64_t n, const int32_t* __restrict__ count,
                                                      const int32_t* __restrict__ where, int ot, int tn, int cap,
                                                      int64_t steps, const float* __restrict__ rest,
                                                      const int32_t* __restrict__ tgt, const char* __restrict__ w,
                                                      int64_t ldw, void* __restrict__ dx) {
  const int64_t quads = width / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / quads, c = (i - row * quads) * 4;
  if (row >= n) return;
  const int cnt = *count, k = where[row];
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  if (k >= 0) {
    const int split = dx_split((cnt + ot - 1) / ot * tn, cap, steps);
    const float* at = slots + (int64_t)k * width + c;
    v = *(const f32x4_t*)at;
#pragma unroll 4
    for (int s = 1; s < split; ++s) v = v + *(const f32x4_t*)(at + (int64_t)s * cnt * width);
    if (DT == ODP_DTYPE_BF16 && tgt[k] >= 0) {
      const u32x2_t h = *(const u32x2_t*)(w + 2 * (tgt[k] * ldw + c));
      const float r = rest[k];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(r, odp_bf2f((uint16_t)(h[e / 2] >> (16 * (e & 1)))), v[e]);
    }
  } else if (k == -2) {
    v[0] = v[1] = v[2] = v[3] = __uint_as_float(0x7fc00000u);
  }
  if (cols == width) {
    if constexpr (DT == ODP_DTYPE_F32) odp_gstore((f32x4_t*)((float*)dx + row * cols + c), v);
    else odp_gstore((u32x2_t*)((uint16_t*)dx + row * cols + c), u32x2_t{odp_f2bf2(v[0], v[1]), odp_f2bf2(v[2], v[3])});
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < cols) odp_store_from_float(dx, row * cols + c + e, DT, v[e]);
}

// dW rows [0, vc) of pitch lddw = d^T x, the contraction over the tokens.
// 64256 x 4096 over 4096 tokens: 1.66 ms, 1300 TFLOP/s.
template <int DT>
__global__ __launch_bounds__((Tile<DT, 0>::THREADS), 2) void k_xent_dw(Xent p, int64_t vc, const void* dl, int64_t ldd,
                                                                  void* dw, int64_t lddw) {
  using T = Tile<DT, 0>;
  const int cnt = *(const ODP_CONST int32_t*)p.count;
  Walk walk((int)((vc + T::OT - 1) / T::OT), (int)((p.width + T::NT - 1) / T::NT));
  Product<DT, 0, false, false> prod;
  int ti, tj;
  auto begin = [&]() {
    prod.begin(Operand{dl, ldd, (int64_t)ti * T::OT, ldd}, Operand{p.xc, p.width, (int64_t)tj * T::NT, p.width}, cnt);
  };
  bool more = walk.tile(ti, tj);
  if (more) begin();
  while (more) {
    const int64_t o0 = (int64_t)ti * T::OT, n0 = (int64_t)tj * T::NT;
    typename T::Acc acc;
    prod.run(acc);
    walk.next();
    more = walk.tile(ti, tj);
    if (more) begin();
    t_store<DT, 0>(dw, lddw, o0, vc, n0, p.width, [&](auto ii, auto jj) __attribute__((always_inline)) {
      return acc[decltype(ii)::value][decltype(jj)::value];
    });
  }
}

// A slice of the tokens of each tile of dW into its slot [vc][width] (float32):
// few tiles of many tokens leave most of the CUs idle otherwise (us, whole and
// in slices: 100 x 64 float32 over 65536 tokens 3877 and 41, 5000 x 512 bfloat16
// over 16384 298 and 87).
template <int DT>
__global__ __launch_bounds__((Tile<DT, 0>::THREADS), 2) void k_xent_dw_part(Xent p, int64_t vc, const void* dl,
                                                                            int64_t ldd, int split,
                                                                            float* __restrict__ slots) {
  using T = Tile<DT, 0>;
  const int cnt = *(const ODP_CONST int32_t*)p.count;
  const int tm = (int)((vc + T::OT - 1) / T::OT), tn = (int)((p.width + T::NT - 1) / T::NT);
  int ti, tj;
  if (!Walk(tm, tn * split).tile(ti, tj)) return;  // a workgroup per tile and slice
  const int s = tj / tn;
  tj -= s * tn;
  const int64_t o0 = (int64_t)ti * T::OT, n0 = (int64_t)tj * T::NT;
  const int64_t per = ((int64_t)cnt + (int64_t)T::EK * split - 1) / ((int64_t)T::EK * split) * T::EK;
  const int64_t k0 = min((int64_t)cnt, s * per);
  typename T::Acc acc;
  Product<DT, 0, false, false> prod;
  prod.begin(Operand{(const char*)dl + k0 * ldd * T::ES, ldd, o0, ldd},
             Operand{(const char*)p.xc + k0 * p.width * T::ES, p.width, n0, p.width}, (int32_t)min(per, cnt - k0));
  prod.run(acc);
  const int wave = threadIdx.x >> 6;
  const int wm = T::wm(wave), wn = T::wn(wave);
  float* out = slots + s * vc * p.width;
  static_for<T::BI * T::BJ>([&](auto q) __attribute__((always_inline)) {
    constexpr int i = decltype(q)::value / T::BJ, j = decltype(q)::value % T::BJ;
    const int64_t o = o0 + wm + t_row(i), n = n0 + wn + t_col(j);
    if (o < vc && n < p.width) odp_gstore((f32x4_t*)(out + o * p.width + n), acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  });
}

// dW from the slots, added in one order: Q threads each take every Q-th slot.
template <int DT, int Q>
__global__ __launch_bounds__(256) void k_xent_dw_rows(const float* __restrict__ slots, int split, int64_t quads,
                                                      void* __restrict__ dw) {
  constexpr int R = 256 / Q;
  __shared__ f32x4_t part[Q][R];
  const int r = threadIdx.x % R, q = threadIdx.x / R;
  const int64_t i = (int64_t)blockIdx.x * R + r;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  if (i < quads) {
#pragma unroll 8
    for (int s = q; s < split; s += Q) v = v + *((const f32x4_t*)slots + s * quads + i);
  }
  if constexpr (Q > 1) {
    part[q][r] = v;
    __syncthreads();
    if (q != 0) return;
    for (int k = 1; k < Q; ++k) v = v + part[k][r];
  }
  if (i >= quads) return;
  if constexpr (DT == ODP_DTYPE_F32) odp_gstore((f32x4_t*)dw + i, v);
  else odp_gstore((u32x2_t*)dw + i, u32x2_t{odp_f2bf2(v[0], v[1]), odp_f2bf2(v[2], v[3])});
}

int check_xent(const char* what, int dtype, int64_t n, int64_t width, int64_t ldw, int64_t vocab) {
  if (dtype != ODP_DTYPE_F32 && dtype != ODP_DTYPE_BF16) {
    odp_set_error("%s: rows must be float32 or bfloat16 (dtype %d)", what, dtype);
    return ODP_ERR_UNSUPPORTED;
  }
  const int64_t per = dtype == ODP_DTYPE_F32 ? 4 : 8;
  if (n < 0 || n >= ((int64_t)1 << 31) - 512 || width <= 0 || width % per != 0 || width >= ODP_XENT_WIDE ||
      ldw < width || ldw % per != 0 || ldw >= ODP_XENT_WIDE || vocab <= 0 || vocab >= ((int64_t)1 << 31) - 512) {
    odp_set_error("%s: invalid sizes (n %lld, width %lld, pitch %lld, vocab %lld)", what, (long long)n,
                  (long long)width, (long long)ldw, (long long)vocab);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  return ODP_OK;
}

int check_cap(const char* what, float softcap) {
  if (softcap == 0.f || (softcap >= FLT_MIN && softcap <= FLT_MAX)) return ODP_OK;
  odp_set_error("%s: softcap %g is neither 0 nor a positive normal number", what, (double)softcap);
  return ODP_ERR_INVALID_ARGUMENT;
}

// Columns a piece of d is padded to, and the edges of the tiles of a kind (Tile's S).
int tile_edge(int dtype) { return dtype == ODP_DTYPE_F32 ? 128 : 256; }
int tile_rows(int dtype, int kind) { return kind == 1 ? 64 : kind == 2 ? 128 : kind == 3 ? 32 : tile_edge(dtype); }
int tile_cols(int dtype, int kind) { return kind == 1 || kind == 3 ? 128 : tile_edge(dtype); }

static_assert(2 * 255 * ODP_XENT_PIECE < T_OOB && 4 * 127 * ODP_XENT_PIECE < T_OOB, "offsets of a tile's rows of d");

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether a product of n rows takes the tiles of few rows.  64 in bfloat16: past
// it the large heads lose a third, while heads that fit the cache would gain an
// eighth up to 128.  Rules go by all n tokens, since the host does not know how
// many bear a loss.  Loss and dx, us, with the small tiles and the large ones: bfloat16, 32000 x 2048, 64 tokens 69
// and 87, 128 84 and 96, 192 109 and 104, 256 130 and 118; 128256 x 4096, 64
// tokens 440 and 421, 65 605 and 409 (W past the cache is read once a row of
// tiles); float32, 50257 x 768, 64 tokens 143 and 231, 256 364 and 394, 384 542
// and 524.
bool few_rows(int dtype, int64_t n) { return n <= (dtype == ODP_DTYPE_F32 ? 256 : 64); }

// The tiles of few rows of n, else the large ones.  float32, 50257 x 768,
// 16 tokens: 42 us with tiles of 32 rows, 61 with 64.
int few_kind(int dtype, int64_t n) { return !few_rows(dtype, n) ? 0 : dtype == ODP_DTYPE_F32 && n <= 32 ? 3 : 1; }

// The tiles (Tile's S) of a product of n rows and `cols` columns.  A tile of
// 128 rows takes about 0.7 of the time of one of 256: bfloat16 takes those
// where that leaves fewer of the larger ones' times, counting whole rounds of
// the CUs.  Loss and dx, us, with 128 and with 256 rows: 32000 x 2048, 128
// tokens 96 and 106, 256 118 and 136, 512 189 and 181; 128256 x 4096, 128
// tokens 469 and 491, 160 568 and 510; 50257 x 768, 600 tokens 187 and 196.
int tile_kind(int dtype, int64_t n, int64_t cols) {
  if (few_rows(dtype, n)) return few_kind(dtype, n);
  if (dtype == ODP_DTYPE_F32) return 0;
  const int64_t tn = up(cols, 256);
  return up(up(n, 128) * tn, 256) * 7 < up(up(n, 256) * tn, 256) * 10 ? 2 : 0;
}

// Whether logits are worth keeping for the backward: 8 bytes of traffic each
// against 2 width operations, or W's share of reading it again where the rows
// are few.  Loss and gradients, us, formed again and kept: bfloat16, 4096 x
// 32000, width 256 439 and 519, 640 749 and 768, 768 815 and 802, 1024 971 and
// 902; 64 x 128256, width 256 106 and 98; float32, 4096 x 32000, width 64 973 and
// 977, 128 1213 and 1092.
bool keeps(int dtype, int64_t n, int64_t width) {
  return width >= (dtype == ODP_DTYPE_F32 ? 128 : 768) || width >= 4 * n;
}

// Workgroups that walk a tm x tn grid of tiles: as many as the CUs hold at a
// time (one of the large bfloat16 tiles, two of the others), or one a tile (`all`).
int grid_of(const char* what, int dtype, int kind, int64_t tm, int64_t tn, bool all, unsigned& blocks) {
  const int64_t b = (tm * tn + 7) / 8 * 8, held = dtype == ODP_DTYPE_F32 || kind == 1 ? 512 : 256;
  if (b >= (int64_t)1 << 31) {
    odp_set_error("%s: %lld tiles", what, (long long)b);
    return ODP_ERR_UNSUPPORTED;
  }
  blocks = (unsigned)(all || b < held ? b : held);
  return ODP_OK;
}

Xent xent_of(const void* xc, const void* w, int64_t ldw, int64_t vocab, int64_t width, int64_t n,
             const int32_t* count, const int32_t* act, const int32_t* tgt, float cap) {
  return Xent{xc, w, ldw, vocab, width, n, count, act, tgt, cap, cap != 0.f ? 1.0f / cap : 0.f};
}

bool on16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

#define ODP_XENT_GO(KERNEL, THREADS, GRID, ...) \
  hipLaunchKernelGGL(KERNEL, dim3(GRID), dim3(THREADS), 0, s, __VA_ARGS__)
// K<dtype, tiles>
#define ODP_XENT_LAUNCH(K, GRID, ...)                                                                \
  do {                                                                                               \
    constexpr int F = ODP_DTYPE_F32, B = ODP_DTYPE_BF16;                                             \
    if (dtype == F && kind == 3) ODP_XENT_GO((K<F, 3>), (Tile<F, 3>::THREADS), GRID, __VA_ARGS__);   \
    else if (dtype == F && kind == 1) ODP_XENT_GO((K<F, 1>), (Tile<F, 1>::THREADS), GRID, __VA_ARGS__); \
    else if (dtype == F) ODP_XENT_GO((K<F, 0>), (Tile<F, 0>::THREADS), GRID, __VA_ARGS__);           \
    else if (kind == 1) ODP_XENT_GO((K<B, 1>), (Tile<B, 1>::THREADS), GRID, __VA_ARGS__);            \
    else ODP_XENT_GO((K<B, 0>), (Tile<B, 0>::THREADS), GRID, __VA_ARGS__);                           \
  } while (0)
// K<dtype, tiles, softcap>
#define ODP_XENT_CAP(K, D, S, GRID, ...)                                                           \
  do {                                                                                             \
    if (softcap != 0.f) ODP_XENT_GO((K<D, S, true>), (Tile<D, S>::THREADS), GRID, __VA_ARGS__);    \
    else ODP_XENT_GO((K<D, S, false>), (Tile<D, S>::THREADS), GRID, __VA_ARGS__);                  \
  } while (0)
#define ODP_XENT_LAUNCH_CAP(K, GRID, ...)                                                          \
  do {                                                                                             \
    constexpr int F = ODP_DTYPE_F32, B = ODP_DTYPE_BF16;                                           \
    if (dtype == F && kind == 3) ODP_XENT_CAP(K, F, 3, GRID, __VA_ARGS__);                         \
    else if (dtype == F && kind == 1) ODP_XENT_CAP(K, F, 1, GRID, __VA_ARGS__);                    \
    else if (dtype == F) ODP_XENT_CAP(K, F, 0, GRID, __VA_ARGS__);                                 \
    else if (kind == 1) ODP_XENT_CAP(K, B, 1, GRID, __VA_ARGS__);                                  \
    else if (kind == 2) ODP_XENT_CAP(K, B, 2, GRID, __VA_ARGS__);                                  \
    else ODP_XENT_CAP(K, B, 0, GRID, __VA_ARGS__);                                                 \
  } while (0)

extern "C" int odp_xent_rows(odp_stream_t stream, int dtype, const void* x, int64_t ldx, int64_t n, int64_t cols,
                             int64_t width, const void* target, int target_bytes, int64_t vocab, int64_t ignore,
                             int keep, void* xc, int32_t* act, int32_t* tgt, int32_t* where, int32_t* count,
                             float* losses, float* stat) {
  if (int rc = check_xent("odp_xent_rows", dtype, n, width, width, vocab)) return rc;
  if (cols <= 0 || cols > width || ldx < cols || (target_bytes != 4 && target_bytes != 8)) {
    odp_set_error("odp_xent_rows: %lld columns of pitch %lld, targets of %d bytes", (long long)cols, (long long)ldx,
                  target_bytes);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (n > 0 && (x == nullptr || target == nullptr || xc == nullptr || act == nullptr || tgt == nullptr ||
                where == nullptr)) {
    odp_set_error("odp_xent_rows: null pointer");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (count == nullptr || !on16(xc)) {
    odp_set_error("odp_xent_rows: null count or packed rows off the 16-byte grid");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const hipStream_t s = odp_hip_stream(stream);
  const int64_t es = dtype == ODP_DTYPE_F32 ? 4 : 2;
  const int64_t blocks = up(n * (width * es / 16), 256);
  if (blocks >= (int64_t)1 << 24) {
    odp_set_error("odp_xent_rows: the launch needs %lld workgroups", (long long)blocks);
    return ODP_ERR_UNSUPPORTED;
  }
  const bool few = n > 0 && n <= XENT_FEW;
  const Pick p{target, target_bytes == 8 ? 1 : 0, keep, n, vocab, ignore, act, tgt, where, count, losses, stat};
  if (!few)
    hipLaunchKernelGGL(k_xent_pick, dim3(1), dim3(1024), 0, s, target, p.wide, n, vocab, ignore, keep, act, tgt, where,
                       count, losses, stat);
  if (blocks > 0) {
    const int vec = cols == width && on16(x) && ldx * es % 16 == 0;
#define ODP_PACK(D, F) \
  hipLaunchKernelGGL((k_xent_pack<D, F>), dim3((unsigned)blocks), dim3(256), 0, s, (const char*)x, ldx, cols, width, p, \
                     vec, (char*)xc)
    if (dtype == ODP_DTYPE_F32) {
      if (few) ODP_PACK(ODP_DTYPE_F32, true); else ODP_PACK(ODP_DTYPE_F32, false);
    } else {
      if (few) ODP_PACK(ODP_DTYPE_BF16, true); else ODP_PACK(ODP_DTYPE_BF16, false);
    }
#undef ODP_PACK
  }
  return odp_check_launch("odp_xent_rows");
}

extern "C" int64_t odp_xent_stats_scratch(int dtype, int64_t n, int64_t vocab) {
  if (n <= 0 || vocab <= 0) return 0;
  return 4 * n * (2 * up(vocab, tile_cols(dtype, few_rows(dtype, n))) + 1);
}

extern "C" int64_t odp_xent_kept(int dtype, int64_t n, int64_t width, int64_t vocab) {
  if (n <= 0 || width <= 0 || vocab <= 0 || !keeps(dtype, n, width)) return 0;
  const int64_t row = 4 * odp_xent_pitch(dtype, vocab);
  return n <= ((int64_t)1 << 60) / row ? n * row : 0;
}

extern "C" int odp_xent_losses(odp_stream_t stream, int dtype, const void* xc, int64_t n, int64_t width,
                               const int32_t* act, const int32_t* tgt, const int32_t* count, const void* w,
                               int64_t ldw, int64_t vocab, float softcap, void* scratch, float* losses, float* stat,
                               float* logits, int64_t ldl) {
  if (int rc = check_xent("odp_xent_losses", dtype, n, width, ldw, vocab)) return rc;
  if (int rc = check_cap("odp_xent_losses", softcap)) return rc;
  if (n == 0) return ODP_OK;
  if (xc == nullptr || act == nullptr || tgt == nullptr || count == nullptr || w == nullptr || scratch == nullptr ||
      losses == nullptr || stat == nullptr || !on16(xc) || !on16(w)) {
    odp_set_error("odp_xent_losses: null pointer, or rows off the 16-byte grid");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (logits != nullptr && (ldl != odp_xent_pitch(dtype, vocab) || !on16(logits))) {
    odp_set_error("odp_xent_losses: logits of pitch %lld for a vocabulary of %lld, or off the 16-byte grid",
                  (long long)ldl, (long long)vocab);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const hipStream_t s = odp_hip_stream(stream);
  const int kind = tile_kind(dtype, n, vocab);
  const int64_t tn = up(vocab, tile_cols(dtype, kind));
  unsigned blocks;
  if (int rc = grid_of("odp_xent_losses", dtype, kind, up(n, tile_rows(dtype, kind)), tn, false, blocks)) return rc;
  const Xent p = xent_of(xc, w, ldw, vocab, width, n, count, act, tgt, softcap);
  float* pmax = (float*)scratch;
  float* psum = pmax + n * tn;
  float* ztgt = psum + n * tn;
  ODP_XENT_LAUNCH_CAP(k_xent_stats, blocks, p, pmax, psum, ztgt, logits, ldl);
  if (kind == 1 || kind == 3)
    hipLaunchKernelGGL(k_xent_losses<1>, dim3((unsigned)n), dim3(256), 0, s, pmax, psum, ztgt, (int)tn, n, count, act,
                       tgt, losses, stat);
  else
    hipLaunchKernelGGL(k_xent_losses<16>, dim3((unsigned)up(n, 16)), dim3(256), 0, s, pmax, psum, ztgt, (int)tn, n,
                       count, act, tgt, losses, stat);
  return odp_check_launch("odp_xent_losses");
}

extern "C" int odp_xent_reduce(odp_stream_t stream, const float* losses, int64_t n, const float* over, float* out) {
  if (n < 0 || out == nullptr || (n > 0 && losses == nullptr)) {
    odp_set_error("odp_xent_reduce: null pointer or %lld losses", (long long)n);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  hipLaunchKernelGGL(k_xent_reduce, dim3(1), dim3(1024), 0, odp_hip_stream(stream), losses, n, over, out);
  return odp_check_launch("odp_xent_reduce");
}

extern "C" int64_t odp_xent_pitch(int dtype, int64_t columns) {
  return columns > 0 ? up(columns, tile_edge(dtype)) * tile_edge(dtype) : 0;
}

extern "C" int odp_xent_dlogits(odp_stream_t stream, int dtype, const void* xc, int64_t n, int64_t width,
                                const int32_t* act, const int32_t* tgt, const int32_t* count, const void* w,
                                int64_t ldw, int64_t vocab, float softcap, int64_t v0, int64_t vc, const float* stat,
                                const float* g, int g_stride, const float* over, const float* logits, int64_t ldl,
                                void* dl, int64_t ldd, float* rest) {
  if (int rc = check_xent("odp_xent_dlogits", dtype, n, width, ldw, vocab)) return rc;
  if (int rc = check_cap("odp_xent_dlogits", softcap)) return rc;
  if (v0 < 0 || vc <= 0 || v0 + vc > vocab || ldd != odp_xent_pitch(dtype, vc)) {
    odp_set_error("odp_xent_dlogits: columns [%lld, %lld) of %lld at pitch %lld", (long long)v0,
                  (long long)(v0 + vc), (long long)vocab, (long long)ldd);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (n == 0) return ODP_OK;
  if (xc == nullptr || act == nullptr || tgt == nullptr || count == nullptr || w == nullptr || stat == nullptr ||
      g == nullptr || dl == nullptr || rest == nullptr || !on16(xc) || !on16(w) || !on16(dl)) {
    odp_set_error("odp_xent_dlogits: null pointer, or rows off the 16-byte grid");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const hipStream_t s = odp_hip_stream(stream);
  if (logits != nullptr) {
    // Pieces start on a tile's edge, so that a piece's padded columns lie inside the logits' row.
    const int64_t parts = up(ldd, KEPT_COLS);
    if (ldl != odp_xent_pitch(dtype, vocab) || !on16(logits) || v0 % tile_edge(dtype) != 0 ||
        n * parts >= (int64_t)1 << 24) {
      odp_set_error("odp_xent_dlogits: logits of pitch %lld from column %lld, %lld workgroups", (long long)ldl,
                    (long long)v0, (long long)(n * parts));
      return ODP_ERR_INVALID_ARGUMENT;
    }
    const Xent p = xent_of(nullptr, nullptr, 0, vocab, width, n, count, act, tgt, softcap);
#define ODP_KEPT(D, C)                                                                                                 \
  ODP_XENT_GO((k_xent_dkept<D, C>), 256, (unsigned)(n * parts), p, logits, ldl, v0, vc, (int)parts, stat, g, g_stride,  \
              over, (char*)dl, ldd, rest)
    if (dtype == ODP_DTYPE_F32) {
      if (softcap != 0.f) ODP_KEPT(ODP_DTYPE_F32, true); else ODP_KEPT(ODP_DTYPE_F32, false);
    } else {
      if (softcap != 0.f) ODP_KEPT(ODP_DTYPE_BF16, true); else ODP_KEPT(ODP_DTYPE_BF16, false);
    }
#undef ODP_KEPT
    return odp_check_launch("odp_xent_dlogits");
  }
  const int kind = tile_kind(dtype, n, ldd);
  unsigned blocks;
  if (int rc = grid_of("odp_xent_dlogits", dtype, kind, up(n, tile_rows(dtype, kind)), ldd / tile_cols(dtype, kind),
                       false, blocks))
    return rc;
  const Xent p = xent_of(xc, w, ldw, vocab, width, n, count, act, tgt, softcap);
  ODP_XENT_LAUNCH_CAP(k_xent_dlogits, blocks, p, v0, vc, stat, g, g_stride, over, dl, ldd, rest);
  return odp_check_launch("odp_xent_dlogits");
}

// Tiles of n rows of dx, and those that the slots hold: as many, or a few times that to split.
static int64_t dx_tiles(int dtype, int64_t n, int64_t width) {
  const int kind = few_kind(dtype, n);
  return up(n, tile_rows(dtype, kind)) * up(width, tile_cols(dtype, kind));
}
static int dx_cap(int dtype, int64_t n, int64_t width) {
  const int64_t tiles = dx_tiles(dtype, n, width);
  const int64_t most = tiles * DX_SPLIT < 512 ? tiles * DX_SPLIT : 512;
  return (int)(tiles > most ? tiles : most);
}

extern "C" int64_t odp_xent_dx_scratch(int dtype, int64_t n, int64_t width) {
  if (n <= 0 || width <= 0) return 0;
  const int kind = few_kind(dtype, n);
  return 4 * (int64_t)dx_cap(dtype, n, width) * tile_rows(dtype, kind) * tile_cols(dtype, kind);
}

extern "C" int odp_xent_dx(odp_stream_t stream, int dtype, int64_t n, int64_t width, const int32_t* count,
                           const void* w, int64_t ldw, int64_t vocab, int64_t v0, int64_t vc, int64_t piece,
                           const void* dl, int64_t ldd, void* scratch) {
  if (int rc = check_xent("odp_xent_dx", dtype, n, width, ldw, vocab)) return rc;
  if (v0 < 0 || vc <= 0 || vc > piece || v0 + vc > vocab || ldd != odp_xent_pitch(dtype, vc) ||
      ldd >= ODP_XENT_PIECE) {
    odp_set_error("odp_xent_dx: columns [%lld, %lld) of %lld in pieces of %lld at pitch %lld", (long long)v0,
                  (long long)(v0 + vc), (long long)vocab, (long long)piece, (long long)ldd);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (n == 0) return ODP_OK;
  if (count == nullptr || w == nullptr || dl == nullptr || scratch == nullptr || !on16(w) || !on16(dl) ||
      !on16(scratch)) {
    odp_set_error("odp_xent_dx: null pointer, or rows off the 16-byte grid");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const hipStream_t s = odp_hip_stream(stream);
  const int cap = dx_cap(dtype, n, width);
  const int kind = few_kind(dtype, n);
  unsigned blocks;
  if (int rc = grid_of("odp_xent_dx", dtype, kind, cap, 1, true, blocks)) return rc;
  const Xent p = xent_of(nullptr, w, ldw, vocab, width, n, count, nullptr, nullptr, 0.f);
  const int64_t whole = odp_xent_pitch(dtype, piece);
  ODP_XENT_LAUNCH(k_xent_dx, blocks, p, v0, vc, whole, dl, ldd, cap, v0 == 0 ? 1 : 0, (float*)scratch);
  return odp_check_launch("odp_xent_dx");
}

extern "C" int odp_xent_dx_rows(odp_stream_t stream, int dtype, int64_t n, int64_t cols, int64_t width,
                                const int32_t* count, const int32_t* where, const int32_t* tgt, const void* w,
                                int64_t ldw, int64_t piece, const void* scratch, const float* rest, void* dx) {
  if (int rc = check_xent("odp_xent_dx_rows", dtype, n, width, ldw, 1)) return rc;
  if (cols <= 0 || cols > width || piece <= 0) {
    odp_set_error("odp_xent_dx_rows: %lld columns of %lld, pieces of %lld", (long long)cols, (long long)width,
                  (long long)piece);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (n == 0) return ODP_OK;
  if (count == nullptr || where == nullptr || tgt == nullptr || w == nullptr || scratch == nullptr ||
      rest == nullptr || dx == nullptr || !on16(scratch) || !on16(w) ||
      (cols == width && !on16(dx))) {
    odp_set_error("odp_xent_dx_rows: null pointer, or rows off the 16-byte grid");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const int64_t blocks = up(n * (width / 4), 256);
  if (blocks >= (int64_t)1 << 24) {
    odp_set_error("odp_xent_dx_rows: the launch needs %lld workgroups", (long long)blocks);
    return ODP_ERR_UNSUPPORTED;
  }
  const hipStream_t s = odp_hip_stream(stream);
  const int kind = few_kind(dtype, n);
  const int ot = tile_rows(dtype, kind), tn = (int)up(width, tile_cols(dtype, kind)), cap = dx_cap(dtype, n, width);
  const int64_t steps = odp_xent_pitch(dtype, piece) / (dtype == ODP_DTYPE_F32 ? 16 : 32);
  if (dtype == ODP_DTYPE_F32)
    hipLaunchKernelGGL((k_xent_dx_rows<ODP_DTYPE_F32>), dim3((unsigned)blocks), dim3(256), 0, s,
                       (const float*)scratch, width, cols, n, count, where, ot, tn, cap, steps, rest, tgt,
                       (const char*)w, ldw, dx);
  else
    hipLaunchKernelGGL((k_xent_dx_rows<ODP_DTYPE_BF16>), dim3((unsigned)blocks), dim3(256), 0, s,
                       (const float*)scratch, width, cols, n, count, where, ot, tn, cap, steps, rest, tgt,
                       (const char*)w, ldw, dx);
  return odp_check_launch("odp_xent_dx_rows");
}

// Slices of the tokens that the tiles of dW are split into: as many as the CUs
// hold, of at least 32 steps.
static int dw_split(int dtype, int64_t n, int64_t vc, int64_t width) {
  const int64_t tiles = up(vc, tile_edge(dtype)) * up(width, tile_edge(dtype)), held = dtype == ODP_DTYPE_F32 ? 512 : 256;
  const int64_t most = n / (32 * (dtype == ODP_DTYPE_F32 ? 16 : 32)), s = held / tiles < most ? held / tiles : most;
  return (int)(s < 2 ? 1 : s);
}

extern "C" int64_t odp_xent_dw_scratch(int dtype, int64_t n, int64_t vc, int64_t width) {
  if (n <= 0 || vc <= 0 || width <= 0) return 0;
  const int split = dw_split(dtype, n, vc, width);
  return split > 1 ? 4 * split * vc * width : 0;
}

extern "C" int odp_xent_dw(odp_stream_t stream, int dtype, const void* xc, int64_t n, int64_t width,
                           const int32_t* count, int64_t vc, const void* dl, int64_t ldd, void* scratch, void* dw,
                           int64_t lddw) {
  if (int rc = check_xent("odp_xent_dw", dtype, n, width, lddw, vc)) return rc;
  if (ldd != odp_xent_pitch(dtype, vc) || ldd >= ODP_XENT_PIECE || count == nullptr || dw == nullptr || !on16(dw) ||
      (n > 0 && (xc == nullptr || dl == nullptr || !on16(xc) || !on16(dl)))) {
    odp_set_error("odp_xent_dw: pitch %lld for %lld columns, null pointer, or rows off the 16-byte grid",
                  (long long)ldd, (long long)vc);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const hipStream_t s = odp_hip_stream(stream);
  const int split = lddw == width ? dw_split(dtype, n, vc, width) : 1;
  unsigned blocks;
  if (split > 1) {
    if (scratch == nullptr || !on16(scratch)) {
      odp_set_error("odp_xent_dw: scratch is null or off the 16-byte grid");
      return ODP_ERR_INVALID_ARGUMENT;
    }
    const int64_t tiles = up(vc, tile_edge(dtype)) * up(width, tile_edge(dtype)), quads = vc * width / 4;
    const bool wide = split > 8;
    blocks = (unsigned)up(tiles * split, 8) * 8;
    const Xent p = xent_of(xc, nullptr, width, vc, width, n, count, nullptr, nullptr, 0.f);
#define ODP_DW(D)                                                                                                    \
  do {                                                                                                               \
    ODP_XENT_GO((k_xent_dw_part<D>), (Tile<D, 0>::THREADS), blocks, p, vc, dl, ldd, split, (float*)scratch);          \
    if (wide) ODP_XENT_GO((k_xent_dw_rows<D, 16>), 256, (unsigned)up(quads, 16), (const float*)scratch, split, quads, dw); \
    else ODP_XENT_GO((k_xent_dw_rows<D, 1>), 256, (unsigned)up(quads, 256), (const float*)scratch, split, quads, dw); \
  } while (0)
    if (dtype == ODP_DTYPE_F32) ODP_DW(ODP_DTYPE_F32); else ODP_DW(ODP_DTYPE_BF16);
#undef ODP_DW
    return odp_check_launch("odp_xent_dw");
  }
  if (int rc = grid_of("odp_xent_dw", dtype, 0, up(vc, tile_edge(dtype)), up(width, tile_edge(dtype)), false, blocks)) return rc;
  const Xent p = xent_of(xc, nullptr, width, vc, width, n, count, nullptr, nullptr, 0.f);
  if (dtype == ODP_DTYPE_F32)
    ODP_XENT_GO((k_xent_dw<ODP_DTYPE_F32>), (Tile<ODP_DTYPE_F32, 0>::THREADS), blocks, p, vc, dl, ldd, dw, lddw);
  else
    ODP_XENT_GO((k_xent_dw<ODP_DTYPE_BF16>), (Tile<ODP_DTYPE_BF16, 0>::THREADS), blocks, p, vc, dl, ldd, dw, lddw);
  return odp_check_launch("odp_xent_dw");
}
