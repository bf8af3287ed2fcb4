// The embedding table: rows looked up and scaled, its gradient by sorted
// tokens, and that gradient's per-example norms and clipped sum.
//
//   out_n  = s W[y_n]                                   k_embed_rows
//   dW_v   = s sum_{n: y_n = v} g_n                     k_embed_sum<EM_GRAD>
//   S_iv   = s sum_{n in example i, y_n = v} g_n
//   |i|^2  = sum_v |S_iv|^2                             k_embed_sum<EM_NORM>
//   out_v  = sum_i c_i S_iv / normalize_by              k_embed_sum<EM_CLIP>
//
// All of it moves rows and adds them: bound by HBM.  Positions are sorted by
// token (stable, so a token's positions stay in row order and an example's
// come together).  The sums walk the sorted positions in windows of EM_WIN;
// a run of equal tokens inside a window is finished where it is read, one
// that crosses windows leaves float32 partials that k_embed_join adds in
// window order.  So the work per wave is the same whatever the tokens'
// frequencies (half of a batch may be one padding token), every gradient row
// is read once per pass, nothing is added atomically, and results do not
// depend on the order of execution.
#include "odp_internal.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int EM_WIN = 32;   // sorted positions per window
constexpr int EM_LOAD = 8;   // rows in flight per wave
constexpr int EM_WAVES = 4;  // waves per workgroup

enum { EM_GRAD = 0, EM_NORM = 1, EM_CLIP = 2 };

__device__ __forceinline__ int uniform_int(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Values a lane takes of a row piece: 16 bytes.
template <int DT>
__host__ __device__ constexpr int em_vec() { return DT == ODP_DTYPE_F32 ? 4 : 8; }

// Column of value i of this lane within piece cb of a row: contiguous 16-byte
// pieces where rows lie on the 16-byte grid, else one value per lane in turn.
template <int DT, bool AL>
__device__ __forceinline__ int em_col(int cb, int i) {
  constexpr int V = em_vec<DT>();
  const int lane = threadIdx.x & 63;
  return cb * 64 * V + (AL ? lane * V + i : lane + 64 * i);
}

// Reads the lane's values of the row at p as 16 raw bytes or as floats.
template <int DT, bool AL>
struct EmPiece {
  static constexpr int V = em_vec<DT>();
  u32x4_t w;
  __device__ __forceinline__ void load(const char* p, int cb, int width) {
    if constexpr (AL) {
      const int c = em_col<DT, AL>(cb, 0);
      w = u32x4_t{0, 0, 0, 0};
      if (c < width)
        w = __builtin_nontemporal_load(
            (const ODP_GMEM u32x4_t*)(const ODP_GMEM void*)(p + (int64_t)c * (DT == ODP_DTYPE_F32 ? 4 : 2)));
    } else {
      uint32_t h[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = em_col<DT, AL>(cb, i);
        h[i] = 0;
        if (c < width) h[i] = DT == ODP_DTYPE_F32 ? ((const uint32_t*)p)[c] : (uint32_t)((const uint16_t*)p)[c];
      }
      if constexpr (DT == ODP_DTYPE_F32) {
        w = u32x4_t{h[0], h[1], h[2], h[3]};
      } else {
        w = u32x4_t{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == ODP_DTYPE_F32) {
        v[i] = __uint_as_float(w[i]);
      } else if constexpr (DT == ODP_DTYPE_BF16) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
        v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
      }
    }
  }
};

// Stores the lane's values of row `row` of a [*, width] tensor of dtype odt.
template <int DT, bool AL>
__device__ __forceinline__ void em_store(void* out, int odt, int64_t row, int width, int cb,
                                         const float (&v)[em_vec<DT>()]) {
  constexpr int V = em_vec<DT>();
  const int64_t at = row * width;
  if (AL && odt == DT) {
    const int c = em_col<DT, AL>(cb, 0);
    if (c >= width) return;
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == ODP_DTYPE_F32) w[i] = __float_as_uint(v[i]);
      else if constexpr (DT == ODP_DTYPE_BF16) w[i] = odp_f2bf2(v[2 * i], v[2 * i + 1]);
      else
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) |
               (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16;
    }
    odp_gstore((u32x4_t*)((char*)out + (at + c) * (DT == ODP_DTYPE_F32 ? 4 : 2)), w);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = em_col<DT, AL>(cb, i);
    if (c < width) odp_store_from_float(out, at + c, odt, v[i]);
  }
}

__device__ __forceinline__ int64_t token_at(const void* tokens, int wide, int64_t i) {
  return wide ? ((const int64_t*)tokens)[i] : (int64_t)((const int32_t*)tokens)[i];
}

// ---------------------------------------------------------------------------
// Lookup.  One wave per (row, 64 pieces of 16 bytes); a token outside the
// table gives a row of NaN.
// ---------------------------------------------------------------------------
template <int DT, bool AL>
__global__ __launch_bounds__(64 * EM_WAVES) void k_embed_rows(const void* __restrict__ tokens, int wide, int64_t n,
                                                              const char* __restrict__ weight, int64_t ldw,
                                                              int64_t vocab, int width, int ncb, float scale,
                                                              void* __restrict__ out) {
  const int64_t item = (int64_t)blockIdx.x * EM_WAVES + uniform_int(threadIdx.x >> 6);
  const int64_t row = item / ncb;
  const int cb = (int)(item - row * ncb);
  if (row >= n) return;
  const int64_t t = token_at(tokens, wide, row);
  constexpr int V = em_vec<DT>();
  float v[V];
  if (t >= 0 && t < vocab) {
    EmPiece<DT, AL> p;
    p.load(weight + t * ldw * (DT == ODP_DTYPE_F32 ? 4 : 2), cb, width);
    p.get(v);
    if (scale != 1.0f) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = __fmul_rn(v[i], scale);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = __uint_as_float(0x7fc00000u);
  }
  em_store<DT, AL>(out, DT, row, width, cb, v);
}

// ---------------------------------------------------------------------------
// Stable sort of the positions by token: least-significant-digit radix passes
// of up to SORT_BITS bits.  A wave owns SORT_KEYS consecutive positions; its
// digit counts, summed exclusively over (digit, wave), are where its keys go,
// and equal digits within 64 keys are ranked by ballots, so order among equal
// tokens is kept.  Dropped positions (outside the table, padding, rows
// outside every segment) get the key `vocab` and end up last.
// ---------------------------------------------------------------------------
constexpr int SORT_BITS = 9, SORT_BINS = 1 << SORT_BITS;
constexpr int SORT_KEYS = 512;                            // positions per wave
constexpr int SORT_WAVES = 16;                            // waves of the one-workgroup sort
constexpr int64_t SORT_SMALL = SORT_WAVES * SORT_KEYS;    // positions it takes

struct SortIn {
  const void* tokens;
  int wide;  // tokens are int64
  int64_t n, vocab, padding;
  const int32_t* sstart;  // segments (nullptr: every row counts)
  const int32_t* slen;
  int n_seg;
  int32_t* row_seg;  // [n] each row's segment, written in the first pass (with segments)
};

__device__ __forceinline__ uint32_t sort_key(const SortIn& a, int64_t i, bool record) {
  const int64_t t = token_at(a.tokens, a.wide, i);
  bool ok = t >= 0 && t < a.vocab && t != a.padding;
  if (a.sstart != nullptr) {
    int lo = 0, hi = a.n_seg - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)a.sstart[mid] <= i) lo = mid; else hi = mid - 1;
    }
    const bool in = a.n_seg > 0 && i >= a.sstart[lo] && i < (int64_t)a.sstart[lo] + a.slen[lo];
    ok = ok && in;
    if (record) a.row_seg[i] = in ? lo : 0;
  }
  return ok ? (uint32_t)t : (uint32_t)a.vocab;
}

// Adds the digits of positions [lo, hi) to the wave's counts h.
template <typename Key>
__device__ __forceinline__ void sort_count(uint32_t* h, int64_t lo, int64_t hi, int shift, uint32_t mask, Key key) {
  for (int64_t i = lo + (threadIdx.x & 63); i < hi; i += 64) atomicAdd(&h[(key(i) >> shift) & mask], 1u);
}

// Sends positions [lo, hi) to where the wave's h says, in order.
template <typename Key, typename Row>
__device__ __forceinline__ void sort_scatter(uint32_t* h, int64_t lo, int64_t hi, int shift, int bits, Key key,
                                             Row row, uint32_t* ok, uint32_t* orow) {
  const int lane = threadIdx.x & 63;
  const uint64_t before = (1ull << lane) - 1;
  for (int64_t i0 = lo; i0 < hi; i0 += 64) {
    const int64_t i = i0 + lane;
    const bool on = i < hi;
    const uint32_t k = on ? key(i) : 0u, r = on ? row(i) : 0u;
    const uint32_t d = (k >> shift) & ((1u << bits) - 1);
    uint64_t peers = __builtin_amdgcn_ballot_w64(on);
    for (int b = 0; b < bits; ++b) {
      const bool set = (d >> b) & 1u;
      const uint64_t m = __builtin_amdgcn_ballot_w64(on && set);
      peers &= set ? m : ~m;
    }
    const uint32_t base = on ? h[d] : 0u;
    __builtin_amdgcn_wave_barrier();
    __asm__ volatile("" ::: "memory");
    // The last of the equal digits moves the count on for the next 64 keys.
    if (on && (peers >> lane) == 1ull) h[d] = base + (uint32_t)__popcll(peers);
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    if (on) {
      const uint32_t to = base + (uint32_t)__popcll(peers & before);
      ok[to] = k;
      orow[to] = r;
    }
  }
}

// Exclusive sum of each thread's value over the workgroup (of 64 * nw
// threads); `red` has nw entries.  Returns the sum of the threads before,
// and the workgroup's total in `total`.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, int nw, uint32_t* red, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t s = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = __shfl_up(s, off);
    if (lane >= off) s += o;
  }
  __syncthreads();
  if (lane == 63) red[wave] = s;
  __syncthreads();
  uint32_t base = 0, all = 0;
  for (int w = 0; w < nw; ++w) {
    const uint32_t t = red[w];
    if (w < wave) base += t;
    all += t;
  }
  total = all;
  return base + s - v;
}

// The whole sort in one workgroup (n <= SORT_SMALL): one launch instead of
// three per pass.
__global__ __launch_bounds__(64 * SORT_WAVES) void k_sort_small(SortIn a, int passes, int bits, uint32_t* k0,
                                                                uint32_t* r0, uint32_t* k1, uint32_t* r1) {
  __shared__ uint32_t hist[SORT_WAVES][SORT_BINS];
  __shared__ uint32_t red[SORT_WAVES];
  const int wave = threadIdx.x >> 6, bins = 1 << bits;
  const int64_t per = (a.n + SORT_WAVES * 64 - 1) / (SORT_WAVES * 64) * 64;
  const int64_t lo = min(a.n, wave * per), hi = min(a.n, lo + per);
  for (int p = 0; p < passes; ++p) {
    for (int i = threadIdx.x; i < SORT_WAVES * SORT_BINS; i += blockDim.x) (&hist[0][0])[i] = 0;
    __syncthreads();
    const int shift = p * bits;
    // The passes alternate buffers so that the last one writes k0, r0.
    const bool to0 = ((passes - 1 - p) & 1) == 0;
    const uint32_t* ik = to0 ? k1 : k0;
    const uint32_t* ir = to0 ? r1 : r0;
    uint32_t* ok = to0 ? k0 : k1;
    uint32_t* orow = to0 ? r0 : r1;
    auto key = [&](int64_t i) { return p == 0 ? sort_key(a, i, false) : ik[i]; };
    auto row = [&](int64_t i) {
      if (p > 0) return ir[i];
      if (a.sstart != nullptr) sort_key(a, i, true);
      return (uint32_t)i;
    };
    sort_count(hist[wave], lo, hi, shift, (uint32_t)bins - 1, key);
    __syncthreads();
    // Exclusive sums over (digit, wave): thread d takes digit d.
    uint32_t mine = 0;
    if ((int)threadIdx.x < bins)
      for (int w = 0; w < SORT_WAVES; ++w) mine += hist[w][threadIdx.x];
    uint32_t total;
    uint32_t at = block_exclusive(mine, SORT_WAVES, red, total);
    if ((int)threadIdx.x < bins)
      for (int w = 0; w < SORT_WAVES; ++w) {
        const uint32_t c = hist[w][threadIdx.x];
        hist[w][threadIdx.x] = at;
        at += c;
      }
    __syncthreads();
    sort_scatter(hist[wave], lo, hi, shift, bits, key, row, ok, orow);
    __threadfence_block();
    __syncthreads();
  }
}

// counts[digit][wave of the launch].
__global__ __launch_bounds__(64 * EM_WAVES) void k_sort_count(SortIn a, const uint32_t* ik, int first, int shift,
                                                              int bits, uint32_t* counts, int nw) {
  __shared__ uint32_t hist[EM_WAVES][SORT_BINS];
  const int wave = threadIdx.x >> 6, bins = 1 << bits;
  for (int i = threadIdx.x; i < EM_WAVES * SORT_BINS; i += blockDim.x) (&hist[0][0])[i] = 0;
  __syncthreads();
  const int64_t w = (int64_t)blockIdx.x * EM_WAVES + wave;
  const int64_t lo = min(a.n, w * SORT_KEYS), hi = min(a.n, lo + SORT_KEYS);
  sort_count(hist[wave], lo, hi, shift, (uint32_t)bins - 1,
             [&](int64_t i) { return first ? sort_key(a, i, false) : ik[i]; });
  __syncthreads();
  if (w < nw)
    for (int d = threadIdx.x & 63; d < bins; d += 64) counts[(int64_t)d * nw + w] = hist[wave][d];
}

// Exclusive sums of counts in place, one workgroup.
__global__ __launch_bounds__(1024) void k_sort_scan(uint32_t* counts, int64_t n) {
  __shared__ uint32_t red[16];
  uint32_t carry = 0;
  for (int64_t i0 = 0; i0 < n; i0 += 4096) {
    uint32_t v[4], s = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t i = i0 + 4 * threadIdx.x + q;
      v[q] = i < n ? counts[i] : 0u;
      s += v[q];
    }
    uint32_t total;
    uint32_t at = carry + block_exclusive(s, 16, red, total);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t i = i0 + 4 * threadIdx.x + q;
      if (i < n) counts[i] = at;
      at += v[q];
    }
    carry += total;
  }
}

__global__ __launch_bounds__(64 * EM_WAVES) void k_sort_scatter(SortIn a, const uint32_t* ik, const uint32_t* ir,
                                                                int first, int shift, int bits,
                                                                const uint32_t* counts, int nw, uint32_t* ok,
                                                                uint32_t* orow) {
  __shared__ uint32_t hist[EM_WAVES][SORT_BINS];
  const int wave = threadIdx.x >> 6, bins = 1 << bits;
  const int64_t w = (int64_t)blockIdx.x * EM_WAVES + wave;
  if (w < nw)
    for (int d = threadIdx.x & 63; d < bins; d += 64) hist[wave][d] = counts[(int64_t)d * nw + w];
  __syncthreads();
  const int64_t lo = min(a.n, w * SORT_KEYS), hi = min(a.n, lo + SORT_KEYS);
  sort_scatter(hist[wave], lo, hi, shift, bits, [&](int64_t i) { return first ? sort_key(a, i, false) : ik[i]; },
               [&](int64_t i) {
                 if (!first) return ir[i];
                 if (a.sstart != nullptr) sort_key(a, i, true);
                 return (uint32_t)i;
               },
               ok, orow);
}

// ---------------------------------------------------------------------------
// Sums over the sorted positions.
// ---------------------------------------------------------------------------
struct EmbedSum {
  const char* g;  // gradient rows
  int64_t ldg;    // elements
  int64_t n;
  int width, ncb;
  const uint32_t* keys;   // sorted tokens, `vocab` for dropped positions
  const uint32_t* rows;   // the positions, sorted
  const int32_t* row_seg;  // NORM, CLIP: segment of each row
  uint32_t vocab;
  float scale;
  float* ws;     // [windows][2][width] partials of runs that cross windows
  float* ws_sq;  // the same of the squares (CLIP with second moments)
  float* whole;  // NORM, CLIP: [windows][width] sums S of the crossing (example, token) runs
  void* out;     // GRAD, CLIP: [vocab][width]
  void* out2;
  int odt;
  // NORM
  double* part;
  int64_t part_stride, slot;
  const int32_t* sstart;
  const int32_t* sex;
  int64_t* nf_flag;  // set when an S entry is not finite
  // CLIP
  const double* scales;
  float normalize_by;
};

template <int V>
__device__ __forceinline__ void em_clear(float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
}

// A float32 workspace row: contiguous per lane, whatever the columns' order.
template <int DT>
__device__ __forceinline__ float* em_ws(float* ws, int64_t row, const EmbedSum& a, int cb) {
  constexpr int V = em_vec<DT>();
  return ws + (row * a.ncb + cb) * 64 * V + (threadIdx.x & 63) * V;
}
template <int V>
__device__ __forceinline__ void em_put(float* p, const float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 4) odp_gstore((f32x4_t*)(p + i), f32x4_t{v[i], v[i + 1], v[i + 2], v[i + 3]});
}
template <int V>
__device__ __forceinline__ void em_add(const float* p, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const f32x4_t x = *(const ODP_GMEM f32x4_t*)(const ODP_GMEM void*)(p + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[i + e] += x[e];
  }
}

// An (example, token) run's S is complete: its squares go to the partial of
// its first row and this piece.
template <int DT>
__device__ __forceinline__ void em_norm(const EmbedSum& a, uint32_t head_row, int seg, int cb,
                                        const float (&v)[em_vec<DT>()]) {
  double s = 0.0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < em_vec<DT>(); ++i) {
    const float x = __fmul_rn(v[i], a.scale);
    const bool fin = isfinite(x);
    bad |= !fin;
    if (fin) s += (double)__fmul_rn(x, x);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
  const uint64_t any = __builtin_amdgcn_ballot_w64(bad);
  if ((threadIdx.x & 63) == 0) {
    a.part[(int64_t)a.sex[seg] * a.part_stride + a.slot + ((int64_t)head_row - a.sstart[seg]) * a.ncb + cb] = s;
    if (any != 0) *a.nf_flag = 1;
  }
}

// A token's sum is complete.
template <int DT, bool AL>
__device__ __forceinline__ void em_finish(const EmbedSum& a, int mode, uint32_t key, int cb,
                                          float (&v)[em_vec<DT>()], float (&q)[em_vec<DT>()]) {
  constexpr int V = em_vec<DT>();
  if (mode == EM_GRAD) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = __fmul_rn(v[i], a.scale);
  } else if (a.normalize_by != 1.0f) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = __fdiv_rn(v[i], a.normalize_by);
  }
  em_store<DT, AL>(a.out, a.odt, key, a.width, cb, v);
  if (mode == EM_CLIP && a.out2 != nullptr) {
    if (a.normalize_by != 1.0f) {
#pragma unroll
      for (int i = 0; i < V; ++i) q[i] = __fdiv_rn(q[i], a.normalize_by);
    }
    em_store<DT, AL>(a.out2, a.odt, key, a.width, cb, q);
  }
}

// One wave per (window, 64 pieces of 16 bytes of the rows).
template <int DT, bool AL, int MODE>
__global__ __launch_bounds__(64 * EM_WAVES) void k_embed_sum(EmbedSum a) {
  constexpr int V = em_vec<DT>(), ES = DT == ODP_DTYPE_F32 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * EM_WAVES + uniform_int(threadIdx.x >> 6);
  const int64_t win = item / a.ncb, p0 = win * EM_WIN;
  const int cb = (int)(item - win * a.ncb);
  if (p0 >= a.n) return;
  // Lane l holds position p0 - 1 + l: the window, the one before and the one after.
  const int64_t pos = p0 - 1 + lane;
  const bool in = pos >= 0 && pos < a.n && lane <= EM_WIN + 1;
  const uint32_t key = in ? a.keys[pos] : a.vocab;
  const uint32_t row = in ? a.rows[pos] : 0u;
  int seg = 0;
  float c = 0.f;
  if (MODE != EM_GRAD && key != a.vocab) {
    seg = a.row_seg[row];
    if (MODE == EM_CLIP) c = (float)a.scales[a.sex[seg]];
  }
  const uint32_t pkey = __shfl_up(key, 1);
  const int pseg = __shfl_up(seg, 1);
  // Bit p: position p0 + p counts / starts a token's run / an (example, token)
  // run (bit EM_WIN: the position after the window).
  const bool live_l = key != a.vocab && lane >= 1;
  const uint64_t live = __builtin_amdgcn_ballot_w64(live_l) >> 1;
  const uint64_t tok = __builtin_amdgcn_ballot_w64(live_l && key != pkey) >> 1;
  const uint64_t sub = MODE == EM_GRAD ? tok : __builtin_amdgcn_ballot_w64(live_l && (key != pkey || seg != pseg)) >> 1;
  const int n_live = __popcll(live & ((1ull << EM_WIN) - 1));  // dropped positions come last
  if (n_live == 0) return;
  const bool more = (live >> EM_WIN) & 1;
  const bool tok_on = more && !((tok >> EM_WIN) & 1);  // the last run goes on in the next window
  const bool sub_on = more && !((sub >> EM_WIN) & 1);
  // Rows of (example, token) runs that cross windows were added by the NORM
  // pass: CLIP takes their sum from `whole` at the run's first window.
  int from = 0, to = n_live;
  if (MODE == EM_CLIP) {
    const uint64_t heads = sub & ((1ull << n_live) - 1);
    from = heads ? __builtin_ctzll(heads) : n_live;
    if (sub_on && heads) to = 63 - __builtin_clzll(heads);
  }

  float acc[V], acc2[V], sum[V];
  em_clear(acc);
  em_clear(acc2);
  em_clear(sum);
  // Position p ends a run of `heads`.
  auto ends = [&](uint64_t heads, int p) { return p == n_live - 1 || ((heads >> (p + 1)) & 1); };
  int run_head = 0;  // first position of the current (example, token) run
  auto close_token = [&](int p) {
    const uint64_t upto = tok & ((2ull << p) - 1);
    const bool began = upto != 0, last = p == n_live - 1;
    const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)key, p + 1);
    float(&v)[V] = MODE == EM_GRAD ? sum : acc;
    if (began && !(last && tok_on)) {
      em_finish<DT, AL>(a, MODE, k, cb, v, acc2);
    } else {
      const int64_t slot = 2 * win + (began ? 1 : 0);
      em_put(em_ws<DT>(a.ws, slot, a, cb), v);
      if (MODE == EM_CLIP && a.out2 != nullptr) em_put(em_ws<DT>(a.ws_sq, slot, a, cb), acc2);
    }
    em_clear(v);
    em_clear(acc2);
  };
  auto close_sub = [&](int p) {
    const bool began = (sub & ((2ull << p) - 1)) != 0, crosses = p == n_live - 1 && sub_on;
    if (MODE == EM_NORM) {
      if (began && !crosses) {
        em_norm<DT>(a, (uint32_t)__builtin_amdgcn_readlane((int)row, run_head + 1),
                    __builtin_amdgcn_readlane(seg, p + 1), cb, sum);
      } else {
        em_put(em_ws<DT>(a.ws, 2 * win + (began ? 1 : 0), a, cb), sum);
      }
    } else if (began) {  // one that began before belongs to the window of its first row
      const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(c), p + 1));
      if (crosses) em_add(em_ws<DT>(a.whole, win, a, cb), sum);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float x = __fmul_rn(sum[i], a.scale);
        x = isfinite(x) ? __fmul_rn(f, x) : 0.f;
        acc[i] += x;
        acc2[i] = __builtin_fmaf(x, x, acc2[i]);
      }
    }
    em_clear(sum);
  };
  EmPiece<DT, AL> piece[EM_LOAD];
  for (int b = 0; b < n_live; b += EM_LOAD) {
#pragma unroll
    for (int q = 0; q < EM_LOAD; ++q) {
      const int p = b + q;
      if (p >= from && p < to) {
        const uint32_t r = (uint32_t)__builtin_amdgcn_readlane((int)row, p + 1);
        piece[q].load(a.g + (int64_t)r * a.ldg * ES, cb, a.width);
      }
    }
#pragma unroll
    for (int q = 0; q < EM_LOAD; ++q) {
      const int p = b + q;
      if (p >= n_live) break;
      if ((sub >> p) & 1) run_head = p;
      if (p >= from && p < to) {
        float v[V];
        piece[q].get(v);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += v[i];
      }
      if (MODE != EM_GRAD && ends(sub, p)) close_sub(p);
      if (MODE != EM_NORM && ends(tok, p)) close_token(p);
    }
  }
}

// Adds the partials of a run that begins in window `win` and crosses into the
// next ones: one workgroup per (window, 64 pieces), whose waves take the
// windows in turn.
template <int DT, bool AL, int MODE>
__global__ __launch_bounds__(64 * EM_WAVES) void k_embed_join(EmbedSum a) {
  constexpr int V = em_vec<DT>();
  const int64_t win = blockIdx.x / a.ncb;
  const int cb = (int)(blockIdx.x - win * a.ncb);
  const int lane = threadIdx.x & 63, wave = uniform_int(threadIdx.x >> 6);
  const int64_t p0 = win * EM_WIN, last = p0 + EM_WIN - 1;
  if (last + 1 >= a.n) return;
  const uint32_t key = a.keys[last];
  if (key == a.vocab || a.keys[last + 1] != key) return;
  int seg = 0;
  if (MODE == EM_NORM) {
    seg = a.row_seg[a.rows[last]];
    if (a.row_seg[a.rows[last + 1]] != seg) return;
  }
  auto same = [&](int64_t p) {
    return a.keys[p] == key && (MODE != EM_NORM || a.row_seg[a.rows[p]] == seg);
  };
  if (p0 > 0 && same(p0) && same(p0 - 1)) return;  // it began before
  // The run's last position: positions after it compare greater.
  int64_t lo = last + 1, hi = a.n - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (same(mid)) lo = mid; else hi = mid - 1;
  }
  const int64_t end = lo / EM_WIN;  // its last window
  __shared__ float red[2][EM_WAVES][64 * V];
  float v[V], q[V];
  em_clear(v);
  em_clear(q);
  const bool second = MODE == EM_CLIP && a.out2 != nullptr;
#pragma unroll 4
  for (int64_t w = win + 1 + wave; w <= end; w += EM_WAVES) em_add(em_ws<DT>(a.ws, 2 * w, a, cb), v);
  if (second)
    for (int64_t w = win + 1 + wave; w <= end; w += EM_WAVES) em_add(em_ws<DT>(a.ws_sq, 2 * w, a, cb), q);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    red[0][wave][i * 64 + lane] = v[i];
    red[1][wave][i * 64 + lane] = q[i];
  }
  __syncthreads();
  if (wave != 0) return;
  em_clear(v);
  em_clear(q);
  em_add(em_ws<DT>(a.ws, 2 * win + 1, a, cb), v);
  if (second) em_add(em_ws<DT>(a.ws_sq, 2 * win + 1, a, cb), q);
#pragma unroll
  for (int w = 0; w < EM_WAVES; ++w)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] += red[0][w][i * 64 + lane];
      q[i] += red[1][w][i * 64 + lane];
    }
  if (MODE != EM_NORM) {
    em_finish<DT, AL>(a, MODE, key, cb, v, q);
    return;
  }
  // The first row of the run: the first of this window's positions in it.
  int64_t h = p0;
  while (!same(h)) ++h;
  em_norm<DT>(a, a.rows[h], seg, cb, v);
  em_put(em_ws<DT>(a.whole, win, a, cb), v);
}

// Zeroes `bytes` bytes.
__global__ __launch_bounds__(256) void k_embed_zero(char* out, int64_t bytes) {
  const int64_t n16 = ((uintptr_t)out & 15) == 0 ? bytes / 16 : 0;
  const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, nt = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = t; i < n16; i += nt) odp_gstore((u32x4_t*)(out + 16 * i), u32x4_t{0, 0, 0, 0});
  for (int64_t i = 16 * n16 + t; i < bytes; i += nt) out[i] = 0;
}

int sort_passes(int64_t vocab, int& bits) {
  int need = 1;
  while ((vocab >> need) != 0) ++need;  // keys 0 .. vocab
  const int passes = (need + SORT_BITS - 1) / SORT_BITS;
  bits = (need + passes - 1) / passes;
  return passes;
}

int64_t sort_waves(int64_t n) { return (n + SORT_KEYS - 1) / SORT_KEYS; }
int64_t pieces(int dtype, int64_t width) {
  const int64_t per = 64 * (dtype == ODP_DTYPE_F32 ? 4 : 8);
  return (width + per - 1) / per;
}
int64_t windows(int64_t n) { return (n + EM_WIN - 1) / EM_WIN; }

int check_rows(const char* what, int dtype, int64_t n, int64_t width, int64_t vocab, int64_t ld) {
  if (dtype != ODP_DTYPE_F32 && dtype != ODP_DTYPE_BF16 && dtype != ODP_DTYPE_F16) {
    odp_set_error("%s: rows must be float32, bfloat16 or float16 (dtype %d)", what, dtype);
    return ODP_ERR_UNSUPPORTED;
  }
  if (n < 0 || n >= ((int64_t)1 << 31) - 64 || width <= 0 || width >= ((int64_t)1 << 24) || vocab <= 0 ||
      vocab >= ((int64_t)1 << 31) - 1 || ld < width) {
    odp_set_error("%s: invalid sizes (n %lld, width %lld, vocab %lld, pitch %lld)", what, (long long)n,
                  (long long)width, (long long)vocab, (long long)ld);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  return ODP_OK;
}

int check_grid(const char* what, int64_t blocks) {
  if (blocks >= (int64_t)1 << 24) {
    odp_set_error("%s: the launch needs %lld workgroups", what, (long long)blocks);
    return ODP_ERR_UNSUPPORTED;
  }
  return ODP_OK;
}

template <int MODE>
int launch_sum(const char* what, hipStream_t s, int dtype, bool aligned, const EmbedSum& a) {
  const int64_t items = windows(a.n) * a.ncb;
  if (int rc = check_grid(what, items)) return rc;
  const dim3 grid((unsigned)((items + EM_WAVES - 1) / EM_WAVES)), block(64 * EM_WAVES), jgrid((unsigned)items);
#define ODP_EM(DT, AL)                                                   \
  do {                                                                   \
    hipLaunchKernelGGL((k_embed_sum<DT, AL, MODE>), grid, block, 0, s, a); \
    hipLaunchKernelGGL((k_embed_join<DT, AL, MODE>), jgrid, block, 0, s, a); \
  } while (0)
  if (dtype == ODP_DTYPE_F32) {
    if (aligned) ODP_EM(ODP_DTYPE_F32, true); else ODP_EM(ODP_DTYPE_F32, false);
  } else if (dtype == ODP_DTYPE_BF16) {
    if (aligned) ODP_EM(ODP_DTYPE_BF16, true); else ODP_EM(ODP_DTYPE_BF16, false);
  } else {
    if (aligned) ODP_EM(ODP_DTYPE_F16, true); else ODP_EM(ODP_DTYPE_F16, false);
  }
#undef ODP_EM
  return odp_check_launch(what);
}

bool rows_aligned(int dtype, const void* p, int64_t ld, int64_t width) {
  const int64_t es = dtype == ODP_DTYPE_F32 ? 4 : 2;
  return ((uintptr_t)p & 15) == 0 && ld * es % 16 == 0 && width * es % 16 == 0;
}

int launch_zero(const char* what, hipStream_t s, void* out, int64_t bytes) {
  int64_t blocks = (bytes + 16383) / 16384;
  if (blocks > 4096) blocks = 4096;
  if (blocks > 0) hipLaunchKernelGGL(k_embed_zero, dim3((unsigned)blocks), dim3(256), 0, s, (char*)out, bytes);
  return odp_check_launch(what);
}

}  // namespace

extern "C" int odp_embed_rows(odp_stream_t stream, int dtype, const void* tokens, int token_bytes, int64_t n,
                              const void* weight, int64_t ldw, int64_t vocab, int64_t width, float scale, void* out) {
  if (int rc = check_rows("odp_embed_rows", dtype, n, width, vocab, ldw)) return rc;
  if (token_bytes != 4 && token_bytes != 8) {
    odp_set_error("odp_embed_rows: tokens of %d bytes", token_bytes);
    return ODP_ERR_UNSUPPORTED;
  }
  if (n == 0) return ODP_OK;
  if (tokens == nullptr || weight == nullptr || out == nullptr) {
    odp_set_error("odp_embed_rows: null pointer");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const int ncb = (int)pieces(dtype, width);
  const int64_t blocks = (n * ncb + EM_WAVES - 1) / EM_WAVES;
  if (int rc = check_grid("odp_embed_rows", blocks)) return rc;
  const bool al = rows_aligned(dtype, weight, ldw, width) && ((uintptr_t)out & 15) == 0;
  const hipStream_t s = odp_hip_stream(stream);
#define ODP_ER(DT, AL)                                                                                              \
  hipLaunchKernelGGL((k_embed_rows<DT, AL>), dim3((unsigned)blocks), dim3(64 * EM_WAVES), 0, s, tokens,              \
                     token_bytes == 8 ? 1 : 0, n, (const char*)weight, ldw, vocab, (int)width, ncb, scale, out)
  if (dtype == ODP_DTYPE_F32) {
    if (al) ODP_ER(ODP_DTYPE_F32, true); else ODP_ER(ODP_DTYPE_F32, false);
  } else if (dtype == ODP_DTYPE_BF16) {
    if (al) ODP_ER(ODP_DTYPE_BF16, true); else ODP_ER(ODP_DTYPE_BF16, false);
  } else {
    if (al) ODP_ER(ODP_DTYPE_F16, true); else ODP_ER(ODP_DTYPE_F16, false);
  }
#undef ODP_ER
  return odp_check_launch("odp_embed_rows");
}

extern "C" int64_t odp_token_sort_scratch(int64_t n, int64_t vocab) {
  if (n <= 0 || vocab <= 0) return 0;
  int bits;
  sort_passes(vocab, bits);
  return 4 * (2 * n + (n > SORT_SMALL ? ((int64_t)1 << bits) * sort_waves(n) : 0));
}

extern "C" int odp_token_sort(odp_stream_t stream, const void* tokens, int token_bytes, int64_t n, int64_t vocab,
                              int64_t padding, const int32_t* seg_row_start, const int32_t* seg_row_len,
                              int32_t n_seg, void* scratch, uint32_t* keys, uint32_t* rows, int32_t* row_seg) {
  if (int rc = check_rows("odp_token_sort", ODP_DTYPE_F32, n, 1, vocab, 1)) return rc;
  if (token_bytes != 4 && token_bytes != 8) {
    odp_set_error("odp_token_sort: tokens of %d bytes", token_bytes);
    return ODP_ERR_UNSUPPORTED;
  }
  if (n == 0) return ODP_OK;
  if (tokens == nullptr || scratch == nullptr || keys == nullptr || rows == nullptr || n_seg < 0 ||
      (seg_row_start != nullptr && (seg_row_len == nullptr || row_seg == nullptr))) {
    odp_set_error("odp_token_sort: null pointer or negative n_seg (%d)", n_seg);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  int bits;
  const int passes = sort_passes(vocab, bits);
  SortIn a{tokens, token_bytes == 8 ? 1 : 0, n, vocab, padding, seg_row_start, seg_row_len, n_seg, row_seg};
  uint32_t* k1 = (uint32_t*)scratch;
  uint32_t* r1 = k1 + n;
  const hipStream_t s = odp_hip_stream(stream);
  if (n <= SORT_SMALL) {
    hipLaunchKernelGGL(k_sort_small, dim3(1), dim3(64 * SORT_WAVES), 0, s, a, passes, bits, keys, rows, k1, r1);
    return odp_check_launch("odp_token_sort");
  }
  uint32_t* counts = r1 + n;
  const int nw = (int)sort_waves(n);
  const dim3 grid((unsigned)((nw + EM_WAVES - 1) / EM_WAVES)), block(64 * EM_WAVES);
  for (int p = 0; p < passes; ++p) {
    const bool to0 = ((passes - 1 - p) & 1) == 0;
    const uint32_t* ik = to0 ? k1 : keys;
    const uint32_t* ir = to0 ? r1 : rows;
    uint32_t* ok = to0 ? keys : k1;
    uint32_t* orow = to0 ? rows : r1;
    hipLaunchKernelGGL(k_sort_count, grid, block, 0, s, a, ik, p == 0 ? 1 : 0, p * bits, bits, counts, nw);
    hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(1024), 0, s, counts, ((int64_t)1 << bits) * nw);
    hipLaunchKernelGGL(k_sort_scatter, grid, block, 0, s, a, ik, ir, p == 0 ? 1 : 0, p * bits, bits, counts, nw, ok,
                       orow);
  }
  return odp_check_launch("odp_token_sort");
}

extern "C" int64_t odp_embed_sum_scratch(int dtype, int64_t n, int64_t width, int second) {
  if (n <= 0 || width <= 0) return 0;
  const int64_t row = pieces(dtype, width) * 64 * (dtype == ODP_DTYPE_F32 ? 4 : 8);
  return 4 * row * windows(n) * (second ? 4 : 2);
}

extern "C" int64_t odp_embed_pieces(int dtype, int64_t width) { return width > 0 ? pieces(dtype, width) : 0; }

extern "C" int odp_embed_grad(odp_stream_t stream, int dtype, const void* g, int64_t ldg, int64_t n, int64_t width,
                              const uint32_t* keys, const uint32_t* rows, int64_t vocab, float scale, void* scratch,
                              void* out) {
  if (int rc = check_rows("odp_embed_grad", dtype, n, width, vocab, ldg)) return rc;
  if (out == nullptr || (n > 0 && (g == nullptr || keys == nullptr || rows == nullptr || scratch == nullptr))) {
    odp_set_error("odp_embed_grad: null pointer");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const hipStream_t s = odp_hip_stream(stream);
  if (int rc = launch_zero("odp_embed_grad", s, out, vocab * width * (dtype == ODP_DTYPE_F32 ? 4 : 2))) return rc;
  if (n == 0) return ODP_OK;
  EmbedSum a{};
  a.g = (const char*)g;
  a.ldg = ldg;
  a.n = n;
  a.width = (int)width;
  a.ncb = (int)pieces(dtype, width);
  a.keys = keys;
  a.rows = rows;
  a.vocab = (uint32_t)vocab;
  a.scale = scale;
  a.ws = (float*)scratch;
  a.out = out;
  a.odt = dtype;
  a.normalize_by = 1.0f;
  return launch_sum<EM_GRAD>("odp_embed_grad", s, dtype,
                             rows_aligned(dtype, g, ldg, width) && ((uintptr_t)out & 15) == 0, a);
}

extern "C" int odp_embed_sqnorm(odp_stream_t stream, int dtype, const void* g, int64_t ldg, int64_t n, int64_t width,
                                const uint32_t* keys, const uint32_t* rows, const int32_t* row_seg, int64_t vocab,
                                float scale, const int32_t* seg_row_start, const int32_t* seg_example, void* scratch,
                                float* whole, double* part, int64_t part_stride, int64_t slot, int64_t* nf_flag) {
  if (int rc = check_rows("odp_embed_sqnorm", dtype, n, width, vocab, ldg)) return rc;
  if (n == 0) return ODP_OK;
  if (g == nullptr || keys == nullptr || rows == nullptr || row_seg == nullptr || seg_row_start == nullptr ||
      seg_example == nullptr || scratch == nullptr || whole == nullptr || part == nullptr || nf_flag == nullptr ||
      slot < 0 || slot >= part_stride) {
    odp_set_error("odp_embed_sqnorm: null pointer or slot %lld outside [0, %lld)", (long long)slot,
                  (long long)part_stride);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  EmbedSum a{};
  a.g = (const char*)g;
  a.ldg = ldg;
  a.n = n;
  a.width = (int)width;
  a.ncb = (int)pieces(dtype, width);
  a.keys = keys;
  a.rows = rows;
  a.row_seg = row_seg;
  a.vocab = (uint32_t)vocab;
  a.scale = scale;
  a.ws = (float*)scratch;
  a.whole = whole;
  a.part = part;
  a.part_stride = part_stride;
  a.slot = slot;
  a.sstart = seg_row_start;
  a.sex = seg_example;
  a.nf_flag = nf_flag;
  return launch_sum<EM_NORM>("odp_embed_sqnorm", odp_hip_stream(stream), dtype, rows_aligned(dtype, g, ldg, width), a);
}

extern "C" int odp_embed_clipped_sum(odp_stream_t stream, int dtype, const void* g, int64_t ldg, int64_t n,
                                     int64_t width, const uint32_t* keys, const uint32_t* rows,
                                     const int32_t* row_seg, int64_t vocab, float scale, const int32_t* seg_example,
                                     void* scratch, const float* whole, const double* scales, float normalize_by,
                                     int out_dtype, void* out, void* out2) {
  if (int rc = check_rows("odp_embed_clipped_sum", dtype, n, width, vocab, ldg)) return rc;
  if (out_dtype < ODP_DTYPE_F32 || out_dtype > ODP_DTYPE_F64) {
    odp_set_error("odp_embed_clipped_sum: out_dtype %d", out_dtype);
    return ODP_ERR_UNSUPPORTED;
  }
  if (out == nullptr || (n > 0 && (g == nullptr || keys == nullptr || rows == nullptr || row_seg == nullptr ||
                                   seg_example == nullptr || scratch == nullptr || whole == nullptr ||
                                   scales == nullptr))) {
    odp_set_error("odp_embed_clipped_sum: null pointer");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const hipStream_t s = odp_hip_stream(stream);
  const int64_t bytes = vocab * width * odp_dtype_size(out_dtype);
  if (int rc = launch_zero("odp_embed_clipped_sum", s, out, bytes)) return rc;
  if (out2 != nullptr)
    if (int rc = launch_zero("odp_embed_clipped_sum", s, out2, bytes)) return rc;
  if (n == 0) return ODP_OK;
  EmbedSum a{};
  a.g = (const char*)g;
  a.ldg = ldg;
  a.n = n;
  a.width = (int)width;
  a.ncb = (int)pieces(dtype, width);
  a.keys = keys;
  a.rows = rows;
  a.row_seg = row_seg;
  a.vocab = (uint32_t)vocab;
  a.scale = scale;
  a.ws = (float*)scratch;
  a.ws_sq = a.ws + odp_embed_sum_scratch(dtype, n, width, 0) / 4;
  a.whole = (float*)whole;
  a.out = out;
  a.out2 = out2;
  a.odt = out_dtype;
  a.sex = seg_example;
  a.scales = scales;
  a.normalize_by = normalize_by;
  return launch_sum<EM_CLIP>("odp_embed_clipped_sum", s, dtype,
                             rows_aligned(dtype, g, ldg, width) && ((uintptr_t)out & 15) == 0 &&
                                 ((uintptr_t)out2 & 15) == 0,
                             a);
}
