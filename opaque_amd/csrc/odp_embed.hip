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
//
// 32768 tokens of a 128256 x 4096 bfloat16 table, lookup and gradient: 340 us
// for 1.86 GB (5.5 TB/s; a copy runs at 5.2).  A clip step's norms and sum over
// 16384 of them: 285 us for 1.19 GB, 1.05 GB of it the table's zeros.
#include <cmath>

#include "odp_internal.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

constexpr int EM_WIN = 32;   // sorted positions per window, at most
constexpr int EM_LOAD = 8;   // rows in flight per wave
constexpr int EM_WAVES = 4;  // waves per workgroup

enum { EM_GRAD = 0, EM_NORM = 1, EM_CLIP = 2, EM_CLIP2 = 3 };  // CLIP2: with second moments

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

// The lane's 16 bytes of a row piece.  NT: a non-temporal load, for gradient
// rows, which a pass reads once (32768 x 4096 bfloat16: 85 us, 125 through the
// caches; the two passes of a clip step over 16384 x 4096: 71 us, 90); table
// rows, of which frequent tokens' come again, are read through the caches
// (66 us, 97).
template <int DT, bool AL, bool NT = false>
struct EmPiece {
  static constexpr int V = em_vec<DT>();
  u32x4_t w;
  __device__ __forceinline__ void load(const char* p, int cb, int width) {
    if constexpr (AL) {
      const int c = em_col<DT, AL>(cb, 0);
      w = u32x4_t{0, 0, 0, 0};
      const ODP_GMEM u32x4_t* src =
          (const ODP_GMEM u32x4_t*)(const ODP_GMEM void*)(p + (int64_t)c * (DT == ODP_DTYPE_F32 ? 4 : 2));
      if (c < width) w = NT ? __builtin_nontemporal_load(src) : *src;
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
// Lookup.  A wave takes EM_ITEMS (row, 64 pieces of 16 bytes) items, their
// loads in flight together; a token outside the table gives a row of NaN.
// 32768 rows of 8 KB in 83 us (6.5 TB/s, a fifth of them one token's); 16
// rows in 3.6 us, which is the launch.
// ---------------------------------------------------------------------------
constexpr int EM_ITEMS = 4;
template <int DT, bool AL>
__global__ __launch_bounds__(64 * EM_WAVES) void k_embed_rows(const void* __restrict__ tokens, int wide, int64_t n,
                                                              const char* __restrict__ weight, int64_t ldw,
                                                              int64_t vocab, int width, int ncb, float scale,
                                                              void* __restrict__ out) {
  constexpr int V = em_vec<DT>();
  const int64_t first = ((int64_t)blockIdx.x * EM_WAVES + uniform_int(threadIdx.x >> 6)) * EM_ITEMS;
  EmPiece<DT, AL> p[EM_ITEMS];
  int64_t row[EM_ITEMS];
  int cb[EM_ITEMS];
  bool ok[EM_ITEMS];
#pragma unroll
  for (int q = 0; q < EM_ITEMS; ++q) {
    row[q] = (first + q) / ncb;
    cb[q] = (int)(first + q - row[q] * ncb);
    const int64_t t = row[q] < n ? token_at(tokens, wide, row[q]) : -1;
    ok[q] = t >= 0 && t < vocab;
    if (ok[q]) p[q].load(weight + t * ldw * (DT == ODP_DTYPE_F32 ? 4 : 2), cb[q], width);
  }
#pragma unroll
  for (int q = 0; q < EM_ITEMS; ++q) {
    if (row[q] >= n) return;
    float v[V];
    if (ok[q]) {
      p[q].get(v);
      if (scale != 1.0f) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = __fmul_rn(v[i], scale);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = __uint_as_float(0x7fc00000u);
    }
    em_store<DT, AL>(out, DT, row[q], width, cb[q], v);
  }
}

// ---------------------------------------------------------------------------
// Stable sort of the positions by token: least-significant-digit radix passes
// of up to SORT_BITS bits.  A wave owns SORT_KEYS consecutive positions; its
// digit counts, summed exclusively over (digit, wave), are where its keys go,
// and equal digits within 64 keys are ranked by ballots, so order among equal
// tokens is kept.  Dropped positions (outside the table, padding, rows
// outside every segment) get the key `vocab` and end up last.  Bound by latency,
// not bytes: 16384 positions take two passes of 8 and 14 us, 1023 in one
// workgroup 8 us.  The launches therefore zero the output table on the side:
// with a table of 1.05 GB the two passes take 2 x (48 + 31) us, 6.6 TB/s of it.
// ---------------------------------------------------------------------------
constexpr int SORT_BITS = 9, SORT_BINS = 1 << SORT_BITS;
constexpr int SORT_KEYS = 512;                            // positions a wave holds at a time
constexpr int SORT_NW = 128;                              // waves of the other, at most
constexpr int SORT_WAVES = 16;                            // waves of the one-workgroup sort
constexpr int64_t SORT_SMALL = SORT_WAVES * SORT_KEYS;    // positions it takes
constexpr int SORT_SEGS = 1024;                           // segments it keeps in LDS

// Memory that the sort's launches zero beside their own work, with
// workgroups the sort leaves idle: pieces [first, first + count) of
// ZERO_BYTES of 16 bytes a thread, one after the other in address order (a
// table of 1.05 GB: 152 us, 6.9 TB/s; with 1024 to 16384 workgroups striding
// over it 195-280 us).
struct ZeroShare {
  char* at;
  int64_t bytes;
  int64_t first, count;
  int per;  // pieces a workgroup
};

__device__ __forceinline__ void zero_pieces(const ZeroShare& z, int64_t wg) {
  const int64_t size = (int64_t)blockDim.x * 16;
  for (int q = 0; q < z.per; ++q) {
    const int64_t p = wg * z.per + q;
    if (p >= z.count) return;
    const int64_t b = (z.first + p) * size + 16 * (int64_t)threadIdx.x;
    if (b + 16 <= z.bytes && ((uintptr_t)z.at & 15) == 0)
      odp_gstore((u32x4_t*)(z.at + b), u32x4_t{0, 0, 0, 0});
    else
      for (int64_t i = b; i < b + 16 && i < z.bytes; ++i) z.at[i] = 0;
  }
}

struct SortIn {
  const void* tokens;
  int wide;  // tokens are int64
  int64_t n, vocab, padding;
  const int32_t* sstart;  // segments (nullptr: every row counts)
  const int32_t* slen;
  int n_seg;
  int32_t* row_seg;  // [n] each row's segment, written when the keys are counted first (with segments)
  int32_t* seg_of;   // [n] the sorted positions' segments, written in the last (with segments)
  ZeroShare zero;
};

// `starts`: the segments' starts, in LDS where they fit.
__device__ __forceinline__ uint32_t sort_key(const SortIn& a, const int32_t* starts, int64_t i, bool record) {
  const int64_t t = token_at(a.tokens, a.wide, i);
  bool ok = t >= 0 && t < a.vocab && t != a.padding;
  if (a.sstart != nullptr) {
    int lo = 0, hi = a.n_seg - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)starts[mid] <= i) lo = mid; else hi = mid - 1;
    }
    const bool in = a.n_seg > 0 && i >= starts[lo] && i < (int64_t)starts[lo] + a.slen[lo];
    ok = ok && in;
    if (record) a.row_seg[i] = in ? lo : 0;
  }
  return ok ? (uint32_t)t : (uint32_t)a.vocab;
}

// Positions [lo, hi), at most 64 R, in the wave's registers: all loads in flight together.
template <int R, typename Key>
__device__ __forceinline__ void sort_load(uint32_t (&v)[R], int64_t lo, int64_t hi, Key key) {
#pragma unroll
  for (int q = 0; q < R; ++q) {
    const int64_t i = lo + 64 * q + (threadIdx.x & 63);
    v[q] = i < hi ? key(i) : 0u;
  }
}

// Adds the digits of the wave's keys to its counts h.
template <int R>
__device__ __forceinline__ void sort_count(uint32_t* h, int64_t lo, int64_t hi, int shift, uint32_t mask,
                                           const uint32_t (&key)[R]) {
#pragma unroll
  for (int q = 0; q < R; ++q)
    if (lo + 64 * q + (threadIdx.x & 63) < hi) atomicAdd(&h[(key[q] >> shift) & mask], 1u);
}

// Sends them to where h says, in order.
template <int R>
__device__ __forceinline__ void sort_scatter(uint32_t* h, int64_t lo, int64_t hi, int shift, int bits,
                                             const uint32_t (&key)[R], const uint32_t (&row)[R],
                                             uint32_t* ok, uint32_t* orow, const int32_t* row_seg, int32_t* seg_of) {
  const int lane = threadIdx.x & 63;
  const uint64_t before = (1ull << lane) - 1;
#pragma unroll
  for (int q = 0; q < R; ++q) {
    const bool on = lo + 64 * q + lane < hi;
    const uint32_t k = key[q], d = (k >> shift) & ((1u << bits) - 1);
    uint64_t peers = __builtin_amdgcn_ballot_w64(on);
    if (peers == 0) break;
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
      orow[to] = row[q];
      if (seg_of != nullptr) seg_of[to] = row_seg[row[q]];
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
template <int R>
__global__ __launch_bounds__(64 * SORT_WAVES) void k_sort_small(SortIn a, int passes, int bits, uint32_t* k0,
                                                                uint32_t* r0, uint32_t* k1, uint32_t* r1) {
  __shared__ uint32_t hist[SORT_WAVES][SORT_BINS];
  __shared__ uint32_t red[SORT_WAVES];
  if (blockIdx.x > 0) {
    zero_pieces(a.zero, blockIdx.x - 1);
    return;
  }
  __shared__ int32_t seg_start[SORT_SEGS];
  const bool kept = a.sstart != nullptr && a.n_seg <= SORT_SEGS;
  if (kept)
    for (int i = threadIdx.x; i < a.n_seg; i += blockDim.x) seg_start[i] = a.sstart[i];
  const int32_t* starts = kept ? seg_start : a.sstart;
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
    // The wave's positions in rounds of 64 R, their loads in flight together.
    uint32_t key[R], row[R];
    for (int64_t c = lo; c < hi; c += 64 * R) {
      sort_load(key, c, hi, [&](int64_t i) { return p == 0 ? sort_key(a, starts, i, a.sstart != nullptr) : ik[i]; });
      sort_count(hist[wave], c, hi, shift, (uint32_t)bins - 1, key);
    }
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
    for (int64_t c = lo; c < hi; c += 64 * R) {
      sort_load(key, c, hi, [&](int64_t i) { return p == 0 ? sort_key(a, starts, i, false) : ik[i]; });
      sort_load(row, c, hi, [&](int64_t i) { return p == 0 ? (uint32_t)i : ir[i]; });
      sort_scatter(hist[wave], c, hi, shift, bits, key, row, ok, orow, a.row_seg,
                   p == passes - 1 ? a.seg_of : nullptr);
    }
    __threadfence_block();
    __syncthreads();
  }
}

// The sort of more positions: per pass a launch that counts, counts[wave][digit],
// and one that sums the counts and scatters.
__global__ __launch_bounds__(64 * EM_WAVES) void k_sort_count(SortIn a, const uint32_t* ik, int first, int shift,
                                                              int bits, uint32_t* counts, int nw, int64_t per) {
  __shared__ uint32_t hist[EM_WAVES][SORT_BINS];
  const int own = (nw + EM_WAVES - 1) / EM_WAVES;
  if ((int)blockIdx.x >= own) {
    zero_pieces(a.zero, blockIdx.x - own);
    return;
  }
  const int wave = threadIdx.x >> 6, bins = 1 << bits;
  for (int i = threadIdx.x; i < EM_WAVES * SORT_BINS; i += blockDim.x) (&hist[0][0])[i] = 0;
  __syncthreads();
  const int w = blockIdx.x * EM_WAVES + wave;
  const int64_t lo = min(a.n, w * per), hi = min(a.n, lo + per);
  for (int64_t c = lo; c < hi; c += SORT_KEYS) {
    uint32_t key[SORT_KEYS / 64];
    sort_load(key, c, hi, [&](int64_t i) { return first ? sort_key(a, a.sstart, i, a.sstart != nullptr) : ik[i]; });
    sort_count(hist[wave], c, hi, shift, (uint32_t)bins - 1, key);
  }
  if (w < nw)
    for (int d = threadIdx.x & 63; d < bins; d += 64) counts[(int64_t)w * SORT_BINS + d] = hist[wave][d];
}

__global__ __launch_bounds__(64 * EM_WAVES) void k_sort_scatter(SortIn a, const uint32_t* ik, const uint32_t* ir,
                                                                int first, int shift, int bits,
                                                                const uint32_t* counts, int nw, int64_t per,
                                                                uint32_t* ok, uint32_t* orow, int last) {
  __shared__ uint32_t hist[EM_WAVES][SORT_BINS];
  __shared__ uint32_t red[EM_WAVES];
  const int own = (nw + EM_WAVES - 1) / EM_WAVES;
  if ((int)blockIdx.x >= own) {
    zero_pieces(a.zero, blockIdx.x - own);
    return;
  }
  const int wave = threadIdx.x >> 6;
  const int w0 = blockIdx.x * EM_WAVES;
  static_assert(SORT_BINS == 2 * 64 * EM_WAVES, "two digits a thread");
  // Where this workgroup's waves' keys of digits 2 t and 2 t + 1 go: after
  // every smaller digit's and the earlier waves' of the same (digits past
  // the pass's have no counts: they are not read).
  const bool on = 2 * (int)threadIdx.x < (1 << bits);
  u32x2_t all = {0, 0}, before = {0, 0}, mine[EM_WAVES];
#pragma unroll
  for (int j = 0; j < EM_WAVES; ++j) mine[j] = u32x2_t{0, 0};
  if (on) {
    const u32x2_t* at = (const u32x2_t*)counts + threadIdx.x;
#pragma unroll 16
    for (int w = 0; w < nw; ++w) {
      const u32x2_t c = at[(int64_t)w * (SORT_BINS / 2)];
      all = all + c;
      if (w < w0) before = before + c;
    }
#pragma unroll
    for (int j = 0; j < EM_WAVES; ++j)
      if (w0 + j < nw) mine[j] = at[(int64_t)(w0 + j) * (SORT_BINS / 2)];
  }
  uint32_t total;
  const uint32_t below = block_exclusive(all[0] + all[1], EM_WAVES, red, total);
  u32x2_t to = {below + before[0], below + all[0] + before[1]};
#pragma unroll
  for (int j = 0; j < EM_WAVES; ++j) {
    hist[j][2 * threadIdx.x] = to[0];
    hist[j][2 * threadIdx.x + 1] = to[1];
    to = to + mine[j];
  }
  __syncthreads();
  const int64_t lo = min(a.n, (w0 + wave) * per), hi = min(a.n, lo + per);
  for (int64_t c = lo; c < hi; c += SORT_KEYS) {
    uint32_t key[SORT_KEYS / 64], row[SORT_KEYS / 64];
    sort_load(key, c, hi, [&](int64_t i) { return first ? sort_key(a, a.sstart, i, false) : ik[i]; });
    sort_load(row, c, hi, [&](int64_t i) { return first ? (uint32_t)i : ir[i]; });
    sort_scatter(hist[wave], c, hi, shift, bits, key, row, ok, orow, a.row_seg, last ? a.seg_of : nullptr);
  }
}

// ---------------------------------------------------------------------------
// Sums over the sorted positions.
// ---------------------------------------------------------------------------
struct EmbedSum {
  const char* g;  // gradient rows
  int64_t ldg;    // elements
  int64_t n;
  int win;      // sorted positions per window: 8, 16 or 32
  int grouped;  // whether k_embed_group has run
  int width, ncb;
  const uint32_t* keys;   // sorted tokens, `vocab` for dropped positions
  const uint32_t* rows;   // the positions, sorted
  const int32_t* seg_of;  // NORM, CLIP: the sorted positions' segments
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

// Adds slot `slot` of windows first, first + step, .. last, JOIN_LOAD rows in flight.
constexpr int JOIN_LOAD = 8, JOIN_GROUP = 16;
template <int DT>
__device__ __forceinline__ void em_gather(const float* ws, int64_t first, int64_t last, int step, int slot,
                                          const EmbedSum& a, int cb, float (&v)[em_vec<DT>()]) {
  constexpr int V = em_vec<DT>();
  for (int64_t w = first; w <= last; w += JOIN_LOAD * step) {
    f32x4_t x[JOIN_LOAD][V / 4];
#pragma unroll
    for (int k = 0; k < JOIN_LOAD; ++k)
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        if (w + k * step <= last)
          x[k][i] = *(const ODP_GMEM f32x4_t*)(const ODP_GMEM void*)(em_ws<DT>((float*)ws, 2 * (w + k * step) + slot,
                                                                               a, cb) +
                                                                     4 * i);
#pragma unroll
    for (int k = 0; k < JOIN_LOAD; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (w + k * step <= last) v[i] += x[k][i / 4][i % 4];
  }
}

// Adds the partials of windows first .. last of a run that ends in `last`,
// whole groups by their sums (a.grouped).
template <int DT>
__device__ __forceinline__ void em_join(const float* ws, int64_t first, int64_t last, const EmbedSum& a, int cb,
                                        float (&v)[em_vec<DT>()]) {
  const int64_t g0 = (first + JOIN_GROUP - 1) / JOIN_GROUP * JOIN_GROUP, g1 = last / JOIN_GROUP * JOIN_GROUP;
  if (!a.grouped || g0 >= g1) {
    em_gather<DT>(ws, first, last, 1, 0, a, cb, v);
    return;
  }
  em_gather<DT>(ws, first, g0 - 1, 1, 0, a, cb, v);
  em_gather<DT>(ws, g0, g1 - 1, JOIN_GROUP, 1, a, cb, v);  // windows before g1 lie wholly inside the run
  em_gather<DT>(ws, g1, last, 1, 0, a, cb, v);
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
  // Across the lanes on the VALU: a window may close a run at every position.
  s = rows_sum4(row_sum16(s));
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
  if (mode == EM_CLIP2) {
    if (a.normalize_by != 1.0f) {
#pragma unroll
      for (int i = 0; i < V; ++i) q[i] = __fdiv_rn(q[i], a.normalize_by);
    }
    em_store<DT, AL>(a.out2, a.odt, key, a.width, cb, q);
  }
}

// One wave per (window, 64 pieces of 16 bytes of the rows).  0.27 GB of gradient
// rows (32768 of 8 KB) read and their tokens' sums written in 86 us; the two
// passes of a clip step over 16384 rows 36 and 37 us.
template <int DT, bool AL, int MODE>
__global__ __launch_bounds__(64 * EM_WAVES) void k_embed_sum(EmbedSum a) {
  constexpr int V = em_vec<DT>(), ES = DT == ODP_DTYPE_F32 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * EM_WAVES + uniform_int(threadIdx.x >> 6);
  const int64_t win = item / a.ncb, p0 = win * a.win;
  const int cb = (int)(item - win * a.ncb);
  if (p0 >= a.n) return;
  // Lane l holds position p0 - 1 + l: the window, the one before and the one after.
  const int64_t pos = p0 - 1 + lane;
  const bool in = pos >= 0 && pos < a.n && lane <= a.win + 1;
  const uint32_t key = in ? a.keys[pos] : a.vocab;
  const uint32_t row = in ? a.rows[pos] : 0u;
  const int seg = MODE != EM_GRAD && in ? a.seg_of[pos] : 0;
  float c = 0.f;
  if (MODE >= EM_CLIP && key != a.vocab) c = (float)a.scales[a.sex[seg]];
  const uint32_t pkey = __shfl_up(key, 1);
  const int pseg = __shfl_up(seg, 1);
  // Bit p: position p0 + p counts / starts a token's run / an (example, token)
  // run (bit a.win: the position after the window).
  const bool live_l = key != a.vocab && lane >= 1;
  const uint64_t live = __builtin_amdgcn_ballot_w64(live_l) >> 1;
  const uint64_t tok = __builtin_amdgcn_ballot_w64(live_l && key != pkey) >> 1;
  const uint64_t sub = MODE == EM_GRAD ? tok : __builtin_amdgcn_ballot_w64(live_l && (key != pkey || seg != pseg)) >> 1;
  const int n_live = __popcll(live & ((1ull << a.win) - 1));  // dropped positions come last
  if (n_live == 0) return;
  const bool more = (live >> a.win) & 1;
  const bool tok_on = more && !((tok >> a.win) & 1);  // the last run goes on in the next window
  const bool sub_on = more && !((sub >> a.win) & 1);
  // Rows of (example, token) runs that cross windows were added by the NORM
  // pass: CLIP takes their sum from `whole` at the run's first window.
  int from = 0, to = n_live;
  if (MODE >= EM_CLIP) {
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
      if (MODE == EM_CLIP2) em_put(em_ws<DT>(a.ws_sq, slot, a, cb), acc2);
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
        if (MODE == EM_CLIP2) acc2[i] = __builtin_fmaf(x, x, acc2[i]);
      }
    }
    em_clear(sum);
  };
  EmPiece<DT, AL, true> piece[EM_LOAD];
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

// Runs of hundreds of windows (a padding token's) are joined in two steps:
// first, the partials of every JOIN_GROUP windows that lie wholly inside a
// run, into the group's first window's second slot (unused there).
template <int DT, int MODE>
__global__ __launch_bounds__(64 * EM_WAVES) void k_embed_group(EmbedSum a) {
  constexpr int V = em_vec<DT>();
  const int64_t item = (int64_t)blockIdx.x * EM_WAVES + uniform_int(threadIdx.x >> 6);
  const int64_t group = item / a.ncb, win = group * JOIN_GROUP;
  const int cb = (int)(item - group * a.ncb);
  const int64_t first = win * a.win, last = first + JOIN_GROUP * a.win - 1;
  if (win == 0 || last >= a.n) return;
  const uint32_t key = a.keys[first];
  if (key == a.vocab || a.keys[first - 1] != key || a.keys[last] != key) return;
  if (MODE == EM_NORM && (a.seg_of[first - 1] != a.seg_of[first] || a.seg_of[last] != a.seg_of[first])) return;
  float v[V];
  em_clear(v);
  em_gather<DT>(a.ws, win, win + JOIN_GROUP - 1, 1, 0, a, cb, v);
  em_put(em_ws<DT>(a.ws, 2 * win + 1, a, cb), v);
  if (MODE == EM_CLIP2) {
    em_clear(v);
    em_gather<DT>(a.ws_sq, win, win + JOIN_GROUP - 1, 1, 0, a, cb, v);
    em_put(em_ws<DT>(a.ws_sq, 2 * win + 1, a, cb), v);
  }
}

// Adds the partials of a run that begins in a window and crosses into the
// next ones, one wave per (window, 64 pieces).  4 us where none is long, 7-12
// for runs of thousands.
template <int DT, bool AL, int MODE>
__global__ __launch_bounds__(64 * EM_WAVES) void k_embed_join(EmbedSum a) {
  constexpr int V = em_vec<DT>();
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * EM_WAVES + uniform_int(threadIdx.x >> 6);
  const int64_t win = item / a.ncb;
  const int cb = (int)(item - win * a.ncb);
  const int64_t p0 = win * a.win, last = p0 + a.win - 1;
  if (last + 1 >= a.n) return;
  const uint32_t key = a.keys[last];
  if (key == a.vocab || a.keys[last + 1] != key) return;
  int seg = 0;
  if (MODE == EM_NORM) {
    seg = a.seg_of[last];
    if (a.seg_of[last + 1] != seg) return;
  }
  auto same = [&](int64_t p) { return a.keys[p] == key && (MODE != EM_NORM || a.seg_of[p] == seg); };
  if (p0 > 0 && same(p0) && same(p0 - 1)) return;  // it began before
  // The run's last window: most often the next one, else that of its last
  // position (positions after it compare greater).
  int64_t end = win + 1;
  const int64_t next = min(last + a.win, a.n - 1);
  if (same(next)) {
    int64_t lo = next, hi = a.n - 1;
    while (lo < hi) {  // 64 places at a time
      const int64_t step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
      const uint64_t in = __builtin_amdgcn_ballot_w64(at <= hi && same(min(at, hi)));
      lo += __popcll(in) * step;
      hi = min(hi, lo + step - 1);
    }
    end = lo / a.win;
  }
  constexpr bool second = MODE == EM_CLIP2;
  float v[V], q[V];
  em_clear(v);
  em_clear(q);
  em_add(em_ws<DT>(a.ws, 2 * win + 1, a, cb), v);
  if (second) em_add(em_ws<DT>(a.ws_sq, 2 * win + 1, a, cb), q);
  em_join<DT>(a.ws, win + 1, end, a, cb, v);
  if (second) em_join<DT>(a.ws_sq, win + 1, end, a, cb, q);
  if (MODE != EM_NORM) {
    em_finish<DT, AL>(a, MODE, key, cb, v, q);
    return;
  }
  // The first row of the run: the first of this window's positions in it.
  const uint64_t in = __builtin_amdgcn_ballot_w64(lane < a.win && same(p0 + min(lane, a.win - 1)));
  em_norm<DT>(a, a.rows[p0 + __builtin_ctzll(in)], seg, cb, v);
  em_put(em_ws<DT>(a.whole, win, a, cb), v);
}

__global__ __launch_bounds__(256) void k_embed_zero(ZeroShare z) { zero_pieces(z, blockIdx.x); }

// Shares [k, l) of n of the pieces, and the workgroups (of `threads`) they take.
ZeroShare zero_share(void* at, int64_t bytes, int threads, int64_t k, int64_t l, int64_t n, unsigned& blocks) {
  ZeroShare z{(char*)at, at != nullptr ? bytes : 0, 0, 0, 1};
  const int64_t size = (int64_t)threads * 16, pieces = (z.bytes + size - 1) / size;
  z.first = pieces * k / n;
  z.count = pieces * l / n - z.first;
  z.per = (int)(1 + z.count / ((int64_t)1 << 21));  // a grid of fewer than 2^32 threads
  blocks = (unsigned)((z.count + z.per - 1) / z.per);
  return z;
}

int sort_passes(int64_t vocab, int& bits) {
  int need = 1;
  while ((vocab >> need) != 0) ++need;  // keys 0 .. vocab
  const int passes = (need + SORT_BITS - 1) / SORT_BITS;
  bits = (need + passes - 1) / passes;
  return passes;
}

// Waves of the sort of n positions and the positions of each.
int64_t sort_waves(int64_t n, int64_t& per) {
  int64_t w = (n + SORT_KEYS - 1) / SORT_KEYS;
  if (w > SORT_NW) w = SORT_NW;
  per = ((n + w - 1) / w + 63) / 64 * 64;
  return (n + per - 1) / per;
}
int64_t pieces(int dtype, int64_t width) {
  const int64_t per = 64 * (dtype == ODP_DTYPE_F32 ? 4 : 8);
  return (width + per - 1) / per;
}
// Sorted positions per window: 32, or 16 or 8 where that leaves fewer than
// EM_FILL waves, which then would each wait for their loads in turn.
constexpr int64_t EM_FILL = 8192;
int window(int64_t n, int64_t ncb) {
  int w = EM_WIN;
  while (w > 8 && (n + w - 1) / w * ncb < EM_FILL) w /= 2;
  return w;
}
int64_t windows(int64_t n, int64_t ncb) { return (n + window(n, ncb) - 1) / window(n, ncb); }

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

int check_scale(const char* what, float scale) {
  if (std::isfinite(scale)) return ODP_OK;
  odp_set_error("%s: scale %g", what, (double)scale);
  return ODP_ERR_INVALID_ARGUMENT;
}

int check_grid(const char* what, int64_t blocks) {
  if (blocks >= (int64_t)1 << 24) {
    odp_set_error("%s: the launch needs %lld workgroups", what, (long long)blocks);
    return ODP_ERR_UNSUPPORTED;
  }
  return ODP_OK;
}

template <int MODE>
int launch_sum(const char* what, hipStream_t s, int dtype, bool aligned, EmbedSum a) {
  a.win = window(a.n, a.ncb);
  const int64_t items = windows(a.n, a.ncb) * a.ncb;
  if (int rc = check_grid(what, items)) return rc;
  const dim3 grid((unsigned)((items + EM_WAVES - 1) / EM_WAVES)), block(64 * EM_WAVES);
  const int64_t groups = windows(a.n, a.ncb) / JOIN_GROUP * a.ncb;
  // Whether long runs are joined in two steps.  A table gradient in one step and
  // in two, us, with no run, one over half of the rows and one over all: 64
  // windows (512 x 768 bfloat16) 18 / 19 / 22 and 21 / 22 / 23; 128 (1024 x 768) 19 /
  // 24 / 28 and 22 / 23 / 24; 256 (2048 x 768) 19 / 32 / 45 and 22 / 26 / 28; 1024
  // (8192 x 4096) 56 / 111 / 167 and 58 / 67 / 74.
  a.grouped = windows(a.n, a.ncb) > 8 * JOIN_GROUP;
  const dim3 ggrid((unsigned)((groups + EM_WAVES - 1) / EM_WAVES));
#define ODP_EM(DT, AL)                                                     \
  do {                                                                     \
    hipLaunchKernelGGL((k_embed_sum<DT, AL, MODE>), grid, block, 0, s, a); \
    if (a.grouped) hipLaunchKernelGGL((k_embed_group<DT, MODE>), ggrid, block, 0, s, a); \
    hipLaunchKernelGGL((k_embed_join<DT, AL, MODE>), grid, block, 0, s, a); \
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
  unsigned blocks;
  const ZeroShare z = zero_share(out, bytes, 256, 0, 1, 1, blocks);
  if (blocks > 0) hipLaunchKernelGGL(k_embed_zero, dim3(blocks), dim3(256), 0, s, z);
  return odp_check_launch(what);
}

}  // namespace

extern "C" int odp_embed_rows(odp_stream_t stream, int dtype, const void* tokens, int token_bytes, int64_t n,
                              const void* weight, int64_t ldw, int64_t vocab, int64_t width, float scale, void* out) {
  if (int rc = check_rows("odp_embed_rows", dtype, n, width, vocab, ldw)) return rc;
  if (int rc = check_scale("odp_embed_rows", scale)) return rc;
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
  const int64_t blocks = (n * ncb + EM_WAVES * EM_ITEMS - 1) / (EM_WAVES * EM_ITEMS);
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
  int64_t per;
  return 4 * ((3 * n + 3) / 4 * 4 + (n > SORT_SMALL ? SORT_BINS * sort_waves(n, per) : 0));
}

extern "C" int odp_token_sort(odp_stream_t stream, const void* tokens, int token_bytes, int64_t n, int64_t vocab,
                              int64_t padding, const int32_t* seg_row_start, const int32_t* seg_row_len,
                              int32_t n_seg, void* scratch, uint32_t* keys, uint32_t* rows, int32_t* seg_of,
                              void* zero, int64_t zero_bytes) {
  if (int rc = check_rows("odp_token_sort", ODP_DTYPE_F32, n, 1, vocab, 1)) return rc;
  if (token_bytes != 4 && token_bytes != 8) {
    odp_set_error("odp_token_sort: tokens of %d bytes", token_bytes);
    return ODP_ERR_UNSUPPORTED;
  }
  if (zero_bytes < 0) {
    odp_set_error("odp_token_sort: %lld bytes to zero", (long long)zero_bytes);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const hipStream_t s = odp_hip_stream(stream);
  if (n == 0) return zero != nullptr ? launch_zero("odp_token_sort", s, zero, zero_bytes) : ODP_OK;
  if (tokens == nullptr || scratch == nullptr || ((uintptr_t)scratch & 15) != 0 || keys == nullptr ||
      rows == nullptr || n_seg < 0 || (seg_row_start != nullptr && (seg_row_len == nullptr || seg_of == nullptr))) {
    odp_set_error("odp_token_sort: null pointer, scratch off the 16-byte grid or negative n_seg (%d)", n_seg);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  int bits;
  const int passes = sort_passes(vocab, bits);
  uint32_t* k1 = (uint32_t*)scratch;
  uint32_t* r1 = k1 + n;
  const bool segs = seg_row_start != nullptr;
  SortIn a{tokens, token_bytes == 8 ? 1 : 0, n, vocab, padding, seg_row_start, seg_row_len, n_seg,
           segs ? (int32_t*)(r1 + n) : nullptr, segs ? seg_of : nullptr, ZeroShare{}};
  unsigned zb;
  if (n <= SORT_SMALL) {
    a.zero = zero_share(zero, zero_bytes, 64 * SORT_WAVES, 0, 1, 1, zb);
#define ODP_SORT(R) \
  hipLaunchKernelGGL(k_sort_small<R>, dim3(1 + zb), dim3(64 * SORT_WAVES), 0, s, a, passes, bits, keys, rows, k1, r1)
    if (n <= SORT_WAVES * 64 * 2) ODP_SORT(2);
    else ODP_SORT(8);
#undef ODP_SORT
    return odp_check_launch("odp_token_sort");
  }
  uint32_t* counts = k1 + (3 * n + 3) / 4 * 4;
  int64_t per;
  const int nw = (int)sort_waves(n, per);
  const unsigned own = (unsigned)((nw + EM_WAVES - 1) / EM_WAVES);
  const dim3 block(64 * EM_WAVES);
  for (int p = 0; p < passes; ++p) {
    const bool to0 = ((passes - 1 - p) & 1) == 0;
    const uint32_t* ik = to0 ? k1 : keys;
    const uint32_t* ir = to0 ? r1 : rows;
    uint32_t* ok = to0 ? keys : k1;
    uint32_t* orow = to0 ? rows : r1;
    // The zeroing goes out in shares of two to three, as the launches' times do.
    a.zero = zero_share(zero, zero_bytes, 64 * EM_WAVES, 5 * p, 5 * p + 2, 5 * passes, zb);
    hipLaunchKernelGGL(k_sort_count, dim3(own + zb), block, 0, s, a, ik, p == 0 ? 1 : 0, p * bits, bits, counts, nw,
                       per);
    a.zero = zero_share(zero, zero_bytes, 64 * EM_WAVES, 5 * p + 2, 5 * p + 5, 5 * passes, zb);
    hipLaunchKernelGGL(k_sort_scatter, dim3(own + zb), block, 0, s, a, ik, ir, p == 0 ? 1 : 0, p * bits, bits, counts,
                       nw, per, ok, orow, p == passes - 1 ? 1 : 0);
  }
  return odp_check_launch("odp_token_sort");
}

extern "C" int64_t odp_embed_sum_scratch(int dtype, int64_t n, int64_t width, int second) {
  if (n <= 0 || width <= 0) return 0;
  const int64_t ncb = pieces(dtype, width), row = ncb * 64 * (dtype == ODP_DTYPE_F32 ? 4 : 8);
  return 4 * row * windows(n, ncb) * (second ? 4 : 2);
}

extern "C" int64_t odp_embed_pieces(int dtype, int64_t width) { return width > 0 ? pieces(dtype, width) : 0; }

extern "C" int odp_embed_grad(odp_stream_t stream, int dtype, const void* g, int64_t ldg, int64_t n, int64_t width,
                              const uint32_t* keys, const uint32_t* rows, int64_t vocab, float scale, void* scratch,
                              void* out) {
  if (int rc = check_rows("odp_embed_grad", dtype, n, width, vocab, ldg)) return rc;
  if (int rc = check_scale("odp_embed_grad", scale)) return rc;
  if (out == nullptr || (n > 0 && (g == nullptr || keys == nullptr || rows == nullptr || scratch == nullptr))) {
    odp_set_error("odp_embed_grad: null pointer");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (n == 0) return ODP_OK;
  const hipStream_t s = odp_hip_stream(stream);
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
                                const uint32_t* keys, const uint32_t* rows, const int32_t* seg_of, int64_t vocab,
                                float scale, const int32_t* seg_row_start, const int32_t* seg_example, void* scratch,
                                float* whole, double* part, int64_t part_stride, int64_t slot, int64_t* nf_flag) {
  if (int rc = check_rows("odp_embed_sqnorm", dtype, n, width, vocab, ldg)) return rc;
  if (int rc = check_scale("odp_embed_sqnorm", scale)) return rc;
  if (n == 0) return ODP_OK;
  if (g == nullptr || keys == nullptr || rows == nullptr || seg_of == nullptr || seg_row_start == nullptr ||
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
  a.seg_of = seg_of;
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
                                     const int32_t* seg_of, int64_t vocab, float scale, const int32_t* seg_example,
                                     void* scratch, const float* whole, const double* scales, float normalize_by,
                                     int out_dtype, void* out, void* out2) {
  if (int rc = check_rows("odp_embed_clipped_sum", dtype, n, width, vocab, ldg)) return rc;
  if (int rc = check_scale("odp_embed_clipped_sum", scale)) return rc;
  if (out_dtype < ODP_DTYPE_F32 || out_dtype > ODP_DTYPE_F64) {
    odp_set_error("odp_embed_clipped_sum: out_dtype %d", out_dtype);
    return ODP_ERR_UNSUPPORTED;
  }
  if (out == nullptr || (n > 0 && (g == nullptr || keys == nullptr || rows == nullptr || seg_of == nullptr ||
                                   seg_example == nullptr || scratch == nullptr || whole == nullptr ||
                                   scales == nullptr))) {
    odp_set_error("odp_embed_clipped_sum: null pointer");
    return ODP_ERR_INVALID_ARGUMENT;
  }
  const hipStream_t s = odp_hip_stream(stream);
  if (out2 != nullptr)
    if (int rc = launch_zero("odp_embed_clipped_sum", s, out2, vocab * width * odp_dtype_size(out_dtype))) return rc;
  if (n == 0) return ODP_OK;
  EmbedSum a{};
  a.g = (const char*)g;
  a.ldg = ldg;
  a.n = n;
  a.width = (int)width;
  a.ncb = (int)pieces(dtype, width);
  a.keys = keys;
  a.rows = rows;
  a.seg_of = seg_of;
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
  const bool aligned = rows_aligned(dtype, g, ldg, width) && ((uintptr_t)out & 15) == 0 && ((uintptr_t)out2 & 15) == 0;
  return out2 != nullptr ? launch_sum<EM_CLIP2>("odp_embed_clipped_sum", s, dtype, aligned, a)
                         : launch_sum<EM_CLIP>("odp_embed_clipped_sum", s, dtype, aligned, a);
}
