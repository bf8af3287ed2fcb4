// The norm of a whole tree of gradients, and the tree scaled to keep below a
// bound.
//
//   norm = sqrt(sum over all leaves of x^2)                k_tree_squares
//   out = x min(1, bound / norm)                           k_tree_scale
//
// Two passes, since no element can be scaled before the last has been read:
// bound by HBM.  Leaves travel in the kernels' arguments (TN_LEAVES a launch),
// so a call copies no table and may be captured.  Squares are exact in float64
// and added there: no overflow, and sums that do not depend on how a tree is cut
// into leaves by more than 2^-53 of their size a step.  Float64 leaves may have
// entries whose squares leave float64: those are added up beside, over 2^1200 or
// times it (Far), so that the norm is infinite only where float64 cannot hold it.
// The second pass walks the chunks backwards, the last read first, which the
// 256 MB cache still holds.  Every workgroup adds the first pass's partials for
// itself, in one order, so neither a third launch nor an atomic is needed.
//
// Four Llama-3-8B-shaped layers in bfloat16 (36 leaves, 1.74 GB): 261 us at 6.7 TB/s
// and 650 at 5.4; 50 leaves of 64 to 4 million float32 (65 MB): 14 and 21 us.
#include <cmath>
#include <type_traits>

#include "odp_internal.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t u32x4_h __attribute__((aligned(2)));  // at any address that a 16-bit type may have

constexpr int TN_LEAVES = 128;   // of a launch: the arguments stay below 4 KB
constexpr int TN_BLOCKS = 512;   // workgroups of a launch, two a compute unit
constexpr int TN_THREADS = 1024;

struct Leaves {
  const char* src[TN_LEAVES];
  char* dst[TN_LEAVES];
  int64_t n[TN_LEAVES];
  int32_t start[TN_LEAVES];  // first chunk
  uint8_t dt[TN_LEAVES];
  int32_t count, chunks, chunk;  // leaves, chunks in all, elements of a chunk
  int32_t once;                  // the tree is larger than the cache (TN_ONCE)
};
static_assert(sizeof(Leaves) + 64 <= 4096, "a launch's arguments");

// The leaf of a chunk.
__device__ __forceinline__ int leaf_of(const Leaves& l, int chunk) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.start[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <bool NT>
__device__ __forceinline__ u32x4_t piece(const char* p) {
  const ODP_GMEM u32x4_h* g = (const ODP_GMEM u32x4_h*)(const ODP_GMEM void*)p;
  return NT ? __builtin_nontemporal_load(g) : *g;
}
template <bool NT>
__device__ __forceinline__ void put(char* p, u32x4_t w) {
  ODP_GMEM u32x4_h* g = (ODP_GMEM u32x4_h*)(ODP_GMEM void*)p;
  if (NT) __builtin_nontemporal_store(w, g);
  else *g = w;
}

// Sums of squares of float64 entries above 2^480, over 2^1200, and below 2^-480,
// times it: the other squares, 2^45 of them, and these lie well within float64.
struct Far {
  double big = 0.0, small = 0.0;
};
constexpr double TN_FAR = 0x1p480, TN_BY = 0x1p600;

__device__ __forceinline__ double square_wide(double v, double s, Far& far) {
  const double m = fabs(v);
  if (m > TN_FAR) {
    const double t = v * (1.0 / TN_BY);
    far.big = fma(t, t, far.big);
  } else if (m < 1.0 / TN_FAR) {
    const double t = v * TN_BY;
    far.small = fma(t, t, far.small);
  } else {
    s = fma(v, v, s);
  }
  return s;
}

__device__ __forceinline__ double norm_of(double s, Far far) {
  if (far.big > 0.0) return TN_BY * sqrt(far.big + s / TN_BY / TN_BY);
  if (s != 0.0) return sqrt(s + far.small / TN_BY / TN_BY);
  return sqrt(far.small) / TN_BY;
}

template <int DT>
__device__ __forceinline__ double squares(u32x4_t w, double s, Far& far) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == ODP_DTYPE_F32) {
      const double v = __uint_as_float(w[i]);
      s = fma(v, v, s);
    } else if constexpr (DT == ODP_DTYPE_F64) {
      if (i & 1) continue;
      s = square_wide(__longlong_as_double((long long)((uint64_t)w[i + 1] << 32 | w[i])), s, far);
    } else {
      double a, b;
      if constexpr (DT == ODP_DTYPE_BF16) {
        a = __uint_as_float(w[i] << 16);
        b = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        a = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
        b = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
      }
      s = fma(a, a, s);
      s = fma(b, b, s);
    }
  }
  return s;
}

template <int DT>
__device__ __forceinline__ u32x4_t scaled(u32x4_t w, float f, double d) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == ODP_DTYPE_F32) {
      w[i] = __float_as_uint(__uint_as_float(w[i]) * f);
    } else if constexpr (DT == ODP_DTYPE_F64) {
      if (i & 1) continue;
      const double v = __longlong_as_double((long long)((uint64_t)w[i + 1] << 32 | w[i])) * d;
      const uint64_t u = (uint64_t)__double_as_longlong(v);
      w[i] = (uint32_t)u;
      w[i + 1] = (uint32_t)(u >> 32);
    } else if constexpr (DT == ODP_DTYPE_BF16) {
      w[i] = odp_f2bf2(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xffff0000u) * f);
    } else {
      const float a = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]) * f;
      const float b = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16)) * f;
      w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) |
             (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
    }
  }
  return w;
}

constexpr int TN_FLIGHT = 4;  // 16-byte pieces of a thread in flight

// One chunk's squares, or its scaled copy.  NT: by non-temporal loads and stores.
template <int DT, bool SCALE, bool NT>
__device__ __forceinline__ double chunk_pass(const char* src, char* dst, int64_t n, float f, double d, double s,
                                             Far& far) {
  constexpr int E = DT == ODP_DTYPE_F64 ? 8 : DT == ODP_DTYPE_F32 ? 4 : 2, V = 16 / E;
  const int pieces = (int)(n / V);
  double part[TN_FLIGHT] = {};
  for (int i = threadIdx.x; i < pieces; i += TN_FLIGHT * TN_THREADS) {
    u32x4_t w[TN_FLIGHT];
#pragma unroll
    for (int k = 0; k < TN_FLIGHT; ++k) {
      w[k] = u32x4_t{0, 0, 0, 0};
      if (i + k * TN_THREADS < pieces) w[k] = piece<NT>(src + 16 * (int64_t)(i + k * TN_THREADS));
    }
#pragma unroll
    for (int k = 0; k < TN_FLIGHT; ++k) {
      if constexpr (SCALE) {
        if (i + k * TN_THREADS < pieces) put<NT>(dst + 16 * (int64_t)(i + k * TN_THREADS), scaled<DT>(w[k], f, d));
      } else {
        part[k] = squares<DT>(w[k], part[k], far);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < TN_FLIGHT; ++k) s += part[k];
  const int64_t at = (int64_t)pieces * V + threadIdx.x;
  if (at < n) {
    const double v = odp_load_as_double(src, at, DT);
    if constexpr (SCALE) {
      if constexpr (DT == ODP_DTYPE_F64) odp_gstore((double*)dst + at, v * d);
      else odp_store_from_float(dst, at, DT, (float)v * f);
    } else if constexpr (DT == ODP_DTYPE_F64) {
      s = square_wide(v, s, far);
    } else {
      s = fma(v, v, s);
    }
  }
  return s;
}

// WIDE: the tree has float64 leaves.
template <bool SCALE, bool WIDE>
__device__ __forceinline__ double one_chunk(const Leaves& l, int c, float f, double d, double s, Far& far) {
  const int leaf = leaf_of(l, c), dt = l.dt[leaf];
  const int64_t first = (int64_t)(c - l.start[leaf]) * l.chunk, n = min((int64_t)l.chunk, l.n[leaf] - first);
  const int64_t at = first * odp_dtype_size(dt);
  const char* src = l.src[leaf] + at;
  char* dst = SCALE ? l.dst[leaf] + at : nullptr;
  const auto pass = [&](auto nt) {
    constexpr bool NT = decltype(nt)::value;
    if (dt == ODP_DTYPE_BF16) return chunk_pass<ODP_DTYPE_BF16, SCALE, NT>(src, dst, n, f, d, s, far);
    if (dt == ODP_DTYPE_F32) return chunk_pass<ODP_DTYPE_F32, SCALE, NT>(src, dst, n, f, d, s, far);
    if (!WIDE || dt == ODP_DTYPE_F16) return chunk_pass<ODP_DTYPE_F16, SCALE, NT>(src, dst, n, f, d, s, far);
    return chunk_pass<ODP_DTYPE_F64, SCALE, NT>(src, dst, n, f, d, s, far);
  };
  return l.once ? pass(std::true_type{}) : pass(std::false_type{});
}

// Sum over the workgroup, the same bits in every thread.
__device__ __forceinline__ double sum_block(double s, double* red) {
  s = rows_sum4(row_sum16(s));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < TN_THREADS / 64; ++i) t += red[i];
  return t;
}

// part: of the squares, and `apart` further on each of what Far holds.
template <bool WIDE>
__global__ __launch_bounds__(TN_THREADS) void k_tree_squares(const Leaves l, double* part, int64_t apart) {
  __shared__ double red[WIDE ? 3 : 1][TN_THREADS / 64];
  double s = 0.0;
  Far far;
  for (int c = blockIdx.x; c < l.chunks; c += gridDim.x) s = one_chunk<false, WIDE>(l, c, 0.0f, 0.0, s, far);
  s = sum_block(s, red[0]);
  if (threadIdx.x == 0) odp_gstore(part + blockIdx.x, s);
  if constexpr (WIDE) {
    const double big = sum_block(far.big, red[1]), small = sum_block(far.small, red[2]);
    if (threadIdx.x != 0) return;
    odp_gstore(part + apart + blockIdx.x, big);
    odp_gstore(part + 2 * apart + blockIdx.x, small);
  }
}

__device__ __forceinline__ double factor_of(double norm, double most) {
  return norm != norm ? norm : norm > most ? most / norm : 1.0;
}

__device__ __forceinline__ void store_norm(void* out, int wide, double norm) {
  if (threadIdx.x != 0) return;
  if (wide) odp_gstore((double*)out, norm);
  else odp_gstore((float*)out, (float)norm);
}

// out: where the norm goes (null but in the first launch).
template <bool WIDE>
__global__ __launch_bounds__(TN_THREADS) void k_tree_scale(const Leaves l, const double* __restrict__ part, int64_t apart,
                                                           int parts, double most, int wide, void* out) {
  __shared__ double red[WIDE ? 3 : 1][TN_THREADS / 64];
  double s = 0.0;
  Far far;
  for (int i = threadIdx.x; i < parts; i += TN_THREADS) {
    s += part[i];
    if constexpr (WIDE) far.big += part[apart + i], far.small += part[2 * apart + i];
  }
  s = sum_block(s, red[0]);
  if constexpr (WIDE) far.big = sum_block(far.big, red[1]), far.small = sum_block(far.small, red[2]);
  const double norm = norm_of(s, far);
  if (out != nullptr && blockIdx.x == 0) store_norm(out, wide, norm);
  const double d = factor_of(norm, most);
  const float f = (float)d;
  for (int c = l.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) one_chunk<true, WIDE>(l, c, f, d, 0.0, far);
}

// A small tree in one launch of one workgroup.
template <bool WIDE>
__global__ __launch_bounds__(TN_THREADS) void k_tree_small(const Leaves l, int clip, double most, int wide, void* out) {
  __shared__ double red[WIDE ? 3 : 1][TN_THREADS / 64];
  double s = 0.0;
  Far far;
  for (int c = 0; c < l.chunks; ++c) s = one_chunk<false, WIDE>(l, c, 0.0f, 0.0, s, far);
  s = sum_block(s, red[0]);
  if constexpr (WIDE) far.big = sum_block(far.big, red[1]), far.small = sum_block(far.small, red[2]);
  const double norm = norm_of(s, far);
  store_norm(out, wide, norm);
  if (!clip) return;
  const double d = factor_of(norm, most);
  const float f = (float)d;
  for (int c = l.chunks - 1; c >= 0; --c) one_chunk<true, WIDE>(l, c, f, d, 0.0, far);
}

// A tree of few and small leaves is one workgroup's.
constexpr int64_t TN_SMALL = 16384, TN_FEW = 8;

// Bytes of a tree from which on both passes load and store non-temporally, as the
// second finds nothing of it in the 256 MB cache: 1.75 GB of bfloat16 261 + 650 us
// (316 + 659 through the caches; with the last 160 MB left to them, 288 + 648), 65 MB
// 15 + 22 us (16 + 27 non-temporally).
constexpr int64_t TN_ONCE = (int64_t)192 << 20;

// The leaves of launch `k`, of a tree of `bytes`.
void fill(Leaves& l, const int64_t* rows, int64_t n_leaves, int64_t k, int64_t chunk, int64_t bytes) {
  int64_t chunks = 0;
  l.count = 0;
  l.chunk = (int)chunk;
  l.once = bytes > TN_ONCE;
  for (int64_t i = k * TN_LEAVES; i < n_leaves && i < (k + 1) * TN_LEAVES; ++i) {
    const int64_t* r = rows + i * ODP_TN_FIELDS;
    if (r[ODP_TN_N] == 0) continue;
    const int j = l.count++;
    l.src[j] = (const char*)r[ODP_TN_SRC];
    l.dst[j] = (char*)r[ODP_TN_DST];
    l.n[j] = r[ODP_TN_N];
    l.dt[j] = (uint8_t)r[ODP_TN_DTYPE];
    l.start[j] = (int32_t)chunks;
    chunks += (r[ODP_TN_N] + chunk - 1) / chunk;
  }
  l.chunks = (int32_t)chunks;
}

}  // namespace

extern "C" int64_t odp_tree_norm_scratch(int64_t n_leaves) {
  return n_leaves <= 0 ? 8 : 8 * 3 * TN_BLOCKS * ((n_leaves + TN_LEAVES - 1) / TN_LEAVES);
}

extern "C" int odp_tree_norm(odp_stream_t stream, const int64_t* leaves, int64_t n_leaves, int clip, double max_norm,
                             int wide, void* scratch, void* norm) {
  const char* what = "odp_tree_norm";
  if (n_leaves < 0 || (n_leaves > 0 && leaves == nullptr) || scratch == nullptr || norm == nullptr) {
    odp_set_error("%s: null pointer or %lld leaves", what, (long long)n_leaves);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (clip && !(max_norm >= 0.0)) {
    odp_set_error("%s: max_norm %g must be 0 or more", what, max_norm);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  int64_t total = 0, used = 0, bytes = 0;
  bool doubles = false;
  for (int64_t i = 0; i < n_leaves; ++i) {
    const int64_t* r = leaves + i * ODP_TN_FIELDS;
    const int64_t n = r[ODP_TN_N], dt = r[ODP_TN_DTYPE];
    if (n < 0 || n > (int64_t)1 << 44 || total > (int64_t)1 << 45) {
      odp_set_error("%s: leaf %lld has %lld elements", what, (long long)i, (long long)n);
      return ODP_ERR_INVALID_ARGUMENT;
    }
    if (dt < ODP_DTYPE_F32 || dt > ODP_DTYPE_F64) {
      odp_set_error("%s: leaf %lld has dtype %lld", what, (long long)i, (long long)dt);
      return ODP_ERR_UNSUPPORTED;
    }
    if (n > 0 && (r[ODP_TN_SRC] == 0 || (clip && r[ODP_TN_DST] == 0))) {
      odp_set_error("%s: leaf %lld has a null pointer", what, (long long)i);
      return ODP_ERR_INVALID_ARGUMENT;
    }
    total += n;
    bytes += n * odp_dtype_size((int)dt);
    used += n > 0;
    doubles = doubles || dt == ODP_DTYPE_F64;
  }
  hipStream_t s = odp_hip_stream(stream);
  Leaves l;
  const int64_t launches = (n_leaves + TN_LEAVES - 1) / TN_LEAVES;
  if (total <= TN_SMALL && used <= TN_FEW && launches <= 1) {
    fill(l, leaves, n_leaves, 0, TN_SMALL, bytes);
    const auto small = doubles ? k_tree_small<true> : k_tree_small<false>;
    small<<<1, TN_THREADS, 0, s>>>(l, clip, max_norm, wide, norm);
    return odp_check_launch(what);
  }
  // Chunks of 32768 elements (of bfloat16 what the threads have in flight at once),
  // down to 2048 where there are fewer than two for every workgroup.
  int64_t chunk = 8 * TN_THREADS * TN_FLIGHT;
  while (chunk > 2048 && total / chunk < 2 * TN_BLOCKS) chunk >>= 1;
  while (total / chunk > (int64_t)1 << 28) chunk <<= 1;
  double* part = (double*)scratch;
  const int64_t apart = TN_BLOCKS * launches;
  const auto squares = doubles ? k_tree_squares<true> : k_tree_squares<false>;
  const auto scale = doubles ? k_tree_scale<true> : k_tree_scale<false>;
  int64_t parts = 0;
  for (int64_t k = 0; k < launches; ++k) {
    fill(l, leaves, n_leaves, k, chunk, bytes);
    if (l.chunks == 0) continue;
    const int blocks = l.chunks < TN_BLOCKS ? l.chunks : TN_BLOCKS;
    squares<<<blocks, TN_THREADS, 0, s>>>(l, part + parts, apart);
    parts += blocks;
  }
  if (!clip || parts == 0) {
    l.chunks = l.count = 0;
    scale<<<1, TN_THREADS, 0, s>>>(l, part, apart, (int)parts, 0.0, wide, norm);  // the norm alone
    return odp_check_launch(what);
  }
  bool told = false;
  for (int64_t k = launches - 1; k >= 0; --k) {
    fill(l, leaves, n_leaves, k, chunk, bytes);
    if (l.chunks == 0) continue;
    const int blocks = l.chunks < TN_BLOCKS ? l.chunks : TN_BLOCKS;
    scale<<<blocks, TN_THREADS, 0, s>>>(l, part, apart, (int)parts, max_norm, wide, told ? nullptr : norm);
    told = true;
  }
  return odp_check_launch(what);
}
