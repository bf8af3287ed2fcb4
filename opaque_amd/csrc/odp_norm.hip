// The root-mean-square norm behind the residual stream's addition, its
// gradients and its output in 8 bits.
//
//   h = x + r, as the stream's type holds it (h = x without a residual)
//   u = h / sqrt(mean(h^2) + eps),  y = u w                        k_rms_norm
//   a = gy w,  dh = (a - u mean(a u)) / sqrt(..) + gh,
//   dw_i = sum of gy u over the rows of gain i      k_rms_norm_grad, k_gain_sum
//   scale = max(max |y| / 448, the least normal float32) of a row or of 128
//   columns of it, q = y / scale in e4m3
//
// Every pass reads and writes its tensors once: bound by HBM.  A row is held in
// registers between the sum of its squares and its output, 8 values a vector:
// T threads of NV vectors, T from 8 (rows of up to 64 values, 32 rows a
// workgroup) through one wave to a workgroup of 1024 (32768 values).  A gain of
// its own for every group of rows (an example's) costs no launch more.  The
// gains' gradient is summed in registers along a strip of rows, then over the
// strips: no atomics, so results do not depend on the order of execution, and a
// row's not on its place in the batch.
//
// 16384 x 4096 bfloat16 with a residual: forward 92-95 us for 537 MB (5.7 TB/s),
// gradients 83-89 + 4 us for as much (6.1); a copy runs at 5.1.
//
// Vectors of 16 bytes are loaded at any address (this target's global loads
// need no more than the type's own alignment).  Rows of odd widths start at odd
// addresses, where each vector spans two lines: 8192 x 8191 118 + 145 us, 8192 x
// 8192 93 + 88.  Aligned vectors shifted into place in registers would give every
// thread the same values; that has not been tried.
#include <cmath>

#include "odp_internal.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
// The same at any 2- or 4-byte address.
typedef u32x4_t u32x4_h __attribute__((aligned(2)));
typedef u32x4_t u32x4_w __attribute__((aligned(4)));
typedef u32x2_t u32x2_h __attribute__((aligned(2)));
typedef u32x2_t u32x2_b __attribute__((aligned(1)));
typedef uint32_t uint32_h __attribute__((aligned(2)));

// What a thread holds of a row: 8 values of float32 (F32) or of a 16-bit type,
// as they lie in memory.
template <bool F32>
struct Eight {
  u32x4_t w[F32 ? 2 : 1];

  // Values c to c + 8 of a row, whatever its width.
  template <bool NT>
  __device__ __forceinline__ void load_whole(const char* row, int c) {
    if constexpr (F32) {
      const ODP_GMEM u32x4_w* p = (const ODP_GMEM u32x4_w*)(const ODP_GMEM void*)(row + 4 * c);
      w[0] = NT ? __builtin_nontemporal_load(p) : p[0];
      w[1] = NT ? __builtin_nontemporal_load(p + 1) : p[1];
    } else {
      const ODP_GMEM u32x4_h* p = (const ODP_GMEM u32x4_h*)(const ODP_GMEM void*)(row + 2 * c);
      w[0] = NT ? __builtin_nontemporal_load(p) : p[0];
    }
  }
  // Values c to c + 8 of a row of `width` (0 past it).
  template <bool NT = false>
  __device__ __forceinline__ void load(const char* row, int c, int width) {
    if (c + 8 <= width) {
      load_whole<NT>(row, c);
      return;
    }
    if (c >= width) {
      w[0] = u32x4_t{0, 0, 0, 0};
      if constexpr (F32) w[1] = w[0];
    } else if (width >= 8) {
      load_whole<NT>(row, width - 8);  // the row's last 8, moved down to c
      down(c + 8 - width);
    } else {
      w[0] = u32x4_t{0, 0, 0, 0};
      if constexpr (F32) w[1] = w[0];
#pragma unroll
      for (int i = 0; i < 7; ++i) {
        if (i >= width) break;
        if constexpr (F32) w[i / 4][i % 4] = ((const uint32_t*)row)[i];
        else w[0][i / 2] |= (uint32_t)((const uint16_t*)row)[i] << 16 * (i % 2);
      }
    }
  }
  // Value i becomes value i + n's, 0 past the last (n below 8).
  __device__ __forceinline__ void down(int n) {
    if constexpr (F32) {
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = w[i / 4][i % 4];
#pragma unroll
      for (int by = 4; by > 0; by >>= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = n & by ? (i + by < 8 ? v[i + by] : 0) : v[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i / 4][i % 4] = v[i];
    } else {
      uint32_t v[4] = {w[0][0], w[0][1], w[0][2], w[0][3]};
#pragma unroll
      for (int by = 2; by > 0; by >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = n & 2 * by ? (i + by < 4 ? v[i + by] : 0) : v[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = n & 1 ? v[i] >> 16 | (i < 3 ? v[i + 1] << 16 : 0) : v[i];
      w[0] = u32x4_t{v[0], v[1], v[2], v[3]};
    }
  }
  __device__ __forceinline__ void get(float (&v)[8], int dt) const {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i / 4][i % 4]);
    } else if (dt == ODP_DTYPE_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[0][i] << 16);
        v[2 * i + 1] = __uint_as_float(w[0][i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[0][i]);
        v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[0][i] >> 16));
      }
    }
  }
  // Rounded to nearest-even.
  __device__ __forceinline__ void set(const float (&v)[8], int dt) {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i / 4][i % 4] = __float_as_uint(v[i]);
    } else if (dt == ODP_DTYPE_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[0][i] = odp_f2bf2(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[0][i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) |
                  (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16;
    }
  }
  __device__ __forceinline__ void store(char* row, int c, int width) const {
    if (c + 8 <= width) {
      if constexpr (F32) {
        ODP_GMEM u32x4_w* p = (ODP_GMEM u32x4_w*)(ODP_GMEM void*)(row + 4 * c);
        p[0] = w[0];
        p[1] = w[1];
      } else {
        *(ODP_GMEM u32x4_h*)(ODP_GMEM void*)(row + 2 * c) = w[0];
      }
      return;
    }
    // The 4, 2 and 1 values that make up what is left.
    int n = width - c;
    if (n <= 0) return;
    Eight rest = *this;
    if constexpr (F32) {
      uint32_t* to = (uint32_t*)row + c;
      if (n & 4) {
        *(ODP_GMEM u32x4_w*)(ODP_GMEM void*)to = rest.w[0];
        rest.w[0] = rest.w[1];
        to += 4;
      }
      if (n & 2) {
        odp_gstore(to, rest.w[0][0]);
        odp_gstore(to + 1, rest.w[0][1]);
        rest.w[0][0] = rest.w[0][2];
        to += 2;
      }
      if (n & 1) odp_gstore(to, rest.w[0][0]);
    } else {
      uint16_t* to = (uint16_t*)row + c;
      if (n & 4) {
        *(ODP_GMEM u32x2_h*)(ODP_GMEM void*)to = u32x2_t{rest.w[0][0], rest.w[0][1]};
        rest.w[0][0] = rest.w[0][2];
        rest.w[0][1] = rest.w[0][3];
        to += 4;
      }
      if (n & 2) {
        *(ODP_GMEM uint32_h*)(ODP_GMEM void*)to = rest.w[0][0];
        rest.w[0][0] = rest.w[0][1];
        to += 2;
      }
      if (n & 1) odp_gstore(to, (uint16_t)rest.w[0][0]);
    }
  }
};

// A thread's vectors of a row; nt: by non-temporal loads (NORM_ONCE).
template <int T, bool F32, int NV>
__device__ __forceinline__ void load_rows(Eight<F32> (&x)[NV], const char* row, int width, int t, int nt) {
  if (!F32 && nt) {
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v].template load<true>(row, 8 * (v * T + t), width);
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) x[v].load(row, 8 * (v * T + t), width);
  }
}

// 8 gains of the run-time type dt, held as they lie in memory: both types use
// the same registers (those of 16 bits the first 4).
struct Gains {
  Eight<true> e;
  __device__ __forceinline__ void load(const char* row, int dt, int c, int width) {
    if (row == nullptr) return;
    if (dt == ODP_DTYPE_F32) {
      e.load(row, c, width);
    } else {
      Eight<false> half;
      half.load(row, c, width);
      e.w[0] = half.w[0];
    }
  }
  // Their values, 1 where there are none.
  __device__ __forceinline__ void get(float (&g)[8], const char* row, int dt, float offset) const {
    if (row == nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = 1.0f;
      return;
    }
    if (dt == ODP_DTYPE_F32) {
      e.get(g, dt);
    } else {
      Eight<false> half;
      half.w[0] = e.w[0];
      half.get(g, dt);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] += offset;
  }
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ float dpp_add(float v, uint32_t o) { return v + __uint_as_float(o); }

// Sum over T threads side by side (T <= 64), the same bits in each.
template <int T>
__device__ __forceinline__ float sum_lanes(float v) {
  v = dpp_add(v, dpp_u32<0xB1>(__float_as_uint(v)));                    // quad_perm 1,0,3,2
  v = dpp_add(v, dpp_u32<0x4E>(__float_as_uint(v)));                    // quad_perm 2,3,0,1
  v = dpp_add(v, dpp_u32<0x141>(__float_as_uint(v)));                   // row_half_mirror
  if constexpr (T >= 16) v = dpp_add(v, dpp_u32<0x140>(__float_as_uint(v)));  // row_mirror
  if constexpr (T >= 32) v += __shfl_xor(v, 16);
  if constexpr (T >= 64) v += __shfl_xor(v, 32);
  return v;
}
template <int T>
__device__ __forceinline__ uint32_t max_lanes(uint32_t v) {
  v = max(v, dpp_u32<0xB1>(v));
  v = max(v, dpp_u32<0x4E>(v));
  v = max(v, dpp_u32<0x141>(v));
  if constexpr (T >= 16) v = max(v, dpp_u32<0x140>(v));
  if constexpr (T >= 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  if constexpr (T >= 64) v = max(v, (uint32_t)__shfl_xor((int)v, 32));
  return v;
}

// Over the T threads of a row; for T > 64 through `red` [2][T / 64], the half
// of it that `turn` names, so that one barrier a row is enough.
template <int T>
__device__ __forceinline__ float sum_row(float v, float* red, int turn) {
  if constexpr (T <= 64) return sum_lanes<T>(v);
  constexpr int W = T / 64;
  float* r = red + W * (turn & 1);
  v = sum_lanes<64>(v);
  if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) s += r[i];
  return s;
}
template <int T>
__device__ __forceinline__ uint32_t max_row(uint32_t v, float* red, int turn) {
  if constexpr (T <= 64) return max_lanes<T>(v);
  constexpr int W = T / 64;
  float* r = red + W * (turn & 1);
  v = max_lanes<64>(v);
  if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = __uint_as_float(v);
  __syncthreads();
  uint32_t s = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) s = max(s, __float_as_uint(r[i]));
  return s;
}

struct NormArgs {
  const char *x, *r, *gain;
  char *y, *h;
  float *rstd, *scales;
  int64_t ldx, ldr, ldg, n;  // pitches in bytes
  int64_t row0;              // the launch's first row
  int64_t rows_per_gain;
  int width, dt, ht, gt, nt;
  float eps, offset;
};

enum { NQ_NONE = 0, NQ_ROW = 1, NQ_BLOCK = 2 };
constexpr int NQ_COLS = 128;          // columns of a block
constexpr float NQ_MOST = 448.0f;     // the largest e4m3 value
constexpr float NQ_LEAST = 1.17549435e-38f;

// The scale of a row or block, and its codes' values y / scale.  With 1 / rms = c
// 2^k, 1 <= c < 2, and t = 2^k h w (of 16-bit values the exact product) these are
// 448 t / max |t|: what a first quotient q leaves of 448 t puts q right, so that a
// border between two codes is met where it is (of 4096 bfloat16 one value in 5000
// lies on one, and goes to the even code).  At the ends of float32's range, t c /
// scale (0 for finite y over an infinite scale).
struct Codes {
  float scale, times, den, over;
  __device__ __forceinline__ Codes(uint32_t most, float c) {  // most: max |t|, its bits
    const float m = __uint_as_float(most), y = m * c;
    scale = y != y ? y : fmaxf(y / NQ_MOST, NQ_LEAST);
    const bool middle = m >= 0x1p-100f && m <= 0x1p100f && scale > NQ_LEAST;
    times = middle ? NQ_MOST : c;
    over = 1.0f / (middle ? m : scale);
    den = middle ? m : scale == INFINITY ? 0.0f : scale;
  }
  __device__ __forceinline__ float operator()(float t) const {
    const float x = t * times, q = x * over;
    return fmaf(fmaf(-q, den, x), over, q);
  }
};

template <int T>
constexpr int norm_threads() { return T < 256 ? 256 : T; }

template <bool XF, bool HF, int T, int NV, int Q>
__global__ __launch_bounds__(norm_threads<T>()) void k_rms_norm(const NormArgs a) {
  constexpr int ROWS = norm_threads<T>() / T;
  __shared__ float red[2][T > 64 ? T / 64 : 1];
  const int t = T < 256 ? (int)(threadIdx.x % T) : (int)threadIdx.x;
  int64_t row = a.row0 + (int64_t)blockIdx.x * ROWS + (T < 256 ? (int)(threadIdx.x / T) : 0);
  const bool live = row < a.n;
  row = live ? row : a.n - 1;
  const int width = a.width;
  Eight<XF> x[NV];
  Eight<HF> r[NV];
  load_rows<T>(x, a.x + row * a.ldx, width, t, a.nt);
  if (a.r != nullptr) load_rows<T>(r, a.r + row * a.ldr, width, t, a.nt);
  // The gains' loads go out with the row's; after its sum they were a second
  // wait (4.1 us for 4.0 at one row of 4096, 95 for 92 at 16384 on one card).
  const char* gain = a.gain == nullptr ? nullptr : a.gain + (a.ldg ? row / a.rows_per_gain * a.ldg : 0);
  Gains gains[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) gains[v].load(gain, a.gt, 8 * (v * T + t), width);
  float f[NV][8], sum = 0.0f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    x[v].get(f[v], a.dt);
    if (a.r != nullptr) {
      const int c = 8 * (v * T + t);
      float o[8];
      r[v].get(o, a.ht);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[v][i] += o[i];
      r[v].set(f[v], a.ht);
      if (live) r[v].store(a.h + row * width * (HF ? 4 : 2), c, width);
      r[v].get(f[v], a.ht);  // the norm is of what is stored
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(f[v][i], f[v][i], sum);
  }
  sum = sum_row<T>(sum, red[0], 0);
  const float inv = 1.0f / sqrtf(sum / (float)width + a.eps);
  if (a.rstd != nullptr && t == 0 && live) odp_gstore(a.rstd + row, inv);
  // For codes by its power of two alone (Codes); a NaN stays with what is left.
  const uint32_t bits = __float_as_uint(inv);
  const float by = Q == NQ_NONE ? inv : __uint_as_float(bits & 0x7f800000u);
  const float rest = inv != inv ? inv : __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
  uint32_t most = 0;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = 8 * (v * T + t);
    float g[8];
    gains[v].get(g, gain, a.gt, a.offset);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[v][i] = f[v][i] * by * g[i];
    if constexpr (Q == NQ_NONE) {
      Eight<XF> y;
      y.set(f[v], a.dt);
      if (live) y.store(a.y + row * width * (XF ? 4 : 2), c, width);
    } else {
      uint32_t m = 0;  // by the bits, above which those of infinities and NaN lie
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, c + i < width ? __float_as_uint(f[v][i]) & 0x7fffffffu : 0u);
      if constexpr (Q == NQ_ROW) {
        most = max(most, m);
      } else {
        const Codes code(max_lanes<(T < 16 ? T : 16)>(m), rest);  // 16 threads of 8 values
        if (live && (t & 15) == 0 && c < width)
          odp_gstore(a.scales + row * ((width + NQ_COLS - 1) / NQ_COLS) + c / NQ_COLS, code.scale);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[v][i] = code(f[v][i]);
      }
    }
  }
  if constexpr (Q == NQ_NONE) return;
  if constexpr (Q == NQ_ROW) {
    const Codes code(max_row<T>(most, red[0], 1), rest);
    if (live && t == 0) odp_gstore(a.scales + row, code.scale);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[v][i] = code(f[v][i]);
    }
  }
  if (!live) return;
  char* q = a.y + row * width;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = 8 * (v * T + t);
    if (c >= width) continue;
    u32x2_t w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(f[v][4 * i], f[v][4 * i + 1], 0, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(f[v][4 * i + 2], f[v][4 * i + 3], p, true);
      w[i] = (uint32_t)p;
    }
    if (c + 8 <= width) {
      *(ODP_GMEM u32x2_b*)(ODP_GMEM void*)(q + c) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (c + i < width) odp_gstore((uint8_t*)q + c + i, (uint8_t)(w[i / 4] >> 8 * (i % 4)));
    }
  }
}

struct NormGradArgs {
  const char *h, *gy, *gh, *gain;
  const float* rstd;
  char *dx, *dr, *dw;
  float* part;
  int64_t ldh, ldy, ldgh, ldg;  // pitches in bytes
  int64_t rows_per_gain, strips;
  int width, dt, ht, gt, nt;
  float offset;
};

// Workgroup (gain, strip): every strips-th ROWS of that gain's rows, so that the
// workgroups together walk the tensors from front to back (4.7 TB/s; each along
// rows of its own, 128 KB apart: 4.4).
template <bool XF, bool HF, int T, int NV>
__global__ __launch_bounds__(norm_threads<T>()) void k_rms_norm_grad(const NormGradArgs a) {
  constexpr int ROWS = norm_threads<T>() / T;
  __shared__ float red[2][T > 64 ? T / 64 : 1];
  __shared__ float joined[ROWS > 1 ? ROWS * T * NV * 8 : 1];
  const int t = T < 256 ? (int)(threadIdx.x % T) : (int)threadIdx.x;
  const int slot = T < 256 ? (int)(threadIdx.x / T) : 0;
  const int64_t group = blockIdx.x / a.strips, strip = blockIdx.x - group * a.strips;
  const int64_t first = group * a.rows_per_gain + strip * ROWS, last = (group + 1) * a.rows_per_gain;
  const int64_t step = a.strips * ROWS;
  const int width = a.width;
  const char* gain = a.gain == nullptr ? nullptr : a.gain + group * a.ldg;
  float g[NV][8], acc[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    Gains own;
    own.load(gain, a.gt, 8 * (v * T + t), width);
    own.get(g[v], gain, a.gt, a.offset);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[v][i] = 0.0f;
  }
  // The next row's loads go out before a row's sum over its threads and its
  // stores, where the registers hold both (AHEAD).
  constexpr bool AHEAD = NV * (XF ? 2 : 1) <= 2;
  Eight<HF> h[NV], gh[NV];
  Eight<XF> gy[NV];
  float inv = 0.0f;
  const bool with_gh = a.gh != nullptr && a.dx != nullptr;
  const auto load = [&](int64_t row) {
    load_rows<T>(h, a.h + row * a.ldh, width, t, a.nt);
    load_rows<T>(gy, a.gy + row * a.ldy, width, t, a.nt);
    if (with_gh) load_rows<T>(gh, a.gh + row * a.ldgh, width, t, a.nt);
    inv = a.rstd[row];
  };
  int turn = 0;
  if (AHEAD) load(min(first + slot, last - 1));
  for (int64_t base = first; base < last; base += step, ++turn) {
    const bool live = base + slot < last;
    const int64_t row = live ? base + slot : last - 1;
    if (!AHEAD) load(row);
    float u[NV][8], dot = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float d[8];
      h[v].get(u[v], a.ht);
      gy[v].get(d, a.dt);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        u[v][i] *= inv;
        const float p = d[i] * u[v][i];
        acc[v][i] += live ? p : 0.0f;
        dot = fmaf(p, g[v][i], dot);
      }
    }
    Eight<XF> gy0[NV];
    Eight<HF> gh0[NV];
    const float inv0 = inv;
#pragma unroll
    for (int v = 0; v < NV; ++v) gy0[v] = gy[v], gh0[v] = gh[v];
    if (AHEAD && base + step < last) load(min(base + step + slot, last - 1));
    if (a.dx == nullptr) continue;
    const float mean = sum_row<T>(dot, red[0], turn) / (float)width;
    if (!live) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = 8 * (v * T + t);
      float d[8];
      gy0[v].get(d, a.dt);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = inv0 * (d[i] * g[v][i] - u[v][i] * mean);
      if (with_gh) {
        float o[8];
        gh0[v].get(o, a.ht);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] += o[i];
      }
      if (a.dr != nullptr) {
        Eight<HF> out;
        out.set(d, a.ht);
        out.store(a.dr + row * width * (HF ? 4 : 2), c, width);
      }
      Eight<XF> out;
      out.set(d, a.dt);
      out.store(a.dx + row * width * (XF ? 4 : 2), c, width);
    }
  }
  if (a.part == nullptr && a.dw == nullptr) return;
  if constexpr (ROWS > 1) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) joined[(slot * NV + v) * T * 8 + t * 8 + i] = acc[v][i];
    __syncthreads();
    if (slot != 0) return;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        for (int s = 1; s < ROWS; ++s) acc[v][i] += joined[(s * NV + v) * T * 8 + t * 8 + i];
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = 8 * (v * T + t);
    if (a.part != nullptr) {
      Eight<true> out;
      out.set(acc[v], ODP_DTYPE_F32);
      out.store((char*)(a.part + (int64_t)blockIdx.x * width), c, width);
    } else if (a.gt == ODP_DTYPE_F32) {
      Eight<true> out;
      out.set(acc[v], a.gt);
      out.store(a.dw + group * width * 4, c, width);
    } else {
      Eight<false> out;
      out.set(acc[v], a.gt);
      out.store(a.dw + group * width * 2, c, width);
    }
  }
}

// dw of COLS columns of one gain: the threads of a workgroup take a strip each per
// column, 8 at a time, then add up over LDS.  64 columns a workgroup, but 16 where
// that leaves fewer than 64 workgroups (1001 columns of 1024 strips: 7 and 4 us).
constexpr int GS_THREADS = 1024;
template <int COLS>
__global__ __launch_bounds__(GS_THREADS) void k_gain_sum(const float* __restrict__ part, int64_t strips, int width,
                                                         int tiles, int gt, void* dw) {
  constexpr int AT = GS_THREADS / COLS;  // strips at a time
  __shared__ float red[AT][COLS + 1];
  const int64_t group = blockIdx.x / tiles;
  const int lane = threadIdx.x % COLS, own = threadIdx.x / COLS;
  const int c = (int)(blockIdx.x - group * tiles) * COLS + lane;
  const float* p = part + group * strips * width + c;
  float s = 0.0f;
  if (c < width) {
    int64_t i = own;
    for (; i + AT * 7 < strips; i += AT * 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = p[(i + AT * k) * width];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    for (; i < strips; i += AT) s += p[i * width];
  }
  red[own][lane] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  // One wave: 64 / COLS shares of the strips' sums a column.
  constexpr int EACH = AT * COLS / 64;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < EACH; ++i) s += red[own * EACH + i][lane];
#pragma unroll
  for (int x = COLS; x < 64; x <<= 1) s += __shfl_xor(s, x);
  if (own == 0 && c < width) odp_store_from_float(dw, group * width + c, gt, s);
}

// Bytes that a launch reads from which on it loads 16-bit rows non-temporally, as
// they cannot lie in the 256 MB cache: 16384 x 4096 bfloat16, gradient (403 MB read)
// 88 us, 116 through the caches, forward pass behind it (268 MB) 96 and 104.  Below,
// what was written just before may be there: 4096 x 4096 (67 MB), 26 us and 21.
constexpr int64_t NORM_ONCE = (int64_t)192 << 20;
// Workgroups of the gradient: two a compute unit, which leave 512 strips to add up
// (16384 x 4096: 88 + 5 us; 1024 strips 104 + 6).
constexpr int64_t NORM_GROUPS = 512;

int norm_tile(int64_t width) {  // threads of a row
  const int64_t v = (width + 7) / 8;
  return v <= 8 ? 8 : v <= 16 ? 16 : v <= 32 ? 32 : v <= 256 ? 64 : v <= 1024 ? 256 : 1024;
}

// Strips of a gain's rows.
int64_t strips_of(int64_t n, int64_t width, int64_t gains) {
  const int t = norm_tile(width), at = t < 256 ? 256 / t : 1;
  const int64_t rows = (n / gains + at - 1) / at, count = (NORM_GROUPS + gains - 1) / gains;
  // A few rows one after the other (below 1 us each) cost no more than the launch that adds strips up.
  return rows <= 8 ? 1 : rows < count ? rows : count;
}

bool norm_type(int dt) { return dt == ODP_DTYPE_F32 || dt == ODP_DTYPE_BF16 || dt == ODP_DTYPE_F16; }

constexpr int64_t NORM_THREADS = (int64_t)1 << 31;  // of a launch: its threads are counted in 32 bits

template <bool XF, bool HF, int T, int NV>
void launch_norm(hipStream_t s, NormArgs a, int q) {
  constexpr int TH = norm_threads<T>(), ROWS = TH / T;
  for (a.row0 = 0; a.row0 < a.n; a.row0 += NORM_THREADS / TH * ROWS) {
    const int64_t left = (a.n - a.row0 + ROWS - 1) / ROWS;
    const uint32_t blocks = (uint32_t)(left < NORM_THREADS / TH ? left : NORM_THREADS / TH);
    if (q == NQ_NONE) k_rms_norm<XF, HF, T, NV, NQ_NONE><<<blocks, TH, 0, s>>>(a);
    else if (q == NQ_ROW) k_rms_norm<XF, HF, T, NV, NQ_ROW><<<blocks, TH, 0, s>>>(a);
    else k_rms_norm<XF, HF, T, NV, NQ_BLOCK><<<blocks, TH, 0, s>>>(a);
  }
}
template <bool XF, bool HF, int T, int NV>
void launch_grad(hipStream_t s, const NormGradArgs& a, int64_t blocks) {
  k_rms_norm_grad<XF, HF, T, NV><<<(uint32_t)blocks, norm_threads<T>(), 0, s>>>(a);
}

// The narrowest form of at most 32 values a thread.  The gradient holds a row's
// h, gy and gh, the gains and their sums beside: with 4 vectors a thread it takes
// 205-241 registers, two waves a SIMD without the next row's loads (16384 x 2048
// bfloat16 81 us, 3.3 TB/s, for 49 forward; 8192 x 8192 88 for 93).  1024 threads
// have 128 registers each, so rows above 8192 values spill: 12 bytes a thread with
// 16-bit streams (4096 x 16384 90 us), 132 with float32 ones (305 us, 3.5 TB/s), and
// 296-428 above 16384 values (2048 x 32768 373 us, 1.4 TB/s).
#define ODP_NORM_FORM(CALL)                                 \
  do {                                                      \
    const int64_t v = (a.width + 7) / 8;                    \
    if (v <= 8) CALL(8, 1);                                 \
    else if (v <= 16) CALL(16, 1);                          \
    else if (v <= 32) CALL(32, 1);                          \
    else if (v <= 64) CALL(64, 1);                          \
    else if (v <= 128) CALL(64, 2);                         \
    else if (v <= 256) CALL(64, 4);                         \
    else if (v <= 512) CALL(256, 2);                        \
    else if (v <= 1024) CALL(256, 4);                       \
    else if (v <= 2048) CALL(1024, 2);                      \
    else CALL(1024, 4);                                     \
  } while (0)

template <bool XF, bool HF>
void norm_form(hipStream_t s, const NormArgs& a, int q) {
#define ODP_CALL(T, NV) launch_norm<XF, HF, T, NV>(s, a, q)
  ODP_NORM_FORM(ODP_CALL);
#undef ODP_CALL
}
template <bool XF, bool HF>
void grad_form(hipStream_t s, const NormGradArgs& a, int64_t blocks) {
#define ODP_CALL(T, NV) launch_grad<XF, HF, T, NV>(s, a, blocks)
  ODP_NORM_FORM(ODP_CALL);
#undef ODP_CALL
}

int norm_check(const char* what, int dt, int ht, int gt, int64_t n, int64_t width, int64_t gains) {
  if (!norm_type(dt) || !(ht == dt || ht == ODP_DTYPE_F32) || !(gt == dt || gt == ODP_DTYPE_F32)) {
    odp_set_error("%s: types %d (rows), %d (stream), %d (gain): a 16-bit type or float32, the others the same or float32",
                  what, dt, ht, gt);
    return ODP_ERR_UNSUPPORTED;
  }
  if (n < 0 || n >= (int64_t)1 << 31 || width < 1 || width > ODP_NORM_WIDE) {
    odp_set_error("%s: %lld rows of %lld: fewer than 2^31 rows of 1 to %lld", what, (long long)n, (long long)width,
                  (long long)ODP_NORM_WIDE);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (gains < 1 ? n != 0 || gains < 0 : n % gains != 0) {  // an empty batch has no gains
    odp_set_error("%s: %lld rows do not divide into %lld gains", what, (long long)n, (long long)gains);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  return ODP_OK;
}

}  // namespace

extern "C" int odp_rms_norm(odp_stream_t stream, int dtype, int stream_dtype, int gain_dtype, const void* x,
                            int64_t ldx, const void* residual, int64_t ldr, int64_t n, int64_t width, const void* gain,
                            int64_t ldg, int64_t gains, float eps, float offset, int quant, void* y, void* sum,
                            float* rstd, float* scales) {
  const char* what = "odp_rms_norm";
  const int rc = norm_check(what, dtype, stream_dtype, gain_dtype, n, width, gains);
  if (rc != ODP_OK) return rc;
  if (quant < NQ_NONE || quant > NQ_BLOCK) {
    odp_set_error("%s: quant %d: 0 (none), 1 (a scale per row) or 2 (per 128 columns)", what, quant);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (n == 0) return ODP_OK;
  if (x == nullptr || y == nullptr || (residual == nullptr) != (sum == nullptr) ||
      (quant != NQ_NONE) != (scales != nullptr)) {
    odp_set_error("%s: null x or y, a residual without its sum, or scales without quant (or the other way round)", what);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (ldx < width || (residual != nullptr && ldr < width) || (gain != nullptr && ldg != 0 && ldg < width)) {
    odp_set_error("%s: a pitch is less than the width %lld", what, (long long)width);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  NormArgs a;
  a.x = (const char*)x;
  a.r = (const char*)residual;
  a.gain = (const char*)gain;
  a.y = (char*)y;
  a.h = (char*)sum;
  a.rstd = rstd;
  a.scales = scales;
  a.ldx = ldx * odp_dtype_size(dtype);
  a.ldr = ldr * odp_dtype_size(stream_dtype);
  a.ldg = ldg * odp_dtype_size(gain_dtype);
  a.n = n;
  a.rows_per_gain = n / gains;
  a.width = (int)width;
  a.dt = dtype;
  a.ht = stream_dtype;
  a.gt = gain_dtype;
  a.eps = eps;
  a.offset = offset;
  a.nt = n * width * (odp_dtype_size(dtype) + (residual != nullptr ? odp_dtype_size(stream_dtype) : 0)) > NORM_ONCE;
  hipStream_t s = odp_hip_stream(stream);
  if (dtype == ODP_DTYPE_F32) norm_form<true, true>(s, a, quant);
  else if (stream_dtype == ODP_DTYPE_F32 && residual != nullptr) norm_form<false, true>(s, a, quant);
  else norm_form<false, false>(s, a, quant);
  return odp_check_launch(what);
}

extern "C" int64_t odp_rms_norm_grad_scratch(int64_t n, int64_t width, int64_t gains) {
  if (n <= 0 || width < 1 || width > ODP_NORM_WIDE || gains < 1 || n % gains != 0) return 0;
  const int64_t strips = strips_of(n, width, gains);
  return strips > 1 ? 4 * gains * strips * width : 0;
}

extern "C" int odp_rms_norm_grad(odp_stream_t stream, int dtype, int stream_dtype, int gain_dtype, const void* h,
                                 int64_t ldh, const float* rstd, const void* gy, int64_t ldy, const void* gh,
                                 int64_t ldgh, int64_t n, int64_t width, const void* gain, int64_t ldg, int64_t gains,
                                 float offset, void* scratch, void* dx, void* dres, void* dgain) {
  const char* what = "odp_rms_norm_grad";
  const int rc = norm_check(what, dtype, stream_dtype, gain_dtype, n, width, gains);
  if (rc != ODP_OK) return rc;
  if (n == 0) return ODP_OK;
  if (h == nullptr || rstd == nullptr || gy == nullptr || (dres != nullptr && dx == nullptr)) {
    odp_set_error("%s: null h, rstd or gy, or the residual's gradient without x's", what);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (ldh < width || ldy < width || (gh != nullptr && ldgh < width) || (gain != nullptr && ldg != 0 && ldg < width)) {
    odp_set_error("%s: a pitch is less than the width %lld", what, (long long)width);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (dx == nullptr && dgain == nullptr) return ODP_OK;
  const int64_t strips = strips_of(n, width, gains);
  if (dgain != nullptr && strips > 1 && scratch == nullptr) {
    odp_set_error("%s: null scratch where odp_rms_norm_grad_scratch is not 0", what);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  NormGradArgs a;
  a.h = (const char*)h;
  a.gy = (const char*)gy;
  a.gh = (const char*)gh;
  a.gain = (const char*)gain;
  a.rstd = rstd;
  a.dx = (char*)dx;
  a.dr = (char*)dres;
  a.dw = dgain != nullptr && strips == 1 ? (char*)dgain : nullptr;
  a.part = dgain != nullptr && strips > 1 ? (float*)scratch : nullptr;
  a.ldh = ldh * odp_dtype_size(stream_dtype);
  a.ldy = ldy * odp_dtype_size(dtype);
  a.ldgh = ldgh * odp_dtype_size(stream_dtype);
  a.ldg = ldg * odp_dtype_size(gain_dtype);
  a.rows_per_gain = n / gains;
  a.strips = strips;
  a.width = (int)width;
  a.dt = dtype;
  a.ht = stream_dtype;
  a.gt = gain_dtype;
  a.offset = offset;
  a.nt = n * width * (odp_dtype_size(dtype) + odp_dtype_size(stream_dtype) * (gh != nullptr ? 2 : 1)) > NORM_ONCE;
  hipStream_t s = odp_hip_stream(stream);
  const int64_t blocks = gains * strips;  // at most n
  if (blocks * (width > 8192 ? 1024 : 256) > NORM_THREADS) {
    static_assert(ODP_NORM_GRAD_GAINS * 1024 <= NORM_THREADS, "what the header promises");
    odp_set_error("%s: %lld gains are more than one launch takes", what, (long long)gains);
    return ODP_ERR_UNSUPPORTED;
  }
  if (dtype == ODP_DTYPE_F32) grad_form<true, true>(s, a, blocks);
  else if (stream_dtype == ODP_DTYPE_F32) grad_form<false, true>(s, a, blocks);
  else grad_form<false, false>(s, a, blocks);
  if (a.part != nullptr) {
    const int cols = gains * ((width + 63) / 64) < 64 ? 16 : 64;
    const int64_t tiles = (width + cols - 1) / cols;  // of fewer than 512 gains
    const auto sum = cols == 16 ? k_gain_sum<16> : k_gain_sum<64>;
    sum<<<(uint32_t)(gains * tiles), GS_THREADS, 0, s>>>(a.part, strips, (int)width, (int)tiles, gain_dtype, dgain);
  }
  return odp_check_launch(what);
}
