// Routing of tokens to experts, and its gradient.
//
//   p = softmax(z) or sigmoid(z) over the experts, key = p + bias
//   groups: the best `top_groups` by the sum of their two best keys, or by
//   their best; the `top_k` best keys of what is left, lower experts first
//   where keys are equal                                          k_route
//   w_j = scale p_j, over the sum of the chosen p with `renormalize`
//   dz from dw; the choice has no gradient                        k_route_grad
//
// A token's logits lie in the registers of L threads, 8 or 16 each (L a power
// of two up to a wave), so that a wave takes 64 / L tokens and a step of the
// search costs a few instructions a value and log2(L) exchanges.  Bound by the
// HBM for the logits, by instructions from about 100 experts and 8 choices on.
//
// The search runs on 32-bit words: a key's leading bits above the expert's
// number, counted from the end.  All words of a token differ, one maximum names
// both the key and the expert, equal keys give the lower expert, and the next
// choice is the largest word below the last: the largest of (word - last) in
// wrapping arithmetic, with nothing to mark.  The leading bits decide as the
// keys in 64 bits would unless two that the choice hangs on lie within the
// error of their float32 computation (BIAS_TOL); such a token is done again from
// float64 keys (`route_exactly`; 0.3 % of the tokens of 256 experts with a bias).
// Keys are the logits themselves where those order as the scores do (no bias,
// and no sums over groups); those of 16-bit types always decide.
#include <cmath>

#include "odp_internal.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// The same at any 2- or 4-byte address (this target's loads need no more).
typedef u32x4_t u32x4_h __attribute__((aligned(2)));
typedef u32x4_t u32x4_w __attribute__((aligned(4)));

constexpr int RT_THREADS = 256;
constexpr int RT_GROUPS = 64;  // groups, at most (a mask of 64 bits)

// e^x: 2^t from the hardware, t = x log2(e) rounded, and what the rounding took
// off as a first-order factor; 2 units in the last place.
__device__ __forceinline__ float exp_near(float x) {
  const float t = x * 1.44269502f;
  const float r = fmaf(x, 1.44269502f, -t) + x * 1.92596299e-8f;
  const float e = __builtin_amdgcn_exp2f(t);
  return fabsf(t) < 126.0f ? fmaf(e, r * 0.693147181f, e) : e;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
// The value of the thread that lies across step S (1, 2, 4, .. 32) of a
// butterfly; for 4 and 8 by mirrors, which pair what the steps before joined.
template <int S>
__device__ __forceinline__ uint32_t across(uint32_t v) {
  if constexpr (S == 1) return dpp_u32<0xB1>(v);
  else if constexpr (S == 2) return dpp_u32<0x4E>(v);
  else if constexpr (S == 4) return dpp_u32<0x141>(v);
  else if constexpr (S == 8) return dpp_u32<0x140>(v);
  else return (uint32_t)__shfl_xor((int)v, S);
}
template <int L, typename F>
__device__ __forceinline__ uint32_t join(uint32_t v, F f) {
  if constexpr (L > 1) v = f(v, across<1>(v));
  if constexpr (L > 2) v = f(v, across<2>(v));
  if constexpr (L > 4) v = f(v, across<4>(v));
  if constexpr (L > 8) v = f(v, across<8>(v));
  if constexpr (L > 16) v = f(v, across<16>(v));
  if constexpr (L > 32) v = f(v, across<32>(v));
  return v;
}
template <int L>
__device__ __forceinline__ uint32_t max_of(uint32_t v) {
  return join<L>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int L>
__device__ __forceinline__ uint32_t or_of(uint32_t v) {
  return join<L>(v, [](uint32_t a, uint32_t b) { return a | b; });
}
template <int L>
__device__ __forceinline__ float fmax_of(float v) {
  return __uint_as_float(join<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
template <int L>
__device__ __forceinline__ float sum_of(float v) {
  return __uint_as_float(join<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
template <int L>
__device__ __forceinline__ double sum_of(double v) {
#pragma unroll
  for (int s = 1; s < L; s <<= 1) v += __shfl_xor(v, s);
  return v;
}
template <int L>
__device__ __forceinline__ double fmax_of(double v) {
#pragma unroll
  for (int s = 1; s < L; s <<= 1) v = fmax(v, __shfl_xor(v, s));
  return v;
}

// LDS written by some threads of a wave and read by others of it.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// float32 as an unsigned integer of the same order.
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __float_as_uint(f);
  return (int32_t)u < 0 ? ~u : u | 0x80000000u;
}
// float64 the same, above 1; NaN is 1, below every other.
__device__ __forceinline__ uint64_t ordered(double f) {
  const uint64_t u = (uint64_t)__double_as_longlong(f);
  return f != f ? 1 : (int64_t)u < 0 ? ~u : u | 0x8000000000000000ull;
}

struct RouteArgs {
  const char* z;
  const float* bias;
  int64_t* index;
  float* weights;
  const float* gw;
  const int64_t* chosen;
  char* dz;
  int64_t ldz, n;         // pitch in bytes
  int64_t rows_per_bias;  // 0: one bias for all
  int64_t ldw;            // pitch of gw
  int experts, top_k, groups, top_groups, size;  // size: of a group
  int dt, sigmoid, best, renorm, bits;           // bits: of an expert's number
  float scale, per_size;                         // 1 / size
};

// One logit.
__device__ __forceinline__ float logit(const char* row, int dt, int e) {
  if (dt == ODP_DTYPE_F32) return ((const float*)row)[e];
  const uint16_t h = ((const uint16_t*)row)[e];
  return dt == ODP_DTYPE_BF16 ? odp_bf2f(h) : (float)__builtin_bit_cast(_Float16, h);
}

// Values first to first + V of a row of `experts` (-inf past it).
template <int V>
__device__ __forceinline__ void load_row(float (&z)[V], const char* row, int dt, int first, int experts) {
  if (first + V <= experts) {
    if (dt == ODP_DTYPE_F32) {
      const ODP_GMEM u32x4_w* p = (const ODP_GMEM u32x4_w*)(const ODP_GMEM void*)(row + 4 * first);
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const u32x4_t w = p[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) z[4 * i + j] = __uint_as_float(w[j]);
      }
    } else {
      const ODP_GMEM u32x4_h* p = (const ODP_GMEM u32x4_h*)(const ODP_GMEM void*)(row + 2 * first);
#pragma unroll
      for (int i = 0; i < V / 8; ++i) {
        const u32x4_t w = p[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (dt == ODP_DTYPE_BF16) {
            z[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
            z[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
          } else {
            z[8 * i + 2 * j] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[j]);
            z[8 * i + 2 * j + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[j] >> 16));
          }
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) z[i] = first + i < experts ? logit(row, dt, first + i) : -INFINITY;
}

// sigmoid without a loss of bits on either side.
__device__ __forceinline__ float sigmoid(float z) {
  const float e = exp_near(-fabsf(z));
  return (z >= 0.0f ? 1.0f : e) / (1.0f + e);
}

// The choice from float64 keys, by the L threads of a token; key: [experts] of
// LDS.  Masked experts (a logit of -inf) come after all others, a NaN key last.
template <int L>
__device__ void route_exactly(const RouteArgs& a, const char* row, const float* bias, int t, uint64_t* key,
                                           int* picked) {
  const int n = a.experts;
  double top = -INFINITY, total = 0.0;
  if (!a.sigmoid) {
    for (int e = t; e < n; e += L) top = fmax(top, (double)logit(row, a.dt, e));
    top = fmax_of<L>(top);
    for (int e = t; e < n; e += L) {
      const double z = logit(row, a.dt, e);
      total += z == -INFINITY ? 0.0 : exp(z - top);
    }
    total = sum_of<L>(total);
  }
  for (int e = t; e < n; e += L) {
    const double z = logit(row, a.dt, e);
    double k = z + 0.0;  // the logits order as the scores do (-0 as 0)
    if (bias != nullptr || (a.groups > 1 && a.best == 0)) {
      k = a.sigmoid ? 1.0 / (1.0 + exp(-z)) : exp(z - top) / total;
      k += bias != nullptr ? (double)bias[e] : 0.0;
    }
    key[e] = ordered(z == -INFINITY ? -INFINITY : k);
  }
  wave_sync();
  if (a.groups > 1) {
    // A group's score as an ordered word too; those that do not come into it (masked) add nothing.
    uint64_t open = 0;
    for (int g = t; g < a.groups; g += L) {
      uint64_t mine = 0;
      int above = 0;
      for (int o = -1; o < a.groups; ++o) {  // -1: this group itself, first
        const uint64_t* k = key + (o < 0 ? g : o) * a.size;
        uint64_t one = 0, two = 0;
        for (int i = 0; i < a.size; ++i) {
          const uint64_t w = k[i];
          two = max(two, min(one, w));
          one = max(one, w);
        }
        if (a.best == 0 && one > 1 && two > ordered(-(double)INFINITY)) {
          const auto value = [](uint64_t w) {
            return __longlong_as_double((long long)((int64_t)w < 0 ? w & 0x7fffffffffffffffull : ~w));
          };
          one = ordered(value(one) + value(two));
        }
        if (o < 0) mine = one;
        else above += one > mine || (one == mine && o < g);
      }
      if (above < a.top_groups) open |= 1ull << g;
    }
    const uint32_t lo = or_of<L>((uint32_t)open), hi = or_of<L>((uint32_t)(open >> 32));
    open = (uint64_t)hi << 32 | lo;
    wave_sync();
    for (int e = t; e < n; e += L)
      if (!(open >> (e / a.size) & 1)) key[e] = 0;
    wave_sync();
  }
  for (int j = 0; j < a.top_k; ++j) {
    uint64_t most = 0;
    int at = t;
    for (int e = t; e < n; e += L) {
      const uint64_t w = key[e];
      if (w > most) most = w, at = e;
    }
#pragma unroll
    for (int s = 1; s < L; s <<= 1) {
      const uint64_t w = (uint64_t)__shfl_xor((long long)most, s);
      const int e = __shfl_xor(at, s);
      if (w > most || (w == most && e < at)) most = w, at = e;
    }
    if (t == 0) picked[j] = at, key[at] = 0;
    wave_sync();
  }
}

// Two words' leading parts within this of each other: the float32 computation
// may have them the wrong way round.  In units of 2^-24 of the keys' range R
// (scores' 1 and the bias's): a score is off by up to 16 (an exponential, a sum
// of up to 1024 of them, a reciprocal), the bias above its least, the sum and
// the product by one each.
constexpr uint32_t BIAS_TOL = 64;

template <int L, int V>
__global__ __launch_bounds__(RT_THREADS) void k_route(const RouteArgs a) {
  constexpr int TOKENS = RT_THREADS / L;
  // A token's words: keys of the groups' search (32 bits), or of route_exactly.
  __shared__ uint64_t lds[TOKENS * L * V];
  constexpr int PICKS = L * V < 64 ? L * V : 64;
  __shared__ int picks[TOKENS * PICKS];
  const int slot = threadIdx.x / L, t = threadIdx.x % L;
  int64_t token = (int64_t)blockIdx.x * TOKENS + slot;
  const bool live = token < a.n;
  token = live ? token : a.n - 1;
  const char* row = a.z + token * a.ldz;
  const float* bias = a.bias;
  if (bias != nullptr && a.rows_per_bias > 0) bias += token / a.rows_per_bias * a.experts;
  int* picked = picks + slot * PICKS;
  const int first = t * V;

  float z[V];
  load_row<V>(z, row, a.dt, first, a.experts);
  const uint32_t mask = (1u << a.bits) - 1;
  float top = -INFINITY, total = 0.0f;
  bool odd = false;  // a NaN or +inf
#pragma unroll
  for (int i = 0; i < V; ++i) {
    top = fmaxf(top, z[i]);
    odd |= !(z[i] < INFINITY);
  }
  const bool whole = !a.sigmoid && (bias != nullptr || !a.renorm || (a.groups > 1 && a.best == 0));
  if (!a.sigmoid) top = fmax_of<L>(top);
  float p[V];
  if (whole) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] = z[i] == -INFINITY ? 0.0f : exp_near(z[i] - top);
      total += p[i];
    }
    total = sum_of<L>(total);
  }
  uint32_t key[V];
  uint32_t tol = 0;
  bool again = false;  // to be done from float64 keys
  if (bias != nullptr || (a.groups > 1 && a.best == 0)) {
    float lo = INFINITY, hi = -INFINITY, b[V];
    if (bias != nullptr) {
      load_row<V>(b, (const char*)bias, ODP_DTYPE_F32, first, a.experts);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (first + i < a.experts) {
          lo = fminf(lo, b[i]);
          hi = fmaxf(hi, b[i]);
          again |= b[i] != b[i];
        }
      }
      lo = -fmax_of<L>(-lo);
      hi = fmax_of<L>(hi);
    } else {
      lo = hi = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = 0.0f;
    }
    const float range = 1.0f + (hi - lo);
    again |= !(range < 1e30f);  // infinities among them, too
    const uint32_t steps = 1u << min(24, 32 - a.bits);
    const float by = (float)(steps - 16) / range;
    tol = BIAS_TOL >> (24 - min(24, 32 - a.bits));
    tol += tol < BIAS_TOL ? 1 : 0;
    const float over = a.sigmoid ? 0.0f : __builtin_amdgcn_rcpf(total);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = first + i;
      const float s = a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + exp_near(-z[i])) : p[i] * over;
      again |= e < a.experts && z[i] == -INFINITY;
      const uint32_t q = 1 + (uint32_t)fminf(((b[i] - lo) + s) * by, (float)(steps - 8));
      key[i] = e < a.experts ? q << a.bits | (mask - (uint32_t)e) : 0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = first + i;
      key[i] = e < a.experts ? (ordered(z[i] + 0.0f) & ~mask) | (mask - (uint32_t)e) : 0;
    }
  }
  again |= odd;

  if (a.groups > 1) {
    uint32_t* words = (uint32_t*)(lds + slot * L * V);
    uint32_t* scores = (uint32_t*)picked;  // [groups], before the choices
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (first + i < a.experts) words[first + i] = key[i];
    wave_sync();
    for (int g = t; g < a.groups; g += L) {
      uint32_t one = 0, two = 0;
      for (int i = 0; i < a.size; ++i) {
        const uint32_t w = words[g * a.size + i];
        two = max(two, min(one, w));
        one = max(one, w);
      }
      // The sum of two leading parts takes up to 25 bits, a group's number 6; a
      // best key stands as it is (its low bits order equal ones by the group).
      scores[g] = a.best == 0 ? ((one >> a.bits) + (two >> a.bits)) << 6 | (uint32_t)(63 - g) : one;
    }
    wave_sync();
    uint64_t open = 0;
    uint32_t last = 0, next = 0;
    for (int g = t; g < a.groups; g += L) {
      const uint32_t mine = scores[g];
      int above = 0;
      for (int o = 0; o < a.groups; ++o) above += scores[o] > mine;
      if (above < a.top_groups) open |= 1ull << g;
      if (above == a.top_groups - 1) last = mine;
      if (above == a.top_groups) next = mine;
    }
    last = max_of<L>(last);
    next = max_of<L>(next);
    const uint32_t lo = or_of<L>((uint32_t)open), hi = or_of<L>((uint32_t)(open >> 32));
    open = (uint64_t)hi << 32 | lo;
    if (a.top_groups < a.groups) {
      const int shift = a.best == 0 ? 6 : a.bits;
      const uint32_t apart = (last >> shift) - (next >> shift);
      again |= a.best == 0 ? apart <= 2 * tol : tol ? apart <= tol : apart == 0 && a.dt == ODP_DTYPE_F32;
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int g = (int)(((float)(first + i) + 0.5f) * a.per_size);
      if (!(open >> (g & 63) & 1)) key[i] = 0;
    }
  }

  uint32_t last = 0;
  // One choice more than wanted, for how near the next one lies.
  for (int j = 0; j <= a.top_k; ++j) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, key[i] - last);
    m = max_of<L>(m) + last;
    // Nothing below the last one: the largest difference belongs to one above it (or to it).
    const bool none = j > 0 && m >= last;
    if (!none && j > 0) {
      if ((last >> a.bits) - (m >> a.bits) <= tol && m != 0) {
        // Equal logits and biases are equal keys, which the words order already.
        const int e0 = (int)(mask - (last & mask)), e1 = (int)(mask - (m & mask));
        again |= logit(row, a.dt, e0) != logit(row, a.dt, e1) || (bias != nullptr && bias[e0] != bias[e1]);
      }
    }
    if (j == a.top_k) break;
    if (t == 0) picked[j] = (int)(mask - (m & mask));
    last = m;
  }
  again = or_of<L>(again ? 1u : 0u) != 0;
  odd = or_of<L>(odd ? 1u : 0u) != 0;
  if (again) route_exactly<L>(a, row, bias, t, lds + slot * L * V, picked);
  wave_sync();

  // The weights of the chosen, a few a thread.
  const bool off = odd && !a.sigmoid;
  float most = -INFINITY, sum = 0.0f;
  if (a.renorm) {
    for (int j = t; j < a.top_k; j += L) most = fmaxf(most, logit(row, a.dt, picked[j]));
    most = fmax_of<L>(most);
  }
  // Over the largest of the chosen, so that the sum is never 0; for sigmoids
  // where all are small.
  const float shift = a.sigmoid ? (a.renorm ? fminf(most, 0.0f) : 0.0f) : a.renorm ? most : top;
  const auto share = [&](float x) {
    if (x == -INFINITY) return 0.0f;
    if (!a.sigmoid) return exp_near(x - shift);
    return x >= 0.0f ? 1.0f / (1.0f + exp_near(-x)) : exp_near(x - shift) / (1.0f + exp_near(x));
  };
  if (a.renorm) {
    for (int j = t; j < a.top_k; j += L) sum += share(logit(row, a.dt, picked[j]));
    sum = sum_of<L>(sum);
  } else {
    sum = a.sigmoid ? 1.0f : total;
  }
  if (!live) return;
  for (int j = t; j < a.top_k; j += L) {
    const int e = picked[j];
    const float s = share(logit(row, a.dt, e));
    const float w = off ? NAN : s == 0.0f ? 0.0f : a.scale * (s / sum);
    odp_gstore(a.index + token * a.top_k + j, (int64_t)e);
    odp_gstore(a.weights + token * a.top_k + j, w);
  }
}

// dz of a token's L threads: the chosen entries through LDS.
template <int L, int V>
__global__ __launch_bounds__(RT_THREADS) void k_route_grad(const RouteArgs a) {
  constexpr int TOKENS = RT_THREADS / L;
  __shared__ float lds[TOKENS * L * V];
  const int slot = threadIdx.x / L, t = threadIdx.x % L;
  int64_t token = (int64_t)blockIdx.x * TOKENS + slot;
  const bool live = token < a.n;
  token = live ? token : a.n - 1;
  const char* row = a.z + token * a.ldz;
  const int64_t* chosen = a.chosen + token * a.top_k;
  const float* gw = a.gw + token * a.ldw;
  float* d = lds + slot * L * V;
  const int first = t * V;
  const bool dense = !a.sigmoid && !a.renorm;  // every expert's score depends on every logit
#pragma unroll
  for (int i = 0; i < V; ++i) d[first + i] = 0.0f;
  float z[V], top = -INFINITY, total = 0.0f;
  bool odd = false;
  if (!a.sigmoid) {
    load_row<V>(z, row, a.dt, first, a.experts);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      top = fmaxf(top, z[i]);
      odd |= !(z[i] < INFINITY);
    }
    odd = or_of<L>(odd ? 1u : 0u) != 0;
  }
  if (dense) {
    top = fmax_of<L>(top);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      z[i] = z[i] == -INFINITY ? 0.0f : exp_near(z[i] - top);
      total += z[i];
    }
    total = sum_of<L>(total);
  }
  const auto place = [&](int j) { return (int)min(max(chosen[j], (int64_t)0), (int64_t)(a.experts - 1)); };
  float most = -INFINITY, sum = 0.0f, dot = 0.0f;
  if (a.renorm) {
    for (int j = t; j < a.top_k; j += L) most = fmaxf(most, logit(row, a.dt, place(j)));
    most = fmax_of<L>(most);
  }
  const float shift = a.sigmoid ? fminf(most, 0.0f) : most;
  const auto share = [&](float x) {
    if (x == -INFINITY) return 0.0f;
    if (!a.sigmoid) return exp_near(x - shift);
    return x >= 0.0f ? 1.0f / (1.0f + exp_near(-x)) : exp_near(x - shift) / (1.0f + exp_near(x));
  };
  if (a.renorm) {
    for (int j = t; j < a.top_k; j += L) {
      const float s = share(logit(row, a.dt, place(j)));
      sum += s;
      dot += s == 0.0f ? 0.0f : s * gw[j];
    }
    sum = sum_of<L>(sum);
    dot = sum_of<L>(dot);
    dot = sum > 0.0f ? dot / sum : 0.0f;
  }
  wave_sync();
  for (int j = t; j < a.top_k; j += L) {
    const int e = place(j);
    const float x = logit(row, a.dt, e);
    float v;
    if (a.renorm) {
      const float s = share(x);
      v = s == 0.0f ? 0.0f : s / sum * (gw[j] - dot);
      if (a.sigmoid) v *= sigmoid(-x);
    } else if (a.sigmoid) {
      v = x == -INFINITY ? 0.0f : sigmoid(x) * sigmoid(-x) * gw[j];
    } else {
      v = gw[j];
    }
    d[e] = odd ? NAN : v * a.scale;
  }
  wave_sync();
  float out[V];
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = d[first + i];
  if (dense) {
    const float over = total > 0.0f ? 1.0f / total : 0.0f;
    float with = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) with += z[i] == 0.0f ? 0.0f : z[i] * out[i];
    with = sum_of<L>(with) * over;
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = odd ? NAN : z[i] == 0.0f ? 0.0f : z[i] * over * (out[i] - with);
  }
  if (!live) return;
  char* to = a.dz + token * a.experts * (a.dt == ODP_DTYPE_F32 ? 4 : 2);
  if (first + V <= a.experts) {
    if (a.dt == ODP_DTYPE_F32) {
      ODP_GMEM u32x4_w* w = (ODP_GMEM u32x4_w*)(ODP_GMEM void*)(to + 4 * first);
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        w[i] = u32x4_t{__float_as_uint(out[4 * i]), __float_as_uint(out[4 * i + 1]), __float_as_uint(out[4 * i + 2]),
                       __float_as_uint(out[4 * i + 3])};
    } else {
      ODP_GMEM u32x4_h* w = (ODP_GMEM u32x4_h*)(ODP_GMEM void*)(to + 2 * first);
#pragma unroll
      for (int i = 0; i < V / 8; ++i) {
        u32x4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = out[8 * i + 2 * j], y = out[8 * i + 2 * j + 1];
          v[j] = a.dt == ODP_DTYPE_BF16 ? odp_f2bf2(x, y)
                                        : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x) |
                                              (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)y) << 16;
        }
        w[i] = v;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (first + i < a.experts) odp_store_from_float(to, first + i, a.dt, out[i]);
}

template <int L, int V>
void launch_route(hipStream_t s, const RouteArgs& a, bool grad) {
  constexpr int TOKENS = RT_THREADS / L;
  const uint32_t blocks = (uint32_t)((a.n + TOKENS - 1) / TOKENS);
  if (grad) k_route_grad<L, V><<<blocks, RT_THREADS, 0, s>>>(a);
  else k_route<L, V><<<blocks, RT_THREADS, 0, s>>>(a);
}

void route_form(hipStream_t s, const RouteArgs& a, bool grad) {
  const int n = a.experts;
  if (n <= 8) launch_route<1, 8>(s, a, grad);
  else if (n <= 16) launch_route<2, 8>(s, a, grad);
  else if (n <= 32) launch_route<4, 8>(s, a, grad);
  else if (n <= 64) launch_route<8, 8>(s, a, grad);
  else if (n <= 128) launch_route<8, 16>(s, a, grad);
  else if (n <= 256) launch_route<16, 16>(s, a, grad);
  else if (n <= 512) launch_route<32, 16>(s, a, grad);
  else launch_route<64, 16>(s, a, grad);
}

int route_check(const char* what, int dt, int64_t ldz, int64_t n, int64_t experts, int64_t top_k, float scale) {
  if (dt != ODP_DTYPE_F32 && dt != ODP_DTYPE_BF16 && dt != ODP_DTYPE_F16) {
    odp_set_error("%s: dtype %d: float32, bfloat16 or float16", what, dt);
    return ODP_ERR_UNSUPPORTED;
  }
  if (n < 0 || n >= (int64_t)1 << 31 || experts < 1 || experts > ODP_ROUTE_EXPERTS || top_k < 1 || top_k > experts ||
      top_k > ODP_ROUTE_CHOICES || ldz < experts) {
    odp_set_error("%s: invalid sizes: %lld tokens (pitch %lld), %lld experts (1 to %d), %lld choices (1 to %d)", what,
                  (long long)n, (long long)ldz, (long long)experts, ODP_ROUTE_EXPERTS, (long long)top_k,
                  ODP_ROUTE_CHOICES);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (!(fabsf(scale) < INFINITY)) {
    odp_set_error("%s: the scale must be finite", what);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  return ODP_OK;
}

RouteArgs route_args(int dt, const void* z, int64_t ldz, int64_t n, int64_t experts, int sigmoid, int64_t top_k,
                     int renorm, float scale) {
  RouteArgs a = {};
  a.z = (const char*)z;
  a.ldz = ldz * odp_dtype_size(dt);
  a.n = n;
  a.experts = (int)experts;
  a.top_k = (int)top_k;
  a.dt = dt;
  a.sigmoid = sigmoid;
  a.renorm = renorm;
  a.scale = scale;
  a.groups = a.top_groups = 1;
  a.size = a.experts;
  a.per_size = 1.0f / (float)a.size;
  a.bits = 8;  // words of 24 bits and more hold float32's error
  while (1 << a.bits < a.experts) ++a.bits;
  return a;
}

}  // namespace

extern "C" int odp_route(odp_stream_t stream, int dtype, const void* logits, int64_t ldz, int64_t n, int64_t experts,
                         int sigmoid, const float* bias, int64_t biases, int64_t groups, int64_t top_groups, int best,
                         int64_t top_k, int renormalize, float scale, int64_t* index, float* weights) {
  const char* what = "odp_route";
  const int rc = route_check(what, dtype, ldz, n, experts, top_k, scale);
  if (rc != ODP_OK) return rc;
  if (groups < 1 || groups > RT_GROUPS || experts % groups != 0 || top_groups < 1 || top_groups > groups ||
      top_k > experts / groups * top_groups || best < 0 || best > 1) {
    odp_set_error("%s: %lld experts in %lld groups (1 to %d), %lld of them open, do not give %lld choices", what,
                  (long long)experts, (long long)groups, RT_GROUPS, (long long)top_groups, (long long)top_k);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (bias != nullptr && (biases < 1 || n % biases != 0)) {
    odp_set_error("%s: %lld tokens do not divide into %lld biases", what, (long long)n, (long long)biases);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  if (n == 0) return ODP_OK;
  if (logits == nullptr || index == nullptr || weights == nullptr) {
    odp_set_error("%s: null pointer", what);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  RouteArgs a = route_args(dtype, logits, ldz, n, experts, sigmoid, top_k, renormalize, scale);
  a.bias = bias;
  a.rows_per_bias = bias != nullptr && biases > 1 ? n / biases : 0;
  a.groups = top_groups == groups ? 1 : (int)groups;  // all open: no groups
  a.top_groups = a.groups == 1 ? 1 : (int)top_groups;
  a.size = a.experts / a.groups;
  a.per_size = 1.0f / (float)a.size;
  a.best = best;
  a.index = index;
  a.weights = weights;
  route_form(odp_hip_stream(stream), a, false);
  return odp_check_launch(what);
}

extern "C" int odp_route_grad(odp_stream_t stream, int dtype, const void* logits, int64_t ldz, int64_t n,
                              int64_t experts, int sigmoid, int64_t top_k, int renormalize, float scale,
                              const int64_t* index, const float* gw, int64_t ldw, void* dlogits) {
  const char* what = "odp_route_grad";
  const int rc = route_check(what, dtype, ldz, n, experts, top_k, scale);
  if (rc != ODP_OK) return rc;
  if (n == 0) return ODP_OK;
  if (logits == nullptr || index == nullptr || gw == nullptr || dlogits == nullptr || ldw < 0) {
    odp_set_error("%s: null pointer or a negative pitch", what);
    return ODP_ERR_INVALID_ARGUMENT;
  }
  RouteArgs a = route_args(dtype, logits, ldz, n, experts, sigmoid, top_k, renormalize, scale);
  a.chosen = index;
  a.gw = gw;
  a.ldw = ldw;
  a.dz = (char*)dlogits;
  route_form(odp_hip_stream(stream), a, true);
  return odp_check_launch(what);
}
