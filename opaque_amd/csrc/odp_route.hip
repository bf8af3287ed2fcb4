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
// error of their float32 computation (`units_apart`); of such a token (one in a
// thousand of 256 experts) the candidates' float64 keys are formed and ranked.  Keys are the
// logits themselves where those order as the scores do (no bias, and no sums over
// groups that shut some), also where scores run together in 64 bits; those of 16-bit
// types always decide.
//
// 32768 tokens, 8 choices: of 64 experts 7 us, 256 15 us (33 MB of float32; a copy
// of it takes 7), 256 with sigmoid scores and a bias 20-21, of 4 of 8 groups 24-26.
#include <cmath>

#include "odp_internal.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// The same at any 2- or 4-byte address (this target's loads need no more).
typedef u32x4_t u32x4_h __attribute__((aligned(2)));
typedef u32x4_t u32x4_w __attribute__((aligned(4)));

constexpr int RT_THREADS = 256;
constexpr int RT_GROUPS = 64;  // groups, at most (a mask of 64 bits)
// Spread of the biases, in largest scores, from which on low ones are cut: 32768 x 256
// by sigmoids with one at -100 take 23 us so and 27 in groups, uncut 28 and 40.  Below it
// the scores keep 19 of a word's 24 bits, and the search for the cut is not paid.
constexpr float ROUTE_DEEP = 32.0f;

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
  int64_t token0;         // the launch's first token
  int64_t rows_per_bias;  // 0: one bias for all
  int64_t ldw;            // pitch of gw
  int experts, top_k, groups, top_groups, size;  // size: of a group
  int dt, sigmoid, best, renorm, bits;           // bits: of an expert's number
  int span;                                      // threads of a group (0: none of their own)
  float scale, per_size;                         // 1 / size
};

// One logit.
__device__ __forceinline__ float logit(const char* row, int dt, int e) {
  if (dt == ODP_DTYPE_F32) return ((const float*)row)[e];
  const uint16_t h = ((const uint16_t*)row)[e];
  return dt == ODP_DTYPE_BF16 ? odp_bf2f(h) : (float)__builtin_bit_cast(_Float16, h);
}

// Values first to first + V of a row of `experts` (`none` past it).
template <int V>
__device__ __forceinline__ void load_row(float (&z)[V], const char* row, int dt, int first, int experts, float none) {
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
  for (int i = 0; i < V; ++i) z[i] = first + i < experts ? logit(row, dt, first + i) : none;
}

// sigmoid without a loss of bits on either side.
__device__ __forceinline__ float sigmoid(float z) {
  const float e = exp_near(-fabsf(z));
  return (z >= 0.0f ? 1.0f : e) / (1.0f + e);
}

// A chosen logit's share of the chosen ones' sum (with renormalize) or its
// score times what the softmax divides by: over the largest of the chosen, so
// that the sum is never 0; for sigmoids where all are small.
struct Shares {
  bool sigmoid;
  float shift;
  __device__ __forceinline__ Shares(const RouteArgs& a, float most, float top)
      : sigmoid(a.sigmoid), shift(a.sigmoid ? (a.renorm ? fminf(most, 0.0f) : 0.0f) : a.renorm ? most : top) {}
  __device__ __forceinline__ float operator()(float x) const {
    if (x == -INFINITY) return 0.0f;
    if (!sigmoid) return exp_near(x - shift);
    return x >= 0.0f ? 1.0f / (1.0f + exp_near(-x)) : exp_near(x - shift) / (1.0f + exp_near(x));
  }
};

// A row's float64 keys, as ordered words: a masked expert (a logit of -inf)
// below all others, a NaN key below those.  What follows is for few tokens: its
// loops hold one value at a time, so that the registers go to the others.
struct Keys64 {
  const RouteArgs& a;
  const char* row;
  const float* bias;
  bool sums;   // the keys are more than the logits
  double top;  // the largest logit
  double total = 1.0;
  template <int L>
  __device__ __forceinline__ void normalise(int t) {
    if (!sums || a.sigmoid) return;
    total = 0.0;
    float next = t < a.experts ? logit(row, a.dt, t) : 0.0f;
#pragma unroll 1
    for (int e = t; e < a.experts; e += L) {
      const double z = next;
      if (e + L < a.experts) next = logit(row, a.dt, e + L);
      total += z == -INFINITY ? 0.0 : exp(z - top);
    }
    total = sum_of<L>(total);
  }
  __device__ __forceinline__ uint64_t operator()(float logit_, float bias_) const {
    const double z = logit_;
    double k = z + 0.0;  // the logits order as the scores do (-0 as 0)
    if (sums) k = (a.sigmoid ? 1.0 / (1.0 + exp(-z)) : exp(z - top) / total) + (double)bias_;
    return ordered(z == -INFINITY ? -INFINITY : k);
  }
  __device__ __forceinline__ float bias_of(int e) const { return bias != nullptr ? bias[e] : 0.0f; }
  // The keys of list[j] (null: j) for j < count, by L threads.
  template <int L>
  __device__ __forceinline__ void fill(uint64_t* key, const int* list, int count, int t) const {
    int e = t < count ? (list != nullptr ? list[t] : t) : 0;
    float z = logit(row, a.dt, e), b = bias_of(e);
#pragma unroll 1
    for (int j = t; j < count; j += L) {
      const float z0 = z, b0 = b;
      if (j + L < count) {
        e = list != nullptr ? list[j + L] : j + L;
        z = logit(row, a.dt, e);
        b = bias_of(e);
      }
      key[j] = (*this)(z0, b0);
    }
    wave_sync();
  }
};

// LDS of a wave, in 64-bit words: the words (32 bits) of all its tokens or the
// float64 keys of one of them, and 64 more (a token's groups' scores, or its
// choices by rank).
template <int L, int V>
constexpr int route_words() { return (L > 32 ? L : 32) * V + 64; }

// All keys of a token in LDS, and a mask of the open groups from them.  Masked
// experts add nothing to a group's score.
template <int L, int V>
__device__ __forceinline__ uint64_t open_exactly(const RouteArgs& a, Keys64& of, int t, uint64_t* key) {
  of.normalise<L>(t);
  of.fill<L>(key, nullptr, a.experts, t);
  if (a.groups == 1) return ~0ull;
  uint64_t* scores = key + route_words<L, V>() - 64;
  const auto value = [](uint64_t w) {
    return __longlong_as_double((long long)((int64_t)w < 0 ? w & 0x7fffffffffffffffull : ~w));
  };
#pragma unroll 1
  for (int g = t; g < a.groups; g += L) {
    uint64_t one = 0, two = 0;
#pragma unroll 2
    for (int k = 0; k < a.size; ++k) {
      const uint64_t w = key[g * a.size + k];
      two = max(two, min(one, w));
      one = max(one, w);
    }
    scores[g] = a.best == 0 && one > 1 && two > ordered(-(double)INFINITY) ? ordered(value(one) + value(two)) : one;
  }
  wave_sync();
  uint64_t open = 0;
#pragma unroll 1
  for (int g = t; g < a.groups; g += L) {
    int above = 0;
#pragma unroll 2
    for (int o = 0; o < a.groups; ++o) above += scores[o] > scores[g] || (scores[o] == scores[g] && o < g);
    if (above < a.top_groups) open |= 1ull << g;
  }
  const uint32_t lo = or_of<L>((uint32_t)open), hi = or_of<L>((uint32_t)(open >> 32));
  return (uint64_t)hi << 32 | lo;
}

// The choice from float64 keys, by the L threads of a token.
template <int L, int V>
__device__ __forceinline__ void route_exactly(const RouteArgs& a, Keys64& of, int t, uint64_t* key, int* picked) {
  const uint64_t open = open_exactly<L, V>(a, of, t, key);
  wave_sync();
  if (a.groups > 1) {
#pragma unroll 1
    for (int e = t; e < a.experts; e += L)
      if (!(open >> (e / a.size) & 1)) key[e] = 0;
    wave_sync();
  }
#pragma unroll 1
  for (int j = 0; j < a.top_k; ++j) {
    uint64_t most = 0;
    int at = t;
#pragma unroll 2
    for (int e = t; e < a.experts; e += L) {
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

// The best top_k of `count` candidates, in the order of their float64 keys.
template <int L, int V>
__device__ __forceinline__ void rank_exactly(const RouteArgs& a, Keys64& of, int t, int count, uint64_t* key,
                                             int* picked) {
  int* ranked = (int*)(key + route_words<L, V>() - 64);
  of.normalise<L>(t);
  of.fill<L>(key, picked, count, t);
#pragma unroll 1
  for (int j = t; j < count; j += L) {
    const uint64_t mine = key[j];
    const int e = picked[j];
    int above = 0;
#pragma unroll 2
    for (int i = 0; i < count; ++i) above += key[i] > mine || (key[i] == mine && picked[i] < e);
    if (above < a.top_k) ranked[above] = e;
  }
  wave_sync();
#pragma unroll 1
  for (int j = t; j < a.top_k; j += L) picked[j] = ranked[j];
  wave_sync();
}

// A token whose words do not decide, from the words of its choices and the one
// below them: the candidates are the choices and, where `on`, all that lie within
// `tol` of each other from the last choice on.
template <int L, int V, int PICKS, typename F>
__device__ __forceinline__ void choose_exactly(const RouteArgs& a, Keys64& of, const F& below, int t, uint32_t tol,
                                               bool weird, bool on, uint64_t* key, uint32_t* chain) {
  const uint32_t mask = (1u << a.bits) - 1;
  int count = a.top_k;
  bool full = weird;
  if (on && !full) {
    uint32_t last = chain[count++];  // the first word below the choices is a candidate
    for (; count < PICKS; ++count) {
      const uint32_t m = below(last);
      if (m == 0 || (last >> a.bits) - (m >> a.bits) > tol) break;
      if (t == 0) chain[count] = m;
      last = m;
    }
    // No room to see whether the run ends here.
    full = count >= PICKS;
  }
  wave_sync();
  if (!full) {
    for (int j = t; j < count; j += L) chain[j] = mask - (chain[j] & mask);
    wave_sync();
    rank_exactly<L, V>(a, of, t, count, key, (int*)chain);
  } else {
    route_exactly<L, V>(a, of, t, key, (int*)chain);
  }
}

// How far apart the leading parts of two words may lie with their keys the
// wrong way round, in units of 2^-24 of the keys' range R (the largest score, for
// sigmoids 1, and the bias's; `largest` is the score's part of it).  A sigmoid's score s is within 4: its exponential's argument and the
// exponential itself are off by s (1 - s) (|z| + 2), at most 1, its sum by 1, its
// reciprocal by 2.  A softmax's by 42 s and one more: s |z - top| and 2 s of the
// exponential, 34 s of the sum of up to 1024 of them (22 additions, and the terms'
// own), 2 s of its reciprocal, s of the product.  The bias over its least, its share
// of the range, their sum and the whole part of it are a unit each.  Twice all
// that, for two words.
__device__ __forceinline__ uint32_t units_apart(bool sigmoid, float largest) {
  return sigmoid ? 16 : 11 + (uint32_t)(84.0f * fminf(largest, 1.0f));
}

// Whether a row's logits are all equal, and its biases (an empty token's, a bias
// still at 0): its words order as the keys do however near they lie.  32768 x 256
// zeros take 18 us so and 25-27 in groups, 263 and 450 by their float64 keys.
// Asked only of rows whose leading parts agree: of all that are slow it cost the
// others 3 us of 26.
template <int L>
__device__ __forceinline__ bool all_equal(const RouteArgs& a, const char* row, const float* bias, int t) {
  const float z = logit(row, a.dt, 0), b = bias != nullptr ? bias[0] : 0.0f;
  bool differ = false;
#pragma unroll 4
  for (int e = t; e < a.experts; e += L) {
    differ |= logit(row, a.dt, e) != z;
    if (bias != nullptr) differ |= bias[e] != b;
  }
  return or_of<L>(differ ? 1u : 0u) == 0;
}

template <int L, int V>
__global__ __launch_bounds__(RT_THREADS) void k_route(const RouteArgs a) {
  constexpr int TOKENS = RT_THREADS / L;
  constexpr int PICKS = L * V < ODP_ROUTE_CHOICES ? L * V : ODP_ROUTE_CHOICES;
  __shared__ uint64_t lds[RT_THREADS / 64][route_words<L, V>()];
  __shared__ uint32_t chains[TOKENS * (PICKS + 1)];
  const int slot = threadIdx.x / L, t = threadIdx.x % L, mine = slot % (64 / L);
  int64_t token = a.token0 + (int64_t)blockIdx.x * TOKENS + slot;
  const bool live = token < a.n;
  token = live ? token : a.n - 1;
  const char* row = a.z + token * a.ldz;
  const float* bias = a.bias;
  if (bias != nullptr && a.rows_per_bias > 0) bias += token / a.rows_per_bias * a.experts;
  uint32_t* chain = chains + slot * (PICKS + 1);
  uint64_t* words = lds[threadIdx.x / 64];
  const int first = t * V;

  float z[V];
  load_row<V>(z, row, a.dt, first, a.experts, -INFINITY);
  const uint32_t mask = (1u << a.bits) - 1;
  // Keys that are sums (of a score and its bias, or of a group's two) are held
  // as their share of their range, logits of float32 as theirs of the row's
  // range, the 128 below the largest of it; 16-bit logits fit as they are.
  const bool sums = bias != nullptr || (a.groups > 1 && a.best == 0);
  const bool fits = !sums && a.dt != ODP_DTYPE_F32;
  const uint32_t steps = 1u << min(24, 32 - a.bits);
  float top = -INFINITY, low = INFINITY, total = 0.0f;
  uint32_t size = 0;  // the largest magnitude, by its bits: NaN above infinity
#pragma unroll
  for (int i = 0; i < V; ++i) {
    top = fmaxf(top, z[i]);
    low = fminf(low, z[i]);
    size = max(size, __float_as_uint(z[i]) & 0x7fffffffu);
  }
  const bool odd0 = size > 0x7f800000u || top == INFINITY;
  bool bounded = low > -INFINITY;  // no expert of this thread masked, none missing
  top = fmax_of<L>(top);
  const bool whole = !a.sigmoid && (sums || !a.renorm);
  float p[V];
  if (whole) {
    if (a.renorm) {  // for keys alone (units_apart)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        p[i] = __builtin_amdgcn_exp2f((z[i] - top) * 1.44269502f);
        total += p[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        p[i] = z[i] == -INFINITY ? 0.0f : exp_near(z[i] - top);
        total += p[i];
      }
    }
    total = sum_of<L>(total);
  }
  uint32_t key[V];  // 0: no expert, or closed; leading parts: 1 masked, 2 and more the others
  uint32_t tol = 0;
  bool weird = false;  // a row for route_exactly
  bool cut = false;    // keys far below the largest bias share a leading part of 2
  const uint32_t place = mask - (uint32_t)first;
  if (sums) {
    float lo = 0.0f, hi = 0.0f, b[V];
    if (bias != nullptr) {
      load_row<V>(b, (const char*)bias, ODP_DTYPE_F32, first, a.experts, -INFINITY);
      lo = INFINITY;
      hi = -INFINITY;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool shut = b[i] == -INFINITY;  // a key of -inf, as a masked expert's
        z[i] = shut ? -INFINITY : z[i];
        bounded &= !shut;
        lo = fminf(lo, shut ? INFINITY : b[i]);
        hi = fmaxf(hi, b[i]);
      }
#pragma unroll
      for (int i = 0; i < V; i += 2) weird |= __builtin_isunordered(b[i], b[i + 1]);  // a NaN
      lo = -fmax_of<L>(-lo);
      hi = fmax_of<L>(hi);
      if (!(lo <= hi)) lo = hi = 0.0f;  // all shut
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = 0.0f;
    }
    const float over = a.sigmoid ? 0.0f : __builtin_amdgcn_rcpf(total);
    // The largest softmax is e^0 over the sum; a row that is all masked has none.
    const float one = total > 0.0f && !a.sigmoid ? over : 1.0f;
    // One bias far below the rest (an expert switched off by -1e4) would coarsen all
    // keys.  Where `enough` experts lie within d of the largest, what is below that
    // shares the least leading part: in order still, and near each other where the
    // choice should come to hang on them after all.  Biases spread out evenly fail at
    // the first d.  32768 tokens of 256 experts, one of them at -1e4: 24 us by sigmoids
    // (20 without it; uncut 234), 27 in groups (23; 149).
    const bool deep = hi - lo > ROUTE_DEEP * one;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(deep) != 0, 0) && deep) {
      const float enough = (float)(a.groups > 1 ? 2 * a.top_k * a.groups / a.top_groups : a.top_k);
#pragma unroll 1
      for (float d = fminf((hi - lo) * 0.0625f, 0x1p15f * one);; d *= 0.125f) {
        float within = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) within += z[i] > -INFINITY && b[i] >= hi - d ? 1.0f : 0.0f;
        if (!(sum_of<L>(within) >= enough)) break;
        cut = true;
        lo = hi - d;
        if (!(d > 8.0f * one)) break;
      }
    }
    const float range = one + (hi - lo);
    weird |= !(range < 1e30f);
    // From 2^20 on keys in 64 bits lose what the words still tell apart.
    weird |= fmaxf(fabsf(lo), fabsf(hi)) >= 0x1p20f;
    const float by = (float)(steps - 16) * __builtin_amdgcn_rcpf(range);
    tol = (units_apart(a.sigmoid, over * __builtin_amdgcn_rcpf(range)) >> (24 - min(24, 32 - a.bits))) + 1;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float s = a.sigmoid ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z[i] * -1.44269502f)) : p[i] * over;
      b[i] = fmaf(s, by, fmaf(b[i] - lo, by, 2.0f));
    }
    if (__builtin_amdgcn_ballot_w64(cut) != 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = fmaxf(b[i], 2.0f);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = (uint32_t)b[i] << a.bits | (place - i);
  } else if (fits) {
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = (ordered(z[i] + 0.0f) & ~mask) | (place - i);
  } else {
    low = fmaxf(-fmax_of<L>(-low), top - 128.0f);
    const float by = (float)(steps - 16) * __builtin_amdgcn_rcpf(fmaxf(top - low, 1e-30f));
#pragma unroll
    for (int i = 0; i < V; ++i)
      key[i] = (uint32_t)fmaf(fmaxf(z[i] - low, 0.0f), by, 2.0f) << a.bits | (place - i);
  }
  if (__builtin_amdgcn_ballot_w64(!bounded) != 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (first + i >= a.experts) {
        key[i] = 0;
      } else if (!fits && z[i] == -INFINITY) {
        key[i] = 1u << a.bits | (place - i);
        weird |= sums && a.groups > 1 && a.best == 0;  // it adds nothing to its group's sum
      }
    }
  }
  const uint32_t both = or_of<L>((odd0 ? 1u : 0u) | (weird ? 2u : 0u));
  const bool odd = (both & 1) != 0;  // a NaN or +inf
  weird = both != 0;
  Keys64 exact{a, row, bias, sums, top};

  if (a.groups > 1) {
    uint32_t* scores = chain;  // [groups], before the choices
    const auto second = [](uint32_t& one, uint32_t& two, uint32_t o1, uint32_t o2) {  // the two largest of four
      two = max(min(one, o1), max(two, o2));
      one = max(one, o1);
    };
    // The sum of two leading parts takes up to 25 bits, a group's number 6; a
    // best key stands as it is (its low bits order equal ones by the group).
    const auto score = [&](uint32_t one, uint32_t two, int g) {
      return a.best == 0 ? ((one >> a.bits) + (two >> a.bits)) << 6 | (uint32_t)(63 - g) : one;
    };
    // A group's sum with a second key that is cut is more than the keys'.
    bool mixed = false;
    const auto cut_in = [&](uint32_t one, uint32_t two) {
      mixed |= cut && a.best == 0 && two >> a.bits == 2 && one >> a.bits > 2;
    };
    const int span = a.span;  // threads of a group; 0: its bounds lie between them
    if (span > 0) {
      uint32_t one = 0, two = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        two = max(two, min(one, key[i]));
        one = max(one, key[i]);
      }
      if (L > 1 && span > 1) second(one, two, across<1>(one), across<1>(two));
      if (L > 2 && span > 2) second(one, two, across<2>(one), across<2>(two));
      if (L > 4 && span > 4) second(one, two, across<4>(one), across<4>(two));
      if (L > 8 && span > 8) second(one, two, across<8>(one), across<8>(two));
      if (L > 16 && span > 16) second(one, two, across<16>(one), across<16>(two));
      const int g = t / span;
      if (t == g * span && g < a.groups) {
        scores[g] = score(one, two, g);
        cut_in(one, two);
      }
    } else {
      uint32_t* all = (uint32_t*)words + mine * L * V;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (first + i < a.experts) all[first + i] = key[i];
      wave_sync();
      for (int g = t; g < a.groups; g += L) {
        uint32_t one = 0, two = 0;
        int i = g % a.size;  // each thread from another bank on
#pragma unroll 4
        for (int k = 0; k < a.size; ++k) {
          const uint32_t w = all[g * a.size + i];
          two = max(two, min(one, w));
          one = max(one, w);
          i = i + 1 == a.size ? 0 : i + 1;
        }
        scores[g] = score(one, two, g);
        cut_in(one, two);
      }
    }
    wave_sync();
    uint64_t open = 0;
    uint32_t last = 0, next = 0;
    for (int g = t; g < a.groups; g += L) {
      const uint32_t own = scores[g];
      int above = 0;
#pragma unroll 4
      for (int o = 0; o < a.groups; ++o) above += scores[o] > own;
      if (above < a.top_groups) open |= 1ull << g;
      if (above == a.top_groups - 1) last = own;
      if (above == a.top_groups) next = own;
    }
    last = max_of<L>(last);
    next = max_of<L>(next);
    const uint32_t lo = or_of<L>((uint32_t)open), hi = a.groups > 32 ? or_of<L>((uint32_t)(open >> 32)) : 0;
    open = (uint64_t)hi << 32 | lo;
    const int shift = a.best == 0 ? 6 : a.bits;
    const uint32_t apart = (last >> shift) - (next >> shift);
    bool unsure = !fits && !weird && apart <= (a.best == 0 ? 2 * tol : tol);
    if (__builtin_amdgcn_ballot_w64(mixed) != 0) unsure |= !weird && or_of<L>(mixed ? 1u : 0u) != 0;
    wave_sync();
    if (__builtin_amdgcn_ballot_w64(unsure && apart == 0) != 0) unsure &= apart != 0 || !all_equal<L>(a, row, bias, t);
    if (__builtin_amdgcn_ballot_w64(unsure) != 0) {
#pragma unroll 1
      for (int k = 0; k < 64 / L; ++k) {
        if (unsure && mine == k) open = open_exactly<L, V>(a, exact, t, words);
        wave_sync();
      }
    }
    if (span > 0) {
      if (!(open >> ((t / span) & 63) & 1)) {
#pragma unroll
        for (int i = 0; i < V; ++i) key[i] = 0;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int g = (int)(((float)(first + i) + 0.5f) * a.per_size);
        if (!(open >> (g & 63) & 1)) key[i] = 0;
      }
    }
  }

  // The largest word below `last` (0: any), 0 where there is none: the largest
  // difference then belongs to one above it, or to itself.
  const auto below = [&](uint32_t last) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) m = max(m, key[i] - last);
    m = max_of<L>(m) + last;
    return last != 0 && m >= last ? 0u : m;
  };
  uint32_t last = 0;
  for (int j = 0; j <= a.top_k; ++j) {  // one more, for how near it lies
    last = below(last);
    if (t == 0) chain[j] = last;
  }
  wave_sync();
  // The pairs that lie near each other: those of equal logits and biases are equal
  // keys, which the words order already, and so are two masked experts.
  bool near = false, last_near = false;
  if (!fits) {
    for (int j = t; j < a.top_k; j += L) {
      const uint32_t w = chain[j], n = chain[j + 1];
      if (n == 0 || (w >> a.bits) - (n >> a.bits) > tol || weird) continue;
      const int e0 = (int)(mask - (w & mask)), e1 = (int)(mask - (n & mask));
      const float z0 = logit(row, a.dt, e0), z1 = logit(row, a.dt, e1);
      near |= z0 != z1 || (z0 != -INFINITY && bias != nullptr && bias[e0] != bias[e1]);
      last_near |= j == a.top_k - 1;
    }
  }
  const uint32_t flags = or_of<L>((near || weird ? 1u : 0u) | (last_near ? 2u : 0u));
  // A choice that equals the next word is one of a run, which may end near others.
  const bool on = (flags & 2) != 0;
  bool slow = weird || (!fits && flags != 0);
  const bool level = slow && !weird && chain[0] >> a.bits == chain[a.top_k] >> a.bits;
  if (__builtin_amdgcn_ballot_w64(level) != 0) slow &= !level || !all_equal<L>(a, row, bias, t);
  if (__builtin_amdgcn_ballot_w64(slow) != 0) {
#pragma unroll 1
    for (int k = 0; k < 64 / L; ++k) {
      if (slow && mine == k) choose_exactly<L, V, PICKS>(a, exact, below, t, tol, weird, on, words, chain);
      wave_sync();
    }
  }

  // The weights of the chosen, PER a thread.
  constexpr int PER = (PICKS + L - 1) / L;
  const bool off = odd && !a.sigmoid;
  int e[PER];
  float x[PER], most = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = t + i * L;
    if (j >= a.top_k) break;
    e[i] = slow ? (int)chain[j] : (int)(mask - (chain[j] & mask));
    x[i] = logit(row, a.dt, e[i]);
    most = fmaxf(most, x[i]);
  }
  if (a.renorm) most = fmax_of<L>(most);
  const Shares share(a, most, top);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (t + i * L >= a.top_k) break;
    x[i] = share(x[i]);
    sum += x[i];
  }
  sum = a.renorm ? sum_of<L>(sum) : a.sigmoid ? 1.0f : total;
  if (!live) return;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = t + i * L;
    if (j >= a.top_k) break;
    const float w = off ? NAN : x[i] == 0.0f ? 0.0f : a.scale * (x[i] / sum);
    odp_gstore(a.index + token * a.top_k + j, (int64_t)e[i]);
    odp_gstore(a.weights + token * a.top_k + j, w);
  }
}

// Values c to c + 8 of a 16-bit row, or to c + 4 of a float32 one (fewer at its end).
__device__ __forceinline__ void store_some(char* row, int dt, int c, int experts, const float* v) {
  const int n = dt == ODP_DTYPE_F32 ? 4 : 8;
  if (c + n > experts) {
    for (int i = 0; c + i < experts; ++i) odp_store_from_float(row, c + i, dt, v[i]);
    return;
  }
  u32x4_t w;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (dt == ODP_DTYPE_F32) w[j] = __float_as_uint(v[j]);
    else if (dt == ODP_DTYPE_BF16) w[j] = odp_f2bf2(v[2 * j], v[2 * j + 1]);
    else
      w[j] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * j]) |
             (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * j + 1]) << 16;
  }
  if (dt == ODP_DTYPE_F32) *(ODP_GMEM u32x4_w*)(ODP_GMEM void*)(row + 4 * c) = w;
  else *(ODP_GMEM u32x4_h*)(ODP_GMEM void*)(row + 2 * c) = w;
}

// Whether one of a row's values is NaN or +inf, for this thread's pieces of N.
template <int L, int V, int N>
__device__ __forceinline__ bool odd_pieces(const RouteArgs& a, const char* row, int t) {
  bool odd = false;
  float z[V / N][N];
#pragma unroll
  for (int j = 0; j < V / N; ++j) load_row<N>(z[j], row, a.dt, N * (t + j * L), a.experts, -INFINITY);
#pragma unroll
  for (int i = 0; i < V; ++i) odd |= !(z[i / N][i % N] < INFINITY);
  return odd;
}

// A token's dz out of its chosen entries d (0 elsewhere): its L threads hold
// pieces of N values side by side, 16 bytes each.  For a softmax that is not
// renormalised every logit has a part.
template <int L, int V, int N>
__device__ __forceinline__ void store_dz(const RouteArgs& a, const char* row, char* to, const float* d, int t,
                                         bool live) {
  if (a.sigmoid || a.renorm) {
    if (!live) return;
    for (int c = N * t; c < a.experts; c += N * L) store_some(to, a.dt, c, a.experts, d + c);
    return;
  }
  float z[V / N][N], top = -INFINITY, total = 0.0f, with = 0.0f;
  bool odd = false;
#pragma unroll
  for (int j = 0; j < V / N; ++j) load_row<N>(z[j], row, a.dt, N * (t + j * L), a.experts, -INFINITY);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    top = fmaxf(top, z[i / N][i % N]);
    odd |= !(z[i / N][i % N] < INFINITY);
  }
  odd = or_of<L>(odd ? 1u : 0u) != 0;
  top = fmax_of<L>(top);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float& p = z[i / N][i % N];
    p = p == -INFINITY ? 0.0f : exp_near(p - top);
    total += p;
    with += p == 0.0f ? 0.0f : p * d[N * (t + i / N * L) + i % N];
  }
  total = sum_of<L>(total);
  const float over = total > 0.0f ? 1.0f / total : 0.0f;
  with = sum_of<L>(with) * over;
  if (!live) return;
#pragma unroll
  for (int j = 0; j < V / N; ++j) {
    const int c = N * (t + j * L);
#pragma unroll
    for (int i = 0; i < N; ++i) z[j][i] = odd ? NAN : z[j][i] == 0.0f ? 0.0f : z[j][i] * over * (d[c + i] - with);
    if (c < a.experts) store_some(to, a.dt, c, a.experts, z[j]);
  }
}

// dz of a token's L threads: the chosen entries through LDS, from which the row
// leaves.  Every store of a wave writes whole lines; with the 8 or 16 values of
// a thread side by side 32768 x 256 of float32 took 16 us, so 9 (33 MB written;
// 12 for a softmax, whose rows are read too, 15 without renormalize, before 33).
template <int L, int V>
__global__ __launch_bounds__(RT_THREADS) void k_route_grad(const RouteArgs a) {
  constexpr int TOKENS = RT_THREADS / L;
  __shared__ __align__(16) float lds[TOKENS * L * V];
  const int slot = threadIdx.x / L, t = threadIdx.x % L;
  int64_t token = a.token0 + (int64_t)blockIdx.x * TOKENS + slot;
  const bool live = token < a.n;
  token = live ? token : a.n - 1;
  const char* row = a.z + token * a.ldz;
  const int64_t* chosen = a.chosen + token * a.top_k;
  const float* gw = a.gw + token * a.ldw;
  float* d = lds + slot * L * V;
#pragma unroll
  for (int i = 0; i < V; ++i) d[4 * (t + i / 4 * L) + i % 4] = 0.0f;
  constexpr int PICKS = L * V < ODP_ROUTE_CHOICES ? L * V : ODP_ROUTE_CHOICES, PER = (PICKS + L - 1) / L;
  int e[PER];
  float x[PER], g[PER], most = -INFINITY, sum = 0.0f, dot = 0.0f;
  bool odd = false;  // a softmax with a NaN or +inf
  if (a.renorm && !a.sigmoid)
    odd = a.dt == ODP_DTYPE_F32 ? odd_pieces<L, V, 4>(a, row, t) : odd_pieces<L, V, 8>(a, row, t);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = t + i * L;
    if (j >= a.top_k) break;
    e[i] = (int)min(max(chosen[j], (int64_t)0), (int64_t)(a.experts - 1));
    g[i] = gw[j];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (t + i * L >= a.top_k) break;
    x[i] = logit(row, a.dt, e[i]);
    most = fmaxf(most, x[i]);
  }
  if (a.renorm) {
    most = fmax_of<L>(most);
    odd = or_of<L>(odd ? 1u : 0u) != 0;
    const Shares share(a, most, 0.0f);
    float s[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (t + i * L >= a.top_k) break;
      s[i] = share(x[i]);
      sum += s[i];
    }
    sum = sum_of<L>(sum);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (t + i * L >= a.top_k) break;
      s[i] = s[i] == 0.0f ? 0.0f : s[i] / sum;  // 1 where it is the only one, whose gradient is then 0
      dot += s[i] == 0.0f ? 0.0f : s[i] * g[i];
    }
    dot = sum_of<L>(dot);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (t + i * L >= a.top_k) break;
      g[i] = s[i] == 0.0f ? 0.0f : s[i] * (g[i] - dot);
      if (a.sigmoid) g[i] *= sigmoid(-x[i]);
    }
  } else if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (t + i * L >= a.top_k) break;
      g[i] = x[i] == -INFINITY ? 0.0f : sigmoid(x[i]) * sigmoid(-x[i]) * g[i];
    }
  }
  wave_sync();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (t + i * L >= a.top_k) break;
    d[e[i]] = odd ? NAN : g[i] * a.scale;
  }
  wave_sync();
  if (a.dt == ODP_DTYPE_F32) store_dz<L, V, 4>(a, row, a.dz + token * a.experts * 4, d, t, live);
  else store_dz<L, V, 8>(a, row, a.dz + token * a.experts * 2, d, t, live);
}

template <int L, int V>
void launch_route(hipStream_t s, RouteArgs a, bool grad) {
  constexpr int TOKENS = RT_THREADS / L;
  const int span = a.size / V;
  a.span = a.size % V == 0 && (span & (span - 1)) == 0 ? span : 0;
  // A launch's threads are counted in 32 bits.
  constexpr int64_t MOST = ((int64_t)1 << 31) / RT_THREADS;
  for (a.token0 = 0; a.token0 < a.n; a.token0 += MOST * TOKENS) {
    const int64_t left = (a.n - a.token0 + TOKENS - 1) / TOKENS;
    const uint32_t blocks = (uint32_t)(left < MOST ? left : MOST);
    if (grad) k_route_grad<L, V><<<blocks, RT_THREADS, 0, s>>>(a);
    else k_route<L, V><<<blocks, RT_THREADS, 0, s>>>(a);
  }
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
  a.bits = 8;  // leaves a leading part of 24 bits; of 23 above 256 experts, of 22 above 512
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
  if (bias != nullptr && (biases < 1 ? n != 0 || biases < 0 : n % biases != 0)) {  // an empty batch has no biases
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
