// C = A B^T over LDS-staged MFMA tiles, for operands in either order of the
// contraction: the products of the vocabulary loss.
//
// Included inside an anonymous namespace, after odp_internal.h.  A workgroup
// owns an OT x NT tile of C: rows o from A, columns n from B.  256 x 256 in
// bfloat16 and 128 x 128 in float32; with S == 1, for few rows, 64 x 128 and a ring
// of more, smaller stages, since such a product waits for B's memory; with S
// == 2 (bfloat16) 128 x 256; with S == 3 (float32, whose MFMAs would take longer
// than that memory for 64 rows) 32 x 128.  An operand is K-contiguous (KC: element
// (row, k) at row * ld + k, as the rows of activations or of a weight) or
// K-major (element (row, k) at k * ld + row: the contraction runs over the
// rows of memory).  A step covers 64 bytes of k; both orders then stage the
// same bytes, 64-byte rows of k or rows of o or n, by buffer loads straight
// into a ring of LDS stages, all but one step ahead of the MFMAs.
//
// 256 x 256 of bfloat16 keeps 128 registers of sums a lane and reads each
// staged byte for 8 MFMAs a wave; a CU then holds one workgroup of 8 waves, and
// what hides latency is the ring (4 stages of 32 KB).  Measured on the loss's
// products: 1240 TFLOP/s with rows of k for both operands, 1360 with one and
// 1300 with both K-major (the vendor library 1421, 1373 and 1102 on the same
// shapes).  float32 has no wider MFMA than 16 x 16 x 4: 119, 114 (library 114, 72).
#pragma once

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t u32x4_alias_t __attribute__((may_alias));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef u32x2_t u32x2_alias_t __attribute__((may_alias));
typedef short v4i16_t __attribute__((ext_vector_type(4)));

#define ODP_LDS __attribute__((address_space(3)))
#define ODP_CONST __attribute__((address_space(4)))

constexpr uint32_t T_RSRC = 0x00020000;  // raw buffer resource, 32-bit offsets
constexpr uint32_t T_OOB = 0x80000000u;  // an offset past every buffer's end: reads as zero

template <int DT, int S>
struct Tile {
  static constexpr bool F32 = DT == ODP_DTYPE_F32;
  static constexpr int ES = F32 ? 4 : 2;          // bytes per element
  static constexpr bool FEW = S == 1 || S == 3;
  static constexpr int OT = S == 1 ? 64 : S == 2 ? 128 : S == 3 ? 32 : 512 / ES;  // rows (o) of the tile
  static constexpr int NT = FEW ? 128 : 512 / ES;                                 // columns (n)
  static constexpr int EK = 64 / ES;              // k per step
  static constexpr int WR = S == 3 ? 1 : 2;       // waves over the rows
  static constexpr int WM = OT / WR, WN = 64;     // a wave's block
  static constexpr int WC = NT / WN, WAVES = WC * WR, THREADS = 64 * WAVES;
  static constexpr int BI = WM / 16, BJ = WN / 16;
  static constexpr int ABYTES = OT * 64, BBYTES = NT * 64, STAGE = ABYTES + BBYTES;  // of a step
  static constexpr int ALOADS = ABYTES / 1024 / WAVES, BLOADS = BBYTES / 1024 / WAVES;  // 1 KB loads per wave
  static constexpr int LOADS = ALOADS + BLOADS;
  static constexpr int RING = FEW ? 6 : 4;
  static_assert(ALOADS * WAVES * 1024 == ABYTES && BLOADS * WAVES * 1024 == BBYTES, "whole loads");
  typedef f32x4_t Acc[BI][BJ];
  // First row and column of a wave's block.
  static __device__ __forceinline__ int wm(int wave) { return WM * (wave % WR); }
  static __device__ __forceinline__ int wn(int wave) { return WN * (wave / WR); }
};

// Stage k of the ring: separate arrays, so that reads of one are not made to
// wait for the loads into another.
template <int BYTES, int K>
__device__ __forceinline__ char* t_array() {
  __shared__ __attribute__((aligned(16))) char s[BYTES];
  return s;
}
template <int DT, int S>
__device__ __forceinline__ char* t_stage(int k) {
  constexpr int B = Tile<DT, S>::STAGE;
  if constexpr (Tile<DT, S>::RING == 4)
    return k == 0 ? t_array<B, 0>() : k == 1 ? t_array<B, 1>() : k == 2 ? t_array<B, 2>() : t_array<B, 3>();
  else
    return k == 0   ? t_array<B, 0>()
           : k == 1 ? t_array<B, 1>()
           : k == 2 ? t_array<B, 2>()
           : k == 3 ? t_array<B, 3>()
           : k == 4 ? t_array<B, 4>()
                    : t_array<B, 5>();
}

// Swizzles.  64-byte rows of k: 16-byte slot s of row r lies at slot
// s ^ ((r >> 1) & 3) (full rate for operand reads, measured on the Gram
// kernels).  Rows of 16-bit columns: 8-byte chunks XOR-ed as the transposing
// reads of the full-weight kernels take them; of 32-bit columns:
// 64-byte groups XOR-ed with the row's quarter, so that the four rows a lane
// group reads lie on different banks.
__device__ __forceinline__ int t_kswz(int row) { return (row >> 1) & 3; }
template <int DT>
__device__ __forceinline__ int t_cswz(int row) {  // in 16-byte pieces
  return DT == ODP_DTYPE_F32 ? ((row >> 2) & 3) << 2 : ((row & 3) | ((row >> 1) & 4)) << 1;
}

// The MFMA operand of 16 rows from row0 of a staged operand: lane & 15 = row,
// 16 bytes of k per lane (the slot lane >> 4).
template <int DT, bool KC, int EXT>
__device__ __forceinline__ u32x4_t t_frag(const char* half, int row0) {
  constexpr int PITCH = EXT * (DT == ODP_DTYPE_F32 ? 4 : 2);  // bytes of a K-major row of EXT columns
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  if constexpr (KC) {
    const int row = row0 + c;
    return *(const u32x4_alias_t*)(half + row * 64 + 16 * (q ^ t_kswz(row)));
  } else if constexpr (DT == ODP_DTYPE_F32) {
    u32x4_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = 4 * q + e;
      v[e] = *(const uint32_t*)(half + k * PITCH + 16 * (((row0 + c) >> 2) ^ t_cswz<DT>(k)) + 4 * (c & 3));
    }
    return v;
  } else {
    // Rows k and k + 4 share the swizzle; each read transposes a 4 x 16 block.
    const int k = 8 * q + (c >> 2);
    const int chunk = ((row0 >> 2) + (c & 3)) ^ (t_cswz<DT>(k) << 1);
    const char* src = half + k * PITCH + 8 * chunk;
    const v4i16_t t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ODP_LDS v4i16_t*)(ODP_LDS void*)src);
    const v4i16_t t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ODP_LDS v4i16_t*)(ODP_LDS void*)(src + 4 * PITCH));
    const v4i16_t tt[2] = {t0, t1};
    return __builtin_bit_cast(u32x4_t, tt);
  }
}

template <int DT>
__device__ __forceinline__ f32x4_t t_mfma(u32x4_t b, u32x4_t a, f32x4_t c) {
  if constexpr (DT == ODP_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b[e]), __uint_as_float(a[e]), c, 0, 0, 0);
    return c;
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, b), __builtin_bit_cast(bf16x8_t, a),
                                                   c, 0, 0, 0);
  }
}

__device__ __forceinline__ uint32_t t_uniform(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
__device__ __forceinline__ uint64_t t_uniform64(uint64_t v) {
  return ((uint64_t)t_uniform((uint32_t)(v >> 32)) << 32) | t_uniform((uint32_t)v);
}

// One operand of a tile: `base` is element (row 0 of the matrix, k = 0),
// `row0` the tile's first row, `rows` the matrix's.  The host's checks of ld keep
// the rows of a tile within 31-bit offsets: rows of x and W lie less than 2^22
// bytes apart, rows of d less than 2^23 (256 of bfloat16) or 2^24 (128 of float32).
struct Operand {
  const void* base;
  int64_t ld;
  int64_t row0;
  int64_t rows;
};

// What a lane needs to issue its N loads of one operand, of EXT rows (o or n) a step.
template <int DT, bool KC, int EXT, int N>
struct Loader {
  static constexpr int ES = DT == ODP_DTYPE_F32 ? 4 : 2, EK = 64 / ES;
  static constexpr int LPR = EXT * ES / 16, RPL = 64 / LPR;  // K-major: lanes per row, rows per load
  uint64_t at;    // base of the step's loads
  uint32_t step;  // bytes the base moves per step
  uint32_t ldb;   // bytes per row of memory
  uint32_t off[N];
  int32_t k8[N];  // KC: first k of the load's 16 bytes

  __device__ __forceinline__ void init(const Operand& op, int wave) {
    const int lane = threadIdx.x & 63;
    ldb = t_uniform((uint32_t)(op.ld * ES));
    if constexpr (KC) {
      at = t_uniform64((uint64_t)op.base + (uint64_t)op.row0 * ldb);
      step = 64;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = 16 * (N * wave + i) + (lane >> 2), slot = (lane & 3) ^ t_kswz(row);
        off[i] = op.row0 + row < op.rows ? (uint32_t)row * ldb + 16u * slot : T_OOB;
        k8[i] = slot * (16 / ES);
      }
    } else {
      at = t_uniform64((uint64_t)op.base + (uint64_t)op.row0 * ES);
      step = t_uniform(ldb * EK);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int k = RPL * (N * wave + i) + lane / LPR;
        const int piece = (lane % LPR) ^ t_cswz<DT>(k), col = piece * (16 / ES);
        off[i] = op.row0 + col < op.rows ? (uint32_t)k * ldb + 16u * piece : T_OOB;
        k8[i] = 0;
      }
    }
  }

  // Load i of the step whose first k is k0 of kn (k0 >= kn: zeros).
  __device__ __forceinline__ void issue(char* half, int wave, int i, int32_t k0, int32_t kn) const {
    uint32_t o = off[i], bytes;
    if constexpr (KC) {
      bytes = 0x7fffffffu;
      if (k8[i] + k0 >= kn) o = T_OOB;
    } else {
      const int32_t left = kn - k0;
      bytes = left <= 0 ? 0u : (uint32_t)(left < EK ? left : EK) * ldb;
    }
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)at, (short)0, (int)bytes, T_RSRC);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (ODP_LDS void*)(half + 1024 * (N * wave + i)), 16, o, 0, 0, 0);
  }
};

// The operands a step starts with, read during the step before it.
template <int DT, int S>
struct Head {
  u32x4_t b[Tile<DT, S>::BJ], a[2];
};

template <int DT, int S, bool AKC, bool BKC>
__device__ __forceinline__ void t_head(const char* st, Head<DT, S>& h) {
  using T = Tile<DT, S>;
  const int wave = threadIdx.x >> 6, wm = T::wm(wave), wn = T::wn(wave);
#pragma unroll
  for (int j = 0; j < T::BJ; ++j) h.b[j] = t_frag<DT, BKC, T::NT>(st + T::ABYTES, wn + 16 * j);
  h.a[0] = t_frag<DT, AKC, T::OT>(st, wm);
  h.a[1] = t_frag<DT, AKC, T::OT>(st, wm + 16);
}

// One step: its MFMAs from `cur` and the operands in h, the loads of a later
// step into `nxt` between the first of them, the next step's first operands
// from `ahead` beside the last.  The stages are restrict parameters so that
// the reads do not wait for the loads into `nxt`.
template <int DT, int S, bool AKC, bool BKC, typename Issue>
__device__ __forceinline__ void t_step(char* __restrict__ nxt, const char* __restrict__ cur,
                                       const char* __restrict__ ahead, Issue issue, Head<DT, S>& h, Head<DT, S>& n,
                                       typename Tile<DT, S>::Acc& acc) {
  using T = Tile<DT, S>;
  const int wave = threadIdx.x >> 6, wm = T::wm(wave), wn = T::wn(wave);
  // Block rows beside which the next step's b is read: the last but one of as
  // many as it takes, or all.
  constexpr int ROWS = T::BJ < T::BI ? T::BJ : T::BI, R0 = T::BJ < T::BI ? T::BI - 1 - T::BJ : 0;
  constexpr int PER = (T::LOADS + T::BI - 1) / T::BI;  // loads a block row, over the first of them
  u32x4_t a[3] = {h.a[0], h.a[1], h.a[1]};
#pragma unroll
  for (int i = 0; i < T::BI; ++i) {
    if (i + 2 < T::BI) a[(i + 2) % 3] = t_frag<DT, AKC, T::OT>(cur, wm + 16 * (i + 2));
#pragma unroll
    for (int l = PER * i; l < PER * (i + 1) && l < T::LOADS; ++l) issue(nxt, l);
    if (i >= R0 && i < R0 + ROWS) {
#pragma unroll
      for (int j = T::BJ * (i - R0) / ROWS; j < T::BJ * (i - R0 + 1) / ROWS; ++j)
        n.b[j] = t_frag<DT, BKC, T::NT>(ahead + T::ABYTES, wn + 16 * j);
    }
    if (i >= T::BI - 2) n.a[i - (T::BI - 2)] = t_frag<DT, AKC, T::OT>(ahead, wm + 16 * (i - (T::BI - 2)));
#pragma unroll
    for (int j = 0; j < T::BJ; ++j) acc[i][j] = t_mfma<DT>(h.b[j], a[i % 3], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The product of a tile in two parts: begin() issues the first steps' loads,
// run() does the rest.  A workgroup that walks several tiles begins the next
// one before it stores the last, so that the loads' latency passes beside the
// epilogue (which must leave the ring alone).
template <int DT, int S, bool AKC, bool BKC>
struct Product {
  using T = Tile<DT, S>;
  Loader<DT, AKC, T::OT, T::ALOADS> la;
  Loader<DT, BKC, T::NT, T::BLOADS> lb;
  int32_t kl, kn;  // first k of the next step to load, and the end
  int wave;

  __device__ __forceinline__ void issue(char* st, int l) const {
    if (l < T::ALOADS) la.issue(st, wave, l, kl, kn);
    else lb.issue(st + T::ABYTES, wave, l - T::ALOADS, kl, kn);
  }
  __device__ __forceinline__ void advance() {
    kl += T::EK;
    la.at += la.step;
    lb.at += lb.step;
  }

  // The ring is idle (no wave reads it, no load into it is in flight).
  __device__ __forceinline__ void begin(const Operand& A, const Operand& B, int32_t k) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    kn = (int32_t)t_uniform((uint32_t)k);
    kl = 0;
    la.init(A, wave);
    lb.init(B, wave);
#pragma unroll
    for (int q = 0; q < T::RING - 1; ++q) {
#pragma unroll
      for (int l = 0; l < T::LOADS; ++l) issue(t_stage<DT, S>(q), l);
      advance();
    }
  }

  // acc = A B^T over k in [0, kn).
  __device__ __forceinline__ void run(typename T::Acc& acc) {
#pragma unroll
    for (int i = 0; i < T::BI; ++i)
#pragma unroll
      for (int j = 0; j < T::BJ; ++j) {
        acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        __asm__ volatile("" : "+v"(acc[i][j]));
      }
    Head<DT, S> h[2];
    // Everything so far, an epilogue's stores among it.
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __asm__ volatile("s_barrier" ::: "memory");
    t_head<DT, S, AKC, BKC>(t_stage<DT, S>(0), h[0]);
    int32_t k = 0;
    while (k < kn) {
#pragma unroll
      for (int u = 0; u < T::RING; ++u) {
        if (k >= kn) break;
        // The next step's loads have landed (this wave's; the barrier says so
        // for the others); those of the steps after it may fly.
        __builtin_amdgcn_s_waitcnt(vmcnt_imm((T::RING - 3) * T::LOADS));
        __asm__ volatile("s_barrier" ::: "memory");
        t_step<DT, S, AKC, BKC>(t_stage<DT, S>((u + T::RING - 1) % T::RING), t_stage<DT, S>(u % T::RING),
                             t_stage<DT, S>((u + 1) % T::RING),
                             [&](char* st, int l) __attribute__((always_inline)) { issue(st, l); }, h[u & 1],
                             h[(u + 1) & 1], acc);
        advance();
        k += T::EK;
      }
    }
    __builtin_amdgcn_s_waitcnt(0);  // no load into LDS may outlive the tile
    __asm__ volatile("s_barrier" ::: "memory");
  }
};

// Entry e of block (i, j) of the wave's accumulators is row o = 16 i +
// (lane & 15) and column n = 16 j + 4 (lane >> 4) + e of the wave's block.
__device__ __forceinline__ int t_row(int i) { return 16 * i + (int)(threadIdx.x & 15); }
__device__ __forceinline__ int t_col(int j) { return 16 * j + 4 * (int)((threadIdx.x & 63) >> 4); }

template <int V>
struct Idx {
  static constexpr int value = V;
};
template <int N, int K = 0, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (K < N) {
    f(Idx<K>{});
    static_for<N, K + 1>(f);
  }
}
