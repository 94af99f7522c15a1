// dm_block_gemm.hip — C[m,n] = sum_k A[m,k] B[n,k] on the 16-bit matrix pipe, the products of the gated feed-forward block.
//
// An operand is stored either with k contiguous ("KC": rows of the operand) or with its own rows contiguous ("KS": k is the slow
// index), so that the forward pass and all three products of the backward pass run from the tensors as they lie in memory; a KS tile
// is transposed on its way out of LDS (ds_read_tr).  A product may have up to 12 terms, each
// over all of k with operands of its own: the two of dx = dg Wg + du Wu, times the six of fp32 operands split into three bf16 planes.
//
// A workgroup owns a BM x BN tile and walks k in steps of GEMM_BK: two LDS stages (three of the smallest tile), filled by buffer loads
// that write LDS directly (16 bytes per lane, rows and columns out of range are bounds-checked to zero by the buffer resource), one
// barrier per step.  The LDS image is swizzled in 16-byte pieces so that fragment reads touch all 64 banks once.  Fragments feed
// v_mfma_f32_16x16x32 (2.13 PFLOP/s of them alone under the power limit; 32x32x16: 1.90) with the n side as the first operand: a lane
// then holds four consecutive n of one m.
// A bias' gradient, the sum of A over k, is one more product with ones from the same fragments.
//
// Bound by the matrix pipe and what is issued beside it: a SIMD's time is nearly the sum of its waves' products and other instructions, so
// everything else in a step is kept short and lies between the products.  Measured, bf16, 8192 rows of width 4096, hidden 11008, a training step: both
// projections with their gate 1.28 ms (1.15 PFLOP/s, with 0.9 GB of what is kept), down 0.55 ms (1.34), dh with dg and du 0.79 ms, dx 1.09 ms (1.36),
// both projections' gradients in one launch 1.29 ms (1.15; 1376 tiles in six rounds of 256 CUs), the third weight's 0.64 ms (1.16; 688 in three); the
// library's products of these shapes reach 1.03 to 1.60.
#ifndef DM_BLOCK_GEMM_HIP
#define DM_BLOCK_GEMM_HIP
#include <atomic>
#include <type_traits>

#include "dm_block_common.h"

namespace dmb {

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
#define DM_LDS __attribute__((address_space(3)))

__device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c, bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c, f16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Three bf16 terms of an fp32 value, each the rest rounded to nearest: together they hold all 24 bits.  A value that would round to
// infinity keeps its leading bits instead; infinities and NaN go into the first term alone.
__device__ __forceinline__ void split3(float v, bf16 (&t)[3]) {
  bf16 a = (bf16)v;
  if (!(fabsf((float)a) <= 3.3895314e38f) && fabsf(v) <= 3.4028235e38f)
    a = __builtin_bit_cast(bf16, (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16));
  const float r = fabsf(v) <= 3.4028235e38f ? v - (float)a : 0.f;
  const bf16 b = (bf16)r;
  t[0] = a; t[1] = b; t[2] = (bf16)(r - (float)b);
}

enum { OUT_16 = 0, OUT_F32 = 1, OUT_PLANES = 2 };
// Where a result goes: rows of `ld` elements; OUT_PLANES: three bf16 planes, `plane` elements apart.  `vec`: rows take 16-byte stores.
struct Out { void* p; int64_t ld, plane; int f32, vec; };

__device__ __forceinline__ void store_f32(float* p, const float (&v)[8]) {
  const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
  store_vec<float, 4>(p, a);
  store_vec<float, 4>(p + 4, b);
}

template <typename T, int MODE>
__device__ __forceinline__ void store8(const Out& o, int64_t m, int n, int N, const float (&v)[8]) {
  const int64_t at = m * o.ld + n;
  if (o.vec && n + 8 <= N) {
    if constexpr (MODE == OUT_16) {
      store_vec<T, 8>((T*)o.p + at, v);
    } else if constexpr (MODE == OUT_F32) {
      store_f32((float*)o.p + at, v);
    } else {
      Vec<bf16, 8> r[3];
#pragma unroll
      for (int i = 0; i < 8; ++i) { bf16 t[3]; split3(v[i], t); r[0].v[i] = t[0]; r[1].v[i] = t[1]; r[2].v[i] = t[2]; }
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<Vec<bf16, 8>*>((bf16*)o.p + k * o.plane + at) = r[k];
    }
    return;
  }
  if constexpr (MODE != OUT_PLANES) {  // (planes are the block's own and take whole pieces)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (n + i >= N) break;
      if constexpr (MODE == OUT_16) ((T*)o.p)[at + i] = (T)v[i];
      else ((float*)o.p)[at + i] = v[i];
    }
  }
}

// Columns behind a row's end hold zeros whatever the row holds: the product of an infinite element with the zeros out there is NaN.
__device__ __forceinline__ void zero_behind(int n, int N, float (&v)[8]) {
  if (n + 8 > N)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = n + e < N ? v[e] : 0.f;
}

// ---- activations: value and slope in fp32, all but the erf form by way of s(z) = 1 / (1 + exp(-z)); tanh's by 1 + tanh(y) = 2 s(2 y).
// Results that are rounded to 16 bits take the hardware's exp2 and reciprocal (relative error below 2^-20 for |z| < 16).
// `rest`: 1 - s(z), where s is near 1 as exp(-z) s: the difference would hold none of its bits (z = 17) or too few (z = 9 for a slope of fp16).
template <bool FAST>
__device__ __forceinline__ float sigmoid(float z, float& rest) {
  const float e = FAST ? __builtin_amdgcn_exp2f(z * -1.44269504f) : expf(-z);
  const float s = FAST ? __builtin_amdgcn_rcpf(1.f + e) : 1.f / (1.f + e);
  rest = s < 0.5f ? 1.f - s : e * s;
  return s;
}
template <int ACT, bool FAST>
__device__ __forceinline__ void activation(float v, float& value, float& slope) {
  float rest;
  if constexpr (ACT == DM_ACT_RELU) {
    value = v > 0.f ? v : (v != v ? v : 0.f);
    slope = v > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == DM_ACT_GELU) {
    const float cdf = 0.5f * erfcf(v * -0.70710678f);
    value = v * cdf;
    slope = cdf + v * expf(-0.5f * v * v) * 0.39894228f;
  } else if constexpr (ACT == DM_ACT_GELU_TANH) {
    const float s = sigmoid<FAST>(1.5957691f * (v + 0.044715f * v * v * v), rest);
    value = v * s;
    slope = s + v * s * rest * 1.5957691f * (1.f + 0.134145f * fminf(v * v, 1e30f));  // (rest or s is 0 long before: not 0 times infinity)
  } else {
    const float s = sigmoid<FAST>(v, rest);
    value = ACT == DM_ACT_SIGMOID ? s : v * s;
    slope = ACT == DM_ACT_SIGMOID ? s * rest : s * (1.f + v * rest);
  }
}
// f(constant) for the activation at run time
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case DM_ACT_RELU: return f(std::integral_constant<int, DM_ACT_RELU>{});
    case DM_ACT_GELU: return f(std::integral_constant<int, DM_ACT_GELU>{});
    case DM_ACT_GELU_TANH: return f(std::integral_constant<int, DM_ACT_GELU_TANH>{});
    case DM_ACT_SIGMOID: return f(std::integral_constant<int, DM_ACT_SIGMOID>{});
    default: return f(std::integral_constant<int, DM_ACT_SILU>{});
  }
}

// h = act(g) u; g and u become what the backward pass needs: act(g) and u act'(g)
template <bool FAST>
__device__ __forceinline__ void gate_values(int act, float (&g)[8], float (&u)[8], float (&h)[8]) {
  with_activation(act, [&](auto a) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float value, slope;
      activation<decltype(a)::value, FAST>(g[e], value, slope);
      h[e] = value * u[e];
      u[e] *= slope;
      g[e] = value;
    }
  });
}

template <typename S>
__device__ __forceinline__ float bias_at(const void* b, int n, int N) { return b && n < N ? (float)((const S*)b)[n] : 0.f; }
template <typename S>
__device__ __forceinline__ void load8(const S* p, float (&v)[8]) {
  if constexpr (sizeof(S) == 4) {
    float a[4], b[4];
    load_vec<float, 4>(p, a);
    load_vec<float, 4>(p + 4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
  } else {
    load_vec<S, 8>(p, v);
  }
}

constexpr int GEMM_BK = 64;
__device__ __forceinline__ void from_lds(const char DM_LDS* p, float (&v)[8]) {
  const f32x4 a = *(const DM_LDS f32x4*)p, b = *(const DM_LDS f32x4*)(p + 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}

constexpr int LDS_BIAS = 3 * 1024;  // see load_to_lds
constexpr uint32_t UNBOUNDED = 0x80000000u;  // bytes of a buffer
// Offsets outside of every buffer (one inside is below 2^30): of a row or column that the tensor does not have; and, as a bit of an offset,
// of k behind a step of fewer k.
constexpr uint32_t OUTSIDE = 0xC0000000u, BEHIND = 0x80000000u;
enum { EPI_STORE, EPI_GATE, EPI_GATE_F32, EPI_DACT, EPI_DACT_F32 };  // _F32: of split fp32 operands

struct GemmArgs {
  const void *a[2], *b[2], *b2;       // b2 (GATE): the second projection's weights
  int64_t plane_a, plane_b;           // bytes from one plane of an operand to the next
  uint64_t terms;                     // five bits per product term: plane of a, plane of b (two bits each), which of the two a and b
  int segments, iters;                // number of terms, k steps of GEMM_BK
  int early;                          // the first terms that are taken over the whole range before the others are
  int64_t lda, ldb;                   // elements
  int64_t M;
  int N, K;                           // N: of one projection for EPI_GATE.  K: true length; a KC row is zero from there to the end of its piece
  int tiles_m, tiles_n, splits;
  Out out, out2, out3;                // STORE: out (out2: see `pair`).  GATE: out = h, and for the backward pass (null: not kept) out2 = u act'(g), out3 = act(g), fp32 or not.
                                      // DACT: out = dg, out2 = du
  const void *bias, *bias2;           // of the result's type; GATE: of the operands'
  const void *ug, *ag;                // DACT: u act'(g) and act(g), rows of ldg, fp32 or (kept16) of the operands' type
  int64_t ldg;
  int kept16;
  int act;
  void* part;                         // splits > 1: fp32 partial products (GATE: of both projections in turn), rows of ldpart,
  int64_t split_stride, ldpart;       // split_stride elements from one to the next; joined by a second launch
  void* sums;                         // STORE with both operands KS: sum over k of A[m, k] over the segments of sum_segments, of the result's type,
  float* sum_part;                    // or null; splits > 1: their parts, M apart
  int sum_segments;
  int64_t pair;                       // STORE with both operands KS: 0, or two products of one B in one launch: the second A lies `pair` bytes
  void* sums2;                        // behind the first, its result in out2.p, its sums in sums2; their partial rows follow the first's
};

// What GATE keeps for DACT, eight columns of a row
template <typename T, bool F32>
__device__ __forceinline__ void store_kept(const GemmArgs& p, int64_t m, int n, int np, const float (&ug)[8], const float (&ag)[8]) {
  if (!p.out2.p) return;
  if (F32 || p.out2.f32) {
    store8<T, OUT_F32>(p.out2, m, n, np, ug);
    store8<T, OUT_F32>(p.out3, m, n, np, ag);
  } else {
    store8<T, OUT_16>(p.out2, m, n, np, ug);
    store8<T, OUT_16>(p.out3, m, n, np, ag);
  }
}

// Where a stage keeps a piece of 16 bytes.  KS (one LDS row per k, R columns): piece c of row k lies at c ^ ks_key(k), so that the 32
// lanes of two fragment reads (k .. k + 3 and k + 8 .. k + 11, two pieces each) find 16 pieces of all 64 banks.  KC (one LDS row per
// operand row, 8 pieces): piece c of a row lies at c ^ kc_key(row), so that 16 rows' pieces do.
__device__ __forceinline__ int ks_key(int k) { return ((k & 3) | ((k >> 1) & 4)) << 1; }
__device__ __forceinline__ int kc_key(int row) { return (row >> 1) & 7; }

// One LDS stage of one operand: R rows (of A or B) x GEMM_BK k, 16-bit elements, by the NW waves of the block.
template <int R, bool KS, int NW>
struct Stager {
  static constexpr int PASSES = R * GEMM_BK / 8 / (64 * NW);  // 16-byte pieces per lane
  static constexpr int CPR = KS ? R / 8 : GEMM_BK / 8;        // pieces per LDS row
  static constexpr int RPW = 64 / CPR;                        // LDS rows that one wave's load fills
  uint32_t off[PASSES];                                       // byte offset from LDS_BIAS before the tile's corner, OUTSIDE where the piece lies outside
  static __device__ __forceinline__ int row_of(int wave, int lane, int j) { return (wave * PASSES + j) * RPW + lane / CPR; }
  static __device__ __forceinline__ int piece_of(int lane, int row) { return (lane % CPR) ^ (KS ? ks_key(row) : kc_key(row)); }
  static __device__ __forceinline__ int k_of(int wave, int lane, int j) {  // k of the piece within the step
    const int row = row_of(wave, lane, j);
    return KS ? row : piece_of(lane, row) * 8;
  }
  // GATE: rows 64 i .. +31 of the tile are rows 32 i of the first projection's weights, +32 .. +63 the second's
  template <bool GATE>
  __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int64_t rows_left) {
#pragma unroll
    for (int j = 0; j < PASSES; ++j) {
      const int row = row_of(wave, lane, j), c = piece_of(lane, row);
      const uint32_t bias = LDS_BIAS - j % 4 * 1024;  // see load_to_lds
      const int r = GATE ? row / 64 * 32 + row % 32 : row;
      off[j] = (KS ? c * 8 : r) < rows_left ? (uint32_t)(r * ld * 2 + c * 16) + bias : OUTSIDE;
    }
  }
};

// Two loads of 16 bytes per lane from a bounds-checked buffer straight into LDS, at `lds` + FIRST + lane * 16 and 1024 bytes further on.
// The instruction's offset (FIRST, FIRST + 1024) counts on both sides: the buffer starts LDS_BIAS bytes before its memory, and `off`
// makes up for the difference.  The caller waits (vmcnt) and synchronises.  (s_nop: five wait states, should a vector instruction
// have written the scalar registers.)
template <int FIRST>
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t off0, uint32_t off1, uint32_t lds) {
  static_assert(FIRST + 1024 <= LDS_BIAS && LDS_BIAS < 4096, "offsets of the instruction");
  asm volatile(
      "s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %2, 0 offen offset:%4 lds\n\tbuffer_load_dwordx4 %1, %2, 0 offen offset:%5 lds" ::"v"(off0),
      "v"(off1), "s"(rsrc), "s"(lds), "n"(FIRST), "n"(FIRST + 1024)
      : "memory", "m0");
}
// (addresses have 48 bits: no stride)
__device__ __forceinline__ i32x4 buffer_of(uint64_t u, uint32_t bytes) {
  return i32x4{(int)(uint32_t)u, (int)(uint32_t)(u >> 32), (int)bytes, 0x00020000};
}
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
// The value, in scalar registers, is formed here: neither sunk to where it is used nor loaded again there.
template <typename V>
__device__ __forceinline__ void pin(V& v) { asm volatile("" : "+s"(v)); }
__device__ __forceinline__ uint64_t product64(uint32_t a, uint32_t b) { return (uint64_t)__umulhi(a, b) << 32 | a * b; }  // (in scalar registers)

// All but the LEFT newest loads of every wave are in LDS, and every wave has its fragments of the stage at hand in registers.
template <int LEFT>
__device__ __forceinline__ void stage_arrived() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory"); }

// Every wave's LDS accesses so far are done; loads and stores of global memory stay under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Fragment of 16 rows x 32 k (the s-th of the step) out of a stage: lane l holds row l & 15, k 8 (l >> 4) .. +7.
template <int R, bool KS>
__device__ __forceinline__ s16x8 fragment(const char DM_LDS* stage, int lane, int tile, int s) {
  if constexpr (KS) {
    // A lane asks for 4 consecutive rows of one k; of 16 lanes' answers, lane i receives row i of four k.  (k's bits 2 and 5 are not in
    // its key, and the stage and k lie above the bits of the tile: one exclusive or per fragment, the rest in the instructions' offsets.)
    const int k0 = (lane >> 4) * 8 + ((lane >> 2) & 3);
    const uint32_t at = ((uint32_t)(uintptr_t)stage + k0 * (R * 2) + (((lane >> 1) & 1) ^ ks_key(k0)) * 16 + (lane & 1) * 8) ^ tile * 32;
    s16x4 h[2];
#pragma unroll
    for (int q = 0; q < 2; ++q)
      h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DM_LDS s16x4*)(uintptr_t)(at + (s * 32 + q * 4) * (R * 2)));
    return s16x8{h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
  } else {
    const int row = tile * 16 + (lane & 15);
    return *(const DM_LDS s16x8*)(stage + row * (GEMM_BK * 2) + ((s * 4 + (lane >> 4)) ^ kc_key(lane & 15)) * 16);
  }
}

// Steps of each part of a split k range: whole eights where it has two or more (see `shift` below).
__host__ __device__ inline int split_steps(int iters, int splits) {
  const int per = (iters + splits - 1) / splits;
  return per < 16 ? per : (per + 7) / 8 * 8;
}

template <typename T, int BM, int BN, int WM, int WN, int GEMM_STAGES, bool AKS, bool BKS, int EPI>
__global__ void __launch_bounds__(WM * WN * 64, 2)
gemm_kernel(const GemmArgs p) {
  constexpr int NW = WM * WN, MI = BM / WM / 16, NI = BN / WN / 16;
  constexpr int ABYTES = BM * GEMM_BK * 2, STAGE = (BM + BN) * GEMM_BK * 2;
  constexpr bool GATE = EPI == EPI_GATE || EPI == EPI_GATE_F32, F32 = EPI == EPI_GATE_F32 || EPI == EPI_DACT_F32,
                 DACT = EPI == EPI_DACT || EPI == EPI_DACT_F32, SUMS = AKS && BKS;
  using Bias = typename std::conditional<F32, float, T>::type;
  constexpr int BETWEEN = F32 ? OUT_PLANES : OUT_16;
  constexpr int XS = MI >= WN ? MI / WN : 1;  // the waves of a tile row share its sums of A: XS blocks of 16 rows each
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // Tiles are dealt so that each of the 8 XCDs (blocks go to them in turn) walks a contiguous run, in bands of 8 tile rows: the blocks
  // that share an L2 share operand panels.
  const int tiles = p.tiles_m * p.tiles_n;
  int tile = blockIdx.x;
  {
    const int full = tiles / 8 * 8;
    if (tile < full) tile = tile % 8 * (full / 8) + tile / 8;
  }
  const int band = 8 * p.tiles_n;
  const int first = tile / band * 8;
  const int rows = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
  const int tm = __builtin_amdgcn_readfirstlane(first + tile % band % rows), tn = __builtin_amdgcn_readfirstlane(tile % band / rows);
  const bool other = SUMS && p.pair && tm >= p.tiles_m / 2;  // of the second of a pair
  const int64_t m0 = (int64_t)(other ? tm - p.tiles_m / 2 : tm) * BM;
  const int n0 = tn * (GATE ? BN / 2 : BN);

  // The block's range: k steps, and every term of the product in each.
  const int per = split_steps(p.iters, p.splits);
  const int step0 = blockIdx.y * per, step1 = step0 + per < p.iters ? step0 + per : p.iters;
  const int turns = step0 < step1 ? (step1 - step0) * p.segments : 0;

  Stager<BM, AKS, NW> sa;
  Stager<BN, BKS, NW> sb;
  sa.template init<false>(wave, lane, p.lda, p.M - m0);
  sb.template init<GATE>(wave, lane, p.ldb, p.N - n0);

  const uint32_t lds0 = (uint32_t)(uintptr_t)(DM_LDS char*)smem;
  // Steps are taken in an order of the tile's own within each eight: the blocks of an XCD would otherwise ask for the same columns of all
  // rows at once, which lie on few of the L2's channels when rows are a power of two apart.  (Eights that the range does not hold whole
  // keep their order, and so does the one with a step of fewer k: that step comes last.)
  const int shift = per % 8 && p.splits > 1 ? 0 : (tm + 2 * tn) & (p.segments > 1 && !(AKS && p.splits > 1) ? 3 : 7);
  const int whole = p.K / GEMM_BK < step1 ? p.K / GEMM_BK : step1;
  // A term takes a group of steps, then the next term takes the same group (the last step, if it has fewer k, is one by itself).  The
  // `early` terms, of split fp32 the small ones, go through the whole range first: an instruction's sum is as exact as the largest of what it adds,
  // so small terms that met the main one's sum would lose as much in each instruction as the main term does (step of 65536 x 256 x 1024, relative
  // to 64 bits: 0.4 to 2.4e-6 so and 1.6 to 3.4e-7 this way; 2180 and 2205 us, as the main term's planes are fetched once more).
  const int group = p.segments > 1 ? AKS && p.splits > 1 ? 1 : 4 : p.iters;
  auto group_end = [&](int from) __attribute__((always_inline)) { return from >= whole ? step1 : from + group < whole ? from + group : whole; };
  int seg = 0, step = step0, group0 = step0, group1 = group_end(step0);  // of the next stage to be asked for
  int seg0 = 0, seg1 = p.early ? p.early : p.segments;                   // terms that take turns now
  bool moved = false;
  int look = GEMM_BK;  // k left at a step: fewer are looked at closer
  const int64_t a0 = (AKS ? m0 : m0 * p.lda) * 2 + (other ? p.pair : 0) - LDS_BIAS, b0 = (BKS ? (int64_t)n0 : (int64_t)n0 * p.ldb) * 2 - LDS_BIAS;
  constexpr int LOADS = sa.PASSES + sb.PASSES;
  // (kept in registers: a scalar load among the products would wait for every LDS read under way)
  int segments = p.segments, k_end = p.K, sum_segments = p.sum_segments;
  uint32_t lda2 = (uint32_t)p.lda * 2, ldb2 = (uint32_t)p.ldb * 2;  // bytes
  pin(segments), pin(k_end), pin(lda2), pin(ldb2);
  const uint32_t astep = (AKS ? lda2 : 2) * GEMM_BK, bstep = (BKS ? ldb2 : 2) * GEMM_BK;  // bytes from one step to the next
  uint64_t corners[3];  // lane i: the corners of the i-th term's operands (GATE: and of the second projection's weights)
  {
    const int term = (int)(p.terms >> 5 * (lane < 12 ? lane : 0)) & 31;
    const int64_t in_b = (term >> 2 & 3) * p.plane_b;
    corners[0] = (uint64_t)(!GATE && term & 16 ? p.a[1] : p.a[0]) + a0 + (term & 3) * p.plane_a;
    corners[1] = (uint64_t)(!GATE && term & 16 ? p.b[1] : p.b[0]) + b0 + in_b;
    corners[2] = GATE ? (uint64_t)p.b2 + b0 + in_b : 0;
  }
  uint64_t term_a, term_b, term_b2 = 0;  // of the term at hand
  auto take_term = [&](int piece) __attribute__((always_inline)) {
    if (piece == 0) {
      term_a = from_lane(corners[0], seg);
    } else {
      term_b = from_lane(corners[1], seg);
      if (GATE) term_b2 = from_lane(corners[2], seg);
    }
  };
  take_term(0), take_term(1);
  // What the loads of the range's turn-th stage have in common, formed in five pieces: scalar instructions, which cost nothing between
  // products and 200 cycles of a step in one go (the asm keeps each piece where it stands).
  struct Request { i32x4 a, b, b2; uint32_t at, a_bytes, b_bytes; bool sum; };
  auto request = [&](Request& r, int piece, int turn) __attribute__((always_inline)) {
    if (piece == 0) {
      uint32_t at = (step | 7) < whole ? step ^ shift : step, a_bytes = UNBOUNDED, b_bytes = UNBOUNDED;
      const int left = turn < turns ? k_end - (int)at * GEMM_BK : 0;
      if (left < look) {   // the last step, of a k range of no whole steps (behind it come its own terms, or the range again), or behind the range
        asm volatile("");  // (a branch: every step would pay for the selection)
        if (look > GEMM_BK) {  // the first step of the range taken again (not where that is found: loads of the step before follow there)
          look = GEMM_BK;
#pragma unroll
          for (int j = 0; j < sa.PASSES; ++j)
            if (!AKS && sa.off[j] < OUTSIDE) sa.off[j] &= ~BEHIND;
#pragma unroll
          for (int j = 0; j < sb.PASSES; ++j)
            if (!BKS && sb.off[j] < OUTSIDE) sb.off[j] &= ~BEHIND;
        }
        if (left < GEMM_BK) {
          a_bytes = !left ? 0 : AKS ? left * lda2 + LDS_BIAS : UNBOUNDED;  // rows of a KS tile end with the k range
          b_bytes = !left ? 0 : BKS ? left * ldb2 + LDS_BIAS : UNBOUNDED;
#pragma unroll
          for (int j = 0; j < sa.PASSES; ++j)
            if (!AKS && sa.k_of(wave, lane, j) >= left) sa.off[j] |= BEHIND;
#pragma unroll
          for (int j = 0; j < sb.PASSES; ++j)
            if (!BKS && sb.k_of(wave, lane, j) >= left) sb.off[j] |= BEHIND;
        }
      }
      r.sum = SUMS && turn < turns && (sum_segments >> seg & 1);
      pin(at), pin(a_bytes), pin(b_bytes);
      r.at = at;
      r.a_bytes = a_bytes;
      r.b_bytes = b_bytes;
    } else if (piece == 1) {
      r.a = buffer_of(term_a + product64(r.at, astep), r.a_bytes);
      pin(r.a);
    } else if (piece == 2) {
      const uint64_t to = product64(r.at, bstep);
      r.b = buffer_of(term_b + to, r.b_bytes);
      r.b2 = GATE ? buffer_of(term_b2 + to, r.b_bytes) : r.b;
      pin(r.b);
      if (GATE) pin(r.b2);
    } else if (piece == 3) {
      ++step;
      moved = segments != 1 && step == group1;
      if (moved) {
        if (++seg == seg1) {
          group0 = group1;
          if (group0 >= step1 && seg1 < segments) {  // the range again, with the other terms
            seg0 = seg1;
            seg1 = segments;
            group0 = step0;
            look = 0x7fffffff;
          }
          seg = seg0;
          group1 = group_end(group0);
        }
        step = group0;
        take_term(0);
      }
    } else if (moved) {
      take_term(1);
    }
  };
  // Pairs [first, last) of a wave's loads of a stage.  A wave fills a contiguous part of each operand's tile.
  auto load = [&](const Request& r, uint32_t stage, int first, int last) __attribute__((always_inline)) {
#pragma unroll
    for (int l = first * 2; l < last * 2; l += 2) {
      const bool A = l < sa.PASSES;
      const int j = A ? l : l - sa.PASSES;
      const uint32_t o0 = A ? sa.off[j] : sb.off[j], o1 = A ? sa.off[j + 1] : sb.off[j + 1];
      const i32x4 rs = A ? r.a : GATE && (wave * sb.PASSES + j) * sb.RPW / 32 % 2 ? r.b2 : r.b;
      const uint32_t to = lds0 + stage + (A ? wave * sa.PASSES * 1024 : ABYTES + wave * sb.PASSES * 1024) + j / 4 * 4096;
      if (j % 4 == 0) load_to_lds<0>(rs, o0, o1, to);
      else load_to_lds<2048>(rs, o0, o1, to);
    }
  };
  static_assert(sa.PASSES % 2 == 0 && sb.PASSES % 2 == 0, "loads go in pairs");

  f32x4 acc[MI][NI], asum[XS];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#pragma unroll
    for (int x = 0; x < XS; ++x) asum[x][e] = 0.f;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j][e] = 0.f;
  }
  const short unit = __builtin_bit_cast(short, (T)1.f);
  const s16x8 ones = {unit, unit, unit, unit, unit, unit, unit, unit};

  // A step is PARTS parts of 32 k.  While a part's products run, the fragments of the part after are read into a second set, the first
  // ones needed first and the last ones early enough to be there.  Before a step's last part every wave's fragments of the stage are in
  // registers: behind the barrier there, the next stage is read and the one just left is asked for again, between the products.
  constexpr int PARTS = GEMM_BK / 32, READS = MI + NI, PER = (READS + MI - 3) / (MI - 2);
  s16x8 fa[2][MI], fb[2][NI];
  auto read = [&](int q, uint32_t from, int s, int l) __attribute__((always_inline)) {  // the l-th fragment: B's, and A's in order
    const char DM_LDS* st = (const char DM_LDS*)smem + from;
    if (l == 0) fa[q][0] = fragment<BM, AKS>(st, lane, wm * MI, s);
    else if (l <= NI) fb[q][l - 1] = fragment<BN, BKS>(st + ABYTES, lane, wn * NI + l - 1, s);
    else fa[q][l - NI] = fragment<BM, AKS>(st, lane, wm * MI + l - NI, s);
  };
  auto part = [&](int q, uint32_t from, int s, bool refill, Request& r, uint32_t to, int turn) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int l = i * PER; l < (i + 1) * PER; ++l)
        if (l < READS) read(q ^ 1, from, s, l);
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = mfma16(fb[q][j], fa[q][i], acc[i][j], T());
      if (refill) load(r, to, i * (LOADS / 2) / MI, (i + 1) * (LOADS / 2) / MI);
      if (i < (refill ? 2 : 3)) request(r, refill ? 3 + i : i, turn);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto add_sums = [&](uint32_t from) __attribute__((always_inline)) {  // the stage's share of the sums of A
    const char DM_LDS* st = (const char DM_LDS*)smem + from;
#pragma unroll
    for (int s = 0; s < PARTS; ++s)
#pragma unroll
      for (int x = 0; x < XS; ++x) asum[x] = mfma16(ones, fragment<BM, AKS>(st, lane, wm * MI + wn * XS + x, s), asum[x], T());
  };
  void* const sums_out = SUMS ? other ? p.sums2 : p.sums : nullptr;
  const bool sums = sums_out && tn == 0;
  if (turns) {
    uint32_t cur = 0;
    bool sum = false, next[GEMM_STAGES];  // do the stage at hand, and those asked for, count for the sums of A
#pragma unroll
    for (int k = 0; k < GEMM_STAGES; ++k) {
      Request r;
#pragma unroll
      for (int piece = 0; piece < 5; ++piece) request(r, piece, k);
      next[k] = sums && r.sum;
      load(r, k * STAGE, 0, LOADS / 2);
    }
    stage_arrived<LOADS * (GEMM_STAGES - 1)>();
    sum = next[0];
#pragma unroll
    for (int l = 0; l < READS; ++l) read(0, 0, 0, l);
    for (int turn = 0; turn < turns; ++turn) {
      Request r;
      static_assert(PARTS == 2 && MI >= 3, "a step ends with the set that it began with; its request takes three rows of products");
      part(0, cur, 1, false, r, 0, turn + GEMM_STAGES);
      if (sum) add_sums(cur);
      const uint32_t left = cur;
      cur = cur + STAGE == GEMM_STAGES * STAGE ? 0 : cur + STAGE;
#pragma unroll
      for (int k = 0; k < GEMM_STAGES - 1; ++k) next[k] = next[k + 1];
      next[GEMM_STAGES - 1] = sums && r.sum;
      sum = next[0];
      stage_arrived<LOADS * (GEMM_STAGES - 2)>();
      part(1, cur, 0, true, r, left, 0);  // (behind the range it reads zeros, and nobody uses them)
    }
  }
  stage_arrived<0>();  // the loads behind the range are done with LDS, and so is every wave

  // acc[i][j][e] belongs to m = lane & 15 and n = 4 (lane >> 4) + e of the 16 x 16 block (i, j).  Two block rows of all waves meet in LDS
  // as rows of fp32 (a pitch of 16 bytes more than the row: no bank conflicts), two buffers in turn, and leave as whole pieces of
  // eight columns, neighbouring lanes next to each other: written straight from the accumulators, rows a power of two apart crowd
  // on few of the L2's channels (41 us of a 256 x 256 tile's time, measured at a row of 8 KB).
  constexpr int ROWS = WM * 32, PITCH = BN * 4 + 16, COLS = GATE ? BN / 2 : BN, PIECES = COLS / 8, TASKS = ROWS * PIECES / (NW * 64);
  const int np = (p.N + 7) & ~7;  // intermediate results are padded to whole pieces of zeros
  static_assert(NW * 64 % PIECES == 0, "a thread keeps its columns");
  const bool ragged = n0 + COLS > p.N;
  Out out = p.out;
  if (other) out.p = p.out2.p;
  float b1[8], b2[8];
  if constexpr (!DACT) {
    const int n = n0 + threadIdx.x % PIECES * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      b1[e] = EPI == EPI_STORE && p.out.f32 ? bias_at<float>(p.bias, n + e, p.N) : bias_at<Bias>(p.bias, n + e, p.N);
      b2[e] = GATE ? bias_at<Bias>(p.bias2, n + e, p.N) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < MI / 2; ++i) {
    char DM_LDS* buf = (char DM_LDS*)smem + (i & 1) * ROWS * PITCH;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NI; ++j)
        *(DM_LDS f32x4*)(buf + (wm * 32 + h * 16 + (lane & 15)) * PITCH + ((wn * NI + j) * 16 + (lane >> 4) * 4) * 4) = acc[i * 2 + h][j];
    f32x4 ug[DACT ? TASKS : 1][2], ag[DACT ? TASKS : 1][2];  // asked for ahead of the barrier (16 bits: the first of two, converted behind it)
    if constexpr (DACT) {
      auto ask = [&](auto type) __attribute__((always_inline)) {
        using S = decltype(type);
#pragma unroll
        for (int t = 0; t < TASKS; ++t) {
          const int id = t * NW * 64 + threadIdx.x, row = id / PIECES, n = n0 + id % PIECES * 8;
          const int64_t m = m0 + row / 32 * (MI * 16) + i * 32 + row % 32;
          if (m >= p.M || n >= np || p.splits > 1) continue;
          const S *a = (const S*)p.ug + m * p.ldg + n, *b = (const S*)p.ag + m * p.ldg + n;
          ug[t][0] = *(const f32x4*)a;
          ag[t][0] = *(const f32x4*)b;
          if (sizeof(S) == 4) { ug[t][1] = *(const f32x4*)(a + 4); ag[t][1] = *(const f32x4*)(b + 4); }
        }
      };
      if (!F32 && p.kept16) ask(T());
      else ask(float());
    }
    lds_barrier();
    if (EPI == EPI_STORE && p.splits == 1 && !p.out.vec) {  // rows off 16-byte boundaries: neighbouring lanes store neighbouring elements
#pragma unroll 8
      for (int id = threadIdx.x; id < ROWS * BN; id += NW * 64) {
        const int row = id / BN, n = n0 + id % BN;
        const int64_t m = m0 + row / 32 * (MI * 16) + i * 32 + row % 32;
        if (m >= p.M || n >= p.N) continue;
        const float v = *(const DM_LDS float*)(buf + row * PITCH + id % BN * 4);
        if (out.f32) ((float*)out.p)[m * out.ld + n] = v + bias_at<float>(p.bias, n, p.N);
        else ((T*)out.p)[m * out.ld + n] = (T)(v + bias_at<T>(p.bias, n, p.N));
      }
      continue;
    }
#pragma unroll
    for (int t = 0; t < TASKS; ++t) {
      const int id = t * NW * 64 + threadIdx.x, row = id / PIECES, col = id % PIECES * 8;
      const int64_t m = m0 + row / 32 * (MI * 16) + i * 32 + row % 32;
      const int n = n0 + col;
      if (m >= p.M || n >= (EPI == EPI_STORE ? p.N : np)) continue;
      const char DM_LDS* at = buf + row * PITCH + (GATE ? col / 32 * 64 + col % 32 : col) * 4;
      float v[8], u[8], h[8];
      from_lds(at, v);
      if constexpr (GATE) from_lds(at + 128, u);
      if (p.splits > 1) {  // joined by a second launch
        float* part = (float*)p.part + blockIdx.y * (GATE ? 2 : 1) * p.split_stride + (other ? p.M + m : m) * p.ldpart + n;
        store_f32(part, v);
        if constexpr (GATE) store_f32(part + p.split_stride, u);
        continue;
      }
      if constexpr (GATE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { v[e] += b1[e]; u[e] += b2[e]; }
        gate_values<!F32>(p.act, v, u, h);
        if (ragged) zero_behind(n, p.N, h), zero_behind(n, p.N, u), zero_behind(n, p.N, v);
        store8<T, BETWEEN>(p.out, m, n, np, h);
        store_kept<T, F32>(p, m, n, np, u, v);
      } else if constexpr (DACT) {
        if (!F32 && p.kept16) {
          using T8 = typename std::conditional<std::is_same<T, bf16>::value, bf16x8, f16x8>::type;
          const T8 a = __builtin_bit_cast(T8, ug[t][0]), b = __builtin_bit_cast(T8, ag[t][0]);
#pragma unroll
          for (int e = 0; e < 8; ++e) { u[e] = v[e] * (float)a[e]; h[e] = v[e] * (float)b[e]; }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) { u[e] = v[e] * ug[t][e / 4][e % 4]; h[e] = v[e] * ag[t][e / 4][e % 4]; }
        }
        if (ragged) zero_behind(n, p.N, u), zero_behind(n, p.N, h);
        store8<T, BETWEEN>(p.out, m, n, np, u);
        store8<T, BETWEEN>(p.out2, m, n, np, h);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += b1[e];
        if (out.f32) store8<T, OUT_F32>(out, m, n, p.N, v);
        else store8<T, OUT_16>(out, m, n, p.N, v);
      }
    }
  }
  if constexpr (EPI == EPI_STORE) {
    if constexpr (SUMS) {  // every n of the product with ones holds the sum
#pragma unroll
      for (int x = 0; x < XS; ++x) {
        const int64_t m = m0 + (wm * MI + wn * XS + x) * 16 + lane;
        if (!sums || lane >= 16 || m >= p.M) continue;
        if (p.splits > 1) p.sum_part[(blockIdx.y * (p.pair ? 2 : 1) + other) * p.M + m] = asum[x][0];
        else if (out.f32) ((float*)sums_out)[m] = asum[x][0];
        else ((T*)sums_out)[m] = (T)asum[x][0];
      }
    }
  }
}

// Eight columns' sums over the partial products of a split k range, in a fixed order: by one thread each, or where there are many parts
// by four groups of 64 threads, every fourth part each, that meet in LDS.  Threads of the first group get the result.
__device__ __forceinline__ bool join8(const float* part, int splits, int64_t stride, bool grouped, bool live, float (&v)[8]) {
  __shared__ float sum[3][64][9];
  const int lane = threadIdx.x & 63, group = grouped ? threadIdx.x >> 6 : 0, groups = grouped ? 4 : 1;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  if (live)
#pragma unroll 4
    for (int s = group; s < splits; s += groups) {
      float w[8];
      load8(part + s * stride, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += w[e];
    }
  if (!grouped) return live;
  __syncthreads();
  if (group)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[group - 1][lane][e] = v[e];
  __syncthreads();
  if (group) return false;
#pragma unroll
  for (int g = 0; g < 3; ++g)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += sum[g][lane][e];
  return live;
}

// The second launch of a product whose k range was split: partial products added, then what the epilogue would have done.
template <typename T, int EPI>
__global__ void __launch_bounds__(256) join_kernel(const GemmArgs p) {
  constexpr bool GATE = EPI == EPI_GATE || EPI == EPI_GATE_F32, F32 = EPI == EPI_GATE_F32 || EPI == EPI_DACT_F32;
  using Bias = typename std::conditional<F32, float, T>::type;
  constexpr int BETWEEN = F32 ? OUT_PLANES : OUT_16;
  const int np = (p.N + 7) & ~7, pieces = np / 8;
  const int64_t rows = EPI == EPI_STORE && p.pair ? 2 * p.M : p.M, all = rows * pieces;
  const bool grouped = p.splits > 4;
  const int count = grouped ? 64 : 256;
  for (int64_t base = (int64_t)blockIdx.x * count; base < all; base += (int64_t)gridDim.x * count) {
    const int64_t id = base + (threadIdx.x & (count - 1)), m = id / pieces;
    const int n = (int)(id % pieces) * 8;
    const float* part = (const float*)p.part + m * p.ldpart + n;
    float v[8], u[8], h[8];
    const bool mine = join8(part, p.splits, (GATE ? 2 : 1) * p.split_stride, grouped, id < all, v);
    if constexpr (GATE) join8(part + p.split_stride, p.splits, 2 * p.split_stride, grouped, id < all, u);
    if (!mine) continue;
    if constexpr (GATE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) { v[e] += bias_at<Bias>(p.bias, n + e, p.N); u[e] += bias_at<Bias>(p.bias2, n + e, p.N); }
      gate_values<!F32>(p.act, v, u, h);
      zero_behind(n, p.N, h), zero_behind(n, p.N, u), zero_behind(n, p.N, v);
      store8<T, BETWEEN>(p.out, m, n, np, h);
      store_kept<T, F32>(p, m, n, np, u, v);
    } else if constexpr (EPI == EPI_STORE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += p.out.f32 ? bias_at<float>(p.bias, n + e, p.N) : bias_at<T>(p.bias, n + e, p.N);
      Out o = p.out;
      if (m >= p.M) o.p = p.out2.p;
      if (o.f32) store8<T, OUT_F32>(o, m >= p.M ? m - p.M : m, n, p.N, v);
      else store8<T, OUT_16>(o, m >= p.M ? m - p.M : m, n, p.N, v);
    } else {
      float ag[8];
      if (!F32 && p.kept16) {
        load8((const T*)p.ug + m * p.ldg + n, u);
        load8((const T*)p.ag + m * p.ldg + n, ag);
      } else {
        load8((const float*)p.ug + m * p.ldg + n, u);
        load8((const float*)p.ag + m * p.ldg + n, ag);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) { u[e] *= v[e]; h[e] = ag[e] * v[e]; }
      zero_behind(n, p.N, u), zero_behind(n, p.N, h);
      store8<T, BETWEEN>(p.out, m, n, np, u);
      store8<T, BETWEEN>(p.out2, m, n, np, h);
    }
  }
  if (EPI == EPI_STORE && (p.sums || p.sums2))
    for (int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x; m < rows; m += (int64_t)gridDim.x * 256) {
      void* const out = m >= p.M ? p.sums2 : p.sums;
      if (!out) continue;
      float s = 0.f;
#pragma unroll 16
      for (int i = 0; i < p.splits; ++i) s += p.sum_part[i * rows + m];
      if (p.out.f32) ((float*)out)[m >= p.M ? m - p.M : m] = s;
      else ((T*)out)[m >= p.M ? m - p.M : m] = (T)s;
    }
}

// Tiles.  WIDE, 256 x 256: one workgroup of 8 waves per CU; the fewest bytes and LDS reads per product.  MID, 128 x 128: two of 4 waves per
// CU.  SLIM, 64 x 128: two of 4 waves per CU with three stages each, for rows so few that the n side's bytes are what counts.
enum { TILE_WIDE, TILE_MID, TILE_SLIM, TILES };
constexpr int TILE_M[TILES] = {256, 128, 64}, TILE_N[TILES] = {256, 128, 128}, TILE_PER_CU[TILES] = {1, 2, 2};

struct GemmPlan { int tile, splits; size_t part_bytes; };
inline size_t gemm_part_bytes(int64_t M, int N, int outs, int splits) {
  return splits > 1 ? (size_t)splits * outs * M * (round_up(N, 8) + 1) * 4 : 0;  // products, and sums of A
}

// Tests run every product with every tile: dm_debug_ffn_plan, of the calling thread.  FORCED_COLUMNS: column_kernel wherever it can.
constexpr int FORCED_COLUMNS = TILES;
inline thread_local int forced_tile = -1, forced_splits = 1;

// Tile and split of the k range: the least of an estimate in microseconds.  A product's time is that of its stages - alone on a CU, or two
// workgroups to a CU where they fit (WIDE: two rounds) - but not less than the n side's bytes take, then for each round of workgroups
// a start and the tile's results on their way (`bytes` per element of the tile), and for a split k range the joining launch.  The
// constants are fitted to the measured times of every tile and split at 48 sizes of the block (6 to 65536 rows, widths 64 to 11008,
// bf16 and fp32, all products of both passes): what it picks takes 2 % longer than the best on average and 30 % at worst, where always
// taking MID unsplit would take 66 % longer.  `outs`: products per n (2: both projections).
inline GemmPlan gemm_plan(int64_t M, int N, int steps, int terms, int outs, int bytes, bool slim) {
  if (forced_tile >= 0 && forced_tile < TILES) {
    GemmPlan forced = {forced_tile == TILE_SLIM && !slim ? (int)TILE_MID : forced_tile, 1, 0};
    const int per = split_steps(steps, forced_splits);
    forced.splits = (steps + per - 1) / per;
    forced.part_bytes = gemm_part_bytes(M, N, outs, forced.splits);
    return forced;
  }
  const int cus = 256;
  constexpr double ALONE[TILES] = {1.6, 0.97, 0.54}, PAIR[TILES] = {4.0, 1.08, 0.8}, START[TILES] = {2.1, 1.7, 2.1};
  GemmPlan best = {TILE_MID, 1, 0};
  double cost = 1e300;
  const double stream = (double)N * outs * steps * (terms > 1 ? 3 : 1) * GEMM_BK * 2 / 4.4e6;
  for (int t = 0; t < TILES; ++t) {
    if (t == TILE_SLIM && !slim) continue;
    const int64_t tiles = ((M + TILE_M[t] - 1) / TILE_M[t]) * (((int64_t)N * outs + TILE_N[t] - 1) / TILE_N[t]);
    for (int want = 1; want <= 64; want *= 2) {
      const int s = (steps + split_steps(steps, want) - 1) / split_steps(steps, want), per = split_steps(steps, s);
      if (want > 1 && (s <= want / 2 || per * terms < 4 || tiles * (want / 2) >= cus)) break;
      const int64_t blocks = tiles * s, full = blocks / (2 * cus), rest = blocks % (2 * cus);
      const double alone = blocks <= cus / 2 ? 1.4 * ALONE[t] : ALONE[t];
      double c = per * terms * (full * PAIR[t] + (rest > cus ? PAIR[t] : rest ? alone : 0.0));
      if (c < stream) c = stream;
      c += (double)((blocks + cus - 1) / cus) * (START[t] + TILE_M[t] * TILE_N[t] * (s > 1 ? 4 : bytes) / 22.0e3);
      if (s > 1) c += 9.0 + (double)M * N * outs * 4 * s / 2.3e6;
      if (c < cost) { cost = c; best.tile = t; best.splits = s; }
    }
  }
  best.part_bytes = gemm_part_bytes(M, N, outs, best.splits);
  return best;
}

// The kernel's dynamic LDS on the current device, set at its first launch there (`done`: of the caller's own).
inline hipError_t allow_lds(const void* f, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return hipSuccess;
  e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

template <typename T, int EPI>
int join_launch(const GemmArgs& a, hipStream_t st) {
  const int64_t count = a.splits > 4 ? 64 : 256, blocks = (a.M * (a.pair ? 2 : 1) * ((a.N + 7) / 8) + count - 1) / count;
  join_kernel<T, EPI><<<dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st>>>(a);
  return launched("gated feed-forward block");
}

template <typename T, bool AKS, bool BKS, int EPI>
int gemm_launch(GemmArgs a, int tile, hipStream_t st) {
  constexpr bool GATE = EPI == EPI_GATE || EPI == EPI_GATE_F32, SLIM = !AKS;
  const int bm = TILE_M[tile], bn = TILE_N[tile];
  a.tiles_m = (int)((a.M + bm - 1) / bm) * (a.pair ? 2 : 1);
  a.tiles_n = GATE ? (a.N + bn / 2 - 1) / (bn / 2) : (a.N + bn - 1) / bn;
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
  if (tiles > (1 << 22)) return fail("gated feed-forward block: %lld output tiles in one product", (long long)tiles);
  const dim3 grid((unsigned)tiles, a.splits);
  const void* f;
  int bytes;  // the stages, or the epilogue's two buffers of rows
  if (tile == TILE_WIDE) {
    f = (const void*)gemm_kernel<T, 256, 256, 2, 4, 2, AKS, BKS, EPI>;
    bytes = 2 * 64 * (256 * 4 + 16);
  } else if (!SLIM || tile == TILE_MID) {
    f = (const void*)gemm_kernel<T, 128, 128, 2, 2, 2, AKS, BKS, EPI>;
    bytes = 2 * 64 * (128 * 4 + 16);
  } else {
    if constexpr (SLIM) f = (const void*)gemm_kernel<T, 64, 128, 1, 4, 3, AKS, BKS, EPI>;
    bytes = 3 * (64 + 128) * GEMM_BK * 2;
  }
  static std::atomic<uint64_t> done[TILES];
  hipError_t e = allow_lds(f, bytes, done[tile]);
  if (e == hipSuccess) {
    void* args[] = {&a};
    e = hipLaunchKernel(f, grid, dim3(tile == TILE_WIDE ? 512 : 256), args, bytes, st);
  }
  if (e == hipSuccess && a.splits > 1) return join_launch<T, EPI>(a, st);
  return e == hipSuccess ? 0 : fail("gated feed-forward block: launch failed: %s", hipGetErrorString(e));
}

// The fused products are compiled in translation units of their own (dm_block_ffn_gate.hip, dm_block_ffn_dact.hip).
extern template int gemm_launch<bf16, false, false, EPI_GATE>(GemmArgs, int, hipStream_t);
extern template int gemm_launch<f16, false, false, EPI_GATE>(GemmArgs, int, hipStream_t);
extern template int gemm_launch<bf16, false, false, EPI_GATE_F32>(GemmArgs, int, hipStream_t);
extern template int gemm_launch<bf16, false, true, EPI_DACT>(GemmArgs, int, hipStream_t);
extern template int gemm_launch<f16, false, true, EPI_DACT>(GemmArgs, int, hipStream_t);
extern template int gemm_launch<bf16, false, true, EPI_DACT_F32>(GemmArgs, int, hipStream_t);

}  // namespace dmb
#endif
