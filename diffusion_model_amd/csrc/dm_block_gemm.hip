// dm_block_gemm.hip — C[m,n] = sum_k A[m,k] B[n,k] on the 16-bit matrix pipe, the products of the gated feed-forward block.
//
// An operand is stored either with k contiguous ("KC": rows of the operand) or with its own rows contiguous ("KS": k is the slow
// index), so that the forward pass and all three products of the backward pass run from the tensors as they lie in memory; a KS tile
// is transposed on its way out of LDS (ds_read_tr).  The k range may be a chain of up to 12 segments, each with base pointers of its
// own: the two terms of dx = dg Wg + du Wu, and the six products of fp32 operands that were split into three bf16 terms.
//
// A workgroup owns a BM x BN tile and walks k in steps of GEMM_BK: GEMM_STAGES LDS stages, filled by buffer loads that write LDS directly (16 bytes
// per lane, rows and columns out of range are bounds-checked to zero by the buffer resource), one barrier per step.  The LDS image
// is swizzled in 16-byte pieces so that fragment reads touch all 64 banks once.  Fragments feed v_mfma_f32_32x32x16 with the n side as
// the first operand, its rows permuted: a lane then holds sixteen consecutive n of one m, which the epilogue stores as whole vectors.
// A bias' gradient, the sum of A over k, is one more product with ones from the same fragments.
#ifndef DM_BLOCK_GEMM_HIP
#define DM_BLOCK_GEMM_HIP
#include <type_traits>

#include "dm_block_common.h"

namespace dmb {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
#define DM_LDS __attribute__((address_space(3)))

__device__ __forceinline__ f32x16 mfma16(s16x8 a, s16x8 b, f32x16 c, bf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma16(s16x8 a, s16x8 b, f32x16 c, f16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
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

template <typename T, int MODE>
__device__ __forceinline__ void store8(const Out& o, int64_t m, int n, int N, const float (&v)[8]) {
  const int64_t at = m * o.ld + n;
  if (o.vec && n + 8 <= N) {
    if constexpr (MODE == OUT_16) {
      store_vec<T, 8>((T*)o.p + at, v);
    } else if constexpr (MODE == OUT_F32) {
      const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
      store_vec<float, 4>((float*)o.p + at, a);
      store_vec<float, 4>((float*)o.p + at + 4, b);
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

// ---- activations: value and slope in fp32, all but the erf form by way of s(z) = 1 / (1 + exp(-z)); tanh's by 1 + tanh(y) = 2 s(2 y).
// Results that are rounded to 16 bits take the hardware's exp2 and reciprocal (relative error below 2^-20 for |z| < 16).
template <bool FAST>
__device__ __forceinline__ float sigmoid(float z) {
  if (FAST) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f));
  return 1.f / (1.f + expf(-z));
}
template <int ACT, bool FAST>
__device__ __forceinline__ void activation(float v, float& value, float& slope) {
  if constexpr (ACT == DM_ACT_RELU) {
    value = v > 0.f ? v : (v != v ? v : 0.f);
    slope = v > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == DM_ACT_GELU) {
    const float cdf = 0.5f * erfcf(v * -0.70710678f);
    value = v * cdf;
    slope = cdf + v * expf(-0.5f * v * v) * 0.39894228f;
  } else if constexpr (ACT == DM_ACT_GELU_TANH) {
    const float s = sigmoid<FAST>(1.5957691f * (v + 0.044715f * v * v * v));
    value = v * s;
    slope = s + v * s * (1.f - s) * 1.5957691f * (1.f + 0.134145f * v * v);
  } else {
    const float s = sigmoid<FAST>(v);
    value = ACT == DM_ACT_SIGMOID ? s : v * s;
    slope = ACT == DM_ACT_SIGMOID ? s * (1.f - s) : s * (1.f + v * (1.f - s));
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

#ifndef DM_BK
#define DM_BK 64
#define DM_ST 2
#endif
constexpr int GEMM_BK = DM_BK, GEMM_STAGES = DM_ST;
__device__ __forceinline__ void from_lds(const char DM_LDS* p, float (&v)[8]) {
  const f32x4 a = *(const DM_LDS f32x4*)p, b = *(const DM_LDS f32x4*)(p + 16);
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}

constexpr int GEMM_MAX_SEGMENTS = 12;
enum { EPI_STORE, EPI_GATE, EPI_GATE_F32, EPI_DACT, EPI_DACT_F32 };  // _F32: of split fp32 operands

struct GemmArgs {
  const void* a[GEMM_MAX_SEGMENTS];
  const void* b[GEMM_MAX_SEGMENTS];
  const void* b2[GEMM_MAX_SEGMENTS];  // EPI_GATE: the second projection's weights
  int segments, iters;                // iters: k steps of GEMM_BK per segment
  int64_t lda, ldb;                   // elements
  int64_t M;
  int N, K;                           // N: of one projection for EPI_GATE.  K: true length; a KC row is zero from there to the end of its piece
  int tiles_m, tiles_n, splits;
  Out out, out2, out3;                // STORE: out.  GATE: out = h, and for the backward pass (null: not kept) out2 = u act'(g), out3 = act(g).
                                      // DACT: out = dg, out2 = du
  const void *bias, *bias2;           // of the result's type; GATE: of the operands'
  const void *ug, *ag;                // DACT: u act'(g) and act(g), rows of ldg
  int64_t ldg;
  int act;
  int64_t split_stride;               // STORE with splits > 1: fp32 partial products, elements from one split to the next
  void* sums;                         // STORE with both operands KS: sum over k of A[m, k] over the segments of sum_segments, or null.  One split:
  int sum_segments, sums_f32;         // of the type that sums_f32 gives; several: fp32, M apart
};

template <int N>  // piece of 16 bytes that holds piece `c` of row k of a KS tile with N columns
__device__ __forceinline__ int ks_swizzle(int k, int c) { return N >= 128 ? c ^ ((k & 3) << 2) : c ^ (((k >> 1) & 1) << 2); }

// The n side of a 32 x 32 product is permuted in blocks of four rows, so that a lane's sixteen results are sixteen consecutive n: row r of
// the instruction is n = permuted(r), and its piece c of a KC stage lies at c ^ key(n): sixteen lanes read sixteen pieces of all 64 banks.
__device__ __forceinline__ int permuted(int r) { return ((r >> 2) & 1) * 16 + (r >> 3) * 4 + (r & 3); }
template <bool PERM>
__device__ __forceinline__ int kc_key(int row) {
  if constexpr (GEMM_BK == 64) return PERM ? ((row >> 1) & 3) | ((row >> 2) & 4) : (row >> 1) & 7;
  else return PERM ? ((row >> 2) & 1) | ((row >> 3) & 2) : (row >> 2) & 3;
}

// One LDS stage of one operand: R rows (of A or B) x GEMM_BK k, 16-bit elements, by the NW waves of the block.
template <int R, bool KS, int NW, bool PERM>
struct Stager {
  static constexpr int PASSES = R * GEMM_BK / 8 / (64 * NW);  // 16-byte pieces per lane
  static constexpr int CPR = KS ? R / 8 : GEMM_BK / 8;        // pieces per LDS row
  static constexpr int RPW = 64 / CPR;                        // LDS rows that one wave's load fills
  uint32_t off[PASSES];                                       // byte offset from the tile's corner, 2^31 where the piece lies outside
  int kpos[PASSES];                                           // k of the piece within the step
  // GATE: rows 64 i .. +31 of the tile are rows 32 i of the first projection's weights, +32 .. +63 the second's
  template <bool GATE>
  __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int64_t rows_left) {
#pragma unroll
    for (int j = 0; j < PASSES; ++j) {
      const int row = (j * NW + wave) * RPW + lane / CPR, slot = lane % CPR;
      if constexpr (KS) {
        const int c = ks_swizzle<R>(row, slot);
        off[j] = c * 8 < rows_left ? (uint32_t)(row * ld * 2 + c * 16) : 0x80000000u;
        kpos[j] = row;
      } else {
        const int c = slot ^ kc_key<PERM>(row);
        const int r = GATE ? row / 64 * 32 + row % 32 : row;
        off[j] = r < rows_left ? (uint32_t)(r * ld * 2 + c * 16) : 0x80000000u;
        kpos[j] = c * 8;
      }
    }
  }
};

// 16 bytes per lane from a bounds-checked buffer straight into LDS at `lds` + lane * 16.  The caller waits (vmcnt) and synchronises.
// (Five wait states, should a vector instruction have written the scalar registers.)
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc), "s"(lds) : "memory");
}
__device__ __forceinline__ i32x4 buffer_of(const void* p) {
  const uint64_t u = (uint64_t)p;
  return i32x4{(int)(uint32_t)u, (int)(uint32_t)(u >> 32) & 0xffff, (int)0x80000000u, 0x00020000};
}
// All but the LEFT newest loads of every wave are in LDS, and every wave has its fragments of the stage at hand in registers.
template <int LEFT>
__device__ __forceinline__ void stage_arrived() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory"); }

// Fragments of 32 rows x 16 k (the s-th of the step) out of a stage.
template <int R, bool KS, bool PERM>
__device__ __forceinline__ s16x8 fragment(const char DM_LDS* stage, int lane, int tile, int s) {
  if constexpr (KS) {
    // A lane asks for 4 consecutive rows of one k; of 16 lanes' answers, lane i receives row i of four k.
    const int g = lane >> 4, j = (lane >> 2) & 3;
    const int blk = (g & 1) * 4 + (lane & 3), four = PERM ? (blk & 1) * 4 + (blk >> 1) : blk;
    const int piece = tile * 4 + (four >> 1);
    s16x4 h[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = s * 16 + (g >> 1) * 8 + q * 4 + j;
      h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DM_LDS s16x4*)(stage + k * (R * 2) + ks_swizzle<R>(k, piece) * 16 + (four & 1) * 8));
    }
    return s16x8{h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
  } else {
    const int r = PERM ? permuted(lane & 31) : lane & 31;
    return *(const DM_LDS s16x8*)(stage + (tile * 32 + r) * (GEMM_BK * 2) + ((2 * s + (lane >> 5)) ^ kc_key<PERM>(r)) * 16);
  }
}

template <typename T, int BM, int BN, int WM, int WN, bool AKS, bool BKS, int EPI>
__global__ void __launch_bounds__(WM * WN * 64, 2)
gemm_kernel(const GemmArgs p) {
  constexpr int NW = WM * WN, MI = BM / WM / 32, NI = BN / WN / 32;
  constexpr int ABYTES = BM * GEMM_BK * 2, STAGE = (BM + BN) * GEMM_BK * 2;
  constexpr bool GATE = EPI == EPI_GATE || EPI == EPI_GATE_F32, F32 = EPI == EPI_GATE_F32 || EPI == EPI_DACT_F32, SUMS = AKS && BKS;
  using Kept = typename std::conditional<F32, float, T>::type;  // what GATE keeps for DACT
  constexpr int BETWEEN = F32 ? OUT_PLANES : OUT_16, KEPT = F32 ? OUT_F32 : OUT_16;
  constexpr int XS = (MI + WN - 1) / WN;  // the waves of a tile row share its sums of A: XS blocks of 32 rows each
  static_assert(!GATE || (NI % 2 == 0 && !BKS), "blocks of 32 columns of the two projections alternate");
  extern __shared__ __attribute__((aligned(16))) char smem[];
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
  const int tm = first + tile % band % rows, tn = tile % band / rows;
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * (GATE ? BN / 2 : BN);

  const int total = p.segments * p.iters;
  const int per = ((total + p.splits - 1) / p.splits + 7) / 8 * 8;  // whole eights: see `place`
  const int it0 = blockIdx.y * per, it1 = it0 + per < total ? it0 + per : total;

  Stager<BM, AKS, NW, false> sa;
  Stager<BN, BKS, NW, true> sb;
  sa.template init<false>(wave, lane, p.lda, p.M - m0);
  sb.template init<GATE>(wave, lane, p.ldb, p.N - n0);

  // (the segments' pointers are read where the launch put the arguments: indexing the parameter itself would copy it to scratch)
  const auto* args = (const __attribute__((address_space(4))) GemmArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  const uint32_t lds0 = (uint32_t)(uintptr_t)(DM_LDS char*)smem;
  // Steps are taken in an order of the tile's own within each eight (where the range has all eight): the blocks of an XCD would
  // otherwise ask for the same columns of all rows at once, which lie on few of the L2's channels when rows are a power of two apart.
#ifndef DM_SHIFT
#define DM_SHIFT ((tm + 2 * tn) & 7)
#endif
  const int shift = DM_SHIFT;
  const uint32_t magic = (uint32_t)((1ull << 32) / (uint32_t)p.iters - (p.iters == 1));
  auto place = [&](int it, int& seg, int& step) {  // segment, and step within it, of the range's it-th step
    const int at = (it | 7) < it1 ? it ^ shift : it;
    seg = (int)(((uint64_t)(uint32_t)at * magic) >> 32);
    if (at - seg * p.iters >= p.iters) ++seg;
    step = at - seg * p.iters;
  };
  const int64_t astep = (AKS ? p.lda : 1) * GEMM_BK * 2, bstep = (BKS ? p.ldb : 1) * GEMM_BK * 2;  // bytes from one step to the next
  const int64_t a0 = (AKS ? m0 : m0 * p.lda) * 2, b0 = (BKS ? (int64_t)n0 : (int64_t)n0 * p.ldb) * 2;
  const char *sega = nullptr, *segb = nullptr, *segb2 = nullptr;  // the corners of the segment last asked for
  int have = -1;
  constexpr int LOADS = sa.PASSES + sb.PASSES;
  struct Request { i32x4 a, b, b2; int left; uint32_t to; };
  auto request = [&](int it, uint32_t stage) {  // what the loads of a stage have in common; behind the range every piece lies outside
    int seg, step;
    place(it < it1 ? it : it1 - 1, seg, step);
    if (seg != have) {
      have = seg;
      sega = (const char*)args->a[seg] + a0;
      segb = (const char*)args->b[seg] + b0;
      if (GATE) segb2 = (const char*)args->b2[seg] + b0;
    }
    Request r;
    r.a = buffer_of(sega + step * astep);
    r.b = buffer_of(segb + step * bstep);
    r.b2 = GATE ? buffer_of(segb2 + step * bstep) : r.b;
    r.left = it < it1 ? p.K - step * GEMM_BK : 0;
    r.to = lds0 + stage + wave * 1024;
    return r;
  };
  auto load = [&](const Request& r, int l) __attribute__((always_inline)) {  // the l-th of a wave's LOADS loads of a stage
    if (l < sa.PASSES) {
      load_to_lds(r.a, sa.kpos[l] < r.left ? sa.off[l] : 0x80000000u, r.to + l * NW * 1024);
    } else {
      const int j = l - sa.PASSES;
      load_to_lds(GATE && (j * NW + wave) * sb.RPW / 32 % 2 ? r.b2 : r.b, sb.kpos[j] < r.left ? sb.off[j] : 0x80000000u,
                  r.to + ABYTES + j * NW * 1024);
    }
  };

  f32x16 acc[MI][NI], asum[XS];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int x = 0; x < XS; ++x) asum[x][e] = 0.f;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j][e] = 0.f;
  }
  const short unit = __builtin_bit_cast(short, (T)1.f);
  const s16x8 ones = {unit, unit, unit, unit, unit, unit, unit, unit};

  // Fragments are read 16 k ahead of the products that take them.  The last ones of a step are in registers before the barrier, so their
  // products run while the next stage's first fragments arrive and the stage just left is filled again.
  struct Frag { s16x8 a[MI], b[NI], x[XS]; } f[2];
  auto read = [&](Frag& f, uint32_t stage, int s, bool sum) __attribute__((always_inline)) {
    const char DM_LDS* st = (const char DM_LDS*)smem + stage;
#pragma unroll
    for (int j = 0; j < NI; ++j) f.b[j] = fragment<BN, BKS, true>(st + ABYTES, lane, wn * NI + j, s);
#pragma unroll
    for (int i = 0; i < MI; ++i) f.a[i] = fragment<BM, AKS, false>(st, lane, wm * MI + i, s);
    if (SUMS && sum)
#pragma unroll
      for (int x = 0; x < XS; ++x) f.x[x] = fragment<BM, AKS, false>(st, lane, wm * MI + wn * XS + x, s);
  };
  auto multiply_row = [&](const Frag& f, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = mfma16(f.b[j], f.a[i], acc[i][j], T());
  };
  auto multiply_sums = [&](const Frag& f, bool sum) __attribute__((always_inline)) {
    if (SUMS && sum)
#pragma unroll
      for (int x = 0; x < XS; ++x) asum[x] = mfma16(ones, f.x[x], asum[x], T());
  };
  auto interleave = []() __attribute__((always_inline)) {  // a read, a product, and so on
    constexpr int READS = (AKS ? 2 : 1) * MI + (BKS ? 2 : 1) * NI, PER = (READS + MI * NI - 1) / (MI * NI);
#pragma unroll
    for (int i = 0; i < MI * NI; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr int PARTS = GEMM_BK / 16;
  const bool sums = SUMS && p.sums && tn == 0;
  auto summed = [&](int it) {  // does the range's it-th step count for the sums of A
    int seg, step;
    if (!sums) return false;
    place(it, seg, step);
    return (p.sum_segments >> seg & 1) != 0;
  };
  if (it0 < it1) {
    uint32_t cur = 0;
#pragma unroll
    for (int k = 0; k < GEMM_STAGES; ++k) {
      const Request r = request(it0 + k, k * STAGE);
#pragma unroll
      for (int l = 0; l < LOADS; ++l) load(r, l);
    }
    stage_arrived<LOADS * (GEMM_STAGES - 1)>();
    bool sum = summed(it0);
    read(f[0], 0, 0, sum);
    for (int it = it0; it < it1; ++it) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < PARTS - 1; ++s) {
        read(f[(s + 1) & 1], cur, s + 1, sum);
#pragma unroll
        for (int i = 0; i < MI; ++i) multiply_row(f[s & 1], i);
        multiply_sums(f[s & 1], sum);
        interleave();
      }
      const bool last = sum;
      const uint32_t left = cur;
      cur = cur + STAGE == GEMM_STAGES * STAGE ? 0 : cur + STAGE;
      sum = it + 1 < it1 && summed(it + 1);
      stage_arrived<LOADS * (GEMM_STAGES - 2)>();
      read(f[0], cur, 0, sum);  // (behind the range: zeros, and nobody's)
      const Request r = request(it + GEMM_STAGES, left);
#pragma unroll
      for (int i = 0; i < MI; ++i) {  // loads among the products: a burst of them would hold up the wave
        __builtin_amdgcn_sched_barrier(0);
        multiply_row(f[(PARTS - 1) & 1], i);
#pragma unroll
        for (int l = i * LOADS / MI; l < (i + 1) * LOADS / MI; ++l) load(r, l);
      }
      __builtin_amdgcn_sched_barrier(0);
      multiply_sums(f[(PARTS - 1) & 1], last);
    }
  }
  stage_arrived<0>();  // the loads behind the range are done with LDS, and so is every wave

  // acc[i][j][e] belongs to m = lane & 31 and n = 16 (lane >> 5) + e of the 32 x 32 block (i, j).  The i-th blocks of all waves meet in LDS
  // as rows of fp32 (a pitch of 16 bytes more than the row: no bank conflicts), two buffers in turn, and leave as whole pieces of
  // eight columns, neighbouring lanes next to each other: written straight from the accumulators, rows a power of two apart crowd
  // on few of the L2's channels (41 us of a 256 x 256 tile's time, measured at a row of 8 KB).
  constexpr int ROWS = WM * 32, PITCH = BN * 4 + 16, COLS = GATE ? BN / 2 : BN, PIECES = COLS / 8, TASKS = ROWS * PIECES / (NW * 64);
  const int np = (p.N + 7) & ~7;  // intermediate results are padded to whole pieces (with zeros: rows of B out of range are zero)
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    char DM_LDS* buf = (char DM_LDS*)smem + (i & 1) * ROWS * PITCH;
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& c = acc[i][j];
        *(DM_LDS f32x4*)(buf + (wm * 32 + (lane & 31)) * PITCH + ((wn * NI + j) * 32 + (lane >> 5) * 16 + q * 4) * 4) =
            f32x4{c[q * 4], c[q * 4 + 1], c[q * 4 + 2], c[q * 4 + 3]};
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TASKS; ++t) {
      const int id = t * NW * 64 + threadIdx.x, row = id / PIECES, col = id % PIECES * 8;
      const int64_t m = m0 + (row / 32 * MI + i) * 32 + row % 32;
      const int n = n0 + col;
      if (m >= p.M || n >= (EPI == EPI_STORE ? p.N : np)) continue;
      const char DM_LDS* at = buf + row * PITCH + (GATE ? col / 32 * 64 + col % 32 : col) * 4;
      float v[8];
      from_lds(at, v);
      if constexpr (GATE) {
        float u[8], h[8];
        from_lds(at + 128, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] += bias_at<Kept>(p.bias, n + e, p.N);
          u[e] += bias_at<Kept>(p.bias2, n + e, p.N);
        }
        with_activation(p.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float value, slope;
            activation<decltype(act)::value, !F32>(v[e], value, slope);
            h[e] = value * u[e];
            u[e] *= slope;
            v[e] = value;
          }
        });
        store8<T, BETWEEN>(p.out, m, n, np, h);
        if (p.out2.p) { store8<T, KEPT>(p.out2, m, n, np, u); store8<T, KEPT>(p.out3, m, n, np, v); }
      } else if constexpr (EPI == EPI_STORE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += p.out.f32 ? bias_at<float>(p.bias, n + e, p.N) : bias_at<T>(p.bias, n + e, p.N);
        Out o = p.out;
        if (p.splits > 1) o.p = (float*)o.p + blockIdx.y * p.split_stride;
        if (o.f32) store8<T, OUT_F32>(o, m, n, p.N, v);
        else store8<T, OUT_16>(o, m, n, p.N, v);
      } else {
        float ug[8], ag[8];
        load8((const Kept*)p.ug + m * p.ldg + n, ug);
        load8((const Kept*)p.ag + m * p.ldg + n, ag);
#pragma unroll
        for (int e = 0; e < 8; ++e) { ug[e] *= v[e]; ag[e] *= v[e]; }
        store8<T, BETWEEN>(p.out, m, n, np, ug);
        store8<T, BETWEEN>(p.out2, m, n, np, ag);
      }
    }
  }
  if constexpr (EPI == EPI_STORE) {
    if constexpr (SUMS) {  // every n of the product with ones holds the sum
#pragma unroll
      for (int x = 0; x < XS; ++x) {
        const int64_t m = m0 + (wm * MI + wn * XS + x) * 32 + lane;
        if (!p.sums || tn || lane >= 32 || m >= p.M) continue;
        if (p.splits > 1) ((float*)p.sums)[blockIdx.y * p.M + m] = asum[x][0];
        else if (p.sums_f32) ((float*)p.sums)[m] = asum[x][0];
        else ((T*)p.sums)[m] = (T)asum[x][0];
      }
    }
  }
}

// Adds the partial products of a split k range (and the partial sums of A), the bias, and rounds once.
template <typename T>
__global__ void __launch_bounds__(256)
gemm_join_kernel(const float* __restrict__ part, int splits, int64_t stride, const void* bias, const Out out, int64_t M, int N, int ldp,
                 const float* __restrict__ sum_part, void* sums) {
  const int pieces = ldp / 8;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < M * pieces; id += (int64_t)gridDim.x * 256) {
    const int64_t m = id / pieces;
    const int n = (int)(id % pieces) * 8;
    float v[8] = {};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      float w[8];
      load8(part + s * stride + m * ldp + n, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += out.f32 ? bias_at<float>(bias, n + e, N) : bias_at<T>(bias, n + e, N);
    if (out.f32) store8<T, OUT_F32>(out, m, n, N, v);
    else store8<T, OUT_16>(out, m, n, N, v);
  }
  if (!sums) return;
  for (int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x; m < M; m += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += sum_part[s * M + m];
    if (out.f32) ((float*)sums)[m] = v;
    else ((T*)sums)[m] = (T)v;
  }
}

struct GemmPlan { int big, splits; size_t part_bytes; };

// Tile and split of the k range.  A big tile (256 x 256, one workgroup per CU) moves half the bytes per product of a small one (128 x 128,
// two per CU); the smaller one fills the chip with fewer rows.  Where even small tiles leave CUs idle and the k range is long, it is
// split and the partial products are joined by a second launch.  The estimate is in units of one 64-step of a big tile on one CU.
inline GemmPlan gemm_plan(int64_t M, int N, int iters, bool can_split) {
  const int cus = 256;
  GemmPlan best = {0, 1, 0};
  double cost = 1e300;
  for (int big = 0; big < 2; ++big) {
    const int bm = big ? 256 : 128;
    const int64_t tiles = ((M + bm - 1) / bm) * ((N + bm - 1) / bm);
    for (int s = 1; s <= 64; s *= 2) {
      if (s > 1 && (!can_split || s > iters / 2 || tiles * (s / 2) >= 2 * cus)) break;
      const int slots = big ? cus : 2 * cus;
      const double rounds = (double)((tiles * s + slots - 1) / slots);
      const double step = big ? 1.0 : 0.7;  // two small tiles share a CU
      double c = rounds * ((iters + s - 1) / s + 4.0) * step;
      if (s > 1) c += 4.0 + (double)M * N * 4 * (s + 1) / 4.0e6;  // the joining launch at 4 TB/s, a step being about a microsecond
      if (c < cost) { cost = c; best.big = big; best.splits = s; }
    }
  }
  if (best.splits > 1) best.part_bytes = (size_t)best.splits * M * (round_up(N, 8) + 1) * 4;  // products, and sums of A
  return best;
}

template <typename T, bool AKS, bool BKS, int EPI>
int gemm_launch(GemmArgs a, bool big, hipStream_t st) {
  const int bm = big ? 256 : 128, bn = EPI == EPI_GATE || EPI == EPI_GATE_F32 ? bm / 2 : bm;
  a.tiles_m = (int)((a.M + bm - 1) / bm);
  a.tiles_n = (a.N + bn - 1) / bn;
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
  if (tiles > (1 << 22)) return fail("gated feed-forward block: %lld output tiles in one product", (long long)tiles);
  const dim3 grid((unsigned)tiles, a.splits);
  const int stages = GEMM_STAGES * 2 * bm * GEMM_BK * 2, rows = 2 * 64 * (bm * 4 + 16), bytes = stages > rows ? stages : rows;
  const void* f = big ? (const void*)gemm_kernel<T, 256, 256, 2, 4, AKS, BKS, EPI> : (const void*)gemm_kernel<T, 128, 128, 2, 2, AKS, BKS, EPI>;
  hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) {
    void* args[] = {&a};
    e = hipLaunchKernel(f, grid, dim3(big ? 512 : 256), args, bytes, st);
  }
  return e == hipSuccess ? 0 : fail("gated feed-forward block: launch failed: %s", hipGetErrorString(e));
}

// The fused products are compiled in translation units of their own (dm_block_ffn_gate.hip, dm_block_ffn_dact.hip).
extern template int gemm_launch<bf16, false, false, EPI_GATE>(GemmArgs, bool, hipStream_t);
extern template int gemm_launch<f16, false, false, EPI_GATE>(GemmArgs, bool, hipStream_t);
extern template int gemm_launch<bf16, false, false, EPI_GATE_F32>(GemmArgs, bool, hipStream_t);
extern template int gemm_launch<bf16, false, true, EPI_DACT>(GemmArgs, bool, hipStream_t);
extern template int gemm_launch<f16, false, true, EPI_DACT>(GemmArgs, bool, hipStream_t);
extern template int gemm_launch<bf16, false, true, EPI_DACT_F32>(GemmArgs, bool, hipStream_t);

}  // namespace dmb
#endif
