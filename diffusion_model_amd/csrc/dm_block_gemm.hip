// dm_block_gemm.hip — C[m,n] = sum_k A[m,k] B[n,k] on the 16-bit matrix pipe, the products of the gated feed-forward block.
//
// An operand is stored either with k contiguous ("KC": rows of the operand) or with its own rows contiguous ("KS": k is the slow
// index), so that the forward pass and all three products of the backward pass run from the tensors as they lie in memory; a KS tile
// is transposed on its way out of LDS (ds_read_tr).  The k range may be a chain of up to 12 segments, each with base pointers of its
// own: the two terms of dx = dg Wg + du Wu, and the six products of fp32 operands that were split into three bf16 terms.
//
// A workgroup owns a BM x BN tile and walks k in steps of GEMM_BK: two LDS stages (three of the smallest tile), filled by buffer loads that write LDS directly (16 bytes
// per lane, rows and columns out of range are bounds-checked to zero by the buffer resource), one barrier per step.  The LDS image
// is swizzled in 16-byte pieces so that fragment reads touch all 64 banks once.  Fragments feed v_mfma_f32_16x16x32 with the n side as
// the first operand: a lane then holds four consecutive n of one m.
// A bias' gradient, the sum of A over k, is one more product with ones from the same fragments.
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

constexpr int LDS_BIAS = 3072;  // see load_to_lds
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
  void* part;                         // splits > 1: fp32 partial products (GATE: of both projections in turn), rows of ldpart,
  int64_t split_stride, ldpart;       // split_stride elements from one to the next; joined by a second launch
  void* sums;                         // STORE with both operands KS: sum over k of A[m, k] over the segments of sum_segments, or null.  One split:
  int sum_segments, sums_f32;         // of the type that sums_f32 gives; several: fp32, M apart
};

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
  uint32_t off[PASSES];                                       // byte offset from the tile's corner, 2^31 where the piece lies outside
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
      off[j] = (KS ? c * 8 : r) < rows_left ? (uint32_t)(r * ld * 2 + c * 16) + bias : 0x80000000u;
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
      : "memory");
}
__device__ __forceinline__ i32x4 buffer_of(const void* p) {
  const uint64_t u = (uint64_t)p - LDS_BIAS;
  return i32x4{(int)(uint32_t)u, (int)(uint32_t)(u >> 32), (int)0x80000000u, 0x00020000};  // (addresses have 48 bits: no stride)
}
// All but the LEFT newest loads of every wave are in LDS, and every wave has its fragments of the stage at hand in registers.
template <int LEFT>
__device__ __forceinline__ void stage_arrived() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory"); }

// Fragment of 16 rows x 32 k (the s-th of the step) out of a stage: lane l holds row l & 15, k 8 (l >> 4) .. +7.
template <int R, bool KS>
__device__ __forceinline__ s16x8 fragment(const char DM_LDS* stage, int lane, int tile, int s) {
  if constexpr (KS) {
    // A lane asks for 4 consecutive rows of one k; of 16 lanes' answers, lane i receives row i of four k.
    const int k0 = s * 32 + (lane >> 4) * 8 + ((lane >> 2) & 3), piece = tile * 2 + ((lane >> 1) & 1);
    s16x4 h[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = k0 + q * 4;
      h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DM_LDS s16x4*)(stage + k * (R * 2) + (piece ^ ks_key(k)) * 16 + (lane & 1) * 8));
    }
    return s16x8{h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
  } else {
    const int row = tile * 16 + (lane & 15);
    return *(const DM_LDS s16x8*)(stage + row * (GEMM_BK * 2) + ((s * 4 + (lane >> 4)) ^ kc_key(lane & 15)) * 16);
  }
}

template <typename T, int BM, int BN, int WM, int WN, int GEMM_STAGES, bool AKS, bool BKS, int EPI>
__global__ void __launch_bounds__(WM * WN * 64, 2)
gemm_kernel(const GemmArgs p) {
  constexpr int NW = WM * WN, MI = BM / WM / 16, NI = BN / WN / 16;
  constexpr int ABYTES = BM * GEMM_BK * 2, STAGE = (BM + BN) * GEMM_BK * 2;
  constexpr bool GATE = EPI == EPI_GATE || EPI == EPI_GATE_F32, F32 = EPI == EPI_GATE_F32 || EPI == EPI_DACT_F32, SUMS = AKS && BKS;
  using Kept = typename std::conditional<F32, float, T>::type;  // what GATE keeps for DACT
  constexpr int BETWEEN = F32 ? OUT_PLANES : OUT_16, KEPT = F32 ? OUT_F32 : OUT_16;
  constexpr int XS = MI >= WN ? MI / WN : 1;  // the waves of a tile row share its sums of A: XS blocks of 16 rows each
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

  Stager<BM, AKS, NW> sa;
  Stager<BN, BKS, NW> sb;
  sa.template init<false>(wave, lane, p.lda, p.M - m0);
  sb.template init<GATE>(wave, lane, p.ldb, p.N - n0);

  // (the segments' pointers are read where the launch put the arguments: indexing the parameter itself would copy it to scratch)
  const auto* args = (const __attribute__((address_space(4))) GemmArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  const uint32_t lds0 = (uint32_t)(uintptr_t)(DM_LDS char*)smem;
  // Steps are taken in an order of the tile's own within each eight of a segment: the blocks of an XCD would otherwise ask for the same
  // columns of all rows at once, which lie on few of the L2's channels when rows are a power of two apart.  An eight that the block's
  // range or the segment does not hold whole keeps its order (several segments of no whole eights: all of them).
  const int shift = p.segments > 1 && p.iters % 8 ? 0 : (tm + 2 * tn) & 7;
  int seg = it0 / p.iters, step = it0 - seg * p.iters;  // of the next stage to be asked for
  const int whole = p.segments > 1 ? p.iters : it1;     // the end of the segment's steps in this range
  const int64_t astep = (AKS ? p.lda : 1) * GEMM_BK * 2, bstep = (BKS ? p.ldb : 1) * GEMM_BK * 2;  // bytes from one step to the next
  const int64_t a0 = (AKS ? m0 : m0 * p.lda) * 2, b0 = (BKS ? (int64_t)n0 : (int64_t)n0 * p.ldb) * 2;
  const char *sega = (const char*)args->a[seg] + a0, *segb = (const char*)args->b[seg] + b0;  // the corners of the segment at hand
  const char* segb2 = GATE ? (const char*)args->b2[seg] + b0 : nullptr;
  constexpr int LOADS = sa.PASSES + sb.PASSES;
  struct Request { i32x4 a, b, b2; int left; bool sum; };
  auto request = [&](int it) __attribute__((always_inline)) {  // what the loads of the range's it-th step have in common
    const int at = (step | 7) < whole ? step ^ shift : step;
    Request r;
    r.a = buffer_of(sega + at * astep);
    r.b = buffer_of(segb + at * bstep);
    r.b2 = GATE ? buffer_of(segb2 + at * bstep) : r.b;
    r.left = it < it1 ? p.K - at * GEMM_BK : 0;  // behind the range every piece lies outside
    r.sum = SUMS && it < it1 && (p.sum_segments >> seg & 1);
    if (++step == p.iters && seg + 1 < p.segments) {
      step = 0;
      ++seg;
      sega = (const char*)args->a[seg] + a0;
      segb = (const char*)args->b[seg] + b0;
      if (GATE) segb2 = (const char*)args->b2[seg] + b0;
    }
    return r;
  };
  // Pairs [first, last) of a wave's loads of a stage.  A wave fills a contiguous part of each operand's tile.
  auto load = [&](const Request& r, uint32_t stage, int first, int last) __attribute__((always_inline)) {
#pragma unroll
    for (int l = first * 2; l < last * 2; l += 2) {
      const bool A = l < sa.PASSES;
      const int j = A ? l : l - sa.PASSES;
      uint32_t o0 = A ? sa.off[j] : sb.off[j], o1 = A ? sa.off[j + 1] : sb.off[j + 1];
      if (r.left < GEMM_BK) {  // the last step of a k range of no whole steps
        if ((A ? sa.k_of(wave, lane, j) : sb.k_of(wave, lane, j)) >= r.left) o0 = 0x80000000u;
        if ((A ? sa.k_of(wave, lane, j + 1) : sb.k_of(wave, lane, j + 1)) >= r.left) o1 = 0x80000000u;
      }
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
  auto part = [&](int q, uint32_t from, int s, bool refill, const Request& r, uint32_t to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int l = i * PER; l < (i + 1) * PER; ++l)
        if (l < READS) read(q ^ 1, from, s, l);
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = mfma16(fb[q][j], fa[q][i], acc[i][j], T());
      if (refill) load(r, to, i * (LOADS / 2) / MI, (i + 1) * (LOADS / 2) / MI);
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
  const bool sums = SUMS && p.sums && tn == 0;
  if (it0 < it1) {
    uint32_t cur = 0;
    bool sum = false, next[GEMM_STAGES];  // do the stage at hand, and those asked for, count for the sums of A
#pragma unroll
    for (int k = 0; k < GEMM_STAGES; ++k) {
      const Request r = request(it0 + k);
      next[k] = sums && r.sum;
      load(r, k * STAGE, 0, LOADS / 2);
    }
    stage_arrived<LOADS * (GEMM_STAGES - 1)>();
    sum = next[0];
#pragma unroll
    for (int l = 0; l < READS; ++l) read(0, 0, 0, l);
    for (int it = it0; it < it1; ++it) {
      const Request r = request(it + GEMM_STAGES);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < PARTS - 1; ++s) part(s & 1, cur, s + 1, false, r, 0);
      static_assert(PARTS % 2 == 0, "a step ends with the set that it began with");
      if (sum) add_sums(cur);
      const uint32_t left = cur;
      cur = cur + STAGE == GEMM_STAGES * STAGE ? 0 : cur + STAGE;
#pragma unroll
      for (int k = 0; k < GEMM_STAGES - 1; ++k) next[k] = next[k + 1];
      next[GEMM_STAGES - 1] = sums && r.sum;
      sum = next[0];
      stage_arrived<LOADS * (GEMM_STAGES - 2)>();
      part((PARTS - 1) & 1, cur, 0, true, r, left);  // (behind the range it reads zeros, and nobody uses them)
    }
  }
  stage_arrived<0>();  // the loads behind the range are done with LDS, and so is every wave

  // acc[i][j][e] belongs to m = lane & 15 and n = 4 (lane >> 4) + e of the 16 x 16 block (i, j).  Two block rows of all waves meet in LDS
  // as rows of fp32 (a pitch of 16 bytes more than the row: no bank conflicts), two buffers in turn, and leave as whole pieces of
  // eight columns, neighbouring lanes next to each other: written straight from the accumulators, rows a power of two apart crowd
  // on few of the L2's channels (41 us of a 256 x 256 tile's time, measured at a row of 8 KB).
  constexpr int ROWS = WM * 32, PITCH = BN * 4 + 16, COLS = GATE ? BN / 2 : BN, PIECES = COLS / 8, TASKS = ROWS * PIECES / (NW * 64);
  const int np = (p.N + 7) & ~7;  // intermediate results are padded to whole pieces (with zeros: rows of B out of range are zero)
#pragma unroll
  for (int i = 0; i < MI / 2; ++i) {
    char DM_LDS* buf = (char DM_LDS*)smem + (i & 1) * ROWS * PITCH;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NI; ++j)
        *(DM_LDS f32x4*)(buf + (wm * 32 + h * 16 + (lane & 15)) * PITCH + ((wn * NI + j) * 16 + (lane >> 4) * 4) * 4) = acc[i * 2 + h][j];
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TASKS; ++t) {
      const int id = t * NW * 64 + threadIdx.x, row = id / PIECES, col = id % PIECES * 8;
      const int64_t m = m0 + row / 32 * (MI * 16) + i * 32 + row % 32;
      const int n = n0 + col;
      if (m >= p.M || n >= (EPI == EPI_STORE ? p.N : np)) continue;
      const char DM_LDS* at = buf + row * PITCH + (GATE ? col / 32 * 64 + col % 32 : col) * 4;
      float v[8];
      from_lds(at, v);
      if constexpr (GATE) {
        float u[8], h[8];
        from_lds(at + 128, u);
        if (p.splits > 1) {  // finished by gate_join_kernel
          float* part = (float*)p.part + 2 * blockIdx.y * p.split_stride + m * p.ldpart + n;
          store_f32(part, v);
          store_f32(part + p.split_stride, u);
          continue;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] += bias_at<Kept>(p.bias, n + e, p.N);
          u[e] += bias_at<Kept>(p.bias2, n + e, p.N);
        }
        gate_values<!F32>(p.act, v, u, h);
        store8<T, BETWEEN>(p.out, m, n, np, h);
        if (p.out2.p) { store8<T, KEPT>(p.out2, m, n, np, u); store8<T, KEPT>(p.out3, m, n, np, v); }
      } else if constexpr (EPI == EPI_STORE) {
#pragma unroll
        for (int e = 0; e < 8 && p.splits == 1; ++e) v[e] += p.out.f32 ? bias_at<float>(p.bias, n + e, p.N) : bias_at<T>(p.bias, n + e, p.N);
        if (p.splits > 1) store_f32((float*)p.part + blockIdx.y * p.split_stride + m * p.ldpart + n, v);
        else if (p.out.f32) store8<T, OUT_F32>(p.out, m, n, p.N, v);
        else store8<T, OUT_16>(p.out, m, n, p.N, v);
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
        const int64_t m = m0 + (wm * MI + wn * XS + x) * 16 + lane;
        if (!p.sums || tn || lane >= 16 || m >= p.M) continue;
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

// The same for the gated product: bias, activation and product of the joined projections.
template <typename T, bool F32>
__global__ void __launch_bounds__(256) gate_join_kernel(const GemmArgs p) {
  using Kept = typename std::conditional<F32, float, T>::type;
  const int np = (p.N + 7) & ~7, pieces = np / 8;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < p.M * pieces; id += (int64_t)gridDim.x * 256) {
    const int64_t m = id / pieces;
    const int n = (int)(id % pieces) * 8;
    const float* part = (const float*)p.part + m * p.ldpart + n;
    float g[8] = {}, u[8] = {}, h[8];
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
      float a[8], b[8];
      load8(part + 2 * s * p.split_stride, a);
      load8(part + (2 * s + 1) * p.split_stride, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) { g[e] += a[e]; u[e] += b[e]; }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) { g[e] += bias_at<Kept>(p.bias, n + e, p.N); u[e] += bias_at<Kept>(p.bias2, n + e, p.N); }
    gate_values<!F32>(p.act, g, u, h);
    store8<T, F32 ? OUT_PLANES : OUT_16>(p.out, m, n, np, h);
    if (p.out2.p) { store8<T, F32 ? OUT_F32 : OUT_16>(p.out2, m, n, np, u); store8<T, F32 ? OUT_F32 : OUT_16>(p.out3, m, n, np, g); }
  }
}

// Tiles.  WIDE, 256 x 256: one workgroup of 8 waves per CU; the fewest bytes and LDS reads per product.  MID, 128 x 128: two of 4 waves per
// CU.  SLIM, 64 x 128: two of 4 waves per CU with three stages each, for rows so few that the n side's bytes are what counts.
enum { TILE_WIDE, TILE_MID, TILE_SLIM, TILES };
constexpr int TILE_M[TILES] = {256, 128, 64}, TILE_N[TILES] = {256, 128, 128}, TILE_PER_CU[TILES] = {1, 2, 2};

struct GemmPlan { int tile, splits; size_t part_bytes; };

// Tile and split of the k range.  Estimated in microseconds: rounds of workgroups over the chip, each of its k steps (measured: 1.6 us a
// step of a WIDE tile, 1.2 and 0.8 us of two MID or SLIM tiles on a CU) and a start and an end; not less than the bytes of the n side at
// 5.5 TB/s; and, where the k range is split to fill the chip, the joining launch.  `outs`: products per n (2: both projections).
inline GemmPlan gemm_plan(int64_t M, int N, int iters, int outs, bool can_split, bool slim) {
  const int cus = 256;
  constexpr double STEP[TILES] = {1.6, 1.2, 0.8};
  GemmPlan best = {TILE_MID, 1, 0};
  double cost = 1e300;
  for (int t = 0; t < TILES; ++t) {
    if (t == TILE_SLIM && !slim) continue;
    const int64_t tiles = ((M + TILE_M[t] - 1) / TILE_M[t]) * (((int64_t)N * outs + TILE_N[t] - 1) / TILE_N[t]);
    const int slots = cus * TILE_PER_CU[t];
    for (int s = 1; s <= 64; s *= 2) {
      if (s > 1 && (!can_split || s * 8 > iters || tiles * (s / 2) >= slots)) break;
      const double rounds = (double)((tiles * s + slots - 1) / slots);
      const double fill = tiles * s < slots / 2 && TILE_PER_CU[t] > 1 ? 0.6 : 1.0;  // alone on its CU a workgroup is faster
      double c = rounds * (((iters + s - 1) / s) * STEP[t] * fill + 4.0);
      const double stream = (double)N * outs * iters * GEMM_BK * 2 / 5.5e6;
      if (c < stream) c = stream;
      if (s > 1) c += 3.0 + (double)M * N * outs * 4 * 2 * s / 5.0e6;
      if (c < cost) { cost = c; best.tile = t; best.splits = s; }
    }
  }
  if (best.splits > 1) best.part_bytes = (size_t)best.splits * outs * M * (round_up(N, 8) + 1) * 4;  // products, and sums of A
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

template <typename T, bool AKS, bool BKS, int EPI>
int gemm_launch(GemmArgs a, int tile, hipStream_t st) {
  constexpr bool GATE = EPI == EPI_GATE || EPI == EPI_GATE_F32, SLIM = !AKS && (EPI == EPI_STORE || GATE);
  const int bm = TILE_M[tile], bn = TILE_N[tile];
  a.tiles_m = (int)((a.M + bm - 1) / bm);
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
  if (e == hipSuccess && GATE && a.splits > 1) {  // (a.splits is 1 elsewhere: product joins its own)
    const int64_t blocks = (a.M * ((a.N + 7) / 8) + 255) / 256;
    gate_join_kernel<T, EPI == EPI_GATE_F32><<<dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st>>>(a);
    e = hipGetLastError();
  }
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
