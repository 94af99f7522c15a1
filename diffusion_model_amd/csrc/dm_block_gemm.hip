// dm_block_gemm.hip — C[m,n] = sum_k A[m,k] B[n,k] on the 16-bit matrix pipe, the products of the gated feed-forward block.
//
// An operand is stored either with k contiguous ("KC": rows of the operand) or with its own rows contiguous ("KS": k is the slow
// index), so that the forward pass and all three products of the backward pass run from the tensors as they lie in memory; a KS tile
// is transposed on its way out of LDS (ds_read_tr).  The k range may be a chain of up to 12 segments, each with base pointers of its
// own: the two terms of dx = dg Wg + du Wu, and the six products of fp32 operands that were split into three bf16 terms.
//
// A workgroup owns a BM x BN tile and walks k in steps of 64: two LDS stages, filled by buffer loads that write LDS directly (16 bytes
// per lane, rows and columns out of range are bounds-checked to zero by the buffer resource), one barrier per step.  The LDS image
// is swizzled in 16-byte pieces so that fragment reads touch all 64 banks once.  Fragments feed v_mfma_f32_32x32x16 with the n side as
// the first operand: a lane then holds four consecutive n of one m, which the epilogue stores as one vector.
#ifndef DM_BLOCK_GEMM_HIP
#define DM_BLOCK_GEMM_HIP
#include "dm_block_common.h"

namespace dmb {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
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
// Where a result goes: rows of `ld` elements; OUT_PLANES: three bf16 planes, `plane` elements apart.  `vec`: rows take 4-element stores.
struct Out { void* p; int64_t ld, plane; int mode, vec; };

template <typename T>
__device__ __forceinline__ void store4(const Out& o, int64_t m, int n, int N, const float (&v)[4]) {
  const int64_t at = m * o.ld + n;
  if (o.vec && n + 4 <= N) {
    if (o.mode == OUT_F32) {
      store_vec<float, 4>((float*)o.p + at, v);
    } else if (o.mode == OUT_16) {
      store_vec<T, 4>((T*)o.p + at, v);
    } else {
      Vec<bf16, 4> r[3];
#pragma unroll
      for (int i = 0; i < 4; ++i) { bf16 t[3]; split3(v[i], t); r[0].v[i] = t[0]; r[1].v[i] = t[1]; r[2].v[i] = t[2]; }
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<Vec<bf16, 4>*>((bf16*)o.p + k * o.plane + at) = r[k];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= N) break;
    if (o.mode == OUT_F32) ((float*)o.p)[at + i] = v[i];
    else if (o.mode == OUT_16) ((T*)o.p)[at + i] = (T)v[i];
    else { bf16 t[3]; split3(v[i], t); for (int k = 0; k < 3; ++k) ((bf16*)o.p)[k * o.plane + at + i] = t[k]; }
  }
}

// ---- activations: value and slope, fp32
__device__ __forceinline__ float act_value(int act, float v) {
  switch (act) {
    case DM_ACT_RELU: return v > 0.f ? v : (v != v ? v : 0.f);
    case DM_ACT_GELU: return v * (0.5f * (1.f + erff(v * 0.70710678f)));
    case DM_ACT_GELU_TANH: return 0.5f * v * (1.f + tanhf(0.79788456f * (v + 0.044715f * v * v * v)));
    case DM_ACT_SIGMOID: return 1.f / (1.f + expf(-v));
    default: return v / (1.f + expf(-v));
  }
}
__device__ __forceinline__ void act_slope(int act, float v, float& value, float& slope) {
  switch (act) {
    case DM_ACT_RELU: value = v > 0.f ? v : (v != v ? v : 0.f); slope = v > 0.f ? 1.f : 0.f; break;
    case DM_ACT_GELU: {
      const float cdf = 0.5f * (1.f + erff(v * 0.70710678f));
      value = v * cdf;
      slope = cdf + v * expf(-0.5f * v * v) * 0.39894228f;
      break;
    }
    case DM_ACT_GELU_TANH: {
      const float t = tanhf(0.79788456f * (v + 0.044715f * v * v * v));
      value = 0.5f * v * (1.f + t);
      slope = 0.5f * (1.f + t) + 0.5f * v * (1.f - t * t) * 0.79788456f * (1.f + 0.134145f * v * v);
      break;
    }
    case DM_ACT_SIGMOID: { const float s = 1.f / (1.f + expf(-v)); value = s; slope = s * (1.f - s); break; }
    default: { const float s = 1.f / (1.f + expf(-v)); value = v * s; slope = s * (1.f + v * (1.f - s)); }
  }
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) { load_vec<T, 4>(p, v); }

constexpr int GEMM_MAX_SEGMENTS = 12;
enum { EPI_STORE = 0, EPI_GATE = 1, EPI_DACT = 2 };

struct GemmArgs {
  const void* a[GEMM_MAX_SEGMENTS];
  const void* b[GEMM_MAX_SEGMENTS];
  const void* b2[GEMM_MAX_SEGMENTS];  // EPI_GATE: the second projection's weights
  int segments, iters;                // iters: k steps of 64 per segment
  int64_t lda, ldb;                   // elements
  int64_t M;
  int N, K;                           // N: of one projection for EPI_GATE.  K: true length; a KC row is zero from there to the end of its piece
  int tiles_m, tiles_n, splits;
  Out out, out2, out3;                // STORE: out.  GATE: out = h, out2 = g, out3 = u (null: not kept).  DACT: dg, du, h
  const void *bias, *bias2;           // of the element type given by bias_f32
  int bias_f32;
  const void *g, *u;                  // DACT: saved projections, rows of ldg
  int64_t ldg;
  int gu_f32, act;
  int64_t split_stride;               // STORE with splits > 1: fp32 partial products, elements from one split to the next
};

template <int N>  // piece of 16 bytes that holds piece `c` of row k of a KS tile with N columns
__device__ __forceinline__ int ks_swizzle(int k, int c) { return N >= 128 ? c ^ ((k & 3) << 2) : c ^ (((k >> 1) & 1) << 2); }

// One LDS stage of one operand: R rows (of A or B) x 64 k, 16-bit elements, by the NW waves of the block.
template <int R, bool KS, int NW>
struct Stager {
  static constexpr int PASSES = R * 8 / (64 * NW);  // 16-byte pieces per lane
  static constexpr int CPR = KS ? R / 8 : 8;        // pieces per LDS row
  static constexpr int RPW = 64 / CPR;              // LDS rows that one wave's load fills
  uint32_t off[PASSES];                             // byte offset from the tile's corner, 2^31 where the piece lies outside
  int kpos[PASSES];                                 // k of the piece within the step
  __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int64_t rows_left) {
#pragma unroll
    for (int j = 0; j < PASSES; ++j) {
      const int row = (j * NW + wave) * RPW + lane / CPR, slot = lane % CPR;
      if constexpr (KS) {
        const int c = ks_swizzle<R>(row, slot);
        off[j] = c * 8 < rows_left ? (uint32_t)(row * ld * 2 + c * 16) : 0x80000000u;
        kpos[j] = row;
      } else {
        const int c = slot ^ ((row >> 1) & 7);
        off[j] = row < rows_left ? (uint32_t)(row * ld * 2 + c * 16) : 0x80000000u;
        kpos[j] = c * 8;
      }
    }
  }
};

// 16 bytes per lane from a bounds-checked buffer straight into LDS at `lds` + lane * 16.  The caller waits (vmcnt) and synchronises.
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc), "s"(lds) : "memory");
}
__device__ __forceinline__ i32x4 buffer_of(const void* p) {
  const uint64_t u = (uint64_t)p;
  return i32x4{(int)(uint32_t)u, (int)(uint32_t)(u >> 32) & 0xffff, (int)0x80000000u, 0x00020000};
}
__device__ __forceinline__ void stage_arrived() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Fragments of 32 rows x 16 k (step s of 4) out of a stage.
template <int R, bool KS>
struct Fragments {
  uint32_t base;
  int tile;  // first 32-row tile of this wave
  __device__ __forceinline__ void init(int lane, int tile0) {
    tile = tile0;
    if constexpr (KS) {
      const int g = lane >> 4, j = (lane >> 2) & 3, c = lane & 3;
      base = ((g >> 1) * 8 + j) * R * 2 + (c & 1) * 8;  // + the swizzled piece
    } else {
      base = (lane & 31) * 128;
    }
  }
  __device__ __forceinline__ s16x8 get(const char DM_LDS* stage, int lane, int t, int s) const {
    if constexpr (KS) {
      const int g = lane >> 4, j = (lane >> 2) & 3, c = lane & 3;
      const int k = (g >> 1) * 8 + j;  // plus multiples of 4: the swizzle sees only its low bits
      const int piece = (tile + t) * 4 + (g & 1) * 2 + (c >> 1);
      s16x4 h[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int kk = s * 16 + q * 4 + k;
        h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DM_LDS s16x4*)(stage + kk * (R * 2) + ks_swizzle<R>(kk, piece) * 16 + (c & 1) * 8));
      }
      return s16x8{h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
    } else {
      const int row = (tile + t) * 32 + (lane & 31);
      const int c = (2 * s + (lane >> 5)) ^ ((lane >> 1) & 7);  // (row >> 1) & 7 of a row that is lane & 31 above a multiple of 32
      return *(const DM_LDS s16x8*)(stage + row * 128 + c * 16);
    }
  }
};

template <typename T, int BM, int BN, int WM, int WN, bool AKS, bool BKS, int EPI>
__global__ void __launch_bounds__(WM * WN * 64, WM * WN == 8 ? 2 : 2)
gemm_kernel(const GemmArgs p) {
  constexpr int NW = WM * WN, MI = BM / WM / 32, NI = BN / WN / 32;
  constexpr int ABYTES = BM * 128, STAGE = (BM + BN) * 128;
  static_assert(EPI != EPI_GATE || (NI == 2 && !BKS), "a wave of the gated product owns 32 columns of each projection");
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
  constexpr int BROWS = EPI == EPI_GATE ? BN / 2 : BN;  // columns of one projection in the tile
  const int n0 = tn * BROWS;

  const int total = p.segments * p.iters;
  const int per = (total + p.splits - 1) / p.splits;
  const int it0 = blockIdx.y * per, it1 = it0 + per < total ? it0 + per : total;

  Stager<BM, AKS, NW> sa;
  Stager<BN, BKS, NW> sb;
  sa.init(wave, lane, p.lda, p.M - m0);
  if constexpr (EPI == EPI_GATE) {  // rows 64 i .. +31 of the tile are the first projection's, +32 .. +63 the second's
#pragma unroll
    for (int j = 0; j < sb.PASSES; ++j) {
      const int row = (j * NW + wave) * 8 + lane / 8, slot = lane % 8, c = slot ^ ((row >> 1) & 7);
      const int f = row / 64 * 32 + row % 32;
      sb.off[j] = n0 + f < p.N ? (uint32_t)(f * p.ldb * 2 + c * 16) : 0x80000000u;
      sb.kpos[j] = c * 8;
    }
  } else {
    sb.init(wave, lane, p.ldb, p.N - n0);
  }
  Fragments<BM, AKS> fa;
  Fragments<BN, BKS> fb;
  fa.init(lane, wm * MI);
  fb.init(lane, wn * NI);

  const uint32_t lds0 = (uint32_t)(uintptr_t)(DM_LDS char*)smem;
  // (the segments' pointers are read where the launch put the arguments: indexing the parameter itself would copy it to scratch)
  const auto* args = (const __attribute__((address_space(4))) GemmArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  auto issue = [&](int it, uint32_t stage) {
    const int seg = it / p.iters, k0 = (it - seg * p.iters) * 64;
    const int left = p.K - k0;
    const i32x4 ra = buffer_of((const char*)args->a[seg] + (AKS ? (int64_t)k0 * p.lda + m0 : m0 * p.lda + k0) * 2);
#pragma unroll
    for (int j = 0; j < sa.PASSES; ++j)
      load_to_lds(ra, sa.kpos[j] < left ? sa.off[j] : 0x80000000u, lds0 + stage + (j * NW + wave) * 1024);
    const int64_t bo = (BKS ? (int64_t)k0 * p.ldb + n0 : (int64_t)n0 * p.ldb + k0) * 2;
    const i32x4 rb = buffer_of((const char*)args->b[seg] + bo);
    if constexpr (EPI == EPI_GATE) {
      const i32x4 rb2 = buffer_of((const char*)args->b2[seg] + bo);
#pragma unroll
      for (int j = 0; j < sb.PASSES; ++j)
        load_to_lds((j * NW + wave) / 4 % 2 ? rb2 : rb, sb.kpos[j] < left ? sb.off[j] : 0x80000000u,
                    lds0 + stage + ABYTES + (j * NW + wave) * 1024);
    } else {
#pragma unroll
      for (int j = 0; j < sb.PASSES; ++j)
        load_to_lds(rb, sb.kpos[j] < left ? sb.off[j] : 0x80000000u, lds0 + stage + ABYTES + (j * NW + wave) * 1024);
    }
  };

  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  uint32_t cur = 0;
  if (it0 < it1) issue(it0, 0);
  for (int it = it0; it < it1; ++it) {
    stage_arrived();  // this step's tiles are in LDS, and every wave is done with the other stage
    if (it + 1 < it1) issue(it + 1, cur ^ STAGE);
    const char DM_LDS* st = (const char DM_LDS*)smem + cur;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      s16x8 a[MI], b[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) a[i] = fa.get(st, lane, i, s);
#pragma unroll
      for (int j = 0; j < NI; ++j) b[j] = fb.get(st + ABYTES, lane, j, s);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mfma16(b[j], a[i], acc[i][j], T());
    }
    cur ^= STAGE;
  }

  // acc[i][j][4 q + e] belongs to m = lane & 31 and n = 8 q + 4 (lane >> 5) + e of the 32 x 32 block (i, j).
  const int np = (p.N + 7) & ~7;  // intermediate results are padded to whole pieces (with zeros: rows of B out of range are zero)
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = m0 + (wm * MI + i) * 32 + (lane & 31);
    if (m >= p.M) continue;
    if constexpr (EPI == EPI_GATE) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + wn * 32 + q * 8 + (lane >> 5) * 4;
        if (n >= np) continue;
        float g[4], u[4], h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[e] = acc[i][0][q * 4 + e];
          u[e] = acc[i][1][q * 4 + e];
          if (n + e < p.N) {
            if (p.bias) g[e] += p.bias_f32 ? ((const float*)p.bias)[n + e] : (float)((const T*)p.bias)[n + e];
            if (p.bias2) u[e] += p.bias_f32 ? ((const float*)p.bias2)[n + e] : (float)((const T*)p.bias2)[n + e];
          }
          h[e] = act_value(p.act, g[e]) * u[e];
        }
        store4<T>(p.out, m, n, np, h);
        if (p.out2.p) { store4<T>(p.out2, m, n, np, g); store4<T>(p.out3, m, n, np, u); }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = n0 + (wn * NI + j) * 32 + q * 8 + (lane >> 5) * 4;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[i][j][q * 4 + e];
          if constexpr (EPI == EPI_STORE) {
            if (n >= p.N) continue;
            if (p.bias)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n + e < p.N) v[e] += p.bias_f32 ? ((const float*)p.bias)[n + e] : (float)((const T*)p.bias)[n + e];
            Out o = p.out;
            if (p.splits > 1) o.p = (float*)o.p + blockIdx.y * p.split_stride;
            store4<T>(o, m, n, p.N, v);
          } else {
            if (n >= np) continue;
            float g[4], u[4], dg[4], du[4], h[4];
            if (p.gu_f32) { load4((const float*)p.g + m * p.ldg + n, g); load4((const float*)p.u + m * p.ldg + n, u); }
            else { load4((const T*)p.g + m * p.ldg + n, g); load4((const T*)p.u + m * p.ldg + n, u); }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float value, slope;
              act_slope(p.act, g[e], value, slope);
              dg[e] = v[e] * u[e] * slope;
              du[e] = v[e] * value;
              h[e] = value * u[e];
            }
            store4<T>(p.out, m, n, np, dg);
            store4<T>(p.out2, m, n, np, du);
            store4<T>(p.out3, m, n, np, h);
          }
        }
    }
  }
}

// Adds the partial products of a split k range, the bias, and rounds once.
template <typename T>
__global__ void __launch_bounds__(256)
gemm_join_kernel(const float* __restrict__ part, int splits, int64_t stride, const void* bias, int bias_f32, Out out, int64_t M, int N, int ldp) {
  const int quads = ldp / 4;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < M * quads; id += (int64_t)gridDim.x * 256) {
    const int64_t m = id / quads;
    const int n = (int)(id % quads) * 4;
    if (n >= N) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
      float w[4];
      load4(part + s * stride + m * ldp + n, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += w[e];
    }
    if (bias)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < N) v[e] += bias_f32 ? ((const float*)bias)[n + e] : (float)((const T*)bias)[n + e];
    store4<T>(out, m, n, N, v);
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
  if (best.splits > 1) best.part_bytes = (size_t)best.splits * M * round_up(N, 4) * 4;
  return best;
}

template <typename T, bool AKS, bool BKS, int EPI>
int gemm_launch(GemmArgs a, bool big, hipStream_t st) {
  const int bm = big ? 256 : 128, bn = EPI == EPI_GATE ? bm / 2 : bm;
  a.tiles_m = (int)((a.M + bm - 1) / bm);
  a.tiles_n = (a.N + bn - 1) / bn;
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
  if (tiles > (1 << 22)) return fail("gated feed-forward block: %lld output tiles in one product", (long long)tiles);
  const dim3 grid((unsigned)tiles, a.splits);
  const int bytes = 2 * 2 * bm * 128;
  const void* f = big ? (const void*)gemm_kernel<T, 256, 256, 2, 4, AKS, BKS, EPI> : (const void*)gemm_kernel<T, 128, 128, 2, 2, AKS, BKS, EPI>;
  hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) {
    void* args[] = {&a};
    e = hipLaunchKernel(f, grid, dim3(big ? 512 : 256), args, bytes, st);
  }
  return e == hipSuccess ? 0 : fail("gated feed-forward block: launch failed: %s", hipGetErrorString(e));
}

}  // namespace dmb
#endif
