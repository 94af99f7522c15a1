// dm_block_norm.hip — layer norm and its backward pass.
//   z = (x - mean) rstd, y = z w + b;  gz = dy w, dx = rstd (gz - mean(gz) - z mean(gz z)), dw = sum dy z, db = sum dy.
// Both are bound by memory: a row is read once into registers, its mean and centred sum of squares (two sums over the
// registers, no cancellation) follow from there, and the result is written once.  All sums are fp32.  The parameters'
// gradients are summed per workgroup over the rows it walks, written as partial rows and added in a fixed order by a second
// launch: no atomics, the same bits every time.
#include <type_traits>

#include "dm_block_common.h"

namespace dmb {

// Sum over the TPR threads of a row: within a wave by shuffles, across the waves of a block through `red`.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (TPR <= 64) {
    return group_sum<TPR>(v);
  } else {
    constexpr int NW = TPR / 64;
    v = group_sum<64>(v);
    __syncthreads();  // the previous sum's readers are done with `red`
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) s += red[i];
    return s;
  }
}

// TPR threads hold a row as NCH vectors of V elements each: C <= TPR * V * NCH, C % V == 0, rows V-aligned.
template <typename T, typename P, int V, int TPR, int NCH>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
layer_norm_kernel(const T* __restrict__ x, int64_t xs, const P* __restrict__ w, const P* __restrict__ b, T* __restrict__ y,
                  float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t M, int C, float eps) {
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;  // rows per block
  const int t = threadIdx.x % TPR;
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < M; base += (int64_t)gridDim.x * RPB) {
  const int64_t row0 = base + threadIdx.x / TPR;
  const bool live = row0 < M;
  const int64_t row = live ? row0 : M - 1;  // surplus rows repeat the last one and store nothing
  const T* xr = x + row * xs;
  float v[NCH][V];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (i * TPR + t) * V;
    if (c < C) load_vec<T, V>(xr + c, v[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (c >= C) v[i][j] = 0.f;
      s += v[i][j];
    }
  }
  const float mean = row_sum<TPR>(s, red) / C;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i)
    if ((i * TPR + t) * V < C)
#pragma unroll
      for (int j = 0; j < V; ++j) { const float d = v[i][j] - mean; q += d * d; }
  const float rstd = 1.f / sqrtf(row_sum<TPR>(q, red) / C + eps);
  if (!live) continue;
  T* yr = y + row * C;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (i * TPR + t) * V;
    if (c >= C) continue;
    float o[V], wv[V], bv[V];
    if (w) load_vec<P, V>(w + c, wv);
    if (b) load_vec<P, V>(b + c, bv);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      o[j] = (v[i][j] - mean) * rstd;
      if (w) o[j] *= wv[j];
      if (b) o[j] += bv[j];
    }
    store_vec<T, V>(yr + c, o);
  }
  if (t == 0) {
    if (mean_out) mean_out[row] = mean;
    if (rstd_out) rstd_out[row] = rstd;
  }
  }
}

// Rows too wide for registers: three walks over the row (it stays in the caches), one block per row.
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
layer_norm_wide_kernel(const T* __restrict__ x, int64_t xs, const P* __restrict__ w, const P* __restrict__ b, T* __restrict__ y,
                       float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t M, int C, float eps) {
  __shared__ float red[16];
  for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
  const T* xr = x + row * xs;
  float s = 0.f, q = 0.f;
  for (int c = threadIdx.x; c < C; c += 1024) s += (float)xr[c];
  const float mean = row_sum<1024>(s, red) / C;
  for (int c = threadIdx.x; c < C; c += 1024) { const float d = (float)xr[c] - mean; q += d * d; }
  const float rstd = 1.f / sqrtf(row_sum<1024>(q, red) / C + eps);
  for (int c = threadIdx.x; c < C; c += 1024) {
    float o = ((float)xr[c] - mean) * rstd;
    if (w) o *= (float)w[c];
    if (b) o += (float)b[c];
    y[row * C + c] = (T)o;
  }
  if (threadIdx.x == 0) {
    if (mean_out) mean_out[row] = mean;
    if (rstd_out) rstd_out[row] = rstd;
  }
  }
}

// dx, and the block's share of dw / db over the rows it walks (grid-stride): part[block][2][C].
template <typename T, typename P, int V, int TPR, int NCH>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
layer_norm_bwd_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs, const P* __restrict__ w,
                      const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, float* __restrict__ part,
                      int64_t M, int C) {
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  float aw[NCH][V], ab[NCH][V], wv[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (i * TPR + t) * V;
    if (w && c < C) load_vec<P, V>(w + c, wv[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      aw[i][j] = ab[i][j] = 0.f;
      if (!w || c >= C) wv[i][j] = 1.f;
    }
  }
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < M; base += (int64_t)gridDim.x * RPB) {
    const int64_t row0 = base + threadIdx.x / TPR;
    const bool live = row0 < M;
    const int64_t row = live ? row0 : M - 1;
    const float mu = mean[row], rs = rstd[row];
    float z[NCH][V], g[NCH][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (i * TPR + t) * V;
      if (c < C) {
        load_vec<T, V>(x + row * xs + c, z[i]);
        load_vec<T, V>(dy + row * dys + c, g[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          z[i][j] = (z[i][j] - mu) * rs;
          if (live) { aw[i][j] += g[i][j] * z[i][j]; ab[i][j] += g[i][j]; }
          g[i][j] *= wv[i][j];
          s1 += g[i][j];
          s2 += g[i][j] * z[i][j];
        }
      }
    }
    s1 = row_sum<TPR>(s1, red) / C;
    s2 = row_sum<TPR>(s2, red) / C;
    if (live)
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = (i * TPR + t) * V;
        if (c >= C) continue;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = rs * (g[i][j] - s1 - z[i][j] * s2);
        store_vec<T, V>(dx + row * C + c, o);
      }
  }
  if (!part) return;
  float* pw = part + (int64_t)blockIdx.x * 2 * C;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (i * TPR + t) * V;
      if (c >= C) continue;
#pragma unroll
      for (int j = 0; j < V; ++j) { pw[c + j] = aw[i][j]; pw[C + c + j] = ab[i][j]; }
    }
  } else {  // the block's row groups are added in order through LDS, one vector column at a time
    __shared__ float sum[2][RPB][TPR][V];
    const int r = threadIdx.x / TPR;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j) { sum[0][r][t][j] = aw[i][j]; sum[1][r][t][j] = ab[i][j]; }
      __syncthreads();
      for (int e = threadIdx.x; e < 2 * TPR * V; e += 256) {
        const int k = e / (TPR * V), o = e % (TPR * V), c = i * TPR * V + o;
        if (c >= C) continue;
        float v = 0.f;
        for (int q = 0; q < RPB; ++q) v += (&sum[k][q][0][0])[o];
        pw[(int64_t)k * C + c] = v;
      }
    }
  }
}

// Rows too wide for registers: dx alone (two walks over the row); dw / db by column_sums_kernel.
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
layer_norm_bwd_wide_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs, const P* __restrict__ w,
                           const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, int64_t M, int C) {
  __shared__ float red[16];
  for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
  const float mu = mean[row], rs = rstd[row];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < C; c += 1024) {
    const float g = (float)dy[row * dys + c] * (w ? (float)w[c] : 1.f), z = ((float)x[row * xs + c] - mu) * rs;
    s1 += g;
    s2 += g * z;
  }
  s1 = row_sum<1024>(s1, red) / C;
  s2 = row_sum<1024>(s2, red) / C;
  for (int c = threadIdx.x; c < C; c += 1024) {
    const float g = (float)dy[row * dys + c] * (w ? (float)w[c] : 1.f), z = ((float)x[row * xs + c] - mu) * rs;
    dx[row * C + c] = (T)(rs * (g - s1 - z * s2));
  }
  }
}
template <typename T>
__global__ void __launch_bounds__(256)
layer_norm_bwd_wide_params_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
                                  const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part, int64_t M, int C) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float aw = 0.f, ab = 0.f;
  for (int64_t row = blockIdx.y; row < M; row += gridDim.y) {
    const float g = (float)dy[row * dys + c];
    aw += g * ((float)x[row * xs + c] - mean[row]) * rstd[row];
    ab += g;
  }
  float* pw = part + (int64_t)blockIdx.y * 2 * C;
  pw[c] = aw;
  pw[C + c] = ab;
}

constexpr int NORM_BWD_BLOCKS = 1024;
constexpr int64_t NORM_MAX_BLOCKS = 1 << 20;  // further rows are walked by the same blocks (a launch holds fewer than 2^32 threads)
inline unsigned norm_grid(int64_t n) { return (unsigned)(n < NORM_MAX_BLOCKS ? n : NORM_MAX_BLOCKS); }

struct NormShape { int V, TPR, NCH; };

// Vectors of 16 bytes where the width and every row allow it, else single elements.  A wave per row (a quarter of one for narrow rows)
// while the row fits `most` vectors per lane, else a block of 256 or 1024 threads; {0,0,0}: the row does not fit registers.
inline NormShape norm_shape(int C, int full, bool vec, int most, bool few_rows) {
  NormShape s = {0, 0, 0};
  s.V = vec ? full : 1;
  const int64_t n = (C + s.V - 1) / s.V;  // vectors per row
  auto up = [](int64_t v) { int p = 1; while (p < v) p *= 2; return p; };
  if (n <= 16) { s.TPR = 16; s.NCH = 1; return s; }
  if (n <= 64 * (few_rows ? 1 : most)) { s.TPR = 64; s.NCH = up((n + 63) / 64); return s; }
  if (n <= 256 * most) { s.TPR = 256; s.NCH = up((n + 255) / 256); return s; }
  if (n <= 1024 * most) { s.TPR = 1024; s.NCH = up((n + 1023) / 1024); return s; }
  s.TPR = 0;
  return s;
}

template <typename T, typename P, int V, typename F>
int norm_dispatch(const NormShape& s, F&& f) {
#define DM_NORM_CASE(tpr, nch) \
  if (s.TPR == tpr && s.NCH == nch) return f(std::integral_constant<int, tpr>{}, std::integral_constant<int, nch>{});
  DM_NORM_CASE(16, 1) DM_NORM_CASE(64, 1) DM_NORM_CASE(64, 2) DM_NORM_CASE(64, 4) DM_NORM_CASE(256, 1) DM_NORM_CASE(256, 2)
  DM_NORM_CASE(256, 4) DM_NORM_CASE(1024, 2) DM_NORM_CASE(1024, 4)
#undef DM_NORM_CASE
  return fail("layer norm: no kernel for %d threads x %d vectors", s.TPR, s.NCH);
}

template <typename T, typename P, int V>
int norm_fwd_run(const NormShape& s, const T* x, int64_t xs, const P* w, const P* b, T* y, float* mean, float* rstd, int64_t M, int C,
                 float eps, hipStream_t st) {
  return norm_dispatch<T, P, V>(s, [&](auto tpr, auto nch) {
    constexpr int TPR = decltype(tpr)::value, NCH = decltype(nch)::value, RPB = TPR < 256 ? 256 / TPR : 1;
    layer_norm_kernel<T, P, V, TPR, NCH><<<dim3(norm_grid((M + RPB - 1) / RPB)), dim3(TPR < 256 ? 256 : TPR), 0, st>>>(
        x, xs, w, b, y, mean, rstd, M, C, eps);
    return launched("dm_layer_norm");
  });
}

template <typename T, typename P>
int norm_fwd(const void* x, int64_t xs, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t M, int C, float eps,
             hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = C % V == 0 && xs % V == 0 && aligned(x, 16) && aligned(y, 16) && (!w || aligned(w, V * sizeof(P))) &&
                   (!b || aligned(b, V * sizeof(P)));
  const NormShape s = norm_shape(C, V, vec, 4, M < 1024);
  if (!s.TPR) {
    layer_norm_wide_kernel<T, P><<<dim3(norm_grid(M)), dim3(1024), 0, st>>>((const T*)x, xs, (const P*)w, (const P*)b, (T*)y, mean, rstd, M, C, eps);
    return launched("dm_layer_norm");
  }
  return s.V == V ? norm_fwd_run<T, P, V>(s, (const T*)x, xs, (const P*)w, (const P*)b, (T*)y, mean, rstd, M, C, eps, st)
                  : norm_fwd_run<T, P, 1>(s, (const T*)x, xs, (const P*)w, (const P*)b, (T*)y, mean, rstd, M, C, eps, st);
}

template <typename T, typename P, int V>
int norm_bwd_run(const NormShape& s, const T* dy, int64_t dys, const T* x, int64_t xs, const P* w, const float* mean, const float* rstd,
                 T* dx, P* dw, P* db, float* part, int64_t M, int C, hipStream_t st) {
  const bool params = dw || db;
  int blocks = 0;
  const int rc = norm_dispatch<T, P, V>(s, [&](auto tpr, auto nch) {
    constexpr int TPR = decltype(tpr)::value, NCH = decltype(nch)::value, RPB = TPR < 256 ? 256 / TPR : 1;
    const int64_t need = (M + RPB - 1) / RPB;
    blocks = (int)(need < NORM_BWD_BLOCKS ? need : NORM_BWD_BLOCKS);
    layer_norm_bwd_kernel<T, P, V, TPR, NCH><<<dim3(blocks), dim3(TPR < 256 ? 256 : TPR), 0, st>>>(
        dy, dys, x, xs, w, mean, rstd, dx, params ? part : nullptr, M, C);
    return launched("dm_layer_norm_backward");
  });
  if (rc || !params) return rc;
  partial_rows_kernel<P><<<dim3((unsigned)((2 * (int64_t)C + 15) / 16)), dim3(256), 0, st>>>(part, blocks, C, dw, db);
  return launched("dm_layer_norm_backward");
}

template <typename T, typename P>
int norm_bwd(const void* dy, int64_t dys, const void* x, int64_t xs, const void* w, const float* mean, const float* rstd, void* dx,
             void* dw, void* db, float* part, int64_t M, int C, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = C % V == 0 && xs % V == 0 && dys % V == 0 && aligned(x, 16) && aligned(dy, 16) && aligned(dx, 16) &&
                   (!w || aligned(w, V * sizeof(P)));
  const NormShape s = norm_shape(C, V, vec, 4, false);
  if (!s.TPR) {
    layer_norm_bwd_wide_kernel<T, P><<<dim3(norm_grid(M)), dim3(1024), 0, st>>>((const T*)dy, dys, (const T*)x, xs, (const P*)w, mean, rstd,
                                                                              (T*)dx, M, C);
    int rc = launched("dm_layer_norm_backward");
    if (rc || !(dw || db)) return rc;
    const int rows = (int)(M < 64 ? M : 64);
    layer_norm_bwd_wide_params_kernel<T><<<dim3((unsigned)((C + 255) / 256), rows), dim3(256), 0, st>>>((const T*)dy, dys, (const T*)x, xs, mean,
                                                                                             rstd, part, M, C);
    if ((rc = launched("dm_layer_norm_backward"))) return rc;
    partial_rows_kernel<P><<<dim3((unsigned)((2 * (int64_t)C + 15) / 16)), dim3(256), 0, st>>>(part, rows, C, (P*)dw, (P*)db);
    return launched("dm_layer_norm_backward");
  }
  return s.V == V ? norm_bwd_run<T, P, V>(s, (const T*)dy, dys, (const T*)x, xs, (const P*)w, mean, rstd, (T*)dx, (P*)dw, (P*)db, part, M, C, st)
                  : norm_bwd_run<T, P, 1>(s, (const T*)dy, dys, (const T*)x, xs, (const P*)w, mean, rstd, (T*)dx, (P*)dw, (P*)db, part, M, C, st);
}

template <typename P>
__global__ void fill_zero_kernel(P* a, P* b, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  if (a) a[i] = (P)0.f;
  if (b) b[i] = (P)0.f;
}

inline int norm_check(const char* who, int64_t M, int C, int dtype, int param_dtype) {
  if (!dtype_ok(dtype)) return fail("%s: unknown dtype %d", who, dtype);
  if (param_dtype != dtype && param_dtype != DM_F32) return fail("%s: the parameters are of the input's type or fp32", who);
  if (M < 0 || M > 0x7fffffffLL) return fail("%s: %lld rows", who, (long long)M);
  if (C < 1 || C > (1 << 24)) return fail("%s: width %d (1 to 2^24)", who, C);
  return 0;
}

#define DM_NORM_TYPES(call)                                                        \
  switch (dtype) {                                                                 \
    case DM_F32: return call(float, float);                                        \
    case DM_BF16: return param_dtype == DM_F32 ? call(bf16, float) : call(bf16, bf16); \
    default: return param_dtype == DM_F32 ? call(f16, float) : call(f16, f16);     \
  }

}  // namespace dmb

extern "C" {

int dm_layer_norm(const void* x_dev, int64_t x_stride, const void* weight_dev, const void* bias_dev, int param_dtype, void* y_dev,
                  float* mean_dev, float* rstd_dev, int64_t M, int C, float eps, int dtype, void* stream) {
  using namespace dmb;
  if (const int rc = norm_check("dm_layer_norm", M, C, dtype, param_dtype)) return rc;
  if (M == 0) return 0;
  if (!x_dev || !y_dev) return fail("dm_layer_norm: null argument");
  if (x_stride < C && M > 1) return fail("dm_layer_norm: row stride %lld below the width %d", (long long)x_stride, C);
  if (!(eps >= 0.f)) return fail("dm_layer_norm: eps must not be negative");
  const hipStream_t st = (hipStream_t)stream;
#define DM_CALL(T, P) norm_fwd<T, P>(x_dev, x_stride, weight_dev, bias_dev, y_dev, mean_dev, rstd_dev, M, C, eps, st)
  DM_NORM_TYPES(DM_CALL)
#undef DM_CALL
}

size_t dm_layer_norm_backward_workspace_bytes(int64_t M, int C) {
  if (M <= 0 || C < 1) return 0;
  return (size_t)(M < dmb::NORM_BWD_BLOCKS ? M : dmb::NORM_BWD_BLOCKS) * 2 * (size_t)C * sizeof(float);
}

int dm_layer_norm_backward(const void* dy_dev, int64_t dy_stride, const void* x_dev, int64_t x_stride, const void* weight_dev,
                           int param_dtype, const float* mean_dev, const float* rstd_dev, void* dx_dev, void* dweight_dev, void* dbias_dev,
                           int64_t M, int C, int dtype, void* workspace_dev, size_t workspace_bytes, void* stream) {
  using namespace dmb;
  if (const int rc = norm_check("dm_layer_norm_backward", M, C, dtype, param_dtype)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (M == 0) {  // no rows: the parameters' gradients are zero
    if (!dweight_dev && !dbias_dev) return 0;
    const dim3 grid((C + 255) / 256);
    if (param_dtype == DM_F32) fill_zero_kernel<float><<<grid, dim3(256), 0, st>>>((float*)dweight_dev, (float*)dbias_dev, C);
    else fill_zero_kernel<uint16_t><<<grid, dim3(256), 0, st>>>((uint16_t*)dweight_dev, (uint16_t*)dbias_dev, C);
    return launched("dm_layer_norm_backward");
  }
  if (!dy_dev || !x_dev || !mean_dev || !rstd_dev || !dx_dev) return fail("dm_layer_norm_backward: null argument");
  if (M > 1 && (dy_stride < C || x_stride < C)) return fail("dm_layer_norm_backward: row stride below the width %d", C);
  if ((dweight_dev || dbias_dev) && (!workspace_dev || workspace_bytes < dm_layer_norm_backward_workspace_bytes(M, C)))
    return fail("dm_layer_norm_backward: workspace of %zu bytes, %zu needed", workspace_dev ? workspace_bytes : (size_t)0,
                dm_layer_norm_backward_workspace_bytes(M, C));
#define DM_CALL(T, P) norm_bwd<T, P>(dy_dev, dy_stride, x_dev, x_stride, weight_dev, mean_dev, rstd_dev, dx_dev, dweight_dev, dbias_dev, \
                                     (float*)workspace_dev, M, C, st)
  DM_NORM_TYPES(DM_CALL)
#undef DM_CALL
}

}  // extern "C"
