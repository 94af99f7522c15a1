// dm_block_norm.hip — layer norm and its backward pass.
//   z = (x - mean) rstd, y = z w + b;  gz = dy w, dx = rstd (gz - mean(gz) - z mean(gz z)), dw = sum dy z, db = sum dy.
// Both are bound by memory: a row is read once into registers, its mean and centred sum of squares (two sums over the
// registers, no cancellation) follow from there, and the result is written once.  All sums are fp32.  The parameters'
// gradients are summed per workgroup over the rows it walks, written as partial rows and added in a fixed order by a second
// launch: no atomics, the same bits every time.
// Measured, tensors' bytes per time (a large copy: 4.7 TB/s, what the caches hold faster): forward 262144 x 256 fp32 100 us (5.4 TB/s),
// forward and backward 32768 x 4096 bf16 287 us (4.7), backward 8192 x 8192 bf16 92 us (4.4), 4096 x 8191 bf16 46 us (4.4).
#include <type_traits>

#include "dm_block_common.h"

namespace dmb {

// Two sums over the TPR threads of a row: within a wave by shuffles, across the waves of a block through `red`, whose halves are used in
// turn (`half`): one barrier, behind which nobody still reads the half that is written next.
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float (*red)[2][TPR > 64 ? TPR / 64 : 1], int& half) {
  constexpr int W = TPR < 64 ? TPR : 64;
  a = group_sum<W>(a);
  b = group_sum<W>(b);
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    if ((threadIdx.x & 63) == 0) { red[half][0][threadIdx.x >> 6] = a; red[half][1][threadIdx.x >> 6] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) { a += red[half][0][i]; b += red[half][1][i]; }
    half ^= 1;
  }
}
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float (*red)[2][TPR > 64 ? TPR / 64 : 1], int& half) {
  float none = 0.f;
  row_sums<TPR>(v, none, red, half);
  return v;
}

// The Piece of a row that a thread holds from column c on.  WHOLE (C a multiple of V): the piece lies inside the row or behind it.  Else the
// last piece is moved back to end with the row: its first `skip` elements are a neighbour's too, which counts them in sums over the row;
// both write the same values.  Behind the row all of it is skipped.
template <int V, bool WHOLE>
struct Place {
  int at, skip;
  bool in;
  __device__ __forceinline__ Place(int c, int C) : at(WHOLE || c + V <= C ? c : C - V), skip(WHOLE ? 0 : c - at), in(c < C) {}
  template <typename T>
  __device__ __forceinline__ void load(const T* row, Piece<T, V>& r) const {
    if (!WHOLE || in) {
      r = *reinterpret_cast<const Piece<T, V>*>(row + at);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) r.v[j] = (T)0.f;
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&v)[V]) const {
    Piece<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = (T)v[j];
    *reinterpret_cast<Piece<T, V>*>(row + at) = r;
  }
  __device__ __forceinline__ bool counts(int j) const { return WHOLE ? in : j >= skip; }
};

// TPR threads hold a row as NCH pieces each: C <= TPR * V * NCH.
template <typename T, typename P, bool WHOLE, int TPR, int NCH>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
layer_norm_kernel(const T* __restrict__ x, int64_t xs, const P* __restrict__ w, const P* __restrict__ b, T* __restrict__ y,
                  float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t M, int C, float eps) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float red[2][2][TPR > 64 ? TPR / 64 : 1];
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;  // rows per block
  const int t = threadIdx.x % TPR;
  int half = 0;
  for (int64_t base = (int64_t)blockIdx.x * RPB; base < M; base += (int64_t)gridDim.x * RPB) {
    const int64_t row0 = base + threadIdx.x / TPR;
    const bool live = row0 < M;
    const int64_t row = live ? row0 : M - 1;  // surplus rows repeat the last one and store nothing
    const T* xr = x + row * xs;
    float v[NCH][V];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Place<V, WHOLE> at((i * TPR + t) * V, C);
      Piece<T, V> r;
      at.load(xr, r);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[i][j] = (float)r.v[j];
        s += WHOLE || at.counts(j) ? v[i][j] : 0.f;
      }
    }
    const float mean = row_sum<TPR>(s, red, half) / C;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Place<V, WHOLE> at((i * TPR + t) * V, C);
      if (at.in)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float d = v[i][j] - mean;
          q += at.counts(j) ? d * d : 0.f;
        }
    }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(q, red, half) / C + eps);
    if (!live) continue;
    T* yr = y + row * C;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Place<V, WHOLE> at((i * TPR + t) * V, C);
      if (!at.in) continue;
      float o[V];
      Piece<P, V> wv, bv;
      if (w) at.load(w, wv);
      if (b) at.load(b, bv);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        o[j] = (v[i][j] - mean) * rstd;
        if (w) o[j] *= (float)wv.v[j];
        if (b) o[j] += (float)bv.v[j];
      }
      at.store(yr, o);
    }
    if (t == 0) {
      if (mean_out) mean_out[row] = mean;
      if (rstd_out) rstd_out[row] = rstd;
    }
  }
}

// Rows too wide for registers (or narrower than a vector: V = 1): three walks over the row (it stays in the caches), one block per row.
template <typename T, typename P, int V>
__global__ void __launch_bounds__(1024)
layer_norm_wide_kernel(const T* __restrict__ x, int64_t xs, const P* __restrict__ w, const P* __restrict__ b, T* __restrict__ y,
                       float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t M, int C, float eps) {
  __shared__ float red[2][2][16];
  int half = 0;
  for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
    const T* xr = x + row * xs;
    float s = 0.f, q = 0.f;
#pragma unroll 4
    for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
      const Place<V, false> at(c, C);
      Piece<T, V> v;
      at.load(xr, v);
#pragma unroll
      for (int j = 0; j < V; ++j) s += at.counts(j) ? (float)v.v[j] : 0.f;
    }
    const float mean = row_sum<1024>(s, red, half) / C;
#pragma unroll 4
    for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
      const Place<V, false> at(c, C);
      Piece<T, V> v;
      at.load(xr, v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = (float)v.v[j] - mean;
        q += at.counts(j) ? d * d : 0.f;
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<1024>(q, red, half) / C + eps);
#pragma unroll 2
    for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
      const Place<V, false> at(c, C);
      Piece<T, V> v;
      Piece<P, V> wv, bv;
      at.load(xr, v);
      if (w) at.load(w, wv);
      if (b) at.load(b, bv);
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        o[j] = ((float)v.v[j] - mean) * rstd;
        if (w) o[j] *= (float)wv.v[j];
        if (b) o[j] += (float)bv.v[j];
      }
      at.store(y + row * C, o);
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[row] = mean;
      if (rstd_out) rstd_out[row] = rstd;
    }
  }
}

// dx, and the block's share of dw / db over the rows it walks (grid-stride): part[block][2][C].  The next row's loads are under way while a
// row is summed; rows stay in their own type in registers, so that the two rows and the two running sums of every column fit.
// (Pieces are moved back at the end of every row: with a branch around each load, 8192 x 8192 bf16 take 151 us instead of 92.)
template <typename T, typename P, int TPR, int NCH>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
layer_norm_bwd_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs, const P* __restrict__ w,
                      const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, float* __restrict__ part,
                      int64_t M, int C) {
  constexpr int V = 16 / sizeof(T), RPB = TPR < 256 ? 256 / TPR : 1;
  constexpr bool AHEAD = NCH * V <= 16;  // (32 pairs of sums leave no registers for a second row)
  __shared__ float red[2][2][TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  int half = 0;
  float aw[NCH][V], ab[NCH][V];
  Piece<P, V> wv[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const Place<V, false> at((i * TPR + t) * V, C);
    if (w) at.load(w, wv[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      aw[i][j] = ab[i][j] = 0.f;
      if (!w) wv[i].v[j] = (P)1.f;
    }
  }
  struct Row { Piece<T, V> x[NCH], g[NCH]; float mu, rs; } cur, next;
  auto load = [&](Row& r, int64_t base) __attribute__((always_inline)) {
    int64_t row = base + threadIdx.x / TPR;
    if (row >= M) row = M - 1;
    r.mu = mean[row];
    r.rs = rstd[row];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Place<V, false> at((i * TPR + t) * V, C);
      at.load(x + row * xs, r.x[i]);
      at.load(dy + row * dys, r.g[i]);
    }
  };
  const int64_t first = (int64_t)blockIdx.x * RPB, stride = (int64_t)gridDim.x * RPB;
  load(cur, first);
  for (int64_t base = first; base < M; base += stride) {
    if (AHEAD) load(next, base + stride < M ? base + stride : base);
    const int64_t row = base + threadIdx.x / TPR;
    const bool live = row < M;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Place<V, false> at((i * TPR + t) * V, C);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float z = ((float)cur.x[i].v[j] - cur.mu) * cur.rs, d = (float)cur.g[i].v[j];
        if (live) { aw[i][j] += d * z; ab[i][j] += d; }
        const float g = at.counts(j) ? d * (float)wv[i].v[j] : 0.f;
        s1 += g;
        s2 += at.counts(j) ? g * z : 0.f;
      }
    }
    row_sums<TPR>(s1, s2, red, half);
    s1 /= C;
    s2 /= C;
    if (live)
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const Place<V, false> at((i * TPR + t) * V, C);
        if (!at.in) continue;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float z = ((float)cur.x[i].v[j] - cur.mu) * cur.rs, g = (float)cur.g[i].v[j] * (float)wv[i].v[j];
          o[j] = cur.rs * (g - s1 - z * s2);
        }
        at.store(dx + row * C, o);
      }
    if (AHEAD) cur = next;
    else load(cur, base + stride < M ? base + stride : base);
  }
  if (!part) return;
  float* pw = part + (int64_t)blockIdx.x * 2 * C;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Place<V, false> at((i * TPR + t) * V, C);
      if (!at.in) continue;
      at.store(pw, aw[i]);
      at.store(pw + C, ab[i]);
    }
  } else {  // the block's row groups are added in order through LDS, one piece column at a time
    __shared__ float sum[2][RPB][TPR][V];
    const int r = threadIdx.x / TPR;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Place<V, false> at((i * TPR + t) * V, C);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at.counts(j)) { sum[0][r][t][j - at.skip] = aw[i][j]; sum[1][r][t][j - at.skip] = ab[i][j]; }
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

// Rows too wide for registers (or narrower than a vector: V = 1): dx alone (two walks over the row), and the parameters' gradients by
// columns.
template <typename T, typename P, int V>
__global__ void __launch_bounds__(1024)
layer_norm_bwd_wide_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs, const P* __restrict__ w,
                           const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, int64_t M, int C) {
  __shared__ float red[2][2][16];
  int half = 0;
  for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    auto piece = [&](const Place<V, false>& at, float (&z)[V], float (&g)[V]) __attribute__((always_inline)) {
      Piece<T, V> xv, dv;
      Piece<P, V> wv;
      at.load(x + row * xs, xv);
      at.load(dy + row * dys, dv);
      if (w) at.load(w, wv);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        z[j] = ((float)xv.v[j] - mu) * rs;
        g[j] = w ? (float)dv.v[j] * (float)wv.v[j] : (float)dv.v[j];
      }
    };
#pragma unroll 2
    for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
      const Place<V, false> at(c, C);
      float z[V], g[V];
      piece(at, z, g);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at.counts(j)) { s1 += g[j]; s2 += g[j] * z[j]; }
    }
    row_sums<1024>(s1, s2, red, half);
    s1 /= C;
    s2 /= C;
#pragma unroll 2
    for (int c = threadIdx.x * V; c < C; c += 1024 * V) {
      const Place<V, false> at(c, C);
      float z[V], g[V];
      piece(at, z, g);
#pragma unroll
      for (int j = 0; j < V; ++j) z[j] = rs * (g[j] - s1 - z[j] * s2);
      at.store(dx + row * C, z);
    }
  }
}
template <typename T, int V>
__global__ void __launch_bounds__(256)
layer_norm_bwd_wide_params_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
                                  const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part, int64_t M, int C) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * V;
  if (c >= C) return;
  const Place<V, false> at(c, C);
  float aw[V] = {}, ab[V] = {};
#pragma unroll 4
  for (int64_t row = blockIdx.y; row < M; row += gridDim.y) {
    Piece<T, V> xv, dv;
    at.load(x + row * xs, xv);
    at.load(dy + row * dys, dv);
    const float mu = mean[row], rs = rstd[row];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float g = (float)dv.v[j];
      aw[j] += g * (((float)xv.v[j] - mu) * rs);
      ab[j] += g;
    }
  }
  float* pw = part + (int64_t)blockIdx.y * 2 * C;
  at.store(pw, aw);
  at.store(pw + C, ab);
}

// Blocks of the backward pass: four to a CU, but sixteen rows each where that leaves one to a CU, as each writes a row of sums for the
// second launch to read (4096 x 16384 bf16: 1024 blocks' sums are two thirds of the tensors' bytes).
inline int norm_bwd_blocks(int64_t M) { return (int)(M < 256 ? M : M < 256 * 16 ? 256 : M < 1024 * 16 ? M / 16 : 1024); }
constexpr int64_t NORM_MAX_BLOCKS = 1 << 20;  // further rows are walked by the same blocks (a launch holds fewer than 2^32 threads)
inline unsigned norm_grid(int64_t n) { return (unsigned)(n < NORM_MAX_BLOCKS ? n : NORM_MAX_BLOCKS); }

struct NormShape { int TPR, NCH; };

// A wave per row (a quarter of one for narrow rows) while the row fits `most` pieces per lane, else a block of 256, else a block of `wide`
// threads with up to 32 elements each; {0, 0}: the row does not fit registers, or is no whole piece.
inline NormShape norm_shape(int C, int V, int most, int wide) {
  const int64_t n = (C + V - 1) / V;  // pieces per row
  auto up = [](int64_t v) { int p = 1; while (p < v) p *= 2; return p; };
  if (C < V) return {0, 0};
  if (n <= 16) return {16, 1};
  if (n <= 64 * most) return {64, up((n + 63) / 64)};
  if (n <= 256 * most) return {256, up((n + 255) / 256)};
  if (C <= 32 * wide) return {wide, up((n + wide - 1) / wide)};
  return {0, 0};
}

// f(TPR, NCH) of the shape (one of those that norm_shape gives in that direction)
template <int V, bool FORWARD, typename F>
int norm_dispatch(const NormShape& s, F&& f) {
#define DM_NORM_CASE(tpr, nch)                                                                                                  \
  if constexpr (FORWARD ? nch * V <= 32 && tpr != 512 : nch * V <= (tpr == 512 ? 32 : 16) && (tpr != 512 || nch * V > 8) && tpr != 1024) \
    if (s.TPR == tpr && s.NCH == nch) return f(std::integral_constant<int, tpr>{}, std::integral_constant<int, nch>{});
  DM_NORM_CASE(16, 1) DM_NORM_CASE(64, 1) DM_NORM_CASE(64, 2) DM_NORM_CASE(64, 4) DM_NORM_CASE(256, 1) DM_NORM_CASE(256, 2)
  DM_NORM_CASE(256, 4) DM_NORM_CASE(512, 2) DM_NORM_CASE(512, 4) DM_NORM_CASE(512, 8) DM_NORM_CASE(1024, 1) DM_NORM_CASE(1024, 2)
  DM_NORM_CASE(1024, 4) DM_NORM_CASE(1024, 8)
#undef DM_NORM_CASE
  return fail("layer norm: no kernel for %d threads x %d pieces", s.TPR, s.NCH);
}

template <typename T, typename P>
int norm_fwd(const void* xp, int64_t xs, const void* wp, const void* bp, void* yp, float* mean, float* rstd, int64_t M, int C, float eps,
             hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const T* x = (const T*)xp;
  const P *w = (const P*)wp, *b = (const P*)bp;
  T* y = (T*)yp;
  const NormShape s = norm_shape(C, V, M < 1024 ? 1 : 4, 1024);  // (few rows: as many threads as there can be)
  if (!s.TPR) {
    const dim3 grid(norm_grid(M)), block(1024);
    if (C < V) layer_norm_wide_kernel<T, P, 1><<<grid, block, 0, st>>>(x, xs, w, b, y, mean, rstd, M, C, eps);
    else layer_norm_wide_kernel<T, P, V><<<grid, block, 0, st>>>(x, xs, w, b, y, mean, rstd, M, C, eps);
    return launched("dm_layer_norm");
  }
  return norm_dispatch<V, true>(s, [&](auto tpr, auto nch) {
    constexpr int TPR = decltype(tpr)::value, NCH = decltype(nch)::value, RPB = TPR < 256 ? 256 / TPR : 1;
    const dim3 grid(norm_grid((M + RPB - 1) / RPB)), block(TPR < 256 ? 256 : TPR);
    if (C % V == 0) layer_norm_kernel<T, P, true, TPR, NCH><<<grid, block, 0, st>>>(x, xs, w, b, y, mean, rstd, M, C, eps);
    else layer_norm_kernel<T, P, false, TPR, NCH><<<grid, block, 0, st>>>(x, xs, w, b, y, mean, rstd, M, C, eps);
    return launched("dm_layer_norm");
  });
}

template <typename T, typename P>
int norm_bwd(const void* dyp, int64_t dys, const void* xp, int64_t xs, const void* wp, const float* mean, const float* rstd, void* dxp,
             void* dwp, void* dbp, float* part, int64_t M, int C, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const T *dy = (const T*)dyp, *x = (const T*)xp;
  const P* w = (const P*)wp;
  T* dx = (T*)dxp;
  P *dw = (P*)dwp, *db = (P*)dbp;
  const bool params = dw || db;
  const NormShape s = norm_shape(C, V, 16 / V, 512);
  int rc, rows = 0;  // of `part`
  if (!s.TPR) {
    const dim3 grid(norm_grid(M)), block(1024);
    if (C < V) layer_norm_bwd_wide_kernel<T, P, 1><<<grid, block, 0, st>>>(dy, dys, x, xs, w, mean, rstd, dx, M, C);
    else layer_norm_bwd_wide_kernel<T, P, V><<<grid, block, 0, st>>>(dy, dys, x, xs, w, mean, rstd, dx, M, C);
    rc = launched("dm_layer_norm_backward");
    if (rc || !params) return rc;
    rows = (int)(M < 256 ? M : 256);
    if (C < V) layer_norm_bwd_wide_params_kernel<T, 1><<<dim3(1, rows), dim3(256), 0, st>>>(dy, dys, x, xs, mean, rstd, part, M, C);
    else layer_norm_bwd_wide_params_kernel<T, V><<<dim3((C + 256 * V - 1) / (256 * V), rows), dim3(256), 0, st>>>(dy, dys, x, xs, mean, rstd, part, M, C);
    rc = launched("dm_layer_norm_backward");
  } else {
    rc = norm_dispatch<V, false>(s, [&](auto tpr, auto nch) {
      constexpr int TPR = decltype(tpr)::value, NCH = decltype(nch)::value, RPB = TPR < 256 ? 256 / TPR : 1;
      const int64_t need = (M + RPB - 1) / RPB;
      rows = (int)(need < norm_bwd_blocks(M) ? need : norm_bwd_blocks(M));
      layer_norm_bwd_kernel<T, P, TPR, NCH><<<dim3(rows), dim3(TPR < 256 ? 256 : TPR), 0, st>>>(dy, dys, x, xs, w, mean, rstd, dx,
                                                                                              params ? part : nullptr, M, C);
      return launched("dm_layer_norm_backward");
    });
  }
  if (rc || !params) return rc;
  partial_rows_kernel<P><<<dim3((unsigned)((2 * (int64_t)C + 15) / 16)), dim3(256), 0, st>>>(part, rows, C, dw, db);
  return launched("dm_layer_norm_backward");
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
  return (size_t)dmb::norm_bwd_blocks(M) * 2 * (size_t)C * sizeof(float);
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
