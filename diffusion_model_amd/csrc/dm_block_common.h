// dm_block_common.h — what the transformer-block operators (layer norm, rotary positions, gated feed-forward block) share:
// element types, vectors of 16 bytes, wave sums, error reporting.  Each is a translation unit of its own,
// compiled without packed fp32 instructions.
#ifndef DM_BLOCK_COMMON_H
#define DM_BLOCK_COMMON_H

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/dm_sampler.h"

// dm_api.hip: stores the message that dm_last_error() returns; always 1.
__attribute__((visibility("hidden"))) int dm_set_error(const char* msg);

namespace dmb {

inline int fail(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return dm_set_error(buf);
}

inline int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("%s: launch failed: %s", what, hipGetErrorString(e));
}

typedef __bf16 bf16;
typedef _Float16 f16;

inline int dtype_size(int dtype) { return dtype == DM_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == DM_F32 || dtype == DM_BF16 || dtype == DM_F16; }
inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// N elements moved by one load or store
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec { T v[N]; };

// ... at any element boundary: the hardware takes such vectors (layer norm of bf16, 16384 rows of odd width 1001: 16 us against 39 us element
// by element)
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Piece { T v[N]; };

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[N]) {
  const Vec<T, N> r = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = (float)r.v[i];
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[N]) {
  Vec<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = (T)in[i];  // round to nearest even
  *reinterpret_cast<Vec<T, N>*>(p) = r;
}

// sum over the W consecutive lanes (W a power of two, <= 64) that hold one row; every lane gets it
template <int W>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = W / 2; o; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

namespace {  // (a kernel of each translation unit's own)
// out_k[c] = sum over n partial rows of part[i][k][c], k < 2, in a fixed order: 16 columns x 16 interleaved row groups per block.
template <typename P>
__global__ void __launch_bounds__(256)
partial_rows_kernel(const float* __restrict__ part, int n, int C, P* __restrict__ out0, P* __restrict__ out1) {
  __shared__ float sum[16][17];
  const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int64_t e = (int64_t)blockIdx.x * 16 + col;
  float s = 0.f;
  if (e < 2 * (int64_t)C)
#pragma unroll 8
    for (int i = grp; i < n; i += 16) s += part[(int64_t)i * 2 * C + e];
  sum[grp][col] = s;
  __syncthreads();
  if (grp == 0 && e < 2 * (int64_t)C) {
    float v = 0.f;
    for (int q = 0; q < 16; ++q) v += sum[q][col];
    P* o = e < C ? out0 : out1;
    if (o) o[e < C ? e : e - C] = (P)v;
  }
}
}  // namespace

}  // namespace dmb
#endif
