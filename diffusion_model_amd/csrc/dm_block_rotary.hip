// dm_block_rotary.hip — rotary positions on query and key heads, in one launch.
//   pair i of a token's head turns by phi = position[axis(i)] * inv_freq[i]:  (a, b) -> s (a cos phi - b sin phi, a sin phi + b cos phi).
// The angle is formed in 64 bits as a number of turns (three roundings: off by 2^-51 of itself, 4e-10 at position 10^6) and reduced to an eighth of
// a turn exactly;
// sine and cosine of the rest are the Taylor polynomials on [-pi/4, pi/4] (next term < 2^-33) in 32 bits.  Bound by memory: a
// thread forms the angles of its V pairs of one token once and walks `hpt` heads with them.  Measured: 4 x 8192 tokens, 32 + 8 heads of 128,
// bf16 155 us (4.3 TB/s of what is read and written); 256 x 256 tokens, 4 + 4 heads of 64, fp32 57 us (4.7 TB/s; the kernel alone 47); a large copy 4.7 TB/s.
#include "dm_block_common.h"

namespace dmb {

struct RotaryArgs {
  const void* in[2];
  void* out[2];
  int64_t is[2][3], os[2][3];  // strides of (image, token, head) in elements
  int heads[2];
  const int64_t* pos;
  int64_t ps[3];               // strides of (axis, image, token)
  const double* inv_freq;
  int64_t tokens, work;        // B * T; threads that have something to do
  int T, D, pairs, per_axis, units, hpt, groups, half;
  float scale;
  int inverse;
};

__device__ __forceinline__ void sincos_turns(double turns, float& s, float& c) {
  const double q = rint(turns * 4.0);                       // quarter turns
  const float y = (float)(turns - q * 0.25) * 6.2831853071795865f;
  const int k = (int)(long long)(q - 4.0 * floor(q * 0.25));  // 0..3
  const float y2 = y * y;
  float ps = -2.5052108e-8f, pc = -2.7557319e-7f;           // 1/11!, 1/10!, and so on down
  ps = fmaf(ps, y2, 2.7557319e-6f);
  ps = fmaf(ps, y2, -1.9841270e-4f);
  ps = fmaf(ps, y2, 8.3333333e-3f);
  ps = fmaf(ps, y2, -1.6666667e-1f);
  ps = fmaf(ps * y2, y, y);
  pc = fmaf(pc, y2, 2.4801587e-5f);
  pc = fmaf(pc, y2, -1.3888889e-3f);
  pc = fmaf(pc, y2, 4.1666667e-2f);
  pc = fmaf(pc, y2, -0.5f);
  pc = fmaf(pc, y2, 1.0f);
  const float a = (k & 1) ? pc : ps, b = (k & 1) ? ps : pc;
  s = (k & 2) ? -a : a;
  c = (k == 1 || k == 2) ? -b : b;
}

// A unit is 2V elements of a head: V pairs (two vectors of one element type's V), or 2V elements behind the rotated part.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < a.work; id += (int64_t)gridDim.x * 256) {
  const int u = (int)(id % a.units);
  const int64_t rest = id / a.units;
  const int grp = (int)(rest % a.groups);
  const int64_t tok = rest / a.groups;
  const int64_t b = tok / a.T, t = tok % a.T;
  const int rot = a.pairs / V;
  const bool turn = u < rot;
  int e0, e1;
  float cs[V], sn[V];
  if (turn) {
    e0 = HALF ? u * V : 2 * u * V;
    e1 = HALF ? a.pairs + u * V : e0 + V;
    const int axis = u * V / a.per_axis;
    const double p = a.pos ? (double)a.pos[axis * a.ps[0] + b * a.ps[1] + t * a.ps[2]] : (double)t;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sincos_turns(p * (a.inv_freq[u * V + j] * 0.15915494309189533577), sn[j], cs[j]);
      cs[j] *= a.scale;
      sn[j] *= a.inverse ? -a.scale : a.scale;
    }
  } else {
    e0 = 2 * a.pairs + (u - rot) * 2 * V;
    e1 = e0 + V;
  }
  // Four heads at a time: all their loads first (input and output may be the same memory, so the compiler keeps the order written).
  const int total = a.heads[0] + a.heads[1];
  const int h0 = grp * a.hpt, h1 = h0 + a.hpt < total ? h0 + a.hpt : total;
  const bool second = turn || e1 < a.D;
  for (int h = h0; h < h1; h += 4) {
    Vec<T, V> x[4], y[4];
    int64_t at[4];
    int which[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int hc = h + i < h1 ? h + i : h1 - 1;
      const int w = hc >= a.heads[0];
      const int hh = w ? hc - a.heads[0] : hc;
      const T* in = (const T*)a.in[w] + b * a.is[w][0] + t * a.is[w][1] + hh * a.is[w][2];
      which[i] = w;
      at[i] = b * a.os[w][0] + t * a.os[w][1] + hh * a.os[w][2];
      x[i] = *reinterpret_cast<const Vec<T, V>*>(in + e0);
      if (second) y[i] = *reinterpret_cast<const Vec<T, V>*>(in + e1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (h + i >= h1) continue;
      if (turn) {
        float p[2 * V], q[2 * V];  // the unit's 2V elements in memory order, and their images
#pragma unroll
        for (int j = 0; j < V; ++j) { p[j] = (float)x[i].v[j]; p[V + j] = (float)y[i].v[j]; }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float ea = HALF ? p[j] : p[2 * j], eb = HALF ? p[V + j] : p[2 * j + 1];
          const float ra = ea * cs[j] - eb * sn[j], rb = ea * sn[j] + eb * cs[j];
          if (HALF) { q[j] = ra; q[V + j] = rb; } else { q[2 * j] = ra; q[2 * j + 1] = rb; }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) { x[i].v[j] = (T)q[j]; y[i].v[j] = (T)q[V + j]; }
      }
      T* out = (T*)a.out[which[i]] + at[i];
      *reinterpret_cast<Vec<T, V>*>(out + e0) = x[i];
      if (second) *reinterpret_cast<Vec<T, V>*>(out + e1) = y[i];
    }
  }
  }
}

template <typename T, int V>
int rotary_run(RotaryArgs a, bool copy_rest, hipStream_t st) {
  a.units = a.pairs / V + (copy_rest ? (a.D - 2 * a.pairs + 2 * V - 1) / (2 * V) : 0);
  const int total = a.heads[0] + a.heads[1];
  // Few tokens: a thread per head, so that the launch is as wide as it can be; many: eight heads share a thread's angles.
  int hpt = 8;
  while (hpt > 1 && a.tokens * a.units * ((total + hpt - 1) / hpt) < 256 * 1024) hpt /= 2;
  a.hpt = hpt;
  a.groups = (total + hpt - 1) / hpt;
  a.work = a.tokens * a.groups * a.units;
  const int64_t blocks = (a.work + 255) / 256;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20));
  if (a.half) rotary_kernel<T, V, true><<<grid, dim3(256), 0, st>>>(a);
  else rotary_kernel<T, V, false><<<grid, dim3(256), 0, st>>>(a);
  return launched("dm_rotary");
}

template <typename T, int FULL>
int rotary_types(const RotaryArgs& a, bool copy_rest, hipStream_t st) {
  auto fits = [&](int v) {
    if (a.pairs % v || a.per_axis % v || a.D % v) return false;
    for (int w = 0; w < 2; ++w) {
      if (!a.heads[w]) continue;
      if (!aligned(a.in[w], v * sizeof(T)) || !aligned(a.out[w], v * sizeof(T))) return false;
      for (int i = 0; i < 3; ++i)
        if (a.is[w][i] % v || a.os[w][i] % v) return false;
    }
    return true;
  };
  if (fits(FULL)) return rotary_run<T, FULL>(a, copy_rest, st);
  if (fits(FULL / 2)) return rotary_run<T, FULL / 2>(a, copy_rest, st);
  return rotary_run<T, 1>(a, copy_rest, st);
}

}  // namespace dmb

extern "C" int dm_rotary(const dm_rotary_tensor* q, const dm_rotary_tensor* k, const int64_t* positions_dev, const int64_t* position_strides,
                         int axes, const double* inv_freq_dev, int64_t B, int64_t T, int head_dim, int rotary_dim, int interleaved, float scale,
                         int inverse, int dtype, void* stream) {
  using namespace dmb;
  if (!dtype_ok(dtype)) return fail("dm_rotary: unknown dtype %d", dtype);
  if (B < 0 || T < 0 || T > 0x7fffffffLL || B > 0x7fffffffLL || B * T > (1LL << 40)) return fail("dm_rotary: bad sizes");
  if (head_dim < 1 || head_dim > 65536 || rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2)
    return fail("dm_rotary: rotary_dim %d must be even and within head_dim %d", rotary_dim, head_dim);
  if (axes < 1 || (rotary_dim / 2) % axes) return fail("dm_rotary: %d pairs do not divide into %d axes", rotary_dim / 2, axes);
  if (axes > 1 && !positions_dev) return fail("dm_rotary: several axes need positions");
  if (positions_dev && !position_strides) return fail("dm_rotary: positions without strides");
  if (!q || (rotary_dim && !inv_freq_dev)) return fail("dm_rotary: null argument");
  RotaryArgs a = {};
  bool copy_rest = false;
  for (int w = 0; w < 2; ++w) {
    const dm_rotary_tensor* t = w ? k : q;
    if (!t) continue;
    if (t->heads < 0 || t->heads > 65536) return fail("dm_rotary: %d heads", t->heads);
    if (!t->heads) continue;
    if (B * T > 0 && (!t->in || !t->out)) return fail("dm_rotary: null argument");
    a.in[w] = t->in; a.out[w] = t->out; a.heads[w] = t->heads;
    for (int i = 0; i < 3; ++i) { a.is[w][i] = t->in_stride[i]; a.os[w][i] = t->out_stride[i]; }
    if (t->in == t->out && B * T > 0) {
      for (int i = 0; i < 3; ++i)
        if (t->in_stride[i] != t->out_stride[i]) return fail("dm_rotary: in place needs the input's strides");
    } else {
      copy_rest = true;
    }
  }
  if (B * T == 0 || a.heads[0] + a.heads[1] == 0) return 0;
  if (rotary_dim == 0 && !copy_rest) return 0;
  a.pos = positions_dev;
  for (int i = 0; i < 3 && positions_dev; ++i) a.ps[i] = position_strides[i];
  a.inv_freq = inv_freq_dev;
  a.tokens = B * T; a.T = (int)T; a.D = head_dim; a.pairs = rotary_dim / 2;
  a.per_axis = a.pairs ? a.pairs / axes : 1;
  a.half = !interleaved; a.scale = scale; a.inverse = inverse;
  copy_rest = copy_rest && rotary_dim < head_dim;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == DM_F32) return rotary_types<float, 4>(a, copy_rest, st);
  if (dtype == DM_BF16) return rotary_types<bf16, 8>(a, copy_rest, st);
  return rotary_types<f16, 8>(a, copy_rest, st);
}
