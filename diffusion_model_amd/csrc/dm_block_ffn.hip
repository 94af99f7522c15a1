// dm_block_ffn.hip — the gated feed-forward block and its gradients.
//   g = x Wg^T + bg, u = x Wu^T + bu, h = act(g) u, y = h Wd^T + bd
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h, biases: column sums.
// Both projections, the activation and the product are one kernel; so are dh, dg and du: for training the forward pass keeps u act'(g),
// act(g) and h, three values where g and u would be two, so that none is rounded twice and nothing is computed again.
// Three paths forward.  Up to TOKEN_ROWS rows, and fp32 up to SKINNY_ROWS, the weights' bandwidth bounds the block, and every wave streams weight rows
// straight into vector (gemv_kernel) or matrix (skinny_kernel) instructions; above that the tiled products of dm_block_gemm.hip, whose
// smallest tile and split k range serve 16-bit decode batches.  Backward, dh and dx of few fp32 rows by large weights are sums over the weights as they
// lie (column_kernel, columns_fit), in plain fp32; everything else the tiled products.
// Rounding: the matrix pipe takes h, dg and du in 16 bits and nothing wider, so 16-bit tensors round them to their type between the products (but h of
// one or two rows: EXACT_ROWS): a gradient has two roundings where results alone would have one, sqrt(2) of its error.  u act'(g) and act(g) are kept
// in fp32, or rounded too where the caller asks for the fewer bytes (Saved; relative to 64 bits, bf16: 2.3e-3 and 2.9e-3 of a gradient).  Steps in us with
// fp32 and 16 bits: 8192 x 4096 x 11008 bf16 5400 and 5280, 1999 x 1001 x 2731 bf16 242 and 235, 28000 x 288 x 992 bf16 472 and 421.  Every sum is fp32.
// fp32 tensors are split into three bf16 terms and multiplied as six products (a1b1 a1b2 a2b1 a2b2 a1b3 a3b1; what is left out is below
// 2^-25 of |a||b|): the fp32 matrix instructions have 1/16 of the bf16 ones' rate.
#include <type_traits>

#include "dm_block_gemm.hip"

namespace dmb {

constexpr int TOKEN_ROWS = 4;  // gemv_kernel
// ... which keeps h in 32 bits up to so many rows of 16-bit tensors.  Every wave reads all of h: 4096 x 11008 bf16 takes 46.9 us of one row with h in 16
// bits and 47.4 with 32, 48.9 and 49.7 of two, but 51.7 and 59.9 of four.
constexpr int EXACT_ROWS = 2;
constexpr int SKINNY_ROWS = 64;  // skinny_kernel, fp32

// ---- operands that the products cannot read as they are: fp32 (three bf16 planes) and rows of no whole number of 16-byte pieces
struct PackJob { const void* src; void* dst; int64_t ld, plane, rows, block0; int cols, pitch; };  // block0: the first of its blocks
struct PackJobs { PackJob job[5]; int count; int64_t blocks; };
constexpr int PACK_PIECES = 1024;  // of eight elements, per block

// All matrices of a call in one launch: bound by memory, and by the launch where they are small.
template <typename T>
__global__ void __launch_bounds__(256) pack_rows_kernel(const PackJobs jobs) {
  constexpr bool PLANES = sizeof(T) == 4;
  using D = typename std::conditional<PLANES, bf16, T>::type;
  PackJob a = jobs.job[0];
#pragma unroll
  for (int i = 1; i < 5; ++i)
    if (i < jobs.count && blockIdx.x >= jobs.job[i].block0) a = jobs.job[i];
  const int pieces = a.pitch / 8;
  const int64_t piece0 = (blockIdx.x - a.block0) * PACK_PIECES, row0 = piece0 / pieces;
  const unsigned rest = (unsigned)(piece0 - row0 * pieces);
#pragma unroll
  for (int k = 0; k < PACK_PIECES / 256; ++k) {
    const unsigned id = rest + k * 256 + threadIdx.x;
    const int64_t r = row0 + id / (unsigned)pieces;
    const int c = (int)(id % (unsigned)pieces) * 8;
    if (r >= a.rows) continue;
    const T* s = (const T*)a.src + r * a.ld + c;
    Piece<T, 8> v;
    if (c + 8 <= a.cols) {
      v = *reinterpret_cast<const Piece<T, 8>*>(s);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v.v[i] = c + i < a.cols ? s[i] : (T)0.f;
    }
    D* dst = (D*)a.dst + r * a.pitch + c;
    if constexpr (PLANES) {
      Vec<bf16, 8> o[3];
#pragma unroll
      for (int i = 0; i < 8; ++i) { bf16 t[3]; split3((float)v.v[i], t); o[0].v[i] = t[0]; o[1].v[i] = t[1]; o[2].v[i] = t[2]; }
#pragma unroll
      for (int j = 0; j < 3; ++j) *reinterpret_cast<Vec<bf16, 8>*>(dst + j * a.plane) = o[j];
    } else {
      Vec<D, 8> o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[i] = v.v[i];
      *reinterpret_cast<Vec<D, 8>*>(dst) = o;
    }
  }
}

// Arguments of gemv_kernel and skinny_kernel: weights of type T, x of X, results of O.  What a backward pass needs of h is written beside it, as
// elements of the weights' type (`kept`) or planes.
template <typename T, typename X, typename O>
struct Streamed {
  const X* x; int64_t xs; const T *w, *w2; int64_t ldw; const T *bias, *bias2; O* out; int64_t ldo; void *ug, *ag; int kept16; T* kept; bf16* planes; int M, N, K, act;
};
using StreamedF32 = Streamed<float, float, float>;

// h, and what the backward pass needs, of one element from its two sums; the padding of a row holds zeros.
template <typename T, typename X, typename O>
__device__ __forceinline__ void finish_gate(const Streamed<T, X, O>& p, int n, int64_t at, float g, float u) {
  if (n >= ((p.N + 7) & ~7)) return;
  float h = 0.f, ag = 0.f;
  if (n < p.N) {
    g += p.bias ? (float)p.bias[n] : 0.f;
    u += p.bias2 ? (float)p.bias2[n] : 0.f;
    float slope;
    with_activation(p.act, [&](auto a) __attribute__((always_inline)) { activation<decltype(a)::value, sizeof(T) == 2>(g, ag, slope); });
    h = ag * u;
    u *= slope;
  } else {
    u = 0.f;
  }
  p.out[at] = (O)h;
  if (p.kept) p.kept[at] = (T)h;
  if (p.ug) {
    if (p.kept16) { ((T*)p.ug)[at] = (T)u; ((T*)p.ag)[at] = (T)ag; }
    else { ((float*)p.ug)[at] = u; ((float*)p.ag)[at] = ag; }
  }
  if (p.planes) {
    bf16 t[3];
    split3(h, t);
    for (int k = 0; k < 3; ++k) p.planes[k * p.M * p.ldo + at] = t[k];
  }
}

// ---- up to TOKEN_ROWS rows: the weights' bandwidth (one token through 4096 x 11008 bf16: 47 us, 5.7 TB/s of 270 MB; fp32 99 us).  A wave takes R rows
// of w (and of w2) and multiplies them with all of x in vector instructions, a row's piece of 64 V elements per load; the KSPLIT waves that share rows split
// the k range and meet in LDS.
template <int NV>  // v[i] summed over the wave; lane l < NV gets the i = l-th sum
__device__ __forceinline__ float wave_sums(float (&v)[NV], int lane) {
  int n = NV;
#pragma unroll
  for (int b = 0; (1 << b) < NV; ++b) {  // half of the values go to the other lane, which keeps those
    n /= 2;
    const bool up = lane >> b & 1;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = up ? v[2 * i + 1] : v[2 * i], send = up ? v[2 * i] : v[2 * i + 1];
      v[i] = keep + __shfl_xor(send, 1 << b, 64);
    }
  }
  float s = v[0];
#pragma unroll
  for (int o = NV; o < 64; o *= 2) s += __shfl_xor(s, o, 64);
  return s;
}

template <typename T, typename X, typename O, int MR, bool GATE, int KSPLIT>
__global__ void __launch_bounds__(256)
gemv_kernel(const Streamed<T, X, O> p) {
  constexpr int V = 16 / sizeof(T), R = 4, P = GATE ? 2 : 1, GROUPS = 4 / KSPLIT, NV = MR * R;
  __shared__ float red[KSPLIT > 1 ? KSPLIT : 1][GROUPS][P][NV];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = wave / KSPLIT, part = wave % KSPLIT;
  const int n0 = (blockIdx.x * GROUPS + group) * R;
  const T* rows[P][R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t n = n0 + r < p.N ? n0 + r : p.N - 1;
    rows[0][r] = p.w + n * p.ldw;
    if (GATE) rows[P - 1][r] = p.w2 + n * p.ldw;
  }
  float acc[P][NV] = {};
  auto multiply = [&](int k, auto pieces) __attribute__((always_inline)) {  // a piece of every row from k on
    constexpr int N = decltype(pieces)::value;
    Piece<T, N> a[P][R];
    Piece<X, N> b[MR];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int q = 0; q < P; ++q) a[q][r] = *reinterpret_cast<const Piece<T, N>*>(rows[q][r] + k);
#pragma unroll
    for (int m = 0; m < MR; ++m) b[m] = *reinterpret_cast<const Piece<X, N>*>(p.x + (m < p.M ? m : p.M - 1) * p.xs + k);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int q = 0; q < P; ++q)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int m = 0; m < MR; ++m) acc[q][m * R + r] = fmaf((float)a[q][r].v[i], (float)b[m].v[i], acc[q][m * R + r]);
  };
  const int whole = p.K / V * V;
#pragma unroll 2
  for (int k = part * 64 * V + lane * V; k < whole; k += KSPLIT * 64 * V) multiply(k, std::integral_constant<int, V>{});
  if (part == 0 && lane < p.K - whole) multiply(whole + lane, std::integral_constant<int, 1>{});
  float s[P];
#pragma unroll
  for (int q = 0; q < P; ++q) s[q] = wave_sums<NV>(acc[q], lane);
  if constexpr (KSPLIT > 1) {
    if (lane < NV)
#pragma unroll
      for (int q = 0; q < P; ++q) red[part][group][q][lane] = s[q];
    __syncthreads();
    if (part || lane >= NV) return;
#pragma unroll
    for (int q = 0; q < P; ++q) {
      s[q] = red[0][group][q][lane];
#pragma unroll
      for (int i = 1; i < KSPLIT; ++i) s[q] += red[i][group][q][lane];
    }
  }
  const int m = lane / R, n = n0 + lane % R;
  if (lane >= NV || m >= p.M) return;
  const int64_t at = (int64_t)m * p.ldo + n;
  if constexpr (GATE) finish_gate(p, n, at, s[0], s[P - 1]);
  else if (n < p.N) p.out[at] = (O)(s[0] + (p.bias ? (float)p.bias[n] : 0.f));
}

template <bool GATE, typename T, typename X, typename O>
int gemv_launch(const Streamed<T, X, O>& a, hipStream_t st) {
  const int groups = (int)(((int64_t)a.N + 7) / 8 * 8 + 3) / 4;  // of four rows, the padding of h among them
  int split = 1;  // sixteen waves for every CU, as long as each has a load of its own
  while (split < 4 && groups * split < 4096 && a.K > split * 64 * (int)(16 / sizeof(T))) split *= 2;
  auto run = [&](auto mr, auto ks) {
    constexpr int MR = decltype(mr)::value, KS = decltype(ks)::value;
    gemv_kernel<T, X, O, MR, GATE, KS><<<dim3((groups + 4 / KS - 1) / (4 / KS)), dim3(256), 0, st>>>(a);
  };
  auto rows = [&](auto ks) {
    if (a.M == 1) run(std::integral_constant<int, 1>{}, ks);
    else if (a.M == 2) run(std::integral_constant<int, 2>{}, ks);
    else if constexpr (sizeof(X) == sizeof(O) || sizeof(T) == 4) run(std::integral_constant<int, 4>{}, ks);  // (EXACT_ROWS)
  };
  if (split == 1) rows(std::integral_constant<int, 1>{});
  else if (split == 2) rows(std::integral_constant<int, 2>{});
  else rows(std::integral_constant<int, 4>{});
  return launched("dm_gated_ffn");
}

// ---- fp32, up to SKINNY_ROWS rows (of 4 elements or more): 16 rows of 2048 x 5504 52 us (2.6 TB/s of 135 MB), 64 rows 113 us.  Tiles of split operands,
// which first write three planes of every weight, take 132 and 144 (256 x 1024: 16 and 30 of 16 rows, 22 and 32 of 64; 4096 x 11008: 132 and 516,
// 288 and 542).
// Four instructions of four k each: instruction i takes element i of every lane's piece, on both sides.
__device__ __forceinline__ f32x4 mfma_f32(const Piece<float, 4>& a, const Piece<float, 4>& b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
  return c;
}

// Elements k .. k + 3 of a row of K >= 4; the row's last ones are a load moved back to end with the row, of which what lies before k counts
// as zero (`behind`, once the load has arrived): both sides of a product place them alike.
__device__ __forceinline__ Piece<float, 4> load_piece(const float* row, int k, int K) {
  return *reinterpret_cast<const Piece<float, 4>*>(row + (k + 4 <= K ? k : K - 4));
}
__device__ __forceinline__ Piece<float, 4> behind(Piece<float, 4> v, int k, int K) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v.v[i] = k + 4 <= K || K - 4 + i >= k ? v.v[i] : 0.f;
  return v;
}

constexpr int SKINNY_WAVES = 8;

// out[m, n] for 16 n per block: the waves deal the k range among themselves in chunks, and their sums meet in LDS.  A chunk is U pieces
// of every row (U * 64 bytes on end), and the next chunk is on its way while one is multiplied.  Blocks begin at different chunks: in
// step they would all ask for the same columns of rows a power of two apart, which lie on few of the memory's channels.
template <int MT, bool GATE>
__global__ void __launch_bounds__(SKINNY_WAVES * 64) skinny_kernel(const StreamedF32 p) {
  constexpr int V = 4, STEP = 4 * V, P = GATE ? 2 : 1;
  constexpr int U = MT == 4 ? 2 : 4;
  __shared__ f32x4 red[SKINNY_WAVES][P][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = blockIdx.x * 16 + (lane & 15);
  const int64_t nc = n < p.N ? n : p.N - 1;
  const float* w1r = p.w + nc * p.ldw;
  const float* w2r = GATE ? p.w2 + nc * p.ldw : nullptr;
  const float* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = t * 16 + (lane & 15);
    xr[t] = p.x + (m < p.M ? m : p.M - 1) * p.xs;
  }
  f32x4 acc[P][MT] = {};
  struct Chunk { Piece<float, V> a[P][U], b[U][MT]; int k; } one, two;  // k: of its first piece
  const int chunks = (p.K + U * STEP - 1) / (U * STEP), turn = (int)(blockIdx.x * 7u % (unsigned)chunks);
  auto load = [&](Chunk& c, int at) __attribute__((always_inline)) {
    if (at >= chunks) return;
    at += turn;
    if (at >= chunks) at -= chunks;
    c.k = at * U * STEP;
    const int k0 = c.k + (lane >> 4) * V;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      c.a[0][i] = load_piece(w1r, k0 + i * STEP, p.K);
      if (GATE) c.a[P - 1][i] = load_piece(w2r, k0 + i * STEP, p.K);
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t) c.b[i][t] = load_piece(xr[t], k0 + i * STEP, p.K);
  };
  auto multiply = [&](const Chunk& c) __attribute__((always_inline)) {
    const bool last = c.k + U * STEP > p.K;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = c.k + (lane >> 4) * V + i * STEP;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const Piece<float, V> b = last ? behind(c.b[i][t], k, p.K) : c.b[i][t];
#pragma unroll
        for (int q = 0; q < P; ++q) acc[q][t] = mfma_f32(last ? behind(c.a[q][i], k, p.K) : c.a[q][i], b, acc[q][t]);
      }
    }
  };
  int at = wave;
  load(one, at);
  while (at < chunks) {
    load(two, at + SKINNY_WAVES);
    multiply(one);
    at += SKINNY_WAVES;
    if (at >= chunks) break;
    load(one, at + SKINNY_WAVES);
    multiply(two);
    at += SKINNY_WAVES;
  }
#pragma unroll
  for (int q = 0; q < P; ++q)
#pragma unroll
    for (int t = 0; t < MT; ++t) red[wave][q][t][lane] = acc[q][t];
  __syncthreads();
  if (wave >= MT) return;
  f32x4 s[P];
#pragma unroll
  for (int q = 0; q < P; ++q) {
    s[q] = red[0][q][wave][lane];
#pragma unroll
    for (int v = 1; v < SKINNY_WAVES; ++v) s[q] += red[v][q][wave][lane];
  }
  const int m = wave * 16 + (lane & 15);
  if (m >= p.M) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = blockIdx.x * 16 + (lane >> 4) * 4 + e;
    const int64_t to = (int64_t)m * p.ldo + c;
    if constexpr (GATE) finish_gate(p, c, to, s[0][e], s[P - 1][e]);
    else if (c < p.N) p.out[to] = s[0][e] + (p.bias ? p.bias[c] : 0.f);
  }
}

template <bool GATE>
int skinny_launch(const StreamedF32& a, hipStream_t st) {
  const dim3 grid((a.N + 15) / 16), block(SKINNY_WAVES * 64);
  if (a.M <= 16) skinny_kernel<1, GATE><<<grid, block, 0, st>>>(a);
  else if (a.M <= 32) skinny_kernel<2, GATE><<<grid, block, 0, st>>>(a);
  else skinny_kernel<4, GATE><<<grid, block, 0, st>>>(a);
  return launched("dm_gated_ffn");
}

template <bool GATE, typename T, typename X, typename O>
int streamed(const Streamed<T, X, O>& a, hipStream_t st) {
  if constexpr (std::is_same<T, float>::value)
    if (a.M > TOKEN_ROWS) return skinny_launch<GATE>(a, st);
  return gemv_launch<GATE>(a, st);
}

// ---- fp32 backward of few rows (columns_fit): part[split][m][n] = sum over the split's k of A[m][k] B[k][n], B's rows in memory.  A thread takes
// four columns of sixteen rows and walks k; A's part lies in LDS.  Bound by B's bytes, where tiles of split operands would first write three
// planes of it; the parts are joined like those of a tile's split range.
constexpr int COLUMN_ROWS = 16, COLUMN_K = 128;  // k per split, at most
struct Columns { const float* a; const bf16* planes; int64_t lda, plane; const float* b; int64_t ldb; float* part; int64_t split_stride, ldpart; int M, N, K, per; };
__global__ void __launch_bounds__(256) column_kernel(const Columns p) {
  __shared__ float a[COLUMN_K][COLUMN_ROWS];
  const int m0 = blockIdx.z * COLUMN_ROWS, k0 = blockIdx.y * p.per, count = p.K - k0 < p.per ? p.K - k0 : p.per;
  for (int e = threadIdx.x; e < count * COLUMN_ROWS; e += 256) {
    const int m = m0 + e / count, k = e % count;
    float v = 0.f;
    if (m < p.M) {
      const int64_t at = m * p.lda + k0 + k;
      v = p.a ? p.a[at] : ((float)p.planes[2 * p.plane + at] + (float)p.planes[p.plane + at]) + (float)p.planes[at];
    }
    a[k][e / count] = v;
  }
  __syncthreads();
  const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (n >= p.N) return;
  const int at = n + 4 <= p.N ? n : p.N - 4;  // (the last piece is moved back; both write the same values)
  float acc[COLUMN_ROWS][4] = {};
  const float* b = p.b + (int64_t)k0 * p.ldb + at;
#pragma unroll 8
  for (int k = 0; k < count; ++k) {
    const Piece<float, 4> v = *reinterpret_cast<const Piece<float, 4>*>(b + k * p.ldb);
#pragma unroll
    for (int m = 0; m < COLUMN_ROWS; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[m][j] = fmaf(a[k][m], v.v[j], acc[m][j]);
  }
  float* part = p.part + blockIdx.y * p.split_stride + at;
#pragma unroll
  for (int m = 0; m < COLUMN_ROWS; ++m)
    if (m0 + m < p.M) {
      Piece<float, 4> r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r.v[j] = acc[m][j];
      float* row = part + (m0 + m) * p.ldpart;
      *reinterpret_cast<Piece<float, 4>*>(row) = r;
      if (n + 4 >= p.N)  // the padding of a row holds zeros
        for (int c = p.N - at; at + c < p.ldpart; ++c) row[c] = 0.f;
    }
}
// k per split: a thousand workgroups where the range gives them, 16 k or more each
inline int column_per(int64_t M, int N, int K) {
  const int blocks = (int)((N + 1023) / 1024 * ((M + COLUMN_ROWS - 1) / COLUMN_ROWS));
  int per = (int)((int64_t)K * blocks / 1024);
  return per < 16 ? 16 : per > COLUMN_K ? COLUMN_K : per;
}
inline int column_splits(int64_t M, int N, int K) { return (K + column_per(M, N, K) - 1) / column_per(M, N, K); }
inline int column_launch(Columns a, hipStream_t st) {
  a.per = column_per(a.M, a.N, a.K);
  column_kernel<<<dim3((a.N + 1023) / 1024, column_splits(a.M, a.N, a.K), (a.M + COLUMN_ROWS - 1) / COLUMN_ROWS), dim3(256), 0, st>>>(a);
  return launched("dm_gated_ffn_backward");
}

// ---- workspace
struct Carver {
  char* base;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};

// A matrix as the products read it: rows of `ld` 16-bit elements; fp32 matrices as three planes.
struct Operand { const void* p; int64_t ld, plane; };

struct FfnSizes { int64_t M; int D, F, N, dtype, kept16; };  // kept16: see Saved (fp32 tensors: 0)

// fp32 backward passes by column_kernel: where splitting the weights into planes costs more than multiplying in vector instructions, so for
// large weights and few rows.  Measured, backward pass in us with it and with tiles of planes, by the elements of a weight:
// 1M (512 x 2048) 62 and 55 of one row; 4.4M (1918 x 2281) 104 and 114 of one, 123 and 116 of 16; 7.6M (1456 x 5223) 112 and 154 of one, 163 and 162
// of 32; 11M (2048 x 5504) 184 and 208 of 17, 223 and 215 of 48; 45M (4096 x 11008) 416 and 742 of one, 605 and 777 of 48, 822 and 791 of 64.
inline bool columns_fit(const FfnSizes& z) {
  if (z.D < 4 || z.F < 4 || z.M > SKINNY_ROWS) return false;  // its pieces; the rows that its tests reach
  if (forced_tile >= 0) return forced_tile == FORCED_COLUMNS;
  return z.M <= 48 && z.M << 18 <= (int64_t)z.F * (2LL * z.D + z.N) / 3 - (1 << 21);
}

template <typename T>
int pack_launch(const PackJobs& jobs, hipStream_t st) {
  if (!jobs.count) return 0;
  if (jobs.blocks > (1LL << 24)) return fail("gated feed-forward block: operands of %lld elements to pack", (long long)jobs.blocks * PACK_PIECES * 8);
  pack_rows_kernel<T><<<dim3((unsigned)jobs.blocks), dim3(256), 0, st>>>(jobs);
  return launched("gated feed-forward block");
}

// Takes room for the packed form of a [rows][cols] matrix where the products cannot read it as it lies; `needed`: it is to be packed.
template <typename T>
Operand prepare_operand(PackJobs& jobs, const void* src, int64_t ld, int64_t rows, int cols, Carver& ws, bool needed = true) {
  constexpr bool F32 = std::is_same<T, float>::value;
  if (!F32 && cols % 8 == 0) return {src, ld, 0};
  const int64_t pitch = round_up(cols, 8);
  void* p = ws.take((size_t)(F32 ? 3 : 1) * rows * pitch * 2);
  if (needed) {
    jobs.job[jobs.count++] = {src, p, ld, rows * pitch, rows, jobs.blocks, cols, (int)pitch};
    jobs.blocks += (rows * (pitch / 8) + PACK_PIECES - 1) / PACK_PIECES;
  }
  return {p, pitch, rows * pitch};
}
template <typename T>
Operand take_operand(int64_t rows, int cols, Carver& ws) {
  const int64_t pitch = round_up(cols, 8);
  Operand o = {nullptr, pitch, rows * pitch};
  o.p = ws.take((size_t)(std::is_same<T, float>::value ? 3 : 1) * rows * pitch * 2);
  return o;
}

// The product terms of two operands (`second`: of two more, of the same shape): one, or the six of split fp32, those with a leading plane on
// both sides last.
template <typename T>
void add_terms(GemmArgs& g, const Operand& a, const Operand& b, bool second = false) {
  g.terms = 0;
  g.segments = 0;
  auto add = [&](uint64_t i, uint64_t j, int s) { g.terms |= (i | j << 2 | (s ? 16 : 0)) << 5 * g.segments++; };
  if (std::is_same<T, float>::value)
    for (int s = 0; s <= second; ++s) { add(2, 0, s); add(1, 0, s); add(1, 1, s); add(0, 1, s); add(0, 2, s); }  // (one plane tile new at once)
  g.early = g.segments;
  for (int s = 0; s <= second; ++s) add(0, 0, s);
  g.a[second] = a.p;
  g.b[second] = b.p;
  g.lda = a.ld;
  g.ldb = b.ld;
  g.plane_a = a.plane * 2;
  g.plane_b = b.plane * 2;
}

template <typename T> using Mat = typename std::conditional<std::is_same<T, float>::value, bf16, T>::type;  // what the matrix pipe sees

template <typename T>
Out result(void* p, int64_t ld) {  // a tensor of the caller's
  return {p, ld, 0, std::is_same<T, float>::value, ld % (16 / sizeof(T)) == 0 && aligned(p, 16)};
}
template <typename T>
Out between(const Operand& o) {  // an operand of a later product
  return {const_cast<void*>(o.p), o.ld, o.plane, 0, 1};
}

// The plan of a product, and where it keeps its parts (`part`: room for them).
inline int planned(GemmArgs& g, const GemmPlan& plan, void* part) {
  g.splits = plan.splits;
  g.part = part;
  g.ldpart = round_up(g.N, 8);
  g.split_stride = (g.pair ? 2 * g.M : g.M) * g.ldpart;
  return plan.tile;
}

// out[M][N] = A B (+ bias); sums: the sum of A over k (both operands KS).  g.pair: of two A, with g.out2 and g.sums2.
template <typename T, bool AKS, bool BKS>
int product(GemmArgs g, const Out& out, const void* bias, void* sums, void* part, hipStream_t st) {
  const int tile = planned(g, gemm_plan(g.pair ? 2 * g.M : g.M, g.N, g.iters, g.segments, 1, sizeof(T), !AKS), part);
  g.out = out;
  g.bias = bias;
  g.sums = sums;
  if (g.pair) g.out.vec = out.vec && g.out2.vec;
  g.sum_part = (float*)part + g.splits * g.split_stride;
  g.sum_segments = std::is_same<T, float>::value ? 1 << 0 | 1 << 1 | 1 << 5 : 1;  // add_terms: each plane of A once
  return gemm_launch<Mat<T>, AKS, BKS, EPI_STORE>(g, tile, st);
}

inline int iters_of(int64_t K) { return (int)((K + GEMM_BK - 1) / GEMM_BK); }
inline int64_t pad8(int64_t v) { return round_up(v, 8); }

struct FfnIn { const void *x, *wg, *wu, *wd, *bg, *bu, *bd; int64_t xs; };

// What the forward pass keeps for the backward pass: u act'(g) and act(g), fp32 or (kept16) of the tensors' type, and h as an operand of dWd = dy^T h.
struct Saved {
  void *ug = nullptr, *ag = nullptr;
  Operand h = {nullptr, 0, 0};
  int kept16;
  Saved(void* p, int64_t M, int F, int kept16_) : kept16(kept16_) {
    if (!p) return;
    const int64_t Fp = pad8(F), bytes = M * Fp * (kept16 ? 2 : 4);
    ug = p;
    ag = (char*)p + bytes;
    h = {(char*)p + 2 * bytes, Fp, M * Fp};
  }
  Out out(void* p) const { return {p, h.ld, 0, !kept16, 1}; }
};

// run: launch; otherwise only count the workspace.
template <typename T>
int ffn_forward(const FfnSizes& z, const FfnIn& in, void* y, void* saved, int act, Carver& ws, bool run, hipStream_t st) {
  constexpr bool F32 = std::is_same<T, float>::value;
  const int64_t Fp = pad8(z.F);
  const Saved kept(saved, z.M, z.F, z.kept16);
  if (z.M <= TOKEN_ROWS || (F32 && z.M <= SKINNY_ROWS && z.D >= 4 && z.F >= 4)) {
    const int M = (int)z.M;
    auto both = [&](auto type) {  // of h
      using H = decltype(type);
      H* h = (H*)ws.take((size_t)z.M * Fp * sizeof(H));
      if (!run) return 0;
      const Streamed<T, T, H> gate = {(const T*)in.x, in.xs, (const T*)in.wg, (const T*)in.wu, z.D, (const T*)in.bg, (const T*)in.bu, h, Fp,
                                      kept.ug, kept.ag, kept.kept16, saved && !F32 ? (T*)kept.h.p : nullptr, saved && F32 ? (bf16*)kept.h.p : nullptr, M, z.F, z.D, act};
      if (const int rc = streamed<true>(gate, st)) return rc;
      const Streamed<T, H, T> down = {h, Fp, (const T*)in.wd, nullptr, z.F, (const T*)in.bd, nullptr, (T*)y, z.N, nullptr, nullptr, 0, nullptr, nullptr,
                                      M, z.N, z.F, act};
      return streamed<false>(down, st);
    };
    return z.M <= EXACT_ROWS ? both(float()) : both(T());
  }
  PackJobs jobs = {};
  const Operand x = prepare_operand<T>(jobs, in.x, in.xs, z.M, z.D, ws), wg = prepare_operand<T>(jobs, in.wg, z.D, z.F, z.D, ws),
                wu = prepare_operand<T>(jobs, in.wu, z.D, z.F, z.D, ws), wd = prepare_operand<T>(jobs, in.wd, z.F, z.N, z.F, ws);
  const Operand h = saved ? kept.h : take_operand<T>(z.M, z.F, ws);
  const int terms = F32 ? 6 : 1;
  const size_t part_bytes = gemm_plan(z.M, z.N, iters_of(z.F), terms, 1, sizeof(T), true).part_bytes;
  const GemmPlan gate = gemm_plan(z.M, z.F, iters_of(z.D), terms, 2, F32 ? 7 : 3, true);
  void* part = ws.take(gate.part_bytes > part_bytes ? gate.part_bytes : part_bytes);  // used by one product after the other
  if (!run) return 0;
  int rc = pack_launch<T>(jobs, st);
  if (rc) return rc;

  GemmArgs g = {};
  add_terms<T>(g, x, wg);
  g.b2 = wu.p;
  g.M = z.M; g.N = z.F; g.K = z.D; g.iters = iters_of(g.K);
  g.out = between<T>(h);
  g.out2 = kept.out(kept.ug);
  g.out3 = kept.out(kept.ag);
  g.bias = in.bg; g.bias2 = in.bu; g.act = act;
  const int tile = planned(g, gate, part);
  if ((rc = gemm_launch<Mat<T>, false, false, F32 ? EPI_GATE_F32 : EPI_GATE>(g, tile, st))) return rc;

  GemmArgs d = {};
  add_terms<T>(d, h, wd);
  d.M = z.M; d.N = z.N; d.K = z.F; d.iters = iters_of(z.F);
  return product<T, false, false>(d, result<T>(y, z.N), in.bd, nullptr, part, st);
}

struct FfnGrads { void *dx, *dwg, *dwu, *dwd, *dbg, *dbu, *dbd; };

template <typename T>
int ffn_backward(const FfnSizes& z, const FfnIn& in, const void* dy, int64_t dys, const void* saved, const FfnGrads& gr, Carver& ws, bool run,
                 hipStream_t st) {
  const int64_t Fp = pad8(z.F);
  const int terms = std::is_same<T, float>::value ? 6 : 1;
  const bool few = std::is_same<T, float>::value && columns_fit(z);
  PackJobs jobs = {};
  const Operand y = prepare_operand<T>(jobs, dy, dys, z.M, z.N, ws), x = prepare_operand<T>(jobs, in.x, in.xs, z.M, z.D, ws, gr.dwg || gr.dwu);
  Operand wd = {}, wg = {}, wu = {};
  if (!few) {
    wd = prepare_operand<T>(jobs, in.wd, z.F, z.N, z.F, ws);
    wg = prepare_operand<T>(jobs, in.wg, z.D, z.F, z.D, ws, gr.dx);
    wu = prepare_operand<T>(jobs, in.wu, z.D, z.F, z.D, ws, gr.dx);
  }
  // dg and du side by side, so that one product gives both projections' gradients: twice the tiles of a launch, one launch less
  const Operand dg = take_operand<T>(z.M, 2 * (int)Fp, ws), du = {(char*)dg.p + 2 * Fp, dg.ld, dg.plane};
  const Saved kept(const_cast<void*>(saved), z.M, z.F, z.kept16);
  size_t part_bytes = gemm_plan(z.M, z.D, iters_of(z.F), terms * 2, 1, sizeof(T), true).part_bytes;
  const GemmPlan dact = gemm_plan(z.M, z.F, iters_of(z.N), terms, 1, terms > 1 ? 20 : 8, true);
  const size_t more[] = {dact.part_bytes, gemm_plan(2LL * z.F, z.D, iters_of(z.M), terms, 1, sizeof(T), false).part_bytes,
                         gemm_plan(z.F, z.D, iters_of(z.M), terms, 1, sizeof(T), false).part_bytes, gemm_plan(z.N, z.F, iters_of(z.M), terms, 1, sizeof(T), false).part_bytes};
  for (size_t b : more) part_bytes = b > part_bytes ? b : part_bytes;
  if (few) {
    const size_t columns[] = {(size_t)column_splits(z.M, z.F, z.N) * z.M * Fp * 4, (size_t)2 * column_splits(z.M, z.D, z.F) * z.M * pad8(z.D) * 4};
    for (size_t b : columns) part_bytes = b > part_bytes ? b : part_bytes;
  }
  void* part = ws.take(part_bytes);  // used by one product after the other, in stream order
  if (!run) return 0;
  int rc = pack_launch<T>(jobs, st);
  if (rc) return rc;

  GemmArgs a = {};  // dh, and from it dg and du
  add_terms<T>(a, y, wd);
  a.M = z.M; a.N = z.F; a.K = z.N; a.iters = iters_of(a.K);
  a.out = between<T>(dg); a.out2 = between<T>(du);
  a.ug = kept.ug; a.ag = kept.ag; a.ldg = Fp; a.kept16 = kept.kept16;
  const int tile = planned(a, dact, part);
  if constexpr (std::is_same<T, float>::value)
    if (few) {
      a.splits = column_splits(z.M, z.F, z.N);
      if ((rc = column_launch({(const float*)dy, nullptr, dys, 0, (const float*)in.wd, z.F, (float*)part, a.split_stride, a.ldpart, (int)z.M, z.F, z.N, 0}, st)))
        return rc;
      if ((rc = join_launch<bf16, EPI_DACT_F32>(a, st))) return rc;
    }
  if (!few && (rc = gemm_launch<Mat<T>, false, true, std::is_same<T, float>::value ? EPI_DACT_F32 : EPI_DACT>(a, tile, st))) return rc;

  if (gr.dx) {
    GemmArgs g = {};
    add_terms<T>(g, dg, wg);
    add_terms<T>(g, du, wu, true);
    g.M = z.M; g.N = z.D; g.K = z.F; g.iters = iters_of(z.F);
    if constexpr (std::is_same<T, float>::value)
      if (few) {
        const int half = column_splits(z.M, z.D, z.F);
        planned(g, {TILE_MID, 2 * half, 0}, part);
        g.out = result<T>(gr.dx, z.D);
        for (int i = 0; i < 2 && !rc; ++i)
          rc = column_launch({nullptr, (const bf16*)(i ? du.p : dg.p), dg.ld, dg.plane, (const float*)(i ? in.wu : in.wg), z.D,
                              (float*)part + i * half * g.split_stride, g.split_stride, g.ldpart, (int)z.M, z.D, z.F, 0}, st);
        if (!rc) rc = join_launch<bf16, EPI_STORE>(g, st);
        if (rc) return rc;
      }
    if (!few && (rc = product<T, false, true>(g, result<T>(gr.dx, z.D), nullptr, nullptr, part, st))) return rc;
  }
  // (the sum of dg^T, du^T, dy^T over the rows of the batch is the bias' gradient)
  auto weight = [&](const Operand& l, const Operand& r, int rows, int cols, void* out, void* bias, void* out2 = nullptr, void* bias2 = nullptr) {
    GemmArgs g = {};
    add_terms<T>(g, l, r);
    g.M = rows; g.N = cols; g.K = (int)z.M; g.iters = iters_of(z.M);
    if (out2) {
      g.pair = 2 * Fp;
      g.out2 = result<T>(out2, cols);
      g.sums2 = bias2;
    }
    return product<T, true, true>(g, result<T>(out, cols), nullptr, bias, part, st);
  };
  if (gr.dwg && gr.dwu) {
    if ((rc = weight(dg, x, z.F, z.D, gr.dwg, gr.dbg, gr.dwu, gr.dbu))) return rc;
  } else {
    if (gr.dwg && (rc = weight(dg, x, z.F, z.D, gr.dwg, gr.dbg))) return rc;
    if (gr.dwu && (rc = weight(du, x, z.F, z.D, gr.dwu, gr.dbu))) return rc;
  }
  if (gr.dwd && (rc = weight(y, kept.h, z.N, z.F, gr.dwd, gr.dbd))) return rc;
  return 0;
}

inline int ffn_check(const char* who, const FfnSizes& z, int act) {
  if (!dtype_ok(z.dtype)) return fail("%s: unknown dtype %d", who, z.dtype);
  if (act < DM_ACT_SILU || act > DM_ACT_SIGMOID) return fail("%s: unknown activation %d", who, act);
  const int most = 1 << 20;
  if (z.D < 1 || z.F < 1 || z.N < 1 || z.D > most || z.F > most || z.N > most)
    return fail("%s: widths %d, %d, %d (1 to 2^20)", who, z.D, z.F, z.N);
  if (z.M < 0 || z.M > (1 << 28)) return fail("%s: %lld rows (up to 2^28)", who, (long long)z.M);
  return 0;
}
// Rows that the kernels read as 16-byte pieces start at multiples of 16 bytes; rows of no whole number of pieces are read element by element.
inline int ffn_check_matrix(const char* who, const char* what, const void* p, int64_t ld, int64_t rows, int cols, int dtype) {
  if (!p) return fail("%s: null argument (%s)", who, what);
  if (ld < cols && rows > 1) return fail("%s: %s: row stride %lld below the width %d", who, what, (long long)ld, cols);
  if (ld > (1 << 21)) return fail("%s: %s: row stride %lld above 2^21", who, what, (long long)ld);
  const int es = dtype_size(dtype);
  if (cols % (16 / es) == 0 && (!aligned(p, 16) || (rows > 1 && ld % (16 / es))))
    return fail("%s: %s: rows must start at multiples of 16 bytes", who, what);
  if (!aligned(p, es)) return fail("%s: %s: not aligned to its elements", who, what);
  return 0;
}

template <typename F>
int ffn_types(int dtype, F&& f) {
  switch (dtype) {
    case DM_F32: return f(float());
    case DM_BF16: return f(bf16());
    default: return f(f16());
  }
}

__global__ void fill_zero_bytes_kernel(uint32_t* p, int64_t words, uint16_t* tail) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) p[i] = 0;
  if (tail && blockIdx.x == 0 && threadIdx.x == 0) *tail = 0;
}

}  // namespace dmb

extern "C" {

int dm_debug_ffn_plan(int tile, int splits) {
  using namespace dmb;
  if (tile < -1 || tile > FORCED_COLUMNS || splits < 1 || splits > 64) return fail("dm_debug_ffn_plan: tile %d (-1 to 3), %d parts (1 to 64)", tile, splits);
  forced_tile = tile;
  forced_splits = splits;
  return 0;
}

size_t dm_gated_ffn_saved_bytes(int64_t M, int F, int dtype) {
  using namespace dmb;
  const bool keep = dtype & DM_FFN_KEEP_F32;
  dtype &= ~DM_FFN_KEEP_F32;
  if (M <= 0 || F < 1 || !dtype_ok(dtype)) return 0;
  return (size_t)M * pad8(F) * (dtype == DM_F32 ? 2 * 4 + 3 * 2 : keep ? 2 * 4 + 2 : 3 * 2);
}

size_t dm_gated_ffn_workspace_bytes(int64_t M, int D, int F, int N, int dtype, int save) {
  using namespace dmb;
  const FfnSizes z = {M, D, F, N, dtype, 0};
  if (M <= 0 || ffn_check("dm_gated_ffn_workspace_bytes", z, DM_ACT_SILU)) return 0;
  Carver ws = {nullptr};
  ffn_types(dtype, [&](auto t) { return ffn_forward<decltype(t)>(z, FfnIn{}, nullptr, save ? &ws : nullptr, 0, ws, false, nullptr); });
  return ws.used;
}

size_t dm_gated_ffn_backward_workspace_bytes(int64_t M, int D, int F, int N, int dtype) {
  using namespace dmb;
  const FfnSizes z = {M, D, F, N, dtype, 0};
  if (M <= 0 || ffn_check("dm_gated_ffn_backward_workspace_bytes", z, DM_ACT_SILU)) return 0;
  Carver ws = {nullptr};
  ffn_types(dtype, [&](auto t) {
    return ffn_backward<decltype(t)>(z, FfnIn{}, nullptr, 0, nullptr, FfnGrads{}, ws, false, nullptr);
  });
  return ws.used;
}

int dm_gated_ffn(const void* x_dev, int64_t x_stride, const void* w_gate_dev, const void* w_up_dev, const void* w_down_dev, const void* b_gate_dev,
                 const void* b_up_dev, const void* b_down_dev, void* y_dev, void* saved_dev, int64_t M, int D, int F, int N, int activation, int dtype,
                 void* workspace_dev, size_t workspace_bytes, void* stream) {
  using namespace dmb;
  const char* who = "dm_gated_ffn";
  const FfnSizes z = {M, D, F, N, dtype, dtype != DM_F32 && !(activation & DM_FFN_KEEP_F32)};
  activation &= ~DM_FFN_KEEP_F32;
  if (const int rc = ffn_check(who, z, activation)) return rc;
  if (M == 0) return 0;
  if (M == 1) x_stride = D;  // (rows of a product's second operand end where the stride says)
  if (ffn_check_matrix(who, "x", x_dev, x_stride, M, D, dtype) || ffn_check_matrix(who, "w_gate", w_gate_dev, D, F, D, dtype) ||
      ffn_check_matrix(who, "w_up", w_up_dev, D, F, D, dtype) || ffn_check_matrix(who, "w_down", w_down_dev, F, N, F, dtype))
    return 1;
  if (!y_dev) return fail("%s: null argument (y)", who);
  if (saved_dev && !aligned(saved_dev, 16)) return fail("%s: saved must be aligned to 16 bytes", who);
  const size_t need = dm_gated_ffn_workspace_bytes(M, D, F, N, dtype, saved_dev != nullptr);
  if (!workspace_dev || workspace_bytes < need || !aligned(workspace_dev, 16))
    return fail("%s: workspace of %zu bytes, %zu needed (aligned to 16)", who, workspace_dev ? workspace_bytes : (size_t)0, need);
  const FfnIn in = {x_dev, w_gate_dev, w_up_dev, w_down_dev, b_gate_dev, b_up_dev, b_down_dev, x_stride};
  Carver ws = {(char*)workspace_dev};
  return ffn_types(dtype, [&](auto t) { return ffn_forward<decltype(t)>(z, in, y_dev, saved_dev, activation, ws, true, (hipStream_t)stream); });
}

int dm_gated_ffn_backward(const void* dy_dev, int64_t dy_stride, const void* x_dev, int64_t x_stride, const void* w_gate_dev, const void* w_up_dev,
                          const void* w_down_dev, const void* saved_dev, void* dx_dev, void* dw_gate_dev, void* dw_up_dev, void* dw_down_dev,
                          void* db_gate_dev, void* db_up_dev, void* db_down_dev, int64_t M, int D, int F, int N, int activation, int dtype,
                          void* workspace_dev, size_t workspace_bytes, void* stream) {
  using namespace dmb;
  const char* who = "dm_gated_ffn_backward";
  const FfnSizes z = {M, D, F, N, dtype, dtype != DM_F32 && !(activation & DM_FFN_KEEP_F32)};
  activation &= ~DM_FFN_KEEP_F32;
  if (const int rc = ffn_check(who, z, activation)) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (M == 0) {  // no rows: the parameters' gradients are zero
    void* const p[] = {dw_gate_dev, dw_up_dev, dw_down_dev, db_gate_dev, db_up_dev, db_down_dev};
    const int64_t n[] = {(int64_t)F * D, (int64_t)F * D, (int64_t)N * F, F, F, N};
    for (int i = 0; i < 6; ++i) {
      if (!p[i]) continue;
      const int64_t bytes = n[i] * dtype_size(dtype), words = bytes / 4;
      fill_zero_bytes_kernel<<<dim3((unsigned)(words / 256 + 1 < 65536 ? words / 256 + 1 : 65536)), dim3(256), 0, st>>>(
          (uint32_t*)p[i], words, bytes % 4 ? (uint16_t*)((char*)p[i] + words * 4) : nullptr);
      if (const int rc = launched(who)) return rc;
    }
    return 0;
  }
  if (M == 1) { dy_stride = N; x_stride = D; }  // (rows of a product's second operand end where the stride says)
  if (ffn_check_matrix(who, "dy", dy_dev, dy_stride, M, N, dtype) || ffn_check_matrix(who, "x", x_dev, x_stride, M, D, dtype) ||
      ffn_check_matrix(who, "w_gate", w_gate_dev, D, F, D, dtype) || ffn_check_matrix(who, "w_up", w_up_dev, D, F, D, dtype) ||
      ffn_check_matrix(who, "w_down", w_down_dev, F, N, F, dtype))
    return 1;
  if ((db_gate_dev && !dw_gate_dev) || (db_up_dev && !dw_up_dev) || (db_down_dev && !dw_down_dev))
    return fail("%s: a bias' gradient comes with its weight's", who);
  if (!saved_dev || !aligned(saved_dev, 16)) return fail("%s: saved must be what dm_gated_ffn wrote, aligned to 16 bytes", who);
  const size_t need = dm_gated_ffn_backward_workspace_bytes(M, D, F, N, dtype);
  if (!workspace_dev || workspace_bytes < need || !aligned(workspace_dev, 16))
    return fail("%s: workspace of %zu bytes, %zu needed (aligned to 16)", who, workspace_dev ? workspace_bytes : (size_t)0, need);
  const FfnIn in = {x_dev, w_gate_dev, w_up_dev, w_down_dev, nullptr, nullptr, nullptr, x_stride};
  const FfnGrads gr = {dx_dev, dw_gate_dev, dw_up_dev, dw_down_dev, db_gate_dev, db_up_dev, db_down_dev};
  Carver ws = {(char*)workspace_dev};
  return ffn_types(dtype,
                   [&](auto t) { return ffn_backward<decltype(t)>(z, in, dy_dev, dy_stride, saved_dev, gr, ws, true, st); });
}

}  // extern "C"
