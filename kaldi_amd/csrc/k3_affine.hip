// k3_affine.hip -- an affine layer in half precision (float16 / bfloat16) with its activation and its bypass in the product's epilogue, and its backward pass (k3_affine_*).
//   forward:  pre = x W^T + b,  y = act(pre) + residual          x [rows x inner], W [cols x inner]
//   backward: dz = dy act'(pre),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
// All three products are C[m][n] = sum_k A(m, k) B(n, k) on the matrix cores (16 x 16 x 32, float32 accumulation); an operand's contraction index is its contiguous one (x, W, dz for dx) or
// its row index (W for dx; dz and x for dW).  The former is read from LDS as it lies (16 bytes of one row per lane), the latter with the transposing LDS read (4 contraction steps of
// 16 rows per 16 lanes), so no operand is ever transposed in memory.
#include "k3_rowops.h"
#include <algorithm>
#include <type_traits>

namespace {
using namespace k3;

enum { kNone = K3_ACT_NONE, kRelu = K3_ACT_RELU, kSigmoid = K3_ACT_SIGMOID, kTanh = K3_ACT_TANH, kSwish = K3_ACT_SWISH, kGelu = K3_ACT_GELU };

__device__ inline float sigmoid(float z) { return 1.0f / (1.0f + expf(-z)); }
__device__ inline float activation(int act, float z) {
  switch (act) {
    case kRelu: return z < 0.0f ? 0.0f : z;      // (a NaN stays one)
    case kSigmoid: return sigmoid(z);
    case kTanh: return tanhf(z);
    case kSwish: return z * sigmoid(z);
    case kGelu: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    default: return z;
  }
}
__device__ inline float slope(int act, float z) {
  switch (act) {
    case kRelu: return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    case kSigmoid: { const float s = sigmoid(z); return s * (1.0f - s); }
    case kTanh: { const float s = tanhf(z); return 1.0f - s * s; }
    case kSwish: { const float s = sigmoid(z); return s * (1.0f + z * (1.0f - s)); }
    case kGelu: return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
    default: return 1.0f;
  }
}

template <typename T> struct Half;
template <> struct Half<f16> {
  typedef f16 frag __attribute__((ext_vector_type(8)));
  static __device__ inline void mfma(frag a, frag b, float __attribute__((ext_vector_type(4))) &c) { c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Half<bf16> {
  typedef bf16 frag __attribute__((ext_vector_type(8)));
  static __device__ inline void mfma(frag a, frag b, float __attribute__((ext_vector_type(4))) &c) { c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

struct Epilogue {
  void *c; long long ldc;
  float *partial;                  // the contraction in parts: float32 planes [part][M][N], joined by k3_affine_join_kernel
  const float *bias;               // [N] or null
  const void *residual; long long ldr;
  void *pre; long long ldp;
  int act;
};
struct Product { const void *a; long long lda; const void *b; long long ldb; int m, n, k; int tiles_m, tiles_n, parts, steps_per_part; Epilogue e; };

constexpr int BK = 64;             // contraction steps per LDS tile

// 4 consecutive outputs of one row
template <typename T> __device__ inline void finish(const Epilogue &e, long long row, int col, int n, f4 v) {
  typedef T t4 __attribute__((ext_vector_type(4), aligned(2)));
  const T *res = e.residual ? (const T *)e.residual + row * e.ldr + col : nullptr;
  T *c = (T *)e.c + row * e.ldc + col, *pre = e.pre ? (T *)e.pre + row * e.ldp + col : nullptr;
  if (n - col >= 4) {
    typedef float fu __attribute__((ext_vector_type(4), aligned(4)));
    if (e.bias) v += *(const fu *)(e.bias + col);
    if (pre) *(t4 *)pre = __builtin_convertvector(v, t4);
    if (e.act != kNone)
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = activation(e.act, v[j]);
    if (res) v += __builtin_convertvector(*(const t4 *)res, f4);
    *(t4 *)c = __builtin_convertvector(v, t4);
  } else
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (col + j < n) {
        float u = v[j] + (e.bias ? e.bias[col + j] : 0.0f);
        if (pre) pre[j] = (T)u;
        u = activation(e.act, u);
        c[j] = (T)(res ? u + to_f32(res[j]) : u);
      }
}

// what the wavefront's lanes have written to LDS before it they read after it
__device__ inline void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// An LDS tile of ROWS rows (of the operand's output index) by BK contraction steps, in chunks of 8 elements.  ACROSS false: [row][8 chunks], a row's chunk c at c ^ (row / 2 % 8): 16
// lanes that read the same chunk of 16 rows touch every 16-byte column of two LDS rows once.  ACROSS true (the contraction index is the memory row): [step][ROWS / 8 chunks], pairs
// of chunks (16 rows of the operand) exchanged by an XOR with bits of the step that differ among the lanes of one transposing read.
template <int ROWS, bool ACROSS> struct Tile {
  static constexpr int kChunks = ROWS * BK / 8, kBytes = kChunks * 16;
  static __device__ inline int spread(int k) {
    return ROWS >= 128 ? (k & 3) | (k >> 3 & 1) << 2 : ROWS == 64 ? (k >> 1 & 1) | (k >> 3 & 1) << 1 : k >> 3 & 1;
  }
  // LDS position p (in chunks) -> row / step and chunk of the operand
  static __device__ inline void source(int p, int &major, int &chunk) {
    if (ACROSS) {
      major = p / (ROWS / 8);
      const int c = p % (ROWS / 8);
      chunk = ((c >> 1) ^ spread(major)) << 1 | (c & 1);
    } else {
      major = p / 8;
      chunk = (p % 8) ^ (major >> 1 & 7);
    }
  }
  // the fragment of 16 rows from `row` (a multiple of 16) and the contraction steps 32 ks + 8 (lane / 16) ..
  template <typename T> static __device__ inline typename Half<T>::frag fragment(const char *tile, int row, int ks, int lane) {
    if constexpr (ACROSS) {
      const int k = 32 * ks + 8 * (lane >> 4) + (lane & 15) / 4;
      const char *p = tile + k * (ROWS * 2) + ((row >> 4) ^ spread(k)) * 32 + (lane & 3) * 8;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 4 * ROWS * 2));
      return __builtin_bit_cast(typename Half<T>::frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int r = row + (lane & 15), c = 4 * ks + (lane >> 4);
      return *(const typename Half<T>::frag *)(tile + r * 128 + (c ^ (r >> 1 & 7)) * 16);
    }
  }
};

// One operand's way into LDS for a workgroup of THREADS.  direct: global memory to LDS without registers (16-byte aligned rows; chunks that begin behind the operand's last row are read from
// its first one, and their products never stored); otherwise through registers, with zeros where the operand ends, at any alignment.
template <typename T, int ROWS, bool ACROSS, int THREADS> struct Loader {
  using L = Tile<ROWS, ACROSS>;
  static constexpr int N = L::kChunks / THREADS;
  typedef T chunk __attribute__((ext_vector_type(8)));
  const T *base; long long ld; int row0, rows, k;      // the operand, its first row in this tile, its number of rows, and the contraction's length
  const T *at[N];
  __device__ inline void start(int k0) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      int major, c;
      L::source((threadIdx.x / 64 * N + i) * 64 + (threadIdx.x & 63), major, c);
      if (ACROSS) at[i] = base + (long long)(k0 + major) * ld + (row0 + c * 8 < rows ? row0 + c * 8 : 0);
      else at[i] = base + (long long)min(row0 + major, rows - 1) * ld + k0 + c * 8;
    }
  }
  __device__ inline void direct(unsigned lds) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const unsigned to = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x / 64 * N + i) * 1024);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)at[i], (__attribute__((address_space(3))) void *)(unsigned long long)to, 16, 0, 0);
      at[i] += ACROSS ? BK * ld : BK;
    }
  }
  __device__ inline void fetch(int k0, chunk (&v)[N]) const {
    typedef T u8 __attribute__((ext_vector_type(8), aligned(2)));
#pragma unroll
    for (int i = 0; i < N; i++) {
      int major, c;
      L::source((threadIdx.x / 64 * N + i) * 64 + (threadIdx.x & 63), major, c);
      const int row = ACROSS ? k0 + major : row0 + major, col = ACROSS ? row0 + c * 8 : k0 + c * 8, last = ACROSS ? rows : k;
      const T *p = base + (long long)row * ld + col;
      if (row < (ACROSS ? k : rows) && col + 8 <= last) v[i] = *(const u8 *)p;
      else
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] = row < (ACROSS ? k : rows) && col + j < last ? p[j] : (T)0.0f;
    }
  }
  static __device__ inline void store(char *tile, const chunk (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) *(chunk *)(tile + ((threadIdx.x / 64 * N + i) * 64 + (threadIdx.x & 63)) * 16) = v[i];
  }
};

// BM x BN outputs per workgroup of WM x WN wavefronts; two LDS tiles per operand, the next one on its way while the present one is multiplied.
template <typename T, int BM, int BN, int WM, int WN, bool A_ACROSS, bool B_ACROSS, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void k3_affine_product_kernel(Product p) {
  constexpr int THREADS = 64 * WM * WN, MI = BM / WM / 16, NI = BN / WN / 16;
  using TA = Tile<BM, A_ACROSS>;
  using TB = Tile<BN, B_ACROSS>;
  __shared__ __attribute__((aligned(1024))) char lds[2][TA::kBytes + TB::kBytes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
  // workgroups go round the 8 XCDs: each XCD takes a run of neighbouring tiles (columns fastest), which share operands in its L2
  const int tiles = p.tiles_m * p.tiles_n, per = tiles / 8, extra = tiles % 8, x = blockIdx.x % 8, i8 = blockIdx.x / 8;
  const int tile = x * per + min(x, extra) + i8, tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
  const int first = blockIdx.y * p.steps_per_part * BK, end = min(p.k, first + p.steps_per_part * BK), whole = (end - first) / BK, steps = (end - first + BK - 1) / BK;
  Loader<T, BM, A_ACROSS, THREADS> la{(const T *)p.a, p.lda, tm * BM, p.m, p.k};
  Loader<T, BN, B_ACROSS, THREADS> lb{(const T *)p.b, p.ldb, tn * BN, p.n, p.k};
  const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char *)lds[0], stage = TA::kBytes + TB::kBytes;
  f4 acc[MI][NI] = {};
  const auto multiply = [&](const char *ta) {
    const char *tb = ta + TA::kBytes;
#pragma unroll
    for (int ks = 0; ks < BK / 32; ks++) {
      typename Half<T>::frag a[MI], b[NI];
#pragma unroll
      for (int j = 0; j < NI; j++) b[j] = TB::template fragment<T>(tb, wn * (BN / WN) + j * 16, ks, lane);
#pragma unroll
      for (int i = 0; i < MI; i++) a[i] = TA::template fragment<T>(ta, wm * (BM / WM) + i * 16, ks, lane);
#pragma unroll
      for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NI; j++) Half<T>::mfma(b[j], a[i], acc[i][j]);      // (n, m): a lane ends with 4 consecutive n of one m
    }
  };
  if constexpr (DIRECT) {
    la.start(first);
    lb.start(first);
    if (whole) {
      la.direct(lds0);
      lb.direct(lds0 + TA::kBytes);
      __syncthreads();
    }
    for (int s = 0; s < whole; s++) {
      if (s + 1 < whole) {
        la.direct(lds0 + ((s + 1) & 1) * stage);
        lb.direct(lds0 + ((s + 1) & 1) * stage + TA::kBytes);
      }
      multiply(lds[s & 1]);
      __syncthreads();
    }
  }
  // what is left of the contraction (everything, where the operands' alignment does not allow the direct way)
  const int from = DIRECT ? whole : 0;
  if (from < steps) {
    typename Loader<T, BM, A_ACROSS, THREADS>::chunk va[Loader<T, BM, A_ACROSS, THREADS>::N];
    typename Loader<T, BN, B_ACROSS, THREADS>::chunk vb[Loader<T, BN, B_ACROSS, THREADS>::N];
    la.fetch(first + from * BK, va);
    lb.fetch(first + from * BK, vb);
    la.store(lds[0], va);
    lb.store(lds[0] + TA::kBytes, vb);
    __syncthreads();
    for (int s = from; s < steps; s++) {
      const int now = (s - from) & 1;
      if (s + 1 < steps) {
        la.fetch(first + (s + 1) * BK, va);
        lb.fetch(first + (s + 1) * BK, vb);
      }
      multiply(lds[now]);
      if (s + 1 < steps) {
        la.store(lds[now ^ 1], va);
        lb.store(lds[now ^ 1] + TA::kBytes, vb);
      }
      __syncthreads();
    }
  }
  // The epilogue goes through LDS, a part of each wavefront's rows at a time (as many as its share of the tiles' memory holds): out of the accumulators' layout (4 columns of one of 16 rows
  // per lane) into runs of whole rows, so that what is read and written beside it are lines, and so that its code stands here once.  A row's chunk c of 4 lies at c ^ a function of the
  // row that differs among the 16 rows that are written at once.
  constexpr int CW = BN / WN, Q = CW / 4, HOLD = (int)sizeof(lds) / (WM * WN) / (CW * 4), PASS = HOLD < BM / WM ? HOLD / 16 * 16 : BM / WM;
  static_assert(PASS >= 16 && (BM / WM) % PASS == 0, "rows per pass");
  f4 *mine = (f4 *)((char *)lds + wave * ((int)sizeof(lds) / (WM * WN)));
  const int m0 = tm * BM + wm * (BM / WM), n0 = tn * BN + wn * CW;
#pragma unroll
  for (int i0 = 0; i0 < MI; i0 += PASS / 16) {
#pragma unroll
    for (int i = 0; i < PASS / 16; i++)
#pragma unroll
      for (int j = 0; j < NI; j++) {
        const int r = i * 16 + (lane & 15), c = j * 4 + (lane >> 4);
        mine[r * Q + (c ^ (r / (16 / Q) & (Q - 1)))] = acc[i0 + i][j];
      }
    wave_fence();
#pragma unroll 1
    for (int e = lane; e < PASS * Q; e += 64) {
      const int r = e / Q, c = e % Q, col = n0 + c * 4;
      const long long row = m0 + i0 * 16 + r;
      if (row >= p.m || col >= p.n) continue;
      const f4 v = mine[r * Q + (c ^ (r / (16 / Q) & (Q - 1)))];
      if (p.e.partial) {
        float *out = p.e.partial + ((long long)blockIdx.y * p.m + row) * p.n + col;
        typedef float fu __attribute__((ext_vector_type(4), aligned(4)));
        if (p.n - col >= 4) *(fu *)out = v;
        else
#pragma unroll
          for (int k = 0; k < 4; k++) if (col + k < p.n) out[k] = v[k];
      } else finish<T>(p.e, row, col, p.n, v);
    }
    wave_fence();
  }
}

// sums of the contraction's parts, in their order, and the epilogue: 4 columns per thread
template <typename T> __global__ __launch_bounds__(256) void k3_affine_join_kernel(Epilogue e, int m, int n, int parts) {
  const int quads = (n + 3) / 4;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x, row = id / quads;
  const int col = (int)(id - row * quads) * 4;
  if (row >= m) return;
  f4 v = {};
  for (int s = 0; s < parts; s++) {
    const float *in = e.partial + ((long long)s * m + row) * n + col;
    typedef float fu __attribute__((ext_vector_type(4), aligned(4)));
    if (n - col >= 4) v += *(const fu *)in;
    else
#pragma unroll
      for (int j = 0; j < 4; j++) if (col + j < n) v[j] += in[j];
  }
  finish<T>(e, row, col, n, v);
}

// dz = dy act'(pre), rounded to the matrices' type for the products (null: dz is dy), and the sums over a strip of rows of the unrounded values: partial [strip][cols]; a workgroup takes 64
// chunks of 8 columns by one strip, each of its 4 wavefronts every 4th row
template <typename T> __global__ __launch_bounds__(256) void k3_affine_slope_kernel(int act, const T *dy, long long lddy, const T *pre, long long ldp, T *dz, long long lddz, float *partial,
                                                                                     int rows, int cols, int strip) {
  __shared__ float sh[3][64][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = (blockIdx.x * 64 + lane) * 8, valid = cols - col;
  const int r0 = blockIdx.y * strip, r1 = min(rows, r0 + strip);
  float s[8] = {};
  if (valid > 0)
    for (int row = r0 + wave; row < r1; row += 4) {
      const typename Chunk<T>::type g = load_chunk(dy + row * lddy, col, valid);
      typename Chunk<T>::type z = {}, o;
      if (act != kNone) z = load_chunk(pre + row * ldp, col, valid);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float d = act == kNone ? to_f32(g[j]) : to_f32(g[j]) * slope(act, to_f32(z[j]));
        s[j] += d;
        o[j] = (T)d;
      }
      if (dz) store_chunk(dz + row * lddz, col, valid, o);
    }
  if (!partial) return;
  if (wave)
#pragma unroll
    for (int j = 0; j < 8; j++) sh[wave - 1][lane][j] = s[j];
  __syncthreads();
  if (wave == 0)
#pragma unroll
    for (int j = 0; j < 8; j++) if (j < valid) partial[(long long)blockIdx.y * cols + col + j] = ((s[j] + sh[0][lane][j]) + sh[1][lane][j]) + sh[2][lane][j];
}
__global__ __launch_bounds__(1024) void k3_affine_bias_join_kernel(const float *partial, int strips, int cols, float *db) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float v = 0.0f;
  if (c < cols)
#pragma unroll 8
    for (int s = wave; s < strips; s += 16) v += partial[(long long)s * cols + c];
  sh[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < cols) {
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; w++) v += sh[w][lane];
    db[c] = v;
  }
}

// ---- plans

struct Plan { int size, tiles_m, tiles_n, parts, steps_per_part; int64_t bytes; };      // size: 0 = 32 x 64, 1 = 64 x 64, 2 = 128 x 128, 3 = 256 x 256 outputs per workgroup
const int kTile[4][2] = {{32, 64}, {64, 64}, {128, 128}, {256, 256}};

// the largest tile whose tiles (with the contraction in parts where they are few) still cover the 256 compute units
Plan plan_product(int m, int n, int k) {
  const int steps = (k + BK - 1) / BK;
  Plan best{};
  for (int size = 3; size >= 0; size--) {
    if (size > 0 && m <= kTile[size - 1][0] && size < 3) { if (m <= kTile[size - 1][0]) continue; }
    Plan p{};
    p.size = size;
    p.tiles_m = (m + kTile[size][0] - 1) / kTile[size][0];
    p.tiles_n = (n + kTile[size][1] - 1) / kTile[size][1];
    const long long tiles = (long long)p.tiles_m * p.tiles_n;
    const int want = size == 3 ? 200 : 256;
    int parts = 1;
    if (tiles < want) parts = std::max(1, std::min<int>(steps / (size == 0 ? 2 : 4), (int)((want + tiles - 1) / tiles)));
    p.steps_per_part = (steps + parts - 1) / parts;
    p.parts = steps ? (steps + p.steps_per_part - 1) / p.steps_per_part : 1;
    best = p;
    if (tiles * p.parts >= want || size == 0) break;
  }
  best.bytes = best.parts > 1 ? (int64_t)best.parts * m * n * 4 : 0;
  return best;
}

template <typename T, bool A_ACROSS, bool B_ACROSS, bool DIRECT> void launch_product(const Plan &pl, const Product &p, hipStream_t st) {
  const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.parts);
  switch (pl.size) {
    case 0: hipLaunchKernelGGL((k3_affine_product_kernel<T, 32, 64, 1, 4, A_ACROSS, B_ACROSS, DIRECT>), grid, dim3(256), 0, st, p); return;
    case 1: hipLaunchKernelGGL((k3_affine_product_kernel<T, 64, 64, 2, 2, A_ACROSS, B_ACROSS, DIRECT>), grid, dim3(256), 0, st, p); return;
    case 2: hipLaunchKernelGGL((k3_affine_product_kernel<T, 128, 128, 2, 2, A_ACROSS, B_ACROSS, DIRECT>), grid, dim3(256), 0, st, p); return;
    default: hipLaunchKernelGGL((k3_affine_product_kernel<T, 256, 256, 2, 4, A_ACROSS, B_ACROSS, DIRECT>), grid, dim3(512), 0, st, p); return;
  }
}
template <bool ACROSS> bool direct_ok(const void *p, long long ld, int rows) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && (!ACROSS || rows % 8 == 0); }
template <typename T, bool A_ACROSS, bool B_ACROSS> int run_product(Product p, void *workspace, hipStream_t st) {
  const Plan pl = plan_product(p.m, p.n, p.k);
  p.tiles_m = pl.tiles_m; p.tiles_n = pl.tiles_n; p.parts = pl.parts; p.steps_per_part = pl.steps_per_part;
  p.e.partial = pl.parts > 1 ? (float *)workspace : nullptr;
  if (direct_ok<A_ACROSS>(p.a, p.lda, p.m) && direct_ok<B_ACROSS>(p.b, p.ldb, p.n)) launch_product<T, A_ACROSS, B_ACROSS, true>(pl, p, st);
  else launch_product<T, A_ACROSS, B_ACROSS, false>(pl, p, st);
  K3_HIP_CHECK(hipGetLastError());
  if (pl.parts > 1) {
    const long long quads = (long long)p.m * ((p.n + 3) / 4);
    hipLaunchKernelGGL((k3_affine_join_kernel<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, p.e, p.m, p.n, pl.parts);
    K3_HIP_CHECK(hipGetLastError());
  }
  return K3_OK;
}

constexpr int kMaxStrips = 256;
constexpr int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
bool sizes_ok(int rows, int inner, int cols) { return (int64_t)rows * ((int64_t)inner + cols) < (1ll << 42) && inner <= (1 << 20) && cols <= (1 << 22); }

template <typename T> int affine_forward(Product p, void *workspace, hipStream_t st) { return run_product<T, false, false>(p, workspace, st); }
struct Backward { const void *x; long long ldx; const void *w; long long ldw; const void *pre; long long ldp; const void *dy; long long lddy; void *dx; long long lddx; void *dw; long long lddw;
                  float *db; int act, rows, inner, cols; };
template <typename T> int affine_backward(const Backward &q, char *workspace, hipStream_t st) {
  const T *dz = (const T *)q.dy;
  long long lddz = q.lddy;
  char *rest = workspace;
  if (q.act != kNone || q.db) {
    T *out = nullptr;
    float *partial = nullptr;
    if (q.act != kNone && (q.dx || q.dw)) {
      out = (T *)rest;
      dz = out;
      lddz = (q.cols + 7) / 8 * 8;
      rest += up256((int64_t)q.rows * lddz * 2);
    }
    if (q.db) { partial = (float *)rest; rest += up256((int64_t)kMaxStrips * q.cols * 4); }
    const int strip = std::max(16, (q.rows + kMaxStrips - 1) / kMaxStrips), strips = (q.rows + strip - 1) / strip;
    if (q.rows) {
      hipLaunchKernelGGL((k3_affine_slope_kernel<T>), dim3((q.cols + 511) / 512, strips), dim3(256), 0, st, q.act, (const T *)q.dy, q.lddy, (const T *)q.pre, q.ldp, out, lddz, partial,
                         q.rows, q.cols, strip);
      K3_HIP_CHECK(hipGetLastError());
    }
    if (q.db) {
      hipLaunchKernelGGL(k3_affine_bias_join_kernel, dim3((q.cols + 63) / 64), dim3(1024), 0, st, partial, strips, q.cols, q.db);
      K3_HIP_CHECK(hipGetLastError());
    }
  }
  if (q.dx) {
    Product p{};
    p.a = dz; p.lda = lddz; p.b = q.w; p.ldb = q.ldw; p.m = q.rows; p.n = q.inner; p.k = q.cols; p.e.c = q.dx; p.e.ldc = q.lddx;
    const int rc = run_product<T, false, true>(p, rest, st);
    if (rc) return rc;
  }
  if (q.dw) {
    Product p{};
    p.a = dz; p.lda = lddz; p.b = q.x; p.ldb = q.ldx; p.m = q.cols; p.n = q.inner; p.k = q.rows; p.e.c = q.dw; p.e.ldc = q.lddw;
    return run_product<T, true, true>(p, rest, st);
  }
  return K3_OK;
}
}  // namespace

extern "C" int64_t k3_affine_forward_workspace(int32_t rows, int32_t inner, int32_t cols) {
  if (rows <= 0 || inner <= 0 || cols <= 0 || !sizes_ok(rows, inner, cols)) return 0;
  return plan_product(rows, cols, inner).bytes;
}

extern "C" int k3_affine_forward(int32_t dtype, int32_t act, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw, const float *d_bias, const void *d_residual, int64_t ldr, void *d_y,
                                 int64_t ldy, void *d_pre, int64_t ldp, void *d_workspace, int64_t workspace_bytes, int32_t rows, int32_t inner, int32_t cols, void *stream) {
  K3_REQUIRE(dtype == K3_F16 || dtype == K3_BF16, "k3_affine_forward: the types are float16 and bfloat16");
  K3_REQUIRE(act >= kNone && act <= kGelu, "k3_affine_forward: unknown activation");
  K3_REQUIRE(rows >= 0 && inner >= 1 && cols >= 1 && ldx >= inner && ldw >= inner && ldy >= cols && (!d_residual || ldr >= cols) && (!d_pre || ldp >= cols), "k3_affine_forward: bad argument");
  if (!sizes_ok(rows, inner, cols)) { set_error("k3_affine_forward: matrix too large"); return K3_ERR_UNSUPPORTED; }
  if (rows == 0) return K3_OK;
  K3_REQUIRE(d_x && d_w && d_y, "k3_affine_forward: null matrix");
  K3_REQUIRE(workspace_bytes >= k3_affine_forward_workspace(rows, inner, cols) && (d_workspace || workspace_bytes == 0) && ((uintptr_t)d_workspace & 15) == 0,
             "k3_affine_forward: workspace too small or not aligned");
  Product p{};
  p.a = d_x; p.lda = ldx; p.b = d_w; p.ldb = ldw; p.m = rows; p.n = cols; p.k = inner;
  p.e.c = d_y; p.e.ldc = ldy; p.e.bias = d_bias; p.e.residual = d_residual; p.e.ldr = ldr; p.e.pre = d_pre; p.e.ldp = ldp; p.e.act = act;
  return dtype == K3_F16 ? affine_forward<f16>(p, d_workspace, (hipStream_t)stream) : affine_forward<bf16>(p, d_workspace, (hipStream_t)stream);
}

extern "C" int64_t k3_affine_backward_workspace(int32_t act, int32_t rows, int32_t inner, int32_t cols) {
  if (rows <= 0 || inner <= 0 || cols <= 0 || !sizes_ok(rows, inner, cols)) return 0;
  return (act == kNone ? 0 : up256((int64_t)rows * ((cols + 7) / 8 * 8) * 2)) + up256((int64_t)kMaxStrips * cols * 4) +
         std::max(plan_product(rows, inner, cols).bytes, plan_product(cols, inner, rows).bytes);
}

extern "C" int k3_affine_backward(int32_t dtype, int32_t act, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw, const void *d_pre, int64_t ldp, const void *d_dy, int64_t lddy,
                                  void *d_dx, int64_t lddx, void *d_dw, int64_t lddw, float *d_db, void *d_workspace, int64_t workspace_bytes, int32_t rows, int32_t inner, int32_t cols,
                                  void *stream) {
  K3_REQUIRE(dtype == K3_F16 || dtype == K3_BF16, "k3_affine_backward: the types are float16 and bfloat16");
  K3_REQUIRE(act >= kNone && act <= kGelu, "k3_affine_backward: unknown activation");
  K3_REQUIRE(rows >= 0 && inner >= 1 && cols >= 1 && (!d_dw || (ldx >= inner && lddw >= inner)) && (!d_dx || (ldw >= inner && lddx >= inner)) && lddy >= cols && (act == kNone || ldp >= cols),
             "k3_affine_backward: bad argument");
  if (!sizes_ok(rows, inner, cols)) { set_error("k3_affine_backward: matrix too large"); return K3_ERR_UNSUPPORTED; }
  K3_REQUIRE(rows == 0 || (d_dy && (d_x || !d_dw) && (d_w || !d_dx) && (d_pre || act == kNone)), "k3_affine_backward: null input");
  K3_REQUIRE(workspace_bytes >= k3_affine_backward_workspace(act, rows, inner, cols) && (d_workspace || workspace_bytes == 0) && ((uintptr_t)d_workspace & 15) == 0,
             "k3_affine_backward: workspace too small or not aligned");
  const Backward q{d_x, ldx, d_w, ldw, d_pre, ldp, d_dy, lddy, rows ? d_dx : nullptr, lddx, d_dw, lddw, d_db, act, rows, inner, cols};
  return dtype == K3_F16 ? affine_backward<f16>(q, (char *)d_workspace, (hipStream_t)stream) : affine_backward<bf16>(q, (char *)d_workspace, (hipStream_t)stream);
}
