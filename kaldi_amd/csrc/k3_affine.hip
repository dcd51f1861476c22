// k3_affine.hip -- an affine layer in half precision (float16 / bfloat16) with its activation and its bypass in the product's epilogue, and its backward pass (k3_affine_*).
//   forward:  pre = x W^T + b,  y = act(pre) + residual          x [rows x inner], W [cols x inner]
//   backward: dz = dy act'(pre),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz
// All three products are C[m][n] = sum_k A(m, k) B(n, k) on the matrix cores (16 x 16 x 32, float32 accumulation); an operand's contraction index is its contiguous one (x, W, dz for dx) or
// its row index (W for dx; dz and x for dW).  The former is read from LDS as it lies (16 bytes of one row per lane), the latter with the transposing LDS read (4 contraction steps of
// 16 rows per 16 lanes), so no operand is ever transposed in memory.
// Measured in bfloat16: 8192 x 8192 x 8192 938 us forward (1.17 PFLOP/s), 1036 dx, 941 dW; 42752 x 1536 x 1536 with ReLU, bypass and the activation's input kept 234 us (187 without them: the
// epilogues of all compute units come at the same time); 25600 x 768 x 6024 286 us dx, 280 dW (matrix cores busy 36 % of the chip's cycles by counters: what their loads wait for stands at
// k3_affine_product_kernel).
#include "k3_rowops.h"
#include <algorithm>
#include <type_traits>

namespace {
using namespace k3;

enum { kNone = K3_ACT_NONE, kRelu = K3_ACT_RELU, kSigmoid = K3_ACT_SIGMOID, kTanh = K3_ACT_TANH, kSwish = K3_ACT_SWISH, kGelu = K3_ACT_GELU };

__device__ inline float exp_fast(float z) { return __builtin_amdgcn_exp2f(z * 1.44269504088896340736f); }
__device__ inline float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-z)); }
// 1 - 2 / (e^2z + 1), and its series to z^5 where that would cancel
__device__ inline float tanh_fast(float z) {
  const float q = z * z;
  return fabsf(z) < 0.1f ? z * (1.0f + q * (-0.33333333f + q * 0.13333333f)) : 1.0f - 2.0f * __builtin_amdgcn_rcpf(exp_fast(2.0f * z) + 1.0f);
}
// 1 + erf(z / sqrt 2), with e = exp(-z^2 / 2) for who needs it too.  erfc(x) e^(x^2) = t P(t), t = 1 / (1 + 0.4 x), to a relative 1.3e-7 for all x >= 0 (P fitted in float64 to
// the smallest largest relative error): for z < 0 the result is erfc itself, which 1 - (1 - erfc) would leave no digits of
__device__ inline float one_plus_erf(float z, float &e) {
  const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(1.0f + 0.4f * x);
  e = exp_fast(-0.5f * z * z);
  const float c = e * t * (0.225675866f + t * (0.225669608f + t * (0.207842514f + t * (0.168543801f + t * (0.141422957f + t * (-0.00558652263f +
                  t * (0.169057027f + t * (-0.182881743f + t * 0.0502566323f))))))));
  return z < 0.0f ? c : 2.0f - c;
}
// (-inf goes in as a number whose exponential is 0 all the same: 0 times it is 0)
__device__ inline float activation(int act, float z) {
  switch (act) {
    case kRelu: return z < 0.0f ? 0.0f : z;      // (a NaN stays one)
    case kSigmoid: return sigmoid(z);
    case kTanh: return tanh_fast(z);
    case kSwish: z = z < -1e4f ? -1e4f : z; return z * sigmoid(z);
    case kGelu: { float e; z = z < -1e4f ? -1e4f : z; return 0.5f * z * one_plus_erf(z, e); }
    default: return z;
  }
}
__device__ inline float slope(int act, float z) {
  z = z < -1e4f ? -1e4f : z > 1e4f ? 1e4f : z;
  switch (act) {
    case kRelu: return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    // (from t = e^-|z|, sigmoid(|z|) = 1 / (1 + t) and sigmoid(-|z|) = t / (1 + t): 1 - sigmoid(z) would cancel where z is large)
    case kSigmoid: { const float t = exp_fast(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + t); return t * r * r; }
    case kTanh: { const float t = exp_fast(-2.0f * fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + t); return 4.0f * t * r * r; }
    case kSwish: { const float t = exp_fast(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + t), s = z < 0.0f ? t * r : r, c = z < 0.0f ? r : t * r; return s * (1.0f + z * c); }
    case kGelu: { float e; const float f = one_plus_erf(z, e); return 0.5f * f + z * 0.39894228040143268f * e; }
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
  const float *bias;               // [N] or null
  const void *residual; long long ldr;
  void *pre; long long ldp;
  int act;
};
// C [m x n] over k contraction steps, in tiles of `steps` LDS tiles of 64 of them.  The first `whole` tiles are one workgroup's each.  Those behind them (what would leave most of the chip
// idle) are cut into `parts` pieces of their steps each, one workgroup's each: their float32 sums go to partial [tile * parts + part][BM][BN] and are joined by k3_affine_join_kernel.
struct Product { const void *a; long long lda; const void *b; long long ldb; int m, n, k; int tiles_m, tiles_n, whole, parts, steps; float *partial; Epilogue e; };

typedef float f8 __attribute__((ext_vector_type(8)));

// (the choice of the activation outside the loop over the elements: short calls are over before much code has been fetched)
template <int ACT> __device__ inline void activate_as(f8 &v) {
#pragma unroll
  for (int j = 0; j < 8; j++) v[j] = activation(ACT, v[j]);
}
__device__ inline void activate(int act, f8 &v) {
  switch (act) {
    case kRelu: activate_as<kRelu>(v); return;
    case kSigmoid: activate_as<kSigmoid>(v); return;
    case kTanh: activate_as<kTanh>(v); return;
    case kSwish: activate_as<kSwish>(v); return;
    case kGelu: activate_as<kGelu>(v); return;
    default: return;
  }
}

// 8 consecutive outputs of a row, `valid` of which exist
template <typename T> __device__ inline void finish(const Epilogue &e, long long row, int col, int valid, f8 v) {
  typedef typename Chunk<T>::type t8;
  t8 res;
  if (e.residual) res = load_chunk((const T *)e.residual + row * e.ldr, col, valid);
  if (e.bias) {
    float b[8];
    load_params<8>(e.bias, col, valid, 0.0f, b);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] += b[j];
  }
  if (e.pre) store_chunk((T *)e.pre + row * e.ldp, col, valid, __builtin_convertvector(v, t8));
  activate(e.act, v);
  if (e.residual) v += __builtin_convertvector(res, f8);
  store_chunk((T *)e.c + row * e.ldc, col, valid, __builtin_convertvector(v, t8));
}
// U times 8 outputs of the same columns, all of which exist, in rows row0 + u step below m: no activation or ReLU, and what is read for all of them on its way before the first is finished
template <typename T, int U, typename V> __device__ inline void finish_rows(const Epilogue &e, long long row0, int step, int m, int col, V value) {
  typedef typename Chunk<T>::type t8;
  t8 res[U];
  if (e.residual)
#pragma unroll
    for (int u = 0; u < U; u++) res[u] = *(const t8 *)((const T *)e.residual + min(row0 + u * step, m - 1ll) * e.ldr + col);
  float b[8] = {};
  if (e.bias) load_params<8>(e.bias, col, 8, 0.0f, b);
#pragma unroll
  for (int u = 0; u < U; u++) {
    const long long row = row0 + u * step;
    f8 v = value(u);
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] += b[j];
    if (row < m) {
      if (e.pre) *(t8 *)((T *)e.pre + row * e.ldp + col) = __builtin_convertvector(v, t8);
      if (e.act == kRelu)
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = activation(kRelu, v[j]);
      if (e.residual) v += __builtin_convertvector(res[u], f8);
      *(t8 *)((T *)e.c + row * e.ldc + col) = __builtin_convertvector(v, t8);
    }
  }
}

// what the wavefront's lanes have written to LDS before it they read after it
__device__ inline void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// An LDS tile of ROWS rows (of the operand's output index) by BK contraction steps, in chunks of 8 elements and blocks of 64 of them (what a wavefront loads at once).
// ACROSS false: [row][BK / 8 chunks], a row's chunk c at c ^ a function of the row such that 16 lanes that read the same chunk of 16 rows touch every 16-byte column of 256 bytes once.
// ACROSS true (the contraction index is the memory row): a block holds 512 / ROWS steps of all rows; the 4 steps that 16 lanes read at once with one transposing read lie in the 4 blocks of
// a set, which are 32 bytes more than their size apart and so start in different banks, and neighbouring groups of lanes read from different sets (or from halves of a block 128 bytes
// apart).  (No XOR: a lane's reads of all its rows differ by constants alone.)
template <int ROWS, int BK, bool ACROSS> struct Tile {
  static constexpr int kChunks = ROWS * BK / 8, CH = BK / 8, kBlock = ACROSS ? 1056 : 1024, kBytes = kChunks / 64 * kBlock, SETS = kChunks / 256;
  static __device__ inline int spread(int row) { return row / (16 / CH) & (CH - 1); }
  // chunk p of the tile in the order of LDS -> row / step and chunk of the operand
  static __device__ inline void source(int p, int &major, int &chunk) {
    if constexpr (ACROSS) {
      const int block = p / 64, slot = p % 64 / (ROWS / 8);
      major = (slot / 2 * SETS + block / 4) * 8 + slot % 2 * 4 + block % 4;
      chunk = p % (ROWS / 8);
    } else {
      major = p / CH;
      chunk = (p % CH) ^ spread(major);
    }
  }
  // the fragment of 16 rows from `row` (a multiple of 16) and the contraction steps 32 ks + 8 (lane / 16) ..
  template <typename T> static __device__ inline typename Half<T>::frag fragment(const char *tile, int row, int ks, int lane) {
    if constexpr (ACROSS) {
      const int set = SETS == 8 ? 4 * ks + (lane >> 4) : (lane >> 4) % SETS, slot = SETS == 8 ? 0 : 2 * ((4 * ks + (lane >> 4)) / SETS), block = set * 4 + (lane & 15) / 4;
      const char *p = tile + block * kBlock + slot * (ROWS * 2) + (lane & 3) * 8 + row * 2;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + ROWS * 2));
      return __builtin_bit_cast(typename Half<T>::frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int r = row + (lane & 15), c = 4 * ks + (lane >> 4);
      return *(const typename Half<T>::frag *)(tile + r * (BK * 2) + (c ^ spread(lane & 15)) * 16);
    }
  }
};

// One operand's way into LDS for a workgroup of THREADS.  direct: global memory to LDS without registers (16-byte aligned rows; chunks that begin behind the operand's last row are read from
// its first one, and their products never stored); otherwise through registers, with zeros where the operand ends, at any alignment.
template <typename T, int ROWS, int BK, bool ACROSS, int THREADS> struct Loader {
  using L = Tile<ROWS, BK, ACROSS>;
  static constexpr int N = L::kChunks / THREADS;
  typedef Packed chunk;
  const T *base; long long ld; int row0, rows, k;      // the operand, its first row in this tile, its number of rows, and the contraction's length
  int wave, lane;
  const char *from;      // uniform: where the next tile's offsets count from
  unsigned offset[N];
  __device__ inline void start(int k0) {
    from = (const char *)(base + (ACROSS ? (long long)k0 * ld : (long long)row0 * ld + k0));
#pragma unroll
    for (int i = 0; i < N; i++) {
      int major, c;
      L::source((wave * N + i) * 64 + lane, major, c);
      if (ACROSS) offset[i] = 2u * (unsigned)(major * (int)ld + (row0 + c * 8 < rows ? row0 + c * 8 : 0));
      else offset[i] = 2u * (unsigned)(min(major, rows - 1 - row0) * (int)ld + c * 8);
    }
  }
  __device__ inline void direct(unsigned lds) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const unsigned to = lds + (wave * N + i) * L::kBlock;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from + offset[i]), (__attribute__((address_space(3))) void *)(unsigned long long)to, 16, 0, 0);
    }
    from += ACROSS ? 2 * BK * ld : 2 * BK;
  }
  __device__ inline void fetch(int k0, chunk (&v)[N]) const {
    typedef T u8 __attribute__((ext_vector_type(8), aligned(2)));
#pragma unroll
    for (int i = 0; i < N; i++) {
      int major, c;
      L::source((wave * N + i) * 64 + lane, major, c);
      const int row = ACROSS ? k0 + major : row0 + major, col = ACROSS ? row0 + c * 8 : k0 + c * 8, last = ACROSS ? rows : k;
      const bool there = row < (ACROSS ? k : rows);      // (a row behind the last one: read from the first, and cleared)
      const T *p = base + (there ? (long long)row * ld : 0);
      Packed w;
      if (last - col >= 8) w = __builtin_bit_cast(Packed, *(const u8 *)(p + col));
      else w = load_packed<T>(p, col, last - col, (T)0.0f);
      v[i] = there ? w : Packed{0, 0, 0, 0};
    }
  }
  __device__ inline void store(char *tile, const chunk (&v)[N]) const {
#pragma unroll
    for (int i = 0; i < N; i++) *(chunk *)(tile + (wave * N + i) * L::kBlock + lane * 16) = v[i];
  }
};

// a barrier behind which the LDS loads that the workgroup's wavefronts issued are there, but for each one's last LEFT, and their LDS reads are done (raw, so that nothing else is waited
// for); no memory operation crosses it
template <int LEFT> __device__ inline void arrive() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory"); }

// tiles in panels of 8 columns of them, row after row within a panel: any 32 neighbours (what an XCD works on at once) share few rows and columns of the operands
__device__ inline void place(const Product &p, int tile, int &tm, int &tn) {
  const int panel = tile / (8 * p.tiles_m), rest = tile - panel * 8 * p.tiles_m, width = min(8, p.tiles_n - panel * 8);
  tm = rest / width;
  tn = panel * 8 + rest - tm * width;
}

// BM x BN outputs per workgroup of WM x WN wavefronts, over STAGES LDS tiles of 64 contraction steps: one is multiplied while the others are loaded.  PIPED (the size of which a compute
// unit holds one workgroup): a tile is two halves of 32 steps for the matrix instructions, and the fragments of a half are read from LDS among the instructions of the half before it, those
// of the next tile's first half too: the one barrier per tile stands between the halves, where every wavefront has read all of this tile (which the loads issued behind the barrier then
// overwrite) and the next one has arrived.
// Where an operand is ACROSS, the compiler takes its transposing LDS reads to depend on every load into LDS under way and waits for all of them first: the loads of a tile, issued right
// before those reads, then have no time but what the compute unit's other wavefronts take, and the rings of 3 and 4 tiles hold nothing in flight.
template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool A_ACROSS, bool B_ACROSS, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void k3_affine_product_kernel(Product p) {
  constexpr int THREADS = 64 * WM * WN, MI = BM / WM / 16, NI = BN / WN / 16, BK = 64;
  constexpr bool PIPED = BM == 256;
  static_assert(!PIPED || STAGES == 2, "the order of a piped tile is that of two");
  using TA = Tile<BM, BK, A_ACROSS>;
  using TB = Tile<BN, BK, B_ACROSS>;
  using LA = Loader<T, BM, BK, A_ACROSS, THREADS>;
  using LB = Loader<T, BN, BK, B_ACROSS, THREADS>;
  constexpr int kStage = TA::kBytes + TB::kBytes;
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * kStage];
  // workgroups go round the 8 XCDs: each XCD takes neighbouring tiles, which share operands in its L2; so do the parts of the last tiles
  const bool split = (int)blockIdx.x >= p.whole;
  const int count = split ? (int)gridDim.x - p.whole : p.whole, u = split ? blockIdx.x - p.whole : blockIdx.x;
  const int per = count / 8, extra = count % 8, x = u % 8, unit = x * per + min(x, extra) + u / 8;
  const int t = split ? unit / p.parts : unit, part = split ? unit - t * p.parts : 0;
  const int step0 = split ? (int)((long long)part * p.steps / p.parts) : 0, step1 = split ? (int)((long long)(part + 1) * p.steps / p.parts) : p.steps;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  int tm, tn;
  place(p, split ? p.whole + t : t, tm, tn);
  const int first = step0 * BK, end = min(p.k, step1 * BK);
  const int direct = DIRECT ? (end - first) / BK : 0, steps = (end - first + BK - 1) / BK;
  LA la{(const T *)p.a, p.lda, tm * BM, p.m, p.k, wave, lane};
  LB lb{(const T *)p.b, p.ldb, tn * BN, p.n, p.k, wave, lane};
  f4 acc[MI][NI] = {};
  typedef typename Half<T>::frag frag;
  const auto read = [&](const char *ta, int ks, frag (&a)[MI], frag (&b)[NI]) {
#pragma unroll
    for (int j = 0; j < NI; j++) b[j] = TB::template fragment<T>(ta + TA::kBytes, wn * (BN / WN) + j * 16, ks, lane);
#pragma unroll
    for (int i = 0; i < MI; i++) a[i] = TA::template fragment<T>(ta, wm * (BM / WM) + i * 16, ks, lane);
  };
  const auto multiply = [&](const frag (&a)[MI], const frag (&b)[NI]) {
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
      for (int j = 0; j < NI; j++) Half<T>::mfma(b[j], a[i], acc[i][j]);      // (n, m): a lane ends with 4 consecutive n of one m
  };
  // the order of a half: its LDS reads spread over the first part of its matrix instructions
  constexpr int READS = (A_ACROSS ? 2 : 1) * MI + (B_ACROSS ? 2 : 1) * NI, PER = MI * NI / READS > 0 ? MI * NI / READS : 1;
  const auto interleave = [&]() {
#pragma unroll
    for (int i = 0; i < READS; i++) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MI * NI, 0);
  };
  if constexpr (DIRECT) {
    if (direct) {
      const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char *)lds;
      la.start(first);
      lb.start(first);
      unsigned load = 0;      // where the next tile goes
      const auto issue = [&](int) {
        la.direct(lds0 + load);
        lb.direct(lds0 + load + TA::kBytes);
        load = load == (STAGES - 1) * kStage ? 0 : load + kStage;
      };
      issue(0);
      if constexpr (PIPED) {
        frag a0[MI], b0[NI], a1[MI], b1[NI];
        arrive<0>();
        if (direct > 1) issue(1);
        read(lds, 0, a0, b0);
        const auto step = [&](int s, auto loads) {
          read(lds + (s & 1) * kStage, 1, a1, b1);
          multiply(a0, b0);
          interleave();
          arrive<0>();
          if constexpr (decltype(loads)::value) issue(s);
          __builtin_amdgcn_sched_barrier(0);      // (the loads at once: left to itself the compiler puts them behind most of the matrix instructions)
          read(lds + ((s & 1) ^ 1) * kStage, 0, a0, b0);      // (behind the last tile: something from LDS, for nothing)
          multiply(a1, b1);
          interleave();
        };
        int s = 0;
        for (; s + 2 < direct; s++) step(s, std::true_type());
        for (; s < direct; s++) step(s, std::false_type());
      } else {
        // STAGES - 1 tiles are on their way while one is multiplied
#pragma unroll
        for (int i = 1; i < STAGES - 1; i++) if (i < direct) issue(i);
        unsigned now = 0;
        for (int s = 0; s < direct; s++) {
          if (s + STAGES - 2 < direct) arrive<(STAGES - 2) * (LA::N + LB::N)>();
          else arrive<0>();
          if (s + STAGES - 1 < direct) issue(s + STAGES - 1);
          frag a[MI], b[NI];
#pragma unroll
          for (int ks = 0; ks < 2; ks++) {
            read(lds + now, ks, a, b);
            multiply(a, b);
          }
          now = now == (STAGES - 1) * kStage ? 0 : now + kStage;
        }
      }
      __syncthreads();
    }
  }
  // what is left of the contraction (everything, where the operands' alignment does not allow the direct way): through registers, R tiles of them on their way
  if (direct < steps) {
    constexpr int R = DIRECT || BM >= 128 ? 1 : 3;      // (two of 128 x 128 would leave a compute unit one workgroup instead of two)
    typename LA::chunk va[R][LA::N];
    typename LB::chunk vb[R][LB::N];
    la.fetch(first + direct * BK, va[0]);
    lb.fetch(first + direct * BK, vb[0]);
    la.store(lds, va[0]);
    lb.store(lds + TA::kBytes, vb[0]);
#pragma unroll
    for (int r = 0; r < R; r++)
      if (direct + 1 + r < steps) {
        la.fetch(first + (direct + 1 + r) * BK, va[r]);
        lb.fetch(first + (direct + 1 + r) * BK, vb[r]);
      }
    __syncthreads();
    for (int s0 = direct; s0 < steps; s0 += R)
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int s = s0 + r, now = (s - direct) & 1;
        if (s >= steps) break;
        frag a[MI], b[NI];
#pragma unroll
        for (int ks = 0; ks < 2; ks++) {
          read(lds + now * kStage, ks, a, b);
          multiply(a, b);
        }
        if (s + 1 < steps) {
          la.store(lds + (now ^ 1) * kStage, va[r]);
          lb.store(lds + (now ^ 1) * kStage + TA::kBytes, vb[r]);
          if (s + 1 + R < steps) {
            la.fetch(first + (s + 1 + R) * BK, va[r]);
            lb.fetch(first + (s + 1 + R) * BK, vb[r]);
          }
        }
        __syncthreads();
      }
  }
  // The epilogue goes through LDS, a part of each wavefront's rows at a time (as many as its share of the tiles' memory holds): out of the accumulators' layout (4 columns of one of 16 rows
  // per lane) into runs of whole rows, so that what is read and written beside it are lines.  A row's chunk c of 4 lies at c ^ a function of the row that differs among the 16 rows that are
  // written at once.
  constexpr int CW = BN / WN, Q = CW / 4, SHARE = (int)sizeof(lds) / (WM * WN) / 16 * 16, HOLD = SHARE / (CW * 4) / 16 * 16;
  constexpr int PASS = HOLD >= BM / WM ? BM / WM : BM / WM / 2, STRIDE = 64 / (Q / 2), U = PASS / STRIDE;      // rows per pass, rows between a lane's, and rows per lane
  static_assert(PASS >= 16 && PASS <= HOLD && (BM / WM) % PASS == 0 && U >= 1, "rows per pass");
  f4 *mine = (f4 *)(lds + wave * SHARE);
  const int m0 = tm * BM + wm * (BM / WM), n0 = tn * BN + wn * CW;
  float *sums = p.partial + (long long)unit * (BM * BN) + wm * (BM / WM) * BN + wn * CW;
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
    const int r0 = lane / (Q / 2), c = lane % (Q / 2) * 2;      // this lane's first row and columns of the pass
    const auto value = [&](int u) {
      const int r = r0 + u * STRIDE, f = r / (16 / Q) & (Q - 1);
      return __builtin_shufflevector(mine[r * Q + (c ^ f)], mine[r * Q + ((c + 1) ^ f)], 0, 1, 2, 3, 4, 5, 6, 7);
    };
    if (split) {
#pragma unroll 1
      for (int u = 0; u < U; u++) *(f8 *)(sums + (i0 * 16 + r0 + u * STRIDE) * BN + c * 4) = value(u);
    } else if (n0 + CW <= p.n && p.e.act <= kRelu) finish_rows<T, U>(p.e, m0 + i0 * 16 + r0, STRIDE, p.m, n0 + c * 4, value);
    else
#pragma unroll 1
      for (int u = 0; u < U; u++) {
        const long long row = m0 + i0 * 16 + r0 + u * STRIDE;
        if (row < p.m && n0 + c * 4 < p.n) finish<T>(p.e, row, n0 + c * 4, p.n - n0 - c * 4, value(u));
      }
    wave_fence();
  }
}

// the sums of a cut tile's pieces, in their order, and the epilogue: 8 columns per thread
template <typename T> __global__ __launch_bounds__(256) void k3_affine_join_kernel(Product p, int bm, int bn) {
  const int groups = bm * bn / 2048, t = blockIdx.x / groups, e = (blockIdx.x - t * groups) * 256 + threadIdx.x, r = e / (bn / 8), c = e % (bn / 8) * 8;
  int tm, tn;
  place(p, p.whole + t, tm, tn);
  const long long row = (long long)tm * bm + r;
  const int col = tn * bn + c;
  if (row >= p.m || col >= p.n) return;
  const float *in = p.partial + (long long)t * p.parts * bm * bn + r * bn + c;
  f8 v = *(const f8 *)in;
#pragma unroll 4
  for (int u = 1; u < p.parts; u++) v += *(const f8 *)(in + (long long)u * bm * bn);
  finish<T>(p.e, row, col, p.n - col, v);
}

template <int ACT, typename T> __device__ inline void slopes_of(Packed z, float (&d)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j++) d[j] = slope(ACT, element<T>(z, j));
}
template <typename T> __device__ inline void slopes(int act, Packed z, float (&d)[8]) {
  switch (act) {
    case kRelu: slopes_of<kRelu, T>(z, d); return;
    case kSigmoid: slopes_of<kSigmoid, T>(z, d); return;
    case kTanh: slopes_of<kTanh, T>(z, d); return;
    case kSwish: slopes_of<kSwish, T>(z, d); return;
    case kGelu: slopes_of<kGelu, T>(z, d); return;
    default: return;
  }
}
// dz = dy act'(pre), rounded to the matrices' type for the products (null: dz is dy), and the sums over a strip of rows of the unrounded values: sums [strip][cols].  The rounding is what
// the matrix cores ask for: float32's other bits would go into a second half and a second product each.  It is as large as that of dy itself (none for ReLU): dx and dW of 4096 x 768 <- 1536
// with gelu are 2.3e-3 off in bfloat16 where one rounding makes 1.7e-3 (2.9e-4 and 2.1e-4 in float16, in which a dz below 2^-25 is lost).  A workgroup takes 64
// chunks of 8 columns by one strip, each of its 4 wavefronts every 4th row, the next one on its way while this one is worked on.  (Small code counts: short calls are over before much of it has
// been fetched.  4 rows at a time, with their activations written out, took 12.8 us on 208 rows of 173 columns.)
template <typename T> __global__ __launch_bounds__(256) void k3_affine_slope_kernel(int act, const T *dy, long long lddy, const T *pre, long long ldp, T *dz, long long lddz, float *sums,
                                                                                     int rows, int cols, int strip) {
  __shared__ float sh[3][64][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = (blockIdx.x * 64 + lane) * 8, valid = cols - col;
  const int r0 = blockIdx.y * strip, r1 = min(rows, r0 + strip);
  float s[8] = {};
  if (valid > 0) {
    Packed g, z = {}, ng = {}, nz = {};
    const auto load = [&](long long row) {
      ng = load_packed<T>(dy + row * lddy, col, valid, (T)0.0f);
      if (act != kNone) nz = load_packed<T>(pre + row * ldp, col, valid, (T)0.0f);
    };
    if (r0 + wave < r1) load(r0 + wave);
#pragma unroll 1
    for (int row = r0 + wave; row < r1; row += 4) {
      g = ng;
      z = nz;
      if (row + 4 < r1) load(row + 4);
      float d[8];
      slopes<T>(act, z, d);
      typename Chunk<T>::type o;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        d[j] = act == kNone ? element<T>(g, j) : element<T>(g, j) * d[j];
        s[j] += d[j];
        o[j] = (T)d[j];
      }
      if (dz) store_chunk(dz + (long long)row * lddz, col, valid, o);
    }
  }
  if (!sums) return;
  if (wave)
#pragma unroll
    for (int j = 0; j < 8; j++) sh[wave - 1][lane][j] = s[j];
  __syncthreads();
  if (wave == 0)
#pragma unroll
    for (int j = 0; j < 8; j++) if (j < valid) sums[(long long)blockIdx.y * cols + col + j] = ((s[j] + sh[0][lane][j]) + sh[1][lane][j]) + sh[2][lane][j];
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

// A workgroup's outputs, how many workgroups the chip holds at once, and how long an LDS tile of 64 steps takes, in us: alone on its compute unit, and each of those that share one when there
// are enough of them to keep it busy.  Measured in bf16 (one size for all of a product): 2048 x 2048 x 2048 in 50.6 / 27.7 / 27.0 / 39.2 us from the largest size to the smallest,
// 512 x 4096 x 2048 in 49.1 / 25.7 / 15.8 / 19.2, 32 x 8192 x 1024 in 25.8 / 13.6 / 7.8 / 7.0, 42752 x 1536 x 1536 in 173 / 192 / - / -.
struct Size { int bm, bn, slots; double alone, shared; };
const Size kSizes[4] = {{32, 64, 1536, 0.25, 0.115}, {64, 64, 1024, 0.3, 0.19}, {128, 128, 512, 0.7, 0.5}, {256, 256, 256, 1.5, 1.7}};
constexpr int kStep = 64;
struct Plan { int size, tiles_m, tiles_n, whole, parts, steps; int64_t bytes; };      // parts 0: no tile is cut

// The size, and the parts of the last tiles, that cost least by a model of rounds over the chip: rounds of whole tiles, the parts, and their sums' way through memory.  A whole number of
// parts per tile: 256 equal runs over 72 tiles of 400 steps keep every unit busy, but no two of them are then at the same step and share an operand, and a weight derivative of
// 6024 x 768 over 25600 rows took 346 us against 293 in 3 parts per tile.
Plan plan_product(int m, int n, int k) {
  Plan best{};
  double least = 1e300;
  for (int size = 0; size < 4; size++) {
    const Size &z = kSizes[size];
    const long long tm = (m + z.bm - 1) / z.bm, tn = (n + z.bn - 1) / z.bn, tiles = tm * tn, steps = std::max(1, (k + kStep - 1) / kStep);
    if ((tiles + 2 * z.slots) * (size == 3 ? 512 : 256) >= 1ll << 32) continue;      // (threads of a launch)
    const auto round = [&](long long units, double each) { return (each + 2.0) * std::max(z.alone, (double)((units + 255) / 256) * z.shared); };
    const auto rounds = [&](long long units, double each) { return (units / z.slots) * round(z.slots, each) + (units % z.slots ? round(units % z.slots, each) : 0.0); };
    const auto consider = [&](long long whole, int parts, double us) {
      if (us >= least) return;
      least = us;
      best = {size, (int)tm, (int)tn, (int)whole, parts, (int)steps, (int64_t)(tiles - whole) * parts * z.bm * z.bn * 4};
    };
    consider(tiles, 0, rounds(tiles, steps));
    const long long whole = tiles / z.slots * z.slots, rest = tiles - whole;
    if (rest == 0) continue;
    for (int parts = 2; parts <= 16 && rest * parts <= 2 * z.slots && steps >= 2 * parts; parts++) {
      const long long units = rest * parts;
      const double bytes = (double)units * z.bm * z.bn * 4, each = (double)steps / parts;
      consider(whole, parts, rounds(whole, steps) + rounds(units, each) + 3.0 + 2.0 * bytes / 5e6);
    }
  }
  return best;
}

template <typename T, bool A_ACROSS, bool B_ACROSS, bool DIRECT> void launch_product(const Plan &pl, const Product &p, hipStream_t st) {
  const dim3 grid((unsigned)(p.whole + (p.tiles_m * p.tiles_n - p.whole) * p.parts));
  switch (pl.size) {
    case 0: hipLaunchKernelGGL((k3_affine_product_kernel<T, 32, 64, 1, 4, 4, A_ACROSS, B_ACROSS, DIRECT>), grid, dim3(256), 0, st, p); return;
    case 1: hipLaunchKernelGGL((k3_affine_product_kernel<T, 64, 64, 2, 2, 3, A_ACROSS, B_ACROSS, DIRECT>), grid, dim3(256), 0, st, p); return;
    case 2: hipLaunchKernelGGL((k3_affine_product_kernel<T, 128, 128, 2, 2, 2, A_ACROSS, B_ACROSS, DIRECT>), grid, dim3(256), 0, st, p); return;
    default: hipLaunchKernelGGL((k3_affine_product_kernel<T, 256, 256, 2, 4, 2, A_ACROSS, B_ACROSS, DIRECT>), grid, dim3(512), 0, st, p); return;
  }
}
// 16-byte aligned rows, whole chunks, and offsets within a tile that fit 32 bits
template <bool ACROSS> bool direct_ok(const void *p, long long ld, int rows) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld <= 1 << 22 && (!ACROSS || rows % 8 == 0); }
template <typename T, bool A_ACROSS, bool B_ACROSS> int run_product(Product p, void *workspace, hipStream_t st) {
  const Plan pl = plan_product(p.m, p.n, p.k);
  K3_REQUIRE(pl.steps > 0, "k3_affine: matrix too large");
  p.tiles_m = pl.tiles_m; p.tiles_n = pl.tiles_n; p.whole = pl.whole; p.parts = pl.parts; p.steps = pl.steps;
  p.partial = (float *)workspace;
  if (direct_ok<A_ACROSS>(p.a, p.lda, p.m) && direct_ok<B_ACROSS>(p.b, p.ldb, p.n)) launch_product<T, A_ACROSS, B_ACROSS, true>(pl, p, st);
  else launch_product<T, A_ACROSS, B_ACROSS, false>(pl, p, st);
  K3_HIP_CHECK(hipGetLastError());
  if (pl.bytes) {
    const Size &z = kSizes[pl.size];
    hipLaunchKernelGGL((k3_affine_join_kernel<T>), dim3((unsigned)((p.tiles_m * p.tiles_n - p.whole) * (z.bm * z.bn / 2048))), dim3(256), 0, st, p, z.bm, z.bn);
    K3_HIP_CHECK(hipGetLastError());
  }
  return K3_OK;
}

constexpr int kMaxStrips = 256;
constexpr int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }
bool sizes_ok(int rows, int inner, int cols) { return rows <= 1 << 30 && (int64_t)rows * ((int64_t)inner + cols) < (1ll << 42) && inner <= (1 << 20) && cols <= (1 << 22); }
int64_t sums_bytes(int rows, int cols) { return up256((int64_t)std::min((rows + 3) / 4, kMaxStrips) * cols * 4); }      // of the slope kernel: a strip is 4 rows at least

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
    if (q.db) { partial = (float *)rest; rest += sums_bytes(q.rows, q.cols); }
    // enough strips to fill the chip, of a row per wavefront at least; a single one writes the sums at their place
    const int across = (q.cols + 511) / 512, least = (q.rows + kMaxStrips - 1) / kMaxStrips;
    const int strip = std::max({4, least, (int)((long long)q.rows * across / 2048)}), strips = (q.rows + strip - 1) / strip;
    if (q.rows) {
      hipLaunchKernelGGL((k3_affine_slope_kernel<T>), dim3(across, strips), dim3(256), 0, st, q.act, (const T *)q.dy, q.lddy, (const T *)q.pre, q.ldp, out, lddz,
                         q.db && strips == 1 ? q.db : partial, q.rows, q.cols, strip);
      K3_HIP_CHECK(hipGetLastError());
    }
    if (q.db && strips != 1) {
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
  const Span x = matrix_span(d_x, ldx, rows, inner, 2), w = matrix_span(d_w, ldw, cols, inner, 2), b = vector_span(d_bias, cols), r = matrix_span(d_residual, ldr, rows, cols, 2),
             y = matrix_span(d_y, ldy, rows, cols, 2), pre = matrix_span(d_pre, ldp, rows, cols, 2);
  K3_REQUIRE(!on_any(y, {x, w, b, pre}) && !on_any(pre, {x, w, b, r}) && (same(y, r) || !overlap(y, r)), "k3_affine_forward: an output lies on another matrix");
  K3_REQUIRE(workspace_bytes >= k3_affine_forward_workspace(rows, inner, cols) && (d_workspace || workspace_bytes == 0) && ((uintptr_t)d_workspace & 15) == 0,
             "k3_affine_forward: workspace too small or not aligned");
  Product p{};
  p.a = d_x; p.lda = ldx; p.b = d_w; p.ldb = ldw; p.m = rows; p.n = cols; p.k = inner;
  p.e.c = d_y; p.e.ldc = ldy; p.e.bias = d_bias; p.e.residual = d_residual; p.e.ldr = ldr; p.e.pre = d_pre; p.e.ldp = ldp; p.e.act = act;
  return dtype == K3_F16 ? affine_forward<f16>(p, d_workspace, (hipStream_t)stream) : affine_forward<bf16>(p, d_workspace, (hipStream_t)stream);
}

extern "C" int64_t k3_affine_backward_workspace(int32_t act, int32_t rows, int32_t inner, int32_t cols) {
  if (rows <= 0 || inner <= 0 || cols <= 0 || !sizes_ok(rows, inner, cols)) return 0;
  return (act == kNone ? 0 : up256((int64_t)rows * ((cols + 7) / 8 * 8) * 2)) + sums_bytes(rows, cols) +
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
  const Span x = matrix_span(ldx >= inner ? d_x : nullptr, ldx, rows, inner, 2), w = matrix_span(ldw >= inner ? d_w : nullptr, ldw, cols, inner, 2), dy = matrix_span(d_dy, lddy, rows, cols, 2),
             pre = matrix_span(act == kNone ? nullptr : d_pre, ldp, rows, cols, 2), dx = matrix_span(d_dx, lddx, rows, inner, 2), dw = matrix_span(d_dw, lddw, cols, inner, 2), db = vector_span(d_db, cols);
  K3_REQUIRE(rows == 0 || (!on_any(dx, {x, w, dy, pre}) && !on_any(dw, {x, w, dy, pre})), "k3_affine_backward: an output lies on an input");
  K3_REQUIRE(!overlap(dx, dw) && !on_any(db, {dx, dw}), "k3_affine_backward: the outputs lie on each other");
  K3_REQUIRE(workspace_bytes >= k3_affine_backward_workspace(act, rows, inner, cols) && (d_workspace || workspace_bytes == 0) && ((uintptr_t)d_workspace & 15) == 0,
             "k3_affine_backward: workspace too small or not aligned");
  K3_REQUIRE(rows == 0 || !on_any(db, {x, w, dy, pre}), "k3_affine_backward: an output lies on an input");
  const Backward q{d_x, ldx, d_w, ldw, d_pre, ldp, d_dy, lddy, rows ? d_dx : nullptr, lddx, d_dw, lddw, d_db, act, rows, inner, cols};
  return dtype == K3_F16 ? affine_backward<f16>(q, (char *)d_workspace, (hipStream_t)stream) : affine_backward<bf16>(q, (char *)d_workspace, (hipStream_t)stream);
}
