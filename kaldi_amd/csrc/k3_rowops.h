// k3_rowops.h -- device helpers shared by the operators that work on rows of float / half / bfloat16 matrices (k3_layernorm.hip, k3_objf.hip) and by k3_affine.hip.
#pragma once
#include "k3_common.h"
#include <type_traits>

namespace k3 {

typedef _Float16 f16;
typedef __bf16 bf16;

// 16 bytes of a row.  The alignment is the element's: rows may start anywhere (odd widths, padded strides), and gfx950's global loads and stores of four registers take any address.
template <typename T> struct Chunk { static constexpr int N = 16 / (int)sizeof(T); typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))); };

template <typename T> __device__ inline float to_f32(T v) { return (float)v; }

template <typename T> __device__ inline void store_chunk(T *row, int col, int valid, typename Chunk<T>::type v) {
  if (valid >= Chunk<T>::N) { *reinterpret_cast<typename Chunk<T>::type *>(row + col) = v; return; }
#pragma unroll
  for (int j = 0; j < Chunk<T>::N; j++) if (j < valid) row[col + j] = v[j];
}
// A chunk as it is stored, in four registers whatever its type (a vector of halves that comes out of two branches is taken apart by the compiler, into a register per element)
typedef int Packed __attribute__((ext_vector_type(4)));
template <typename T> __device__ inline float element(Packed v, int j) {
  const int w = sizeof(T) == 4 ? v[j] : v[j / 2];
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w);
  else if constexpr (std::is_same<T, bf16>::value) return __builtin_bit_cast(float, j & 1 ? w & (int)0xffff0000 : w << 16);
  else return (float)__builtin_bit_cast(f16, (unsigned short)(j & 1 ? (unsigned)w >> 16 : w & 0xffff));
}
// what is widened behind this is widened again, and not kept in float32 from before (twice the registers)
template <typename T, int E> __device__ inline void keep_packed(Packed (&v)[E]) {
  if constexpr (sizeof(T) == 2)
#pragma unroll
    for (int i = 0; i < E; i++) asm volatile("" : "+v"(v[i]));
}
// The chunk at column col of a row of col + valid columns: `valid` elements of it exist (none: <= 0), `otherwise` stands behind them.  Where the row ends inside it, the row's last 16 bytes are
// read and moved down: element by element it would be N loads instead of one, and under conditions they would wait for each other.
template <typename T> __device__ inline Packed load_packed(const T *row, int col, int valid, T otherwise) {
  constexpr int N = Chunk<T>::N, BITS = 8 * (int)sizeof(T);
  typedef unsigned __int128 u128;
  if (valid >= N) return __builtin_bit_cast(Packed, *reinterpret_cast<const typename Chunk<T>::type *>(row + col));
  Packed fill;
  if constexpr (sizeof(T) == 4) fill = Packed{1, 1, 1, 1} * __builtin_bit_cast(int, otherwise);
  else fill = Packed{1, 1, 1, 1} * (int)(__builtin_bit_cast(unsigned short, otherwise) * 0x10001u);
  if (valid <= 0) return fill;
  u128 w;
  if (col + valid >= N) w = __builtin_bit_cast(u128, *reinterpret_cast<const typename Chunk<T>::type *>(row + col + valid - N)) >> ((N - valid) * BITS);
  else {      // (the whole row is shorter than a chunk)
    w = 0;
    for (int j = valid - 1; j >= 0; j--) {
      if constexpr (sizeof(T) == 4) w = w << BITS | __builtin_bit_cast(unsigned, row[col + j]);
      else w = w << BITS | __builtin_bit_cast(unsigned short, row[col + j]);
    }
  }
  return __builtin_bit_cast(Packed, w | (__builtin_bit_cast(u128, fill) & ~(u128)0 << (valid * BITS)));
}
template <typename T> __device__ inline typename Chunk<T>::type load_chunk(const T *row, int col, int valid) { return __builtin_bit_cast(typename Chunk<T>::type, load_packed<T>(row, col, valid, (T)0.0f)); }
// N floats from a vector (null: `otherwise`)
template <int N> __device__ inline void load_params(const float *p, int col, int valid, float otherwise, float *out) {
  typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
  if (p && valid >= N) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const f4 v = *reinterpret_cast<const f4 *>(p + col + j);
#pragma unroll
      for (int k = 0; k < 4; k++) out[j + k] = v[k];
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < N; j++) out[j] = p ? p[min(col + j, col + valid - 1)] : otherwise;
#pragma unroll
  for (int j = 0; j < N; j++) out[j] = j < valid ? out[j] : otherwise;
}

// lanes of a wavefront: inclusive combination over DPP row shifts and the two row broadcasts, complete in lane 63, in a fixed order
template <int CTRL, int ROW_MASK> __device__ inline float dpp_f32(float identity, float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, identity), __builtin_bit_cast(int, v), CTRL, ROW_MASK, 0xf, false));
}
__device__ inline float lane63(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63)); }
__device__ inline float wave_sum(float v) {
  v += dpp_f32<0x111, 0xf>(0.0f, v);      // row_shr 1, 2, 4, 8
  v += dpp_f32<0x112, 0xf>(0.0f, v);
  v += dpp_f32<0x114, 0xf>(0.0f, v);
  v += dpp_f32<0x118, 0xf>(0.0f, v);
  v += dpp_f32<0x142, 0xa>(0.0f, v);      // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
  v += dpp_f32<0x143, 0xc>(0.0f, v);
  return lane63(v);
}
__device__ inline float wave_max(float v) {      // NaNs are passed over (as fmaxf does)
  const float id = -__builtin_inff();
  v = fmaxf(v, dpp_f32<0x111, 0xf>(id, v));
  v = fmaxf(v, dpp_f32<0x112, 0xf>(id, v));
  v = fmaxf(v, dpp_f32<0x114, 0xf>(id, v));
  v = fmaxf(v, dpp_f32<0x118, 0xf>(id, v));
  v = fmaxf(v, dpp_f32<0x142, 0xa>(id, v));
  v = fmaxf(v, dpp_f32<0x143, 0xc>(id, v));
  return lane63(v);
}

// the same over NW wavefronts of a workgroup; `sh` holds NW values per call and is free again after the NEXT barrier: consecutive calls take different buffers
template <int NW> __device__ inline float block_sum(float v, float *sh) {
  v = wave_sum(v);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++) v += sh[w];
  }
  return v;
}
template <int NW> __device__ inline float block_max(float v, float *sh) {
  v = wave_max(v);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < NW; w++) v = fmaxf(v, sh[w]);
  }
  return v;
}
// two sums at once (sh: 2 NW values)
template <int NW> __device__ inline void block_sum2(float &a, float &b, float *sh) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) { sh[2 * (threadIdx.x >> 6)] = a; sh[2 * (threadIdx.x >> 6) + 1] = b; }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++) { a += sh[2 * w]; b += sh[2 * w + 1]; }
  }
}

// A launch has less than 2^32 threads along one dimension: more workgroups go in several rows of 2^20 (those behind the last one return)
constexpr long long kMostGroups = (1ll << 20) * 65535;
inline dim3 grid_of(long long blocks, int threads) {
  if (blocks * threads < (1ll << 32)) return dim3((unsigned)blocks);
  return dim3(1u << 20, (unsigned)((blocks + (1 << 20) - 1) >> 20));
}
__device__ inline long long block_number() { return blockIdx.x + ((long long)blockIdx.y << 20); }

inline bool dtype_ok(int dtype) { return dtype >= K3_F32 && dtype <= K3_BF16; }
inline size_t dtype_size(int dtype) { return dtype == K3_F32 ? 4 : 2; }

// ---- which memory an operand takes: a call that writes a matrix where another of its operands lies is refused, since workgroups read and write in no order
struct Span {      // `rows` pieces of `width` bytes, `stride` apart (at least `width` where there are several); none: p null, or rows or width 0
  uintptr_t p; int64_t stride, rows, width;
  uintptr_t end() const { return p + (rows - 1) * stride + width; }
  bool none() const { return !p || rows <= 0 || width <= 0; }
};
inline Span matrix_span(const void *p, int64_t ld, int64_t rows, int64_t cols, size_t size) { return {(uintptr_t)p, ld * (int64_t)size, rows, cols * (int64_t)size}; }
inline Span vector_span(const void *p, int64_t n, size_t size = 4) { return {(uintptr_t)p, n * (int64_t)size, 1, n * (int64_t)size}; }
// the same elements at the same places
inline bool same(const Span &a, const Span &b) { return a.p == b.p && a.rows == b.rows && a.width == b.width && (a.rows <= 1 || a.stride == b.stride); }
inline bool overlap(const Span &a, const Span &b) {
  if (a.none() || b.none() || a.end() <= b.p || b.end() <= a.p) return false;
  if (a.rows > 1 && b.rows > 1 && a.stride == b.stride) {      // columns of one buffer, side by side or not
    const int64_t d = (int64_t)(b.p - a.p) % a.stride, at = d < 0 ? d + a.stride : d;
    return at < a.width || at + b.width > a.stride;
  }
  const Span &f = a.rows <= b.rows ? a : b, &m = a.rows <= b.rows ? b : a;
  for (int64_t i = 0; i < f.rows; i++) {      // the first piece of the other that ends behind this one's start: does it start before this one's end
    const uintptr_t s = f.p + i * f.stride, e = s + f.width;
    const int64_t j = s < m.p + m.width ? 0 : (int64_t)((s - m.p - m.width) / m.stride) + 1;
    if (j < m.rows && m.p + j * m.stride < e) return true;
  }
  return false;
}
template <size_t N> inline bool on_any(const Span &out, const Span (&others)[N]) {
  for (const Span &o : others) if (overlap(out, o)) return true;
  return false;
}

}  // namespace k3

// f(T{}) for the type of a k3_dtype that has been checked
#define K3_FOR_DTYPE(dtype, f)                                     \
  do {                                                             \
    if ((dtype) == K3_F32) { f(float); }                           \
    else if ((dtype) == K3_F16) { f(k3::f16); }                    \
    else { f(k3::bf16); }                                          \
  } while (0)
