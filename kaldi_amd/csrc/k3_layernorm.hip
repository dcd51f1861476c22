// k3_layernorm.hip -- layer norm of the rows of a float / half / bfloat16 matrix and its backward pass (k3_layer_norm_*).
//   mean = sum x / D, inv_std = 1 / sqrt(sum (x - mean)^2 / D + eps), y = (x - mean) inv_std scale + offset
//   backward, with xhat = (x - mean) inv_std and g = dy scale:  dx = inv_std (g - mean(g) - xhat mean(g xhat)), dscale = sum over rows of dy xhat, doffset = sum over rows of dy
// The reference has the norm without a mean (NormalizeComponent, cudamatrix/cu-math.h:272-300; k3_mat_normalize_rows here) and no half-precision matrices.
// All sums are kept in float32; a value is rounded to the matrix's type once, when it is written.
// Bound by memory: 2 (forward) or 3 (backward) passes over the matrix and nothing else of its size.  Measured: float16 40011 x 1535 forward 55 us (4.5 TB/s, rows that start anywhere),
// bfloat16 32768 x 4096 backward 151 us (5.3 TB/s; a copy of 1 GB runs at 5.0).
#include "k3_rowops.h"
#include <algorithm>
#include <type_traits>

namespace {
using namespace k3;

// What the first mean m0 is off by, from the mean d and the mean square q of the differences from it.  The sum behind m0 is off by steps of the values' size, the one behind d by steps of
// the differences': where the mean is large beside the spread, d is what the first sum lost (4096 +- 0.5 in float32: 1e-3 of the spread); otherwise it is noise, and the first sum (exact,
// as a rule, for half-precision values) stays.
__device__ inline float left_mean(float m0, float d, float q) { return m0 * m0 > 64.0f * q ? d : 0.0f; }

// 1 / sqrt(var + eps) from the mean square q of the differences from m0 and what m0 is off by.  (Not below 0 by rounding; a NaN, of a row that holds NaNs or infinities, stays one, as fmaxf
// would not let it.)
__device__ inline float inv_std_of(float q, float d, float eps) {
  const float var = q - d * d;
  return 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps);
}

// The rows a launch can hold in registers (up to 1024 threads of 16 or 24 elements).  A row belongs to NW wavefronts (one: four rows per workgroup); thread t holds the chunks t, t + 64 NW,
// ... of it, E of them, so each element is read once and both sums of the forward pass run over registers.  A workgroup walks over rows with a stride of the whole launch: scale
// and offset stay in registers, and the next row is on its way while this one is reduced and written.
template <typename T, int NW, int E> __global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void k3_ln_forward_kernel(const T *x, long long ldx, const float *scale, const float *offset,
    float eps, T *y, long long ldy, float *mean, float *inv_std, int rows, int cols) {
  constexpr int N = Chunk<T>::N, RPB = NW == 1 ? 4 : 1;
  __shared__ float sh[3 * NW];
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
  const long long step = (long long)gridDim.x * RPB;
  float sc[E][N], of[E][N];
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int col = (t + i * 64 * NW) * N;
    load_params<N>(scale, col, cols - col, 1.0f, sc[i]);
    load_params<N>(offset, col, cols - col, 0.0f, of[i]);
  }
  long long row = (long long)blockIdx.x * RPB + (NW == 1 ? threadIdx.x >> 6 : 0);
  typename Chunk<T>::type next[E], v[E];
  if (row < rows)
#pragma unroll
    for (int i = 0; i < E; i++) { const int col = (t + i * 64 * NW) * N; next[i] = load_chunk(x + row * ldx, col, cols - col); }
  const float n = (float)cols;
  for (; row < rows; row += step) {
    float s = 0.0f, d = 0.0f, q = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++) {
      v[i] = next[i];
#pragma unroll
      for (int j = 0; j < N; j++) s += to_f32(v[i][j]);
    }
    if (row + step < rows)
#pragma unroll
      for (int i = 0; i < E; i++) { const int col = (t + i * 64 * NW) * N; next[i] = load_chunk(x + (row + step) * ldx, col, cols - col); }
    const float m0 = block_sum<NW>(s, sh) / n;      // (a division: the mean of equal values is that value)
#pragma unroll
    for (int i = 0; i < E; i++) {
      const int valid = cols - (t + i * 64 * NW) * N;
      if (valid >= N) {
#pragma unroll
        for (int j = 0; j < N; j++) { const float u = to_f32(v[i][j]) - m0; d += u; q += u * u; }
      } else {
#pragma unroll
        for (int j = 0; j < N; j++) { const float u = j < valid ? to_f32(v[i][j]) - m0 : 0.0f; d += u; q += u * u; }
      }
    }
    block_sum2<NW>(d, q, sh + NW);
    d = left_mean(m0, d / n, q / n);
    const float r = inv_std_of(q / n, d, eps), m1 = m0 + d;
    if (t == 0) {
      if (mean) mean[row] = m1;
      if (inv_std) inv_std[row] = r;
    }
#pragma unroll
    for (int i = 0; i < E; i++) {
      const int col = (t + i * 64 * NW) * N;
      typename Chunk<T>::type o;
#pragma unroll
      for (int j = 0; j < N; j++) o[j] = (T)((to_f32(v[i][j]) - m0 - d) * r * sc[i][j] + of[i][j]);
      store_chunk(y + row * ldy, col, cols - col, o);
    }
  }
}

// the same shape for the backward pass; dscale and doffset of the rows a workgroup has walked over stay in registers and leave as one strip of `partial` [strip][2][cols]
template <typename T, int NW, int E> __global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void k3_ln_backward_kernel(const T *x, long long ldx, const T *dy, long long lddy,
    const float *scale, const float *mean, const float *inv_std, T *dx, long long lddx, float *partial, int rows, int cols) {
  constexpr int N = Chunk<T>::N, RPB = NW == 1 ? 4 : 1;
  __shared__ float sh[4 * NW];
  __shared__ float fold[NW == 1 ? 3 * 64 * E * N : 1];
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6;
  const long long step = (long long)gridDim.x * RPB;
  float sc[E][N], ds[E][N], db[E][N];
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int col = (t + i * 64 * NW) * N;
    load_params<N>(scale, col, cols - col, 1.0f, sc[i]);
#pragma unroll
    for (int j = 0; j < N; j++) ds[i][j] = db[i][j] = 0.0f;
  }
  long long row = (long long)blockIdx.x * RPB + (NW == 1 ? wave : 0);
  typename Chunk<T>::type vx[E], vg[E], nx[E], ng[E];
  float m = 0.0f, r = 0.0f, nm = 0.0f, nr = 0.0f;
  if (row < rows) {
#pragma unroll
    for (int i = 0; i < E; i++) {
      const int col = (t + i * 64 * NW) * N;
      nx[i] = load_chunk(x + row * ldx, col, cols - col);
      ng[i] = load_chunk(dy + row * lddy, col, cols - col);
    }
    nm = mean[row];
    nr = inv_std[row];
  }
  const float inv_n = 1.0f / (float)cols;
  int parity = 0;
  for (; row < rows; row += step) {
#pragma unroll
    for (int i = 0; i < E; i++) { vx[i] = nx[i]; vg[i] = ng[i]; }
    m = nm;
    r = nr;
    if (row + step < rows) {
#pragma unroll
      for (int i = 0; i < E; i++) {
        const int col = (t + i * 64 * NW) * N;
        nx[i] = load_chunk(x + (row + step) * ldx, col, cols - col);
        ng[i] = load_chunk(dy + (row + step) * lddy, col, cols - col);
      }
      nm = mean[row + step];
      nr = inv_std[row + step];
    }
    float a = 0.0f, b = 0.0f;      // elements behind the row's end have dy = 0 and add nothing
#pragma unroll
    for (int i = 0; i < E; i++)
#pragma unroll
      for (int j = 0; j < N; j++) {
        const float g0 = to_f32(vg[i][j]), h = (to_f32(vx[i][j]) - m) * r, g = g0 * sc[i][j];
        ds[i][j] += g0 * h;
        db[i][j] += g0;
        a += g;
        b += g * h;
      }
    block_sum2<NW>(a, b, sh + parity);
    parity ^= 2 * NW;      // (one barrier per row: the next row's sums go to the other half)
    a *= inv_n;
    b *= inv_n;
    if (dx)
#pragma unroll
      for (int i = 0; i < E; i++) {
        const int col = (t + i * 64 * NW) * N;
        typename Chunk<T>::type o;
#pragma unroll
        for (int j = 0; j < N; j++) o[j] = (T)(r * (to_f32(vg[i][j]) * sc[i][j] - a - (to_f32(vx[i][j]) - m) * r * b));
        store_chunk(dx + row * lddx, col, cols - col, o);
      }
  }
  if (!partial) return;
#pragma unroll
  for (int which = 0; which < 2; which++) {
    float *out = partial + ((long long)blockIdx.x * 2 + which) * cols;
    if constexpr (NW == 1) {
      __syncthreads();
      if (wave)
#pragma unroll
        for (int i = 0; i < E; i++)
#pragma unroll
          for (int j = 0; j < N; j++) fold[((wave - 1) * E * N + i * N + j) * 64 + t] = which ? db[i][j] : ds[i][j];
      __syncthreads();
      if (wave == 0)
#pragma unroll
        for (int i = 0; i < E; i++)
#pragma unroll
          for (int j = 0; j < N; j++)
#pragma unroll
            for (int w = 0; w < 3; w++) (which ? db : ds)[i][j] += fold[(w * E * N + i * N + j) * 64 + t];
    }
    if (NW > 1 || wave == 0)
#pragma unroll
      for (int i = 0; i < E; i++) {
        const int col = (t + i * 64 * NW) * N;
        typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
        if (col + N <= cols)
#pragma unroll
          for (int j = 0; j < N; j += 4)
            *(f4 *)(out + col + j) = which ? f4{db[i][j], db[i][j + 1], db[i][j + 2], db[i][j + 3]} : f4{ds[i][j], ds[i][j + 1], ds[i][j + 2], ds[i][j + 3]};
        else
#pragma unroll
          for (int j = 0; j < N; j++) if (col + j < cols) out[col + j] = which ? db[i][j] : ds[i][j];
      }
  }
}

// one workgroup per row, any width: the row is read once for each of the sums and once more for the result, element by element (float32 2000 x 20011 123 us forward, 154 backward, bfloat16
// 86 and 113: 2.6 and 1.9 TB/s of what has to be moved forward)
template <typename T> __global__ __launch_bounds__(256) void k3_ln_forward_loop_kernel(const T *x, long long ldx, const float *scale, const float *offset, float eps,
                                                                                       T *y, long long ldy, float *mean, float *inv_std, int cols) {
  __shared__ float sh[12];
  const long long row = blockIdx.x;
  const T *xr = x + row * ldx;
  T *yr = y + row * ldy;
  float s = 0.0f, d = 0.0f, q = 0.0f;
  for (int c = threadIdx.x; c < cols; c += 256) s += to_f32(xr[c]);
  const float m0 = block_sum<4>(s, sh) / (float)cols;
  for (int c = threadIdx.x; c < cols; c += 256) { const float v = to_f32(xr[c]) - m0; d += v; q += v * v; }
  block_sum2<4>(d, q, sh + 4);
  d = left_mean(m0, d / (float)cols, q / (float)cols);
  const float r = inv_std_of(q / (float)cols, d, eps);
  if (threadIdx.x == 0) {
    if (mean) mean[row] = m0 + d;
    if (inv_std) inv_std[row] = r;
  }
  for (int c = threadIdx.x; c < cols; c += 256) {
    const float v = (to_f32(xr[c]) - m0 - d) * r;
    yr[c] = (T)(v * (scale ? scale[c] : 1.0f) + (offset ? offset[c] : 0.0f));
  }
}

template <typename T> __global__ __launch_bounds__(256) void k3_ln_backward_loop_kernel(const T *x, long long ldx, const T *dy, long long lddy, const float *scale, const float *mean,
                                                                                        const float *inv_std, T *dx, long long lddx, int cols) {
  __shared__ float sh[8];
  const long long row = blockIdx.x;
  const T *xr = x + row * ldx, *gr = dy + row * lddy;
  const float m = mean[row], r = inv_std[row];
  float a = 0.0f, b = 0.0f;
  for (int c = threadIdx.x; c < cols; c += 256) {
    const float g = to_f32(gr[c]) * (scale ? scale[c] : 1.0f);
    a += g;
    b += g * ((to_f32(xr[c]) - m) * r);
  }
  block_sum2<4>(a, b, sh);
  a /= (float)cols;
  b /= (float)cols;
  for (int c = threadIdx.x; c < cols; c += 256) {
    const float g = to_f32(gr[c]) * (scale ? scale[c] : 1.0f), h = (to_f32(xr[c]) - m) * r;
    dx[row * lddx + c] = (T)(r * (g - a - h * b));
  }
}

// dscale and doffset of 64 columns over one strip of rows: partial [strip][2][cols]
template <typename T> __global__ __launch_bounds__(256) void k3_ln_param_loop_kernel(const T *x, long long ldx, const T *dy, long long lddy, const float *mean, const float *inv_std,
                                                                                     float *partial, int rows, int cols, int strip) {
  __shared__ float sh[2][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const int r0 = blockIdx.y * strip, r1 = min(rows, r0 + strip);
  float ds = 0.0f, db = 0.0f;
  if (c < cols)
    for (int row = r0 + wave; row < r1; row += 4) {
      const float g = to_f32(dy[row * lddy + c]);
      ds += g * ((to_f32(x[row * ldx + c]) - mean[row]) * inv_std[row]);
      db += g;
    }
  sh[0][wave][lane] = ds;
  sh[1][wave][lane] = db;
  __syncthreads();
  if (wave < 2 && c < cols) partial[((long long)blockIdx.y * 2 + wave) * cols + c] = (sh[wave][0][lane] + sh[wave][1][lane]) + (sh[wave][2][lane] + sh[wave][3][lane]);
}

// out[c] (+)= sum over strips of partial[strip][which][c]: 16 interleaved sums in ascending order of the strips, then over the 16
__global__ __launch_bounds__(1024) void k3_ln_param_join_kernel(const float *partial, int strips, int cols, float *dscale, float *doffset, int accumulate) {
  __shared__ float sh[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float *out = blockIdx.y ? doffset : dscale;
  if (!out) return;
  float v = 0.0f;
  if (c < cols)
#pragma unroll 8
    for (int s = wave; s < strips; s += 16) v += partial[((long long)s * 2 + blockIdx.y) * cols + c];
  sh[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < cols) {
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; w++) v += sh[w][lane];
    out[c] = accumulate ? out[c] + v : v;
  }
}

const int kMaxStrips = 512;
const int kMaxCols = 0x7fffffff - 1023;      // column numbers of threads that run ahead of a row's end still fit 32 bits
const int kMaxParamCols = (1 << 28) - 64;    // k3_ln_param_join_kernel has 16 threads per column, and a launch less than 2^32

// wavefronts per row and chunks per thread: the fewest wavefronts that hold the row with at most 16 (float) or 24 elements per thread, and no more than 16 of them (then 12 or 16
// elements: a workgroup of 1024 has 128 registers per thread, of which the backward pass already spills 4 with 12 floats and 34 with 16 halves); {0, 0} = too wide
struct Shape { int nw, e; };
template <typename T> Shape shape_of(int cols) {
  const int chunks = (cols + Chunk<T>::N - 1) / Chunk<T>::N, most = sizeof(T) == 4 ? 4 : 3;
  for (int nw = 1; nw <= 16; nw *= 2)
    if (chunks <= 64 * nw * (nw == 16 ? most - 1 : most)) return {nw, (chunks + 64 * nw - 1) / (64 * nw)};
  return {0, 0};
}
// f.template operator()<NW, E>() for a shape
template <typename T, typename F> void with_shape(Shape s, F f) {
#define K3_LN_E(NW)                                                                   \
  switch (s.e) {                                                                      \
    case 1: if constexpr (NW == 1) f(std::integral_constant<int, NW>(), std::integral_constant<int, 1>()); return; \
    case 2: f(std::integral_constant<int, NW>(), std::integral_constant<int, 2>()); return; \
    case 3: if constexpr (sizeof(T) == 4 || NW < 16) f(std::integral_constant<int, NW>(), std::integral_constant<int, 3>()); return; \
    default: if constexpr (sizeof(T) == 4 && NW < 16) f(std::integral_constant<int, NW>(), std::integral_constant<int, 4>()); return; \
  }
  switch (s.nw) {
    case 1: K3_LN_E(1)
    case 2: K3_LN_E(2)
    case 4: K3_LN_E(4)
    case 8: K3_LN_E(8)
    default: K3_LN_E(16)
  }
#undef K3_LN_E
}
template <typename T> void forward(const void *x, long long ldx, const float *scale, const float *offset, float eps, void *y, long long ldy, float *mean, float *inv_std, int rows,
                                   int cols, hipStream_t st) {
  const Shape s = shape_of<T>(cols);
  if (!s.nw) {
    hipLaunchKernelGGL((k3_ln_forward_loop_kernel<T>), dim3((unsigned)rows), dim3(256), 0, st, (const T *)x, ldx, scale, offset, eps, (T *)y, ldy, mean, inv_std, cols);
    return;
  }
  with_shape<T>(s, [&](auto nw, auto e) {
    constexpr int NW = decltype(nw)::value, E = decltype(e)::value, RPB = NW == 1 ? 4 : 1;
    const int grid = std::min((rows - 1) / RPB + 1, 256 * (NW <= 4 ? 16 / std::max(NW, 4) * 2 : 16 / NW * 2));
    hipLaunchKernelGGL((k3_ln_forward_kernel<T, NW, E>), dim3(grid), dim3(NW == 1 ? 256 : 64 * NW), 0, st, (const T *)x, ldx, scale, offset, eps, (T *)y, ldy, mean, inv_std, rows, cols);
  });
}
// returns the number of strips written to `partial`
template <typename T> int backward(const void *x, long long ldx, const void *dy, long long lddy, const float *scale, const float *mean, const float *inv_std, void *dx, long long lddx,
                                   float *partial, int rows, int cols, hipStream_t st) {
  const Shape s = shape_of<T>(cols);
  if (!s.nw) {
    const int strip = std::max(16, (rows + kMaxStrips - 1) / kMaxStrips), strips = (rows + strip - 1) / strip;
    if (partial)
      hipLaunchKernelGGL((k3_ln_param_loop_kernel<T>), dim3((cols + 63) / 64, strips), dim3(256), 0, st, (const T *)x, ldx, (const T *)dy, lddy, mean, inv_std, partial, rows, cols, strip);
    if (dx)
      hipLaunchKernelGGL((k3_ln_backward_loop_kernel<T>), dim3((unsigned)rows), dim3(256), 0, st, (const T *)x, ldx, (const T *)dy, lddy, scale, mean, inv_std, (T *)dx, lddx, cols);
    return strips;
  }
  int grid = 0;
  with_shape<T>(s, [&](auto nw, auto e) {
    constexpr int NW = decltype(nw)::value, E = decltype(e)::value, RPB = NW == 1 ? 4 : 1;
    grid = std::min((rows - 1) / RPB + 1, NW <= 8 ? kMaxStrips : kMaxStrips / 2);
    hipLaunchKernelGGL((k3_ln_backward_kernel<T, NW, E>), dim3(grid), dim3(NW == 1 ? 256 : 64 * NW), 0, st, (const T *)x, ldx, (const T *)dy, lddy, scale, mean, inv_std, (T *)dx, lddx,
                       partial, rows, cols);
  });
  return grid;
}

}  // namespace

extern "C" int k3_layer_norm_forward(int32_t dtype, const void *d_x, int64_t ldx, const float *d_scale, const float *d_offset, float eps, void *d_y, int64_t ldy,
                                     float *d_mean, float *d_inv_std, int32_t rows, int32_t cols, void *stream) {
  K3_REQUIRE(dtype_ok(dtype), "k3_layer_norm_forward: unknown type");
  K3_REQUIRE(rows >= 0 && cols >= 0 && ldx >= cols && ldy >= cols && eps >= 0.0f, "k3_layer_norm_forward: bad argument");
  if (cols > kMaxCols) { set_error("k3_layer_norm_forward: at most %d columns", kMaxCols); return K3_ERR_UNSUPPORTED; }
  if (rows == 0 || cols == 0) return K3_OK;
  K3_REQUIRE(d_x && d_y, "k3_layer_norm_forward: null matrix");
  const size_t size = dtype_size(dtype);
  const Span x = matrix_span(d_x, ldx, rows, cols, size), y = matrix_span(d_y, ldy, rows, cols, size), sc = vector_span(d_scale, cols), of = vector_span(d_offset, cols),
             mean = vector_span(d_mean, rows), inv = vector_span(d_inv_std, rows);
  K3_REQUIRE((same(x, y) || !overlap(x, y)) && !on_any(y, {sc, of, mean, inv}) && !on_any(mean, {x, sc, of}) && !on_any(inv, {x, sc, of}), "k3_layer_norm_forward: an output lies on another operand");
#define K3_LN_FWD(T) forward<T>(d_x, ldx, d_scale, d_offset, eps, d_y, ldy, d_mean, d_inv_std, rows, cols, (hipStream_t)stream)
  K3_FOR_DTYPE(dtype, K3_LN_FWD);
  K3_HIP_CHECK(hipGetLastError());
  return K3_OK;
}

extern "C" int64_t k3_layer_norm_backward_workspace(int32_t rows, int32_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (int64_t)sizeof(float) * 2 * cols * std::min(rows, kMaxStrips);
}

extern "C" int k3_layer_norm_backward(int32_t dtype, const void *d_x, int64_t ldx, const void *d_dy, int64_t lddy, const float *d_scale, const float *d_mean, const float *d_inv_std,
                                      void *d_dx, int64_t lddx, float *d_dscale, float *d_doffset, int32_t accumulate, void *d_workspace, int64_t workspace_bytes,
                                      int32_t rows, int32_t cols, void *stream) {
  K3_REQUIRE(dtype_ok(dtype), "k3_layer_norm_backward: unknown type");
  K3_REQUIRE(rows >= 0 && cols >= 0 && ldx >= cols && lddy >= cols && (!d_dx || lddx >= cols), "k3_layer_norm_backward: bad argument");
  const bool params = d_dscale || d_doffset;
  if (cols > (params ? kMaxParamCols : kMaxCols)) {
    set_error("k3_layer_norm_backward: at most %d columns, with the derivatives of scale or offset %d", kMaxCols, kMaxParamCols);
    return K3_ERR_UNSUPPORTED;
  }
  if (cols == 0) return K3_OK;
  K3_REQUIRE(rows == 0 || (d_x && d_dy && d_mean && d_inv_std), "k3_layer_norm_backward: null input");
  K3_REQUIRE(!params || rows == 0 || (d_workspace && workspace_bytes >= k3_layer_norm_backward_workspace(rows, cols)), "k3_layer_norm_backward: workspace too small");
  // (d_dscale and d_doffset are written when everything else has been read)
  const size_t size = dtype_size(dtype);
  const Span x = matrix_span(d_x, ldx, rows, cols, size), dy = matrix_span(d_dy, lddy, rows, cols, size), dx = matrix_span(d_dx, lddx, rows, cols, size), sc = vector_span(d_scale, cols),
             mean = vector_span(d_mean, rows), inv = vector_span(d_inv_std, rows), ds = vector_span(d_dscale, cols), doff = vector_span(d_doffset, cols);
  K3_REQUIRE((same(x, dx) || !overlap(x, dx)) && (same(dy, dx) || !overlap(dy, dx)) && !on_any(dx, {sc, mean, inv, ds, doff}) && !overlap(ds, doff), "k3_layer_norm_backward: an output lies on another operand");
  hipStream_t st = (hipStream_t)stream;
  int strips = 0;
  if (rows && (params || d_dx)) {
#define K3_LN_BWD(T) strips = backward<T>(d_x, ldx, d_dy, lddy, d_scale, d_mean, d_inv_std, d_dx, lddx, params ? (float *)d_workspace : nullptr, rows, cols, st)
    K3_FOR_DTYPE(dtype, K3_LN_BWD);
    K3_HIP_CHECK(hipGetLastError());
  }
  if (params) {
    hipLaunchKernelGGL(k3_ln_param_join_kernel, dim3((cols + 63) / 64, 2), dim3(1024), 0, st, (const float *)d_workspace, strips, cols, d_dscale, d_doffset, accumulate);
    K3_HIP_CHECK(hipGetLastError());
  }
  return K3_OK;
}
