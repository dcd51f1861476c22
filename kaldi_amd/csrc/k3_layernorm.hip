// k3_layernorm.hip -- layer norm of the rows of a float / half / bfloat16 matrix and its backward pass (k3_layer_norm_*).
//   mean = sum x / D, inv_std = 1 / sqrt(sum (x - mean)^2 / D + eps), y = (x - mean) inv_std scale + offset
//   backward, with xhat = (x - mean) inv_std and g = dy scale:  dx = inv_std (g - mean(g) - xhat mean(g xhat)), dscale = sum over rows of dy xhat, doffset = sum over rows of dy
// The reference has the norm without a mean (NormalizeComponent, cudamatrix/cu-math.h:272-300; k3_mat_normalize_rows here) and no half-precision matrices.
// All sums are kept in float32; a value is rounded to the matrix's type once, when it is written.
#include "k3_rowops.h"
#include <algorithm>

namespace {
using namespace k3;

// one workgroup per row, any width: the row is read once for each of the sums and once more for the result
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
  d /= (float)cols;      // what the rounding of the first mean left
  const float r = 1.0f / sqrtf(fmaxf(q / (float)cols - d * d, 0.0f) + eps);
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

// out[c] (+)= sum over strips of partial[strip][which][c], in ascending order of the strips within each of 4 interleaved sums
__global__ __launch_bounds__(256) void k3_ln_param_join_kernel(const float *partial, int strips, int cols, float *dscale, float *doffset, int accumulate) {
  __shared__ float sh[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float *out = blockIdx.y ? doffset : dscale;
  if (!out) return;
  float v = 0.0f;
  if (c < cols)
    for (int s = wave; s < strips; s += 4) v += partial[((long long)s * 2 + blockIdx.y) * cols + c];
  sh[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < cols) {
    v = (sh[0][lane] + sh[1][lane]) + (sh[2][lane] + sh[3][lane]);
    out[c] = accumulate ? out[c] + v : v;
  }
}

const int kMaxStrips = 256;

}  // namespace

extern "C" int k3_layer_norm_forward(int32_t dtype, const void *d_x, int64_t ldx, const float *d_scale, const float *d_offset, float eps, void *d_y, int64_t ldy,
                                     float *d_mean, float *d_inv_std, int32_t rows, int32_t cols, void *stream) {
  K3_REQUIRE(dtype_ok(dtype), "k3_layer_norm_forward: unknown type");
  K3_REQUIRE(rows >= 0 && cols >= 0 && ldx >= cols && ldy >= cols && eps >= 0.0f, "k3_layer_norm_forward: bad argument");
  if (rows == 0 || cols == 0) return K3_OK;
  K3_REQUIRE(d_x && d_y, "k3_layer_norm_forward: null matrix");
  hipStream_t st = (hipStream_t)stream;
#define K3_LN_FWD(T) hipLaunchKernelGGL((k3_ln_forward_loop_kernel<T>), dim3((unsigned)rows), dim3(256), 0, st, (const T *)d_x, (long long)ldx, d_scale, d_offset, eps, (T *)d_y, \
                                        (long long)ldy, d_mean, d_inv_std, cols)
  K3_FOR_DTYPE(dtype, K3_LN_FWD);
  K3_HIP_CHECK(hipGetLastError());
  return K3_OK;
}

extern "C" int64_t k3_layer_norm_backward_workspace(int32_t rows, int32_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (int64_t)sizeof(float) * 2 * cols * kMaxStrips;
}

extern "C" int k3_layer_norm_backward(int32_t dtype, const void *d_x, int64_t ldx, const void *d_dy, int64_t lddy, const float *d_scale, const float *d_mean, const float *d_inv_std,
                                      void *d_dx, int64_t lddx, float *d_dscale, float *d_doffset, int32_t accumulate, void *d_workspace, int64_t workspace_bytes,
                                      int32_t rows, int32_t cols, void *stream) {
  K3_REQUIRE(dtype_ok(dtype), "k3_layer_norm_backward: unknown type");
  K3_REQUIRE(rows >= 0 && cols >= 0 && ldx >= cols && lddy >= cols && (!d_dx || lddx >= cols), "k3_layer_norm_backward: bad argument");
  if (cols == 0) return K3_OK;
  K3_REQUIRE(rows == 0 || (d_x && d_dy && d_mean && d_inv_std), "k3_layer_norm_backward: null input");
  const bool params = d_dscale || d_doffset;
  K3_REQUIRE(!params || rows == 0 || (d_workspace && workspace_bytes >= k3_layer_norm_backward_workspace(rows, cols)), "k3_layer_norm_backward: workspace too small");
  hipStream_t st = (hipStream_t)stream;
  const int strip = std::max(16, (rows + kMaxStrips - 1) / kMaxStrips), strips = (rows + strip - 1) / strip;
  const dim3 colgrid((cols + 63) / 64, 2);
#define K3_LN_BWD(T)                                                                                                                                                          \
  if (params && rows)                                                                                                                                                         \
    hipLaunchKernelGGL((k3_ln_param_loop_kernel<T>), dim3((cols + 63) / 64, strips), dim3(256), 0, st, (const T *)d_x, (long long)ldx, (const T *)d_dy, (long long)lddy, d_mean, \
                       d_inv_std, (float *)d_workspace, rows, cols, strip);                                                                                                   \
  if (d_dx && rows)                                                                                                                                                           \
    hipLaunchKernelGGL((k3_ln_backward_loop_kernel<T>), dim3((unsigned)rows), dim3(256), 0, st, (const T *)d_x, (long long)ldx, (const T *)d_dy, (long long)lddy, d_scale,     \
                       d_mean, d_inv_std, (T *)d_dx, (long long)lddx, cols)
  K3_FOR_DTYPE(dtype, K3_LN_BWD);
  if (params) hipLaunchKernelGGL(k3_ln_param_join_kernel, colgrid, dim3(256), 0, st, (const float *)d_workspace, rows ? strips : 0, cols, d_dscale, d_doffset, accumulate);
  K3_HIP_CHECK(hipGetLastError());
  return K3_OK;
}
