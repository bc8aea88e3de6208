// Layer norm over the last dimension, forward and backward, with the reduction of the weight's gradient.
//
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) rstd, y = h w + b
//   u = dy w,  dx = rstd (u - mean(u) - h mean(u h)),  dw = sum over rows of dy h,  db = sum over rows of dy
//
// Everything between a load and a store is fp32; each output is rounded once.  The variance is summed over centred values
// (never as E[x^2] - mu^2, which cancels when |mu| is large against the spread).
// Bound: HBM.  Forward: x read, y written; backward: x and dy read, dx written; w, b and the row statistics are small.
#include "dtypes.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace b200k {

// Sum over the threads of a CTA; every thread gets the result.  `scratch` holds 32 floats and may be reused after the
// next __syncthreads.  The order of the additions depends on the thread count only.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = warp_sum(v);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = warp_sum(lane < warps ? scratch[lane] : 0.f);
  __syncthreads();
  return v;
}

// ---------------------------------------------------------------------------------------------
// Any row length: one CTA per row, the row walked once per pass (the later passes hit L1 / L2).
// ---------------------------------------------------------------------------------------------
template <typename T, typename W>
__global__ void __launch_bounds__(512) ln_fwd_loop_kernel(const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b,
                                                          T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                                                          int64_t rows, int64_t cols, int64_t ldx, int64_t ldy, float eps) {
  __shared__ float scratch[32];
  const float inv_n = 1.f / static_cast<float>(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * ldx;
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) s += to_f32<T>(xr[c]);
    const float mu = block_sum(s, scratch) * inv_n;
    float q = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float d = to_f32<T>(xr[c]) - mu;
      q += d * d;
    }
    const float rs = rsqrtf(block_sum(q, scratch) * inv_n + eps);
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      float v = (to_f32<T>(xr[c]) - mu) * rs;
      if (w != nullptr) v *= to_f32<W>(w[c]);
      if (b != nullptr) v += to_f32<W>(b[c]);
      y[r * ldy + c] = from_f32<T>(v);
    }
    if (threadIdx.x == 0) {
      if (mean != nullptr) mean[r] = mu;
      if (rstd != nullptr) rstd[r] = rs;
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(512) ln_dx_loop_kernel(const T* __restrict__ dy, const T* __restrict__ x, const W* __restrict__ w,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                                                         int64_t rows, int64_t cols, int64_t lddy, int64_t ldx, int64_t lddx) {
  __shared__ float scratch[32];
  const float inv_n = 1.f / static_cast<float>(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * ldx;
    const T* gr = dy + r * lddy;
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float u = to_f32<T>(gr[c]) * (w != nullptr ? to_f32<W>(w[c]) : 1.f);
      s1 += u;
      s2 += u * ((to_f32<T>(xr[c]) - mu) * rs);
    }
    const float c1 = block_sum(s1, scratch) * inv_n;
    const float c2 = block_sum(s2, scratch) * inv_n;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float u = to_f32<T>(gr[c]) * (w != nullptr ? to_f32<W>(w[c]) : 1.f);
      const float h = (to_f32<T>(xr[c]) - mu) * rs;
      dx[r * lddx + c] = from_f32<T>(rs * (u - c1 - h * c2));
    }
  }
}

// Partial sums of dw and db: CTA (i, j) adds the rows of slice j of the columns of tile i, one column per thread.
// part[2][parts][cols]: first dw, then db.
template <typename T>
__global__ void __launch_bounds__(256) ln_dw_loop_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean,
                                                         const float* __restrict__ rstd, float* __restrict__ part, int64_t rows,
                                                         int64_t cols, int64_t lddy, int64_t ldx) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= cols) return;
  const int parts = gridDim.y;
  float sw = 0.f, sb = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += parts) {
    const float g = to_f32<T>(dy[r * lddy + c]);
    sw += g * ((to_f32<T>(x[r * ldx + c]) - mean[r]) * rstd[r]);
    sb += g;
  }
  part[static_cast<int64_t>(blockIdx.y) * cols + c] = sw;
  part[static_cast<int64_t>(parts + blockIdx.y) * cols + c] = sb;
}

// dw[c] and db[c]: the sums over the parts, in a fixed order.
template <typename W>
__global__ void __launch_bounds__(256) ln_dw_join_kernel(const float* __restrict__ part, W* __restrict__ dw, W* __restrict__ db, int parts,
                                                         int64_t cols) {
  __shared__ float sums[8][33];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int slice = threadIdx.x >> 5;
  const float* p = part + static_cast<int64_t>(blockIdx.y) * parts * cols;
  float s = 0.f;
  if (c < cols)
    for (int i = slice; i < parts; i += 8) s += p[static_cast<int64_t>(i) * cols + c];
  sums[slice][threadIdx.x & 31] = s;
  __syncthreads();
  if (slice == 0 && c < cols) {
    for (int i = 1; i < 8; ++i) s += sums[i][threadIdx.x];
    W* out = blockIdx.y == 0 ? dw : db;
    if (out != nullptr) out[c] = from_f32<W>(s);
  }
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
static int ln_parts(int64_t rows) { return static_cast<int>(rows < LN_MAX_PARTS ? rows : LN_MAX_PARTS); }

int64_t layer_norm_bwd_workspace(int64_t rows, int64_t cols) { return 2 * ln_parts(rows) * cols; }

template <typename T, typename W>
static int ln_fwd(const LayerNormArgs& a, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>(a.rows < (1 << 30) ? a.rows : (1 << 30));
  const int threads = a.cols >= 2048 ? 512 : 128;
  ln_fwd_loop_kernel<T, W><<<grid, threads, 0, stream>>>(static_cast<const T*>(a.x), static_cast<const W*>(a.w), static_cast<const W*>(a.b),
                                                         static_cast<T*>(a.y), a.mean, a.rstd, a.rows, a.cols, a.ldx, a.ldy, a.eps);
  count_launch();
  B200K_CHECK_LAUNCH("ln_fwd_loop_kernel");
  return B200K_OK;
}

template <typename T, typename W>
static int ln_bwd(const LayerNormArgs& a, cudaStream_t stream) {
  const T* dy = static_cast<const T*>(a.dy);
  const T* x = static_cast<const T*>(a.x);
  if (a.dx != nullptr && a.rows > 0) {
    const unsigned grid = static_cast<unsigned>(a.rows < (1 << 30) ? a.rows : (1 << 30));
    const int threads = a.cols >= 2048 ? 512 : 128;
    ln_dx_loop_kernel<T, W><<<grid, threads, 0, stream>>>(dy, x, static_cast<const W*>(a.w), a.mean, a.rstd, static_cast<T*>(a.dx), a.rows,
                                                          a.cols, a.lddy, a.ldx, a.lddx);
    count_launch();
    B200K_CHECK_LAUNCH("ln_dx_loop_kernel");
  }
  if (a.dw != nullptr || a.db != nullptr) {
    const int parts = ln_parts(a.rows);
    if (parts > 0) {
      ln_dw_loop_kernel<T><<<dim3(static_cast<unsigned>((a.cols + 255) / 256), parts), 256, 0, stream>>>(dy, x, a.mean, a.rstd, a.workspace,
                                                                                                       a.rows, a.cols, a.lddy, a.ldx);
      count_launch();
      B200K_CHECK_LAUNCH("ln_dw_loop_kernel");
    }
    ln_dw_join_kernel<W><<<dim3(static_cast<unsigned>((a.cols + 31) / 32), 2), 256, 0, stream>>>(a.workspace, static_cast<W*>(a.dw),
                                                                                                static_cast<W*>(a.db), parts, a.cols);
    count_launch();
    B200K_CHECK_LAUNCH("ln_dw_join_kernel");
  }
  return B200K_OK;
}

template <typename F>
static int ln_dispatch(const LayerNormArgs& a, F&& f) {
  const bool wide = a.wdtype == B200K_DTYPE_F32;
  switch (a.dtype) {
    case B200K_DTYPE_F32: return f(float(), float());
    case B200K_DTYPE_BF16: return wide ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
    default: return wide ? f(__half(), float()) : f(__half(), __half());
  }
}

static int ln_check(const LayerNormArgs& a, const char* what) {
  if (a.dtype < B200K_DTYPE_F32 || a.dtype > B200K_DTYPE_F16) return set_error(B200K_ERR_INVALID_ARG, "%s: bad element type %d", what, a.dtype);
  if (a.wdtype != a.dtype && a.wdtype != B200K_DTYPE_F32)
    return set_error(B200K_ERR_INVALID_ARG, "%s: weight and bias have the type of x or fp32 (got %d for x of type %d)", what, a.wdtype, a.dtype);
  if (a.rows < 0 || a.cols < 1 || a.cols > (int64_t(1) << 31) - 512)
    return set_error(B200K_ERR_INVALID_ARG, "%s: rows >= 0 and 1 <= cols < 2^31 - 512 expected (got %lld x %lld)", what, (long long)a.rows, (long long)a.cols);
  if (a.rows > 0 && a.cols > (int64_t(1) << 62) / a.rows) return set_error(B200K_ERR_INVALID_ARG, "%s: too many elements", what);
  return B200K_OK;
}

int layer_norm_fwd(const LayerNormArgs& a, cudaStream_t stream) {
  const int rc = ln_check(a, "layer_norm");
  if (rc != B200K_OK) return rc;
  if (!(a.eps >= 0.f)) return set_error(B200K_ERR_INVALID_ARG, "layer_norm: eps must be >= 0");
  if (a.rows == 0) return B200K_OK;
  if (a.x == nullptr || a.y == nullptr) return set_error(B200K_ERR_INVALID_ARG, "layer_norm: null pointer");
  if (a.ldx < 0 || a.ldy < a.cols) return set_error(B200K_ERR_INVALID_ARG, "layer_norm: bad row stride");
  const DeviceInfo* dev = current_device_info();
  if (dev == nullptr) return B200K_ERR_NO_DEVICE;
  return ln_dispatch(a, [&](auto t, auto w) { return ln_fwd<decltype(t), decltype(w)>(a, stream); });
}

int layer_norm_bwd(const LayerNormArgs& a, cudaStream_t stream) {
  const int rc = ln_check(a, "layer_norm_backward");
  if (rc != B200K_OK) return rc;
  const bool sums = a.dw != nullptr || a.db != nullptr;
  if (a.rows > 0) {
    if (a.dy == nullptr || a.x == nullptr || a.mean == nullptr || a.rstd == nullptr)
      return set_error(B200K_ERR_INVALID_ARG, "layer_norm_backward: null pointer");
    if (a.ldx < 0 || a.lddy < 0 || (a.dx != nullptr && a.lddx < a.cols)) return set_error(B200K_ERR_INVALID_ARG, "layer_norm_backward: bad row stride");
    if (sums && (a.workspace == nullptr || a.workspace_floats < layer_norm_bwd_workspace(a.rows, a.cols)))
      return set_error(B200K_ERR_INVALID_ARG, "layer_norm_backward: a workspace of %lld floats is needed (got %lld)",
                       (long long)layer_norm_bwd_workspace(a.rows, a.cols), (long long)(a.workspace == nullptr ? 0 : a.workspace_floats));
  }
  const DeviceInfo* dev = current_device_info();
  if (dev == nullptr) return B200K_ERR_NO_DEVICE;
  return ln_dispatch(a, [&](auto t, auto w) { return ln_bwd<decltype(t), decltype(w)>(a, stream); });
}

}  // namespace b200k
