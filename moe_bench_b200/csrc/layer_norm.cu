// Layer norm over the last dimension and its gradients.
//
//   mean = sum(x) / hidden, rstd = 1 / sqrt(sum((x - mean)^2) / hidden + eps), y = (x - mean) rstd w + b
//   h = (x - mean) rstd, g = dy w:  dx = rstd (g - mean(g) - h mean(g h)),  dw = sum dy h,  db = sum dy
//
// Statistics, gradients of the parameters and everything in between are fp32; y and dx are rounded once.

#include "../../include/moe_bench_b200.h"
#include "layer.cuh"

namespace mb200 {

namespace {

struct NormArgs {
  const void* x;
  const void* dy;       // backward
  int64_t x_pitch, dy_pitch;
  int64_t rows, hidden;
  const void* weight;   // null: 1
  const void* bias;     // null: 0
  float eps;
  void* out;            // y or dx, dense; backward: null if not wanted
  float* mean;
  float* rstd;
  float* sums;          // backward: [blocks][2][hidden] sums of dy*h and dy over the rows of each block, or null
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// Sum over the block, the same in all threads; `part` holds a value per warp.
__device__ __forceinline__ float block_sum(float v, float* part) {
  const int warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // the readers of an earlier sum are through
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < warps; ++i) s += part[i];
  return s;
}

constexpr int kLongThreads = 512;

// Rows of any length: a block per row, the row read once per pass.
template <typename T, typename P>
__global__ void __launch_bounds__(kLongThreads) norm_long_kernel(const NormArgs p) {
  __shared__ float part[kLongThreads / 32];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(p.x) + r * p.x_pitch;
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < p.hidden; i += kLongThreads) s += to_float(x[i]);
    const float mean = block_sum(s, part) / float(p.hidden);
    s = 0.f;
    for (int64_t i = threadIdx.x; i < p.hidden; i += kLongThreads) {
      const float d = to_float(x[i]) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = 1.f / sqrtf(block_sum(s, part) / float(p.hidden) + p.eps);
    T* y = reinterpret_cast<T*>(p.out) + r * p.hidden;
    for (int64_t i = threadIdx.x; i < p.hidden; i += kLongThreads) {
      float v = (to_float(x[i]) - mean) * rstd;
      if (p.weight) v *= to_float(reinterpret_cast<const P*>(p.weight)[i]);
      if (p.bias) v += to_float(reinterpret_cast<const P*>(p.bias)[i]);
      y[i] = from_float<T>(v);
    }
    if (threadIdx.x == 0) {
      p.mean[r] = mean;
      p.rstd[r] = rstd;
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kLongThreads) norm_grad_long_kernel(const NormArgs p) {
  __shared__ float part[kLongThreads / 32];
  float* sums = p.sums ? p.sums + int64_t(blockIdx.x) * 2 * p.hidden : nullptr;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(p.x) + r * p.x_pitch;
    const T* dy = reinterpret_cast<const T*>(p.dy) + r * p.dy_pitch;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float sg = 0.f, sgh = 0.f;
    for (int64_t i = threadIdx.x; i < p.hidden; i += kLongThreads) {
      const float d = to_float(dy[i]);
      const float g = p.weight ? d * to_float(reinterpret_cast<const P*>(p.weight)[i]) : d;
      sg += g;
      sgh = fmaf(g, (to_float(x[i]) - mean) * rstd, sgh);
    }
    if (p.out) {
      sg = block_sum(sg, part) / float(p.hidden);
      sgh = block_sum(sgh, part) / float(p.hidden);
    }
    T* dx = p.out ? reinterpret_cast<T*>(p.out) + r * p.hidden : nullptr;
    for (int64_t i = threadIdx.x; i < p.hidden; i += kLongThreads) {
      const float d = to_float(dy[i]);
      const float h = (to_float(x[i]) - mean) * rstd;
      const float g = p.weight ? d * to_float(reinterpret_cast<const P*>(p.weight)[i]) : d;
      if (dx) dx[i] = from_float<T>(rstd * (g - sg - h * sgh));
      if (sums) {  // this thread's own column of this block's own sums
        const bool first = r == blockIdx.x;
        sums[i] = first ? d * h : fmaf(d, h, sums[i]);
        sums[p.hidden + i] = first ? d : sums[p.hidden + i] + d;
      }
    }
  }
}

// dweight and dbias: the blocks' sums added in block order.
__global__ void __launch_bounds__(256) norm_param_grad_kernel(const float* sums, int blocks, int64_t hidden, float* dweight,
                                                              float* dbias) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= 2 * hidden) return;
  float s = 0.f;
  for (int b = 0; b < blocks; ++b) s += sums[int64_t(b) * 2 * hidden + i];
  if (i < hidden) {
    if (dweight) dweight[i] = s;
  } else if (dbias) {
    dbias[i - hidden] = s;
  }
}

int grid_blocks(int64_t rows, int device) {
  const int sms = device_sm_count(device);
  const int64_t most = int64_t(sms > 0 ? sms : 1) * 4;
  return int(rows < most ? rows : most);
}

int check_norm(int precision, int64_t rows, int64_t hidden, const char* what) {
  MB200_REQUIRE(precision == MB200_PRECISION_BF16 || precision == MB200_PRECISION_FP16 || precision == MB200_PRECISION_FP32,
                kInvalidArgument, "%s: precision %d (bf16, fp16 or fp32)", what, precision);
  MB200_REQUIRE(rows >= 0 && hidden >= 1, kInvalidArgument, "%s: rows=%lld hidden=%lld", what, (long long)rows,
                (long long)hidden);
  MB200_REQUIRE(hidden <= (int64_t(1) << 30), kUnsupportedShape, "%s: hidden=%lld", what, (long long)hidden);
  return kOk;
}

template <typename T, typename P>
void launch_forward(const NormArgs& a, int blocks, cudaStream_t s) {
  norm_long_kernel<T, P><<<blocks, kLongThreads, 0, s>>>(a);
}
template <typename T, typename P>
void launch_backward(const NormArgs& a, int blocks, cudaStream_t s) {
  norm_grad_long_kernel<T, P><<<blocks, kLongThreads, 0, s>>>(a);
}

}  // namespace

}  // namespace mb200

using namespace mb200;

extern "C" {

int mb200_layer_norm(int precision, const void* x, int64_t x_pitch, int64_t rows, int64_t hidden, const void* weight,
                     const void* bias, int params_fp32, float eps, void* y, float* mean, float* rstd, int device,
                     void* stream) {
  int rc = check_norm(precision, rows, hidden, "layer_norm");
  if (rc) return rc;
  MB200_REQUIRE(x_pitch >= hidden, kInvalidArgument, "layer_norm: pitch %lld < hidden=%lld", (long long)x_pitch,
                (long long)hidden);
  if (rows == 0) return kOk;
  MB200_REQUIRE(x && y && mean && rstd, kInvalidArgument, "layer_norm: null pointer");
  NormArgs a{};
  a.x = x;
  a.x_pitch = x_pitch;
  a.rows = rows;
  a.hidden = hidden;
  a.weight = weight;
  a.bias = bias;
  a.eps = eps;
  a.out = y;
  a.mean = mean;
  a.rstd = rstd;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int blocks = grid_blocks(rows, device);
  if (precision == MB200_PRECISION_FP32) launch_forward<float, float>(a, blocks, s);
  else if (precision == MB200_PRECISION_FP16 && params_fp32) launch_forward<__half, float>(a, blocks, s);
  else if (precision == MB200_PRECISION_FP16) launch_forward<__half, __half>(a, blocks, s);
  else if (params_fp32) launch_forward<__nv_bfloat16, float>(a, blocks, s);
  else launch_forward<__nv_bfloat16, __nv_bfloat16>(a, blocks, s);
  MB200_CHECK_CUDA(cudaGetLastError());
  return kOk;
}

int64_t mb200_layer_norm_backward_workspace_bytes(int64_t rows, int64_t hidden, int device) {
  if (check_norm(MB200_PRECISION_FP32, rows, hidden, "layer_norm_backward_workspace_bytes")) return -1;
  return int64_t(grid_blocks(rows, device)) * 2 * hidden * 4;
}

int mb200_layer_norm_backward(int precision, const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch,
                              int64_t rows, int64_t hidden, const float* mean, const float* rstd, const void* weight,
                              int params_fp32, void* dx, float* dweight, float* dbias, void* workspace,
                              int64_t workspace_bytes, int device, void* stream) {
  int rc = check_norm(precision, rows, hidden, "layer_norm_backward");
  if (rc) return rc;
  MB200_REQUIRE(x_pitch >= hidden && dy_pitch >= hidden, kInvalidArgument,
                "layer_norm_backward: pitches %lld and %lld, hidden=%lld", (long long)x_pitch, (long long)dy_pitch,
                (long long)hidden);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    if (dweight) MB200_CHECK_CUDA(cudaMemsetAsync(dweight, 0, size_t(hidden) * 4, s));
    if (dbias) MB200_CHECK_CUDA(cudaMemsetAsync(dbias, 0, size_t(hidden) * 4, s));
    return kOk;
  }
  MB200_REQUIRE(dy && x && mean && rstd, kInvalidArgument, "layer_norm_backward: null pointer");
  if (!dx && !dweight && !dbias) return kOk;
  const int blocks = grid_blocks(rows, device);
  NormArgs a{};
  a.x = x;
  a.dy = dy;
  a.x_pitch = x_pitch;
  a.dy_pitch = dy_pitch;
  a.rows = rows;
  a.hidden = hidden;
  a.weight = weight;
  a.out = dx;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  if (dweight || dbias) {
    const int64_t need = int64_t(blocks) * 2 * hidden * 4;
    MB200_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, kInvalidArgument,
                  "layer_norm_backward: needs a 16-byte aligned workspace");
    MB200_REQUIRE(workspace_bytes >= need, kWorkspaceTooSmall, "layer_norm_backward: workspace %lld < %lld bytes",
                  (long long)workspace_bytes, (long long)need);
    a.sums = reinterpret_cast<float*>(workspace);
  }
  if (precision == MB200_PRECISION_FP32) launch_backward<float, float>(a, blocks, s);
  else if (precision == MB200_PRECISION_FP16 && params_fp32) launch_backward<__half, float>(a, blocks, s);
  else if (precision == MB200_PRECISION_FP16) launch_backward<__half, __half>(a, blocks, s);
  else if (params_fp32) launch_backward<__nv_bfloat16, float>(a, blocks, s);
  else launch_backward<__nv_bfloat16, __nv_bfloat16>(a, blocks, s);
  MB200_CHECK_CUDA(cudaGetLastError());
  if (a.sums) {
    norm_param_grad_kernel<<<unsigned((2 * hidden + 255) / 256), 256, 0, s>>>(a.sums, blocks, hidden, dweight, dbias);
    MB200_CHECK_CUDA(cudaGetLastError());
  }
  return kOk;
}

}  // extern "C"
