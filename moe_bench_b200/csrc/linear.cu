// extern "C" entry points of the products around the expert FFN (dense with bias, activation and
// residual; ragged row segments) and of their gradients, and the elementwise step ahead of the
// gradients' products.

#include <algorithm>

#include "../../include/moe_bench_b200.h"
#include "linear.cuh"

namespace mb200 {

namespace {

cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// ---- dz = dy * slope, and its column sums ----------------------------------------------------------
// A block takes kColumns columns of a run of rows: kRowLanes rows side by side, summed in fp32 per
// column, then over the row lanes in a fixed order.  The runs' sums are added by bias_sum_kernel.
constexpr int kColumns = 64;
constexpr int kRowLanes = 8;

// chunk sums [chunks][n]; dz null: no product of its own is stored
__global__ void __launch_bounds__(kColumns* kRowLanes)
output_grad_kernel(const void* dy, int dy_fp32, int64_t dy_pitch, const void* slope, int rows, int n, int fp16,
                   int rows_per_chunk, uint16_t* dz, int64_t dz_pitch, float* sums) {
  __shared__ float part[kRowLanes][kColumns];
  const int c = threadIdx.x % kColumns, lane = threadIdx.x / kColumns;
  const int col = blockIdx.x * kColumns + c;
  const int64_t first = int64_t(blockIdx.y) * rows_per_chunk;
  const int64_t last = first + rows_per_chunk < rows ? first + rows_per_chunk : rows;
  float sum = 0.f;
  if (col < n)
    for (int64_t r = first + lane; r < last; r += kRowLanes) {
      float v = dy_fp32 ? reinterpret_cast<const float*>(dy)[r * dy_pitch + col] : load_h16(dy, r * dy_pitch + col, fp16);
      if (slope) v *= load_h16(slope, r * n + col, fp16);
      sum += v;
      if (dz) dz[r * dz_pitch + col] = to_h16(v, fp16);
    }
  if (sums == nullptr) return;
  part[lane][c] = sum;
  __syncthreads();
  if (lane == 0 && col < n) {
    for (int i = 1; i < kRowLanes; ++i) sum += part[i][c];
    sums[int64_t(blockIdx.y) * n + col] = sum;
  }
}

__global__ void __launch_bounds__(256) bias_sum_kernel(const float* sums, int chunks, int n, float* db) {
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= n) return;
  float s = 0.f;
  for (int i = 0; i < chunks; ++i) s += sums[int64_t(i) * n + col];
  db[col] = s;
}

struct GradLayout {
  int64_t dz_pitch, dz_bytes, sum_bytes;
  int chunks, rows_per_chunk;
};
GradLayout grad_layout(int64_t rows, int n) {
  GradLayout l;
  l.dz_pitch = round_up(n, 8);
  l.dz_bytes = round_up(rows * l.dz_pitch * 2, 256);
  l.chunks = int(rows < 64 ? 1 : rows < 64 * 64 ? (rows + 63) / 64 : 64);
  l.rows_per_chunk = int((rows + l.chunks - 1) / l.chunks);
  l.sum_bytes = l.chunks > 1 ? round_up(int64_t(l.chunks) * n * 4, 256) : 0;
  return l;
}

// Bytes behind dz: the column sums, and after them, in the same place, the parts of one product's split sums.
int64_t split_bytes(int64_t rows, int n, int k, int device, bool dx, bool dw, int64_t sum_bytes) {
  int64_t b = sum_bytes;
  if (rows > 0 && dx) b = std::max(b, product_workspace_bytes(kInputGrad, int(rows), k, 0, n, device));
  if (rows > 0 && dw) b = std::max(b, product_workspace_bytes(kWeightGrad, int(rows), k, n, 0, device));
  return b;
}

int check_precision(int precision, const char* what) {
  MB200_REQUIRE(precision == MB200_PRECISION_BF16 || precision == MB200_PRECISION_FP16, kInvalidArgument,
                "%s: precision %d (bf16 or fp16)", what, precision);
  return kOk;
}

// An operand of a product: rows of `cols` elements that tiles are loaded from.
int check_operand(const void* p, int64_t pitch, int64_t cols, const char* what, const char* name) {
  MB200_REQUIRE(p != nullptr, kInvalidArgument, "%s: %s is null", what, name);
  MB200_REQUIRE(aligned16(p), kInvalidArgument, "%s: %s must start on a 16-byte boundary", what, name);
  MB200_REQUIRE(pitch >= cols && pitch % 8 == 0, kUnsupportedShape,
                "%s: %s has %lld elements from row to row: at least %lld and a multiple of 8", what, name,
                (long long)pitch, (long long)cols);
  return kOk;
}

int check_sizes(int64_t rows, int n, int k, const char* what) {
  MB200_REQUIRE(rows >= 0 && n >= 1 && k >= 1, kInvalidArgument, "%s: rows=%lld n=%d k=%d", what, (long long)rows, n, k);
  MB200_REQUIRE(k % 8 == 0, kUnsupportedShape, "%s: k=%d must be a multiple of 8", what, k);
  MB200_REQUIRE(rows < (int64_t(1) << 31) - 4096, kUnsupportedShape, "%s: %lld rows do not fit 32-bit row indices", what,
                (long long)rows);
  MB200_REQUIRE(n <= (1 << 28) && k <= (1 << 28), kUnsupportedShape, "%s: n=%d k=%d", what, n, k);
  return kOk;
}

int check_groups(int experts, const int32_t* offsets, int64_t expert_pitch, int64_t w_pitch, int n, const char* what) {
  MB200_REQUIRE(experts >= 1 && experts <= kMaxExperts, kUnsupportedShape, "%s: %d experts, supported 1..%d", what,
                experts, kMaxExperts);
  MB200_REQUIRE(offsets != nullptr, kInvalidArgument, "%s: offsets is null", what);
  MB200_REQUIRE(expert_pitch % 8 == 0 && (experts == 1 || expert_pitch >= (n - 1) * w_pitch), kUnsupportedShape,
                "%s: %lld elements from expert to expert: a multiple of 8 that holds %d rows", what,
                (long long)expert_pitch, n);
  return kOk;
}

// dy itself, or the copy of it (times slope) in the workspace that the products read; db on the way.
int prepare_output_grad(const char* what, const void*& dy, int dy_fp32, int64_t& dy_pitch, const void* slope,
                        int64_t rows, int n, int fp16, bool products, float* db, void* workspace,
                        int64_t workspace_bytes, cudaStream_t s) {
  const bool copy = products && (slope || dy_fp32 || dy_pitch % 8 || !aligned16(dy));
  if (!copy && !db) return kOk;
  const GradLayout l = grad_layout(rows, n);
  const int64_t need = (copy ? l.dz_bytes : 0) + (db ? l.sum_bytes : 0);
  MB200_REQUIRE(need == 0 || (workspace && aligned16(workspace)), kInvalidArgument,
                "%s: needs a 16-byte aligned workspace", what);
  MB200_REQUIRE(workspace_bytes >= need, kWorkspaceTooSmall, "%s: workspace %lld < %lld bytes", what,
                (long long)workspace_bytes, (long long)need);
  char* ws = reinterpret_cast<char*>(workspace);
  uint16_t* dz = copy ? reinterpret_cast<uint16_t*>(ws) : nullptr;
  float* sums = !db ? nullptr : l.chunks > 1 ? reinterpret_cast<float*>(ws + (copy ? l.dz_bytes : 0)) : db;
  const dim3 grid((n + kColumns - 1) / kColumns, l.chunks);
  output_grad_kernel<<<grid, kColumns * kRowLanes, 0, s>>>(dy, dy_fp32, dy_pitch, slope, int(rows), n, fp16,
                                                           l.rows_per_chunk, dz, l.dz_pitch, sums);
  MB200_CHECK_CUDA(cudaGetLastError());
  if (db && l.chunks > 1) {
    bias_sum_kernel<<<(n + 255) / 256, 256, 0, s>>>(sums, l.chunks, n, db);
    MB200_CHECK_CUDA(cudaGetLastError());
  }
  if (copy) {
    dy = dz;
    dy_pitch = l.dz_pitch;
  }
  return kOk;
}

Epilogue plain_output(void* out, int out_fp32, int fp16) {
  Epilogue e{};
  e.out = out;
  e.out_fp32 = out_fp32;
  e.fp16 = fp16;
  return e;
}

}  // namespace

}  // namespace mb200

using namespace mb200;

extern "C" {

int64_t mb200_linear_workspace_bytes(int64_t rows, int n, int k, int device) {
  if (check_sizes(rows, n, k, "linear_workspace_bytes")) return -1;
  return product_workspace_bytes(kForward, int(rows), n, 0, k, device);
}

int mb200_linear(int precision, const void* x, int64_t x_pitch, int64_t rows, const void* w, int64_t w_pitch, int n,
                 int k, const void* bias, int bias_fp32, int activation, const void* residual, int64_t residual_pitch,
                 void* y, int out_fp32, void* slope, void* workspace, int64_t workspace_bytes, int device,
                 void* stream) {
  const char* what = "linear";
  int rc;
  if ((rc = check_precision(precision, what)) || (rc = check_sizes(rows, n, k, what))) return rc;
  MB200_REQUIRE(activation >= MB200_ACT_NONE && activation <= MB200_ACT_GELU_TANH, kInvalidArgument,
                "linear: activation %d (0..%d)", activation, MB200_ACT_GELU_TANH);
  MB200_REQUIRE(!residual || residual_pitch >= n, kInvalidArgument, "linear: residual pitch %lld < n=%d",
                (long long)residual_pitch, n);
  if (rows == 0) return kOk;
  if ((rc = check_operand(x, x_pitch, k, what, "x")) || (rc = check_operand(w, w_pitch, k, what, "w"))) return rc;
  MB200_REQUIRE(y != nullptr, kInvalidArgument, "linear: y is null");
  ProductArgs p{};
  p.a = w;
  p.a_pitch = w_pitch;
  p.b = x;
  p.b_pitch = x_pitch;
  p.groups = 1;
  p.rows = int(rows);
  p.m = n;
  p.k = k;
  p.epi = plain_output(y, out_fp32 != 0, precision == MB200_PRECISION_FP16);
  p.epi.bias = bias;
  p.epi.bias_fp32 = bias_fp32 != 0;
  p.epi.residual = residual;
  p.epi.residual_pitch = residual_pitch;
  p.epi.slope = slope;
  p.epi.act = activation;
  return launch_product(kForward, p, workspace, workspace_bytes, device, as_stream(stream));
}

int64_t mb200_linear_backward_workspace_bytes(int64_t rows, int n, int k, int device) {
  if (check_sizes(rows, n, k, "linear_backward_workspace_bytes")) return -1;
  const GradLayout l = grad_layout(rows, n);
  return l.dz_bytes + split_bytes(rows, n, k, device, true, true, l.sum_bytes);
}

int mb200_linear_backward(int precision, const void* dy, int dy_fp32, int64_t dy_pitch, const void* slope, const void* x,
                          int64_t x_pitch, int64_t rows, const void* w, int64_t w_pitch, int n, int k, void* dx,
                          void* dw, int dw_fp32, float* db, void* workspace, int64_t workspace_bytes, int device,
                          void* stream) {
  const char* what = "linear_backward";
  int rc;
  if ((rc = check_precision(precision, what)) || (rc = check_sizes(rows, n, k, what))) return rc;
  const int fp16 = precision == MB200_PRECISION_FP16;
  MB200_REQUIRE(!(fp16 && dy_fp32), kInvalidArgument,
                "linear_backward: an fp32 gradient does not fit the range of fp16; scale and round it first");
  MB200_REQUIRE(dy_pitch >= n, kInvalidArgument, "linear_backward: dy pitch %lld < n=%d", (long long)dy_pitch, n);
  cudaStream_t s = as_stream(stream);
  if (rows == 0) {
    if (dw) MB200_CHECK_CUDA(cudaMemsetAsync(dw, 0, size_t(n) * k * (dw_fp32 ? 4 : 2), s));
    if (db) MB200_CHECK_CUDA(cudaMemsetAsync(db, 0, size_t(n) * 4, s));
    return kOk;
  }
  MB200_REQUIRE(dy != nullptr, kInvalidArgument, "linear_backward: dy is null");
  if (dx && (rc = check_operand(w, w_pitch, k, what, "w"))) return rc;
  if (dw && (rc = check_operand(x, x_pitch, k, what, "x"))) return rc;
  const void* given = dy;
  if ((rc = prepare_output_grad(what, dy, dy_fp32, dy_pitch, slope, rows, n, fp16, dx || dw, db, workspace,
                                workspace_bytes, s)))
    return rc;
  const int64_t dz_bytes = dy == given ? 0 : grad_layout(rows, n).dz_bytes;
  void* parts = workspace ? reinterpret_cast<char*>(workspace) + dz_bytes : nullptr;
  const int64_t part_bytes = workspace_bytes - dz_bytes;
  ProductArgs p{};
  p.b = dy;
  p.b_pitch = dy_pitch;
  p.groups = 1;
  p.rows = int(rows);
  p.m = k;
  p.n = n;
  p.k = n;
  if (dx) {
    p.a = w;
    p.a_pitch = w_pitch;
    p.epi = plain_output(dx, 0, fp16);
    if ((rc = launch_product(kInputGrad, p, parts, part_bytes, device, s))) return rc;
  }
  if (dw) {
    p.a = x;
    p.a_pitch = x_pitch;
    p.epi = plain_output(dw, dw_fp32 != 0, fp16);
    if ((rc = launch_product(kWeightGrad, p, parts, part_bytes, device, s))) return rc;
  }
  return kOk;
}

int mb200_grouped_linear(int precision, const void* x, int64_t x_pitch, int64_t rows, const void* w, int64_t w_pitch,
                         int64_t w_expert_pitch, const int32_t* offsets, int experts, int n, int k, void* y, int device,
                         void* stream) {
  const char* what = "grouped_linear";
  int rc;
  if ((rc = check_precision(precision, what)) || (rc = check_sizes(rows, n, k, what)) ||
      (rc = check_groups(experts, offsets, w_expert_pitch, w_pitch, n, what)))
    return rc;
  if (rows == 0) return kOk;
  if ((rc = check_operand(x, x_pitch, k, what, "x")) || (rc = check_operand(w, w_pitch, k, what, "w"))) return rc;
  MB200_REQUIRE(y != nullptr, kInvalidArgument, "grouped_linear: y is null");
  ProductArgs p{};
  p.a = w;
  p.a_pitch = w_pitch;
  p.a_group = w_expert_pitch;
  p.b = x;
  p.b_pitch = x_pitch;
  p.offsets = offsets;
  p.groups = experts;
  p.rows = int(rows);
  p.m = n;
  p.k = k;
  p.epi = plain_output(y, 0, precision == MB200_PRECISION_FP16);
  return launch_product(kForward, p, nullptr, 0, device, as_stream(stream));
}

int64_t mb200_grouped_linear_backward_workspace_bytes(int64_t rows, int n) {
  if (check_sizes(rows, n, 8, "grouped_linear_backward_workspace_bytes")) return -1;
  return grad_layout(rows, n).dz_bytes;
}

int mb200_grouped_linear_backward(int precision, const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch,
                                  int64_t rows, const void* w, int64_t w_pitch, int64_t w_expert_pitch,
                                  const int32_t* offsets, int experts, int n, int k, void* dx, void* dw, int dw_fp32,
                                  void* workspace, int64_t workspace_bytes, int device, void* stream) {
  const char* what = "grouped_linear_backward";
  int rc;
  if ((rc = check_precision(precision, what)) || (rc = check_sizes(rows, n, k, what))) return rc;
  if ((rc = check_groups(experts, offsets, dx ? w_expert_pitch : int64_t(n) * k, dx ? w_pitch : k, n, what))) return rc;
  const int fp16 = precision == MB200_PRECISION_FP16;
  MB200_REQUIRE(dy_pitch >= n, kInvalidArgument, "grouped_linear_backward: dy pitch %lld < n=%d", (long long)dy_pitch, n);
  cudaStream_t s = as_stream(stream);
  if (rows == 0) {
    if (dw) MB200_CHECK_CUDA(cudaMemsetAsync(dw, 0, size_t(experts) * n * k * (dw_fp32 ? 4 : 2), s));
    return kOk;
  }
  MB200_REQUIRE(dy != nullptr, kInvalidArgument, "grouped_linear_backward: dy is null");
  if (dx && (rc = check_operand(w, w_pitch, k, what, "w"))) return rc;
  if (dw && (rc = check_operand(x, x_pitch, k, what, "x"))) return rc;
  if ((rc = prepare_output_grad(what, dy, 0, dy_pitch, nullptr, rows, n, fp16, dx || dw, nullptr, workspace,
                                workspace_bytes, s)))
    return rc;
  ProductArgs p{};
  p.b = dy;
  p.b_pitch = dy_pitch;
  p.offsets = offsets;
  p.groups = experts;
  p.rows = int(rows);
  p.m = k;
  p.n = n;
  p.k = n;
  if (dx) {
    p.a = w;
    p.a_pitch = w_pitch;
    p.a_group = w_expert_pitch;
    p.epi = plain_output(dx, 0, fp16);
    if ((rc = launch_product(kInputGrad, p, nullptr, 0, device, s))) return rc;
  }
  if (dw) {
    p.a = x;
    p.a_pitch = x_pitch;
    p.epi = plain_output(dw, dw_fp32 != 0, fp16);
    if ((rc = launch_product(kWeightGrad, p, nullptr, 0, device, s))) return rc;
  }
  return kOk;
}

int mb200_linear_status(int32_t* status_out, int clear, void* stream) {
  MB200_REQUIRE(status_out != nullptr, kInvalidArgument, "linear_status: null pointer");
  return product_status(status_out, clear, as_stream(stream));
}

}  // extern "C"
