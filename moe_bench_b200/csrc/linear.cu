// extern "C" entry points of the products around the expert FFN (dense with bias, activation and
// residual; ragged row segments) and of their gradients, and the elementwise step ahead of the
// gradients' products.

#include <algorithm>
#include <type_traits>

#include "../../include/moe_bench_b200.h"
#include "linear.cuh"

namespace mb200 {

namespace {

cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// ---- dz = dy * slope, and its column sums ----------------------------------------------------------
// One pass over dy and slope, bound by HBM.  A block takes 32 * kVec columns of a run of rows, 8 rows side by side: a
// thread has kVec neighbouring columns (16 bytes, or one element where rows do not start on vectors) of every eighth
// row, four of them requested ahead, and sums them in fp32; the eight are added in order, and the runs' sums by
// column_sums_kernel, or where there are up to eight runs by the first block of a cluster.  With slope 4096 x 2048 takes 10 us
// and 8192 x 7168 62 us with both kernels, 1.3 and 1.15 times its bytes at the copy rate (one element per thread in 64 runs:
// 22 and 236 us).  With an fp32 dy a thread keeps 41 words in local memory, for four blocks on an SM; db alone of 8192 x 7168
// then takes 46 us and with the slope 72, 1.3 times the bytes of either.
//
// dz is rounded to 16 bits because the tensor cores take operands of 16 bits; two parts of it would double both products, which are
// 190 of the 205 us of 4096 x 7168 -> 2048.  dx and dw are then off by 2.3e-3 of their size in bf16 instead of 1.7e-3, the rounding of
// the outputs alone.  The sums for db are of dz before it.
constexpr int kRowLanes = 8;
constexpr int kRowsAhead = 4;

struct OutputGrad {
  const void* dy;
  const void* slope;   // dense, or null
  uint16_t* dz;        // or null: only the sums
  float* sums;         // [chunks][n], or null
  int64_t dy_pitch, dz_pitch;
  int rows, n, rows_per_chunk;
  int fp16;
  int joined;          // the runs of a column are a cluster
};

// kVec elements as they lie in memory
template <int kVec, bool kFp32>
struct Raw {
  using Word = typename std::conditional<kVec == 8, uint4, typename std::conditional<kFp32, float, uint16_t>::type>::type;
  static constexpr int kWords = kVec == 8 && kFp32 ? 2 : 1;
  Word w[kWords];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    const Word* q = reinterpret_cast<const Word*>(reinterpret_cast<const char*>(p) + at * (kFp32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = __ldcs(q + i);
  }
  __device__ __forceinline__ void read(int fp16, float (&out)[kVec]) const {
    if constexpr (kFp32) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) out[i] = reinterpret_cast<const float*>(w)[i];
    } else if constexpr (kVec == 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = 0.f;
      add_h16x8(w[0], out, fp16);
    } else {
      out[0] = load_h16(w, 0, fp16);
    }
  }
};

template <int kVec, bool kFp32>
__global__ void __launch_bounds__(256, 4) output_grad_kernel(const OutputGrad p) {
  __shared__ float part[kRowLanes][32 * kVec];
  const int lane = threadIdx.x & 31, row_lane = threadIdx.x >> 5;
  const int col = (int(blockIdx.x) * 32 + lane) * kVec;
  const int64_t first = int64_t(blockIdx.y) * p.rows_per_chunk;
  const int64_t last = first + p.rows_per_chunk < p.rows ? first + p.rows_per_chunk : p.rows;
  float sum[kVec] = {};
  if (col < p.n)
    for (int64_t r = first + row_lane; r < last; r += kRowLanes * kRowsAhead) {
      Raw<kVec, kFp32> dy[kRowsAhead];
      Raw<kVec, false> slope[kRowsAhead];
      // a run's last rows are asked for more than once instead of not at all: no branch stands between the loads
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) dy[u].load(p.dy, min(r + u * kRowLanes, last - 1) * p.dy_pitch + col);
      if (p.slope)
#pragma unroll
        for (int u = 0; u < kRowsAhead; ++u) slope[u].load(p.slope, min(r + u * kRowLanes, last - 1) * p.n + col);
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) {
        const int64_t row = r + u * kRowLanes;
        if (row < last) {
          float v[kVec];
          dy[u].read(p.fp16, v);
          if (p.slope) {
            float s[kVec];
            slope[u].read(p.fp16, s);
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[i] *= s[i];
          }
#pragma unroll
          for (int i = 0; i < kVec; ++i) sum[i] += v[i];
          if (p.dz) {
            uint16_t* to = p.dz + row * p.dz_pitch + col;
            if constexpr (kVec == 8) *reinterpret_cast<uint4*>(to) = pack_h16x8(v, p.fp16);
            else *to = to_h16(v[0], p.fp16);
          }
        }
      }
    }
  if (p.sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < kVec; ++i) part[row_lane][lane * kVec + i] = sum[i];
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * kVec; c += 256) {
    const int at = int(blockIdx.x) * 32 * kVec + c;
    if (at >= p.n) continue;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kRowLanes; ++i) t += part[i][c];
    if (p.joined) part[0][c] = t;
    else p.sums[int64_t(blockIdx.y) * p.n + at] = t;
  }
  if (!p.joined) return;
  cluster_sync();
  if (blockIdx.y == 0)
    for (int c = threadIdx.x; c < 32 * kVec; c += 256) {
      const int at = int(blockIdx.x) * 32 * kVec + c;
      if (at >= p.n) continue;
      float t = 0.f;
      for (int k = 0; k < int(gridDim.y); ++k) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(smem_u32(&part[0][c]), k)) : "memory");
        t += v;
      }
      p.sums[at] = t;
    }
  cluster_sync();  // the first block has read the others' sums
}

constexpr int kMostJoined = 8;      // runs that a cluster joins
constexpr int kRowsJoined = 512;    // rows that are cut into so few runs

struct GradLayout {
  int64_t dz_pitch, dz_bytes, sum_bytes;
  int chunks, rows_per_chunk;
};
// `width`: columns of a block, 256 or (single elements) 32; runs of 256 columns are never fewer.
GradLayout grad_layout(int64_t rows, int n, int width, int device) {
  const int sms = device_sm_count(device) > 0 ? device_sm_count(device) : 1;
  GradLayout l;
  l.dz_pitch = round_up(n, 8);
  l.dz_bytes = round_up(rows * l.dz_pitch * 2, 256);
  // eight blocks per SM, as long as each has 32 rows (16384 x 515, single elements: 29 us with as many runs as 256 columns have)
  int64_t chunks = 8 * sms / ((n + width - 1) / width);
  if (rows <= kRowsJoined) chunks = std::min(chunks, int64_t(kMostJoined));
  chunks = std::max(chunks, int64_t(1));
  constexpr int kTurn = kRowLanes * kRowsAhead;
  l.rows_per_chunk = int(((rows + chunks - 1) / chunks + kTurn - 1) / kTurn * kTurn);
  l.chunks = l.rows_per_chunk > 0 ? int((rows + l.rows_per_chunk - 1) / l.rows_per_chunk) : 1;
  l.sum_bytes = l.chunks > kMostJoined ? round_up(int64_t(l.chunks) * n * 4, 256) : 0;
  return l;
}
bool grad_vectors(const void* dy, int64_t dy_pitch, const void* slope, int n) {
  return n % 8 == 0 && dy_pitch % 8 == 0 && aligned16(dy) && aligned16(slope);
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

// Whether the products read a copy of dy (times slope), in the workspace.
bool copies_output_grad(const void* dy, int dy_fp32, int64_t dy_pitch, const void* slope) {
  return slope || dy_fp32 || dy_pitch % 8 || !aligned16(dy);
}

// `need`: bytes of the workspace that the call uses
int check_grad_workspace(const char* what, bool copy, bool sums, int64_t rows, int n, const void* workspace, int64_t workspace_bytes,
                         int device, int64_t& need) {
  need = 0;
  if (!copy && !sums) return kOk;
  const GradLayout l = grad_layout(rows, n, 256, device);
  need = (copy ? l.dz_bytes : 0) + (sums ? l.sum_bytes : 0);
  MB200_REQUIRE(need == 0 || (workspace && aligned16(workspace)), kInvalidArgument,
                "%s: needs a 16-byte aligned workspace", what);
  MB200_REQUIRE(workspace_bytes >= need, kWorkspaceTooSmall, "%s: workspace %lld < %lld bytes", what,
                (long long)workspace_bytes, (long long)need);
  return kOk;
}

// dy itself, or the copy of it (times slope) in the workspace that the products read; db on the way.
int prepare_output_grad(const void*& dy, int dy_fp32, int64_t& dy_pitch, const void* slope, int64_t rows, int n, int fp16, bool copy,
                        float* db, void* workspace, int device, cudaStream_t s) {
  int rc;
  if (!copy && !db) return kOk;
  const bool vec = grad_vectors(dy, dy_pitch, slope, n);
  const GradLayout l = grad_layout(rows, n, vec ? 256 : 32, device);
  char* ws = reinterpret_cast<char*>(workspace);
  OutputGrad g{};
  g.dy = dy;
  g.slope = slope;
  g.dz = copy ? reinterpret_cast<uint16_t*>(ws) : nullptr;
  g.joined = db && l.chunks > 1 && l.chunks <= kMostJoined;
  g.sums = !db ? nullptr : l.chunks > kMostJoined ? reinterpret_cast<float*>(ws + (copy ? l.dz_bytes : 0)) : db;
  g.dy_pitch = dy_pitch;
  g.dz_pitch = l.dz_pitch;
  g.rows = int(rows);
  g.n = n;
  g.rows_per_chunk = l.rows_per_chunk;
  g.fp16 = fp16;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
  attr[0].val.clusterDim.y = unsigned(l.chunks);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((n + (vec ? 255 : 31)) / (vec ? 256 : 32), l.chunks);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = g.joined ? 1 : 0;
  const auto kernel = vec ? (dy_fp32 ? output_grad_kernel<8, true> : output_grad_kernel<8, false>)
                          : (dy_fp32 ? output_grad_kernel<1, true> : output_grad_kernel<1, false>);
  MB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, g));
  if (db && l.chunks > kMostJoined) {
    if ((rc = launch_column_sums(g.sums, l.chunks, n, db, n, nullptr, s))) return rc;
  }
  uint16_t* dz = g.dz;
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

int mb200_linear(int precision, const void* x, int64_t x_pitch, int64_t rows, const void* w, int64_t w_pitch, int n,
                 int k, const void* bias, int bias_fp32, int activation, const void* residual, int64_t residual_pitch,
                 void* y, int out_fp32, void* slope, int device, void* stream) {
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
  const bool in_place = residual == y && !out_fp32 && (residual_pitch == n || rows == 1);
  if ((rc = check_apart(what, {span_of("y", y, rows, n, n, out_fp32 ? 4 : 2), span_of("slope", slope, rows, n, n, 2)},
                        {span_of("x", x, rows, x_pitch, k, 2), span_of("w", w, n, w_pitch, k, 2),
                         span_of("bias", bias, 1, n, n, bias_fp32 ? 4 : 2),
                         span_of("residual", in_place ? nullptr : residual, rows, residual_pitch, n, 2)})))
    return rc;
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
  if (rows <= kFewRows) return launch_few_rows(p, device, as_stream(stream));
  return launch_product(kForward, p, device, as_stream(stream));
}

int64_t mb200_linear_backward_workspace_bytes(int64_t rows, int n, int copies_dy, int device) {
  if (check_sizes(rows, n, 8, "linear_backward_workspace_bytes")) return -1;
  const GradLayout l = grad_layout(rows, n, 256, device);
  return (copies_dy ? l.dz_bytes : 0) + l.sum_bytes;
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
  const bool copy = (dx || dw) && copies_output_grad(dy, dy_fp32, dy_pitch, slope);
  int64_t need;
  if ((rc = check_grad_workspace(what, copy, db, rows, n, workspace, workspace_bytes, device, need)) ||
      (rc = check_apart(what,
                        {span_of("dx", dx, rows, k, k, 2), span_of("dw", dw, n, k, k, dw_fp32 ? 4 : 2), span_of("db", db, 1, n, n, 4),
                         span_of("workspace", workspace, 1, need, need, 1)},
                        {span_of("dy", dy, rows, dy_pitch, n, dy_fp32 ? 4 : 2), span_of("slope", slope, rows, n, n, 2),
                         span_of("x", dw ? x : nullptr, rows, x_pitch, k, 2), span_of("w", dx ? w : nullptr, n, w_pitch, k, 2)})))
    return rc;
  if ((rc = prepare_output_grad(dy, dy_fp32, dy_pitch, slope, rows, n, fp16, copy, db, workspace, device, s))) return rc;
  ProductArgs p{};
  p.b = dy;
  p.b_pitch = dy_pitch;
  p.groups = 1;
  p.rows = int(rows);
  p.m = k;
  p.n = n;
  p.k = n;
  p.epi = plain_output(nullptr, 0, fp16);
  return launch_gradients(p, dx, dw, dw_fp32 != 0, w, w_pitch, 0, x, x_pitch, device, s);
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
  if ((rc = check_apart(what, {span_of("y", y, rows, n, n, 2)},
                        {span_of("x", x, rows, x_pitch, k, 2), span_of("w", w, experts, w_expert_pitch, (n - 1) * w_pitch + k, 2),
                         span_of("offsets", offsets, 1, 0, experts + 1, 4)})))
    return rc;
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
  return launch_product(kForward, p, device, as_stream(stream));
}

int64_t mb200_grouped_linear_backward_workspace_bytes(int64_t rows, int n) {
  if (check_sizes(rows, n, 8, "grouped_linear_backward_workspace_bytes")) return -1;
  return grad_layout(rows, n, 256, 0).dz_bytes;
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
  const bool copy = (dx || dw) && copies_output_grad(dy, 0, dy_pitch, nullptr);
  int64_t need;
  if ((rc = check_grad_workspace(what, copy, false, rows, n, workspace, workspace_bytes, device, need)) ||
      (rc = check_apart(what,
                        {span_of("dx", dx, rows, k, k, 2), span_of("dw", dw, int64_t(experts) * n, k, k, dw_fp32 ? 4 : 2),
                         span_of("workspace", workspace, 1, need, need, 1)},
                        {span_of("dy", dy, rows, dy_pitch, n, 2), span_of("x", dw ? x : nullptr, rows, x_pitch, k, 2),
                         span_of("w", dx ? w : nullptr, experts, w_expert_pitch, (n - 1) * w_pitch + k, 2),
                         span_of("offsets", offsets, 1, 0, experts + 1, 4)})))
    return rc;
  if ((rc = prepare_output_grad(dy, 0, dy_pitch, nullptr, rows, n, fp16, copy, nullptr, workspace, device, s))) return rc;
  ProductArgs p{};
  p.b = dy;
  p.b_pitch = dy_pitch;
  p.offsets = offsets;
  p.groups = experts;
  p.rows = int(rows);
  p.m = k;
  p.n = n;
  p.k = n;
  p.epi = plain_output(nullptr, 0, fp16);
  return launch_gradients(p, dx, dw, dw_fp32 != 0, w, w_pitch, w_expert_pitch, x, x_pitch, device, s);
}

int mb200_linear_status(int32_t* status_out, int clear, void* stream) {
  MB200_REQUIRE(status_out != nullptr, kInvalidArgument, "linear_status: null pointer");
  return product_status(status_out, clear, as_stream(stream));
}

}  // extern "C"
