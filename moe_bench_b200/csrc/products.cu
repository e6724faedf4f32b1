// The products around the expert FFN (linear.cuh): every output element is one dot product.

#include "linear.cuh"

namespace mb200 {

namespace {

constexpr int kTile = 64;   // features and output rows of a block's tile
constexpr int kDepth = 16;  // terms of the sums per step

// 256 threads, 4 x 4 outputs each, operands staged in shared memory as fp32.
template <int kKind>
__global__ void __launch_bounds__(256) product_kernel(const ProductArgs p) {
  __shared__ float sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  const int group = blockIdx.z;
  const int f0 = blockIdx.x * kTile;
  int begin, end;
  segment_of(p, group, begin, end);
  const int count = kKind == kWeightGrad ? p.n : end - begin;   // output rows of the group
  const int depth = kKind == kWeightGrad ? end - begin : p.k;
  const int fp16 = p.epi.fp16;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int j0 = blockIdx.y * kTile; j0 < count; j0 += gridDim.y * kTile) {
    float acc[4][4] = {};
    for (int c0 = 0; c0 < depth; c0 += kDepth) {
      for (int i = threadIdx.x; i < kTile * kDepth; i += 256) {
        // neighbouring threads read neighbouring elements
        const int ca = kKind == kForward ? i % kDepth : i / kTile, fa = kKind == kForward ? i / kDepth : i % kTile;
        float v = 0.f;
        if (f0 + fa < p.m && c0 + ca < depth) {
          const int64_t at = kKind == kForward     ? group * p.a_group + (f0 + fa) * p.a_pitch + c0 + ca
                             : kKind == kInputGrad ? group * p.a_group + (c0 + ca) * p.a_pitch + f0 + fa
                                                   : int64_t(begin + c0 + ca) * p.a_pitch + f0 + fa;
          v = load_h16(p.a, at, fp16);
        }
        sa[ca][fa] = v;
        const int cb = kKind == kWeightGrad ? i / kTile : i % kDepth, jb = kKind == kWeightGrad ? i % kTile : i / kDepth;
        v = 0.f;
        if (j0 + jb < count && c0 + cb < depth) {
          const int64_t at = kKind == kWeightGrad ? int64_t(begin + c0 + cb) * p.b_pitch + j0 + jb
                                                  : int64_t(begin + j0 + jb) * p.b_pitch + c0 + cb;
          v = load_h16(p.b, at, fp16);
        }
        sb[cb][jb] = v;
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < kDepth; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[c][tx + 16 * i], sb[c][ty + 16 * j], acc[i][j]);
      __syncthreads();
    }
    for (int j = 0; j < 4; ++j)
      for (int i = 0; i < 4; ++i) {
        const int row = j0 + ty + 16 * j, f = f0 + tx + 16 * i;
        if (row >= count || f >= p.m) continue;
        const int64_t at = kKind == kWeightGrad ? int64_t(group) * p.n + row : int64_t(begin) + row;
        finish_element(p.epi, p.m, at, f, acc[i][j]);
      }
  }
}

}  // namespace

int launch_product(ProductKind kind, const ProductArgs& args, int device, cudaStream_t stream) {
  (void)device;
  const int64_t most = kind == kWeightGrad ? args.n : args.rows;
  const unsigned by = unsigned(most <= 0 ? 1 : (most + kTile - 1) / kTile < 512 ? (most + kTile - 1) / kTile : 512);
  const dim3 grid((args.m + kTile - 1) / kTile, by, args.groups);
  if (kind == kForward) product_kernel<kForward><<<grid, 256, 0, stream>>>(args);
  else if (kind == kInputGrad) product_kernel<kInputGrad><<<grid, 256, 0, stream>>>(args);
  else product_kernel<kWeightGrad><<<grid, 256, 0, stream>>>(args);
  MB200_CHECK_CUDA(cudaGetLastError());
  return kOk;
}

}  // namespace mb200
