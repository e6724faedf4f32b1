// Internal interface of the products around the expert FFN: one description for the forward product
// and both gradients, dense (one group) or over ragged row segments, and the epilogue they share.
#pragma once

#include "layer.cuh"

namespace mb200 {

enum Activation : int { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };

// What happens to a 32-bit sum z of the product: y = act(z + bias) + residual, slope = act'(z + bias).
// Everything is computed in fp32; y and slope are rounded once, when they are stored.
struct Epilogue {
  void* out;                // [output rows][m], dense
  const void* bias;         // [m] or null
  const void* residual;     // [output rows][residual_pitch] or null; may be `out`
  void* slope;              // [output rows][m] or null
  int64_t residual_pitch;
  int bias_fp32;
  int out_fp32;
  int act;                  // Activation
  int fp16;                 // the 16-bit type is fp16 instead of bf16
};

// out[j][f] = sum over c of A(f, c) B(j, c), f < m side by side in memory:
//   forward      out[row][f] = sum_k  w[g][f][k] x[row][k]         rows of segment g
//   input grad   out[row][f] = sum_n  w[g][n][f] dz[row][n]        rows of segment g
//   weight grad  out[g*n + j][f] = sum_row x[row][f] dz[row][j]    rows of segment g
enum ProductKind : int { kForward = 0, kInputGrad = 1, kWeightGrad = 2 };
struct ProductArgs {
  const void* a;            // feature side: w, w, x
  const void* b;            // row side: x, dz, dz
  int64_t a_pitch, a_group, b_pitch;  // elements from row to row (of w: and from group to group)
  const int* offsets;       // [groups + 1], or null: one group of all rows
  int groups;
  int rows;
  int m;                    // features
  int n;                    // weight grad: output rows per group
  int k;                    // forward, input grad: length of the sum
  Epilogue epi;
};

// Segment g of the rows, cut to [0, rows] whatever the offsets hold.
__device__ __forceinline__ void segment_of(const ProductArgs& p, int g, int& begin, int& end) {
  if (p.offsets == nullptr) {
    begin = 0;
    end = p.rows;
    return;
  }
  begin = min(max(__ldg(p.offsets + g), 0), p.rows);
  end = max(min(max(__ldg(p.offsets + g + 1), 0), p.rows), begin);
}

__device__ __forceinline__ float load_h16(const void* p, int64_t i, int fp16) {
  return fp16 ? __half2float(reinterpret_cast<const __half*>(p)[i])
              : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

// act(z), and with kSlope act'(z).  Both stay finite wherever z is; NaN stays NaN in act(z).
template <bool kSlope>
__device__ __forceinline__ float activate(int act, float z, float& slope) {
  slope = 1.f;
  switch (act) {
    case kActRelu:
      if (kSlope) slope = z > 0.f ? 1.f : 0.f;
      return z < 0.f ? 0.f : z;
    case kActSilu: {
      const float s = 1.f / (1.f + expf(-z));
      if (kSlope) slope = s * (1.f + z * (1.f - s));
      return z * s;
    }
    case kActGelu: {
      const float c = 0.5f + 0.5f * erff(z * 0.70710678118654752f);
      // below -3 the sum of 1/2 and erf/2 cancels: the same value by the complement
      const float cdf = z < -1.f ? 0.5f * erfcf(-z * 0.70710678118654752f) : c;
      if (kSlope) slope = cdf + z * expf(-0.5f * z * z) * 0.39894228040143268f;
      return z * cdf;
    }
    case kActGeluTanh: {
      // (1 + tanh u) / 2 = 1 / (1 + exp(-2u)); past |z| = 30 it is 0 or 1 in fp32, and z^3 stays finite
      const float t = fminf(fmaxf(z, -30.f), 30.f);
      const float u = 0.79788456080286536f * (t + 0.044715f * t * t * t);
      const float c = 1.f / (1.f + expf(-2.f * u));
      if (kSlope) slope = c + 2.f * t * c * (1.f - c) * (0.79788456080286536f * (1.f + 0.134145f * t * t));
      return z * c;
    }
    default:
      return z;
  }
}

// `residual` may be `out`: no promise that it is constant.
struct Bias4 {
  float v[4];
};
__device__ __forceinline__ Bias4 load_bias4(const Epilogue& e, int m, int f) {
  Bias4 b{};
  if (e.bias)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f + i < m) b.v[i] = e.bias_fp32 ? __ldg(reinterpret_cast<const float*>(e.bias) + f + i) : load_h16(e.bias, f + i, e.fp16);
  return b;
}
__device__ __forceinline__ uint2 pack_h16x4(const float (&v)[4], int fp16) {
  return make_uint2(pack_h16x2(v[0], v[1], fp16), pack_h16x2(v[2], v[3], fp16));
}

// One element.
__device__ __forceinline__ void finish_element(const Epilogue& e, int m, int64_t row, int f, float z) {
  if (e.bias) z += e.bias_fp32 ? reinterpret_cast<const float*>(e.bias)[f] : load_h16(e.bias, f, e.fp16);
  float slope = 1.f;
  float y;
  if (e.slope) {
    y = activate<true>(e.act, z, slope);
    reinterpret_cast<uint16_t*>(e.slope)[row * m + f] = to_h16(slope, e.fp16);
  } else {
    y = activate<false>(e.act, z, slope);
  }
  if (e.residual) y += load_h16(e.residual, row * e.residual_pitch + f, e.fp16);
  if (e.out_fp32)
    reinterpret_cast<float*>(e.out)[row * m + f] = y;
  else
    reinterpret_cast<uint16_t*>(e.out)[row * m + f] = to_h16(y, e.fp16);
}

// Four features side by side, f a multiple of 4.  `vec`: every tensor takes them as one access (then m is a multiple of 4).
__device__ __forceinline__ void finish4(const Epilogue& e, int m, int64_t row, int f, float (&z)[4], const Bias4& bias,
                                        bool vec) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f + i < m) finish_element(e, m, row, f + i, z[i]);
    return;
  }
  float slope[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] += bias.v[i];
  if (e.slope) {
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = activate<true>(e.act, z[i], slope[i]);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(e.slope) + row * m + f) = pack_h16x4(slope, e.fp16);
  } else if (e.act) {
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = activate<false>(e.act, z[i], slope[i]);
  }
  if (e.residual) {
    const uint2 r = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(e.residual) + row * e.residual_pitch + f);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] += load_h16(&r, i, e.fp16);
  }
  if (e.out_fp32)
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(e.out) + row * m + f) = make_float4(z[0], z[1], z[2], z[3]);
  else
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(e.out) + row * m + f) = pack_h16x4(z, e.fp16);
}

// products.cu
// Bytes of workspace that launch_product wants for a dense product (one group), 0 where its sums are not split.
int64_t product_workspace_bytes(ProductKind kind, int rows, int m, int n, int k, int device);
// status word of the products on the current device
int product_status(int* status_out, int clear, cudaStream_t stream);
int launch_product(ProductKind kind, const ProductArgs& args, void* workspace, int64_t workspace_bytes, int device,
                   cudaStream_t stream);

}  // namespace mb200
