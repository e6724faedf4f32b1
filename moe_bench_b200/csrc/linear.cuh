// Internal interface of the products around the expert FFN: one description for the forward product
// and both gradients, dense (one group) or over ragged row segments, and the epilogue they share.
#pragma once

#include <initializer_list>

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
// Both gradients can be one launch: they share dz and their features.
enum ProductKind : int { kForward = 0, kInputGrad = 1, kWeightGrad = 2, kBothGrads = 3 };
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
  // both gradients: x and the weight gradient, beside a = w and epi.out = the input gradient
  const void* a2;
  int64_t a2_pitch;
  void* out2;
  int out2_fp32;
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

// 1 / (1 + exp(-v)), with an error that grows with |v| where v is negative, since the exponential's argument is rounded: at
// most (9 + 2.35 |v|) 2^-24 of the value by CUDA's bounds of __expf and __fdividef, for v >= 0 9 of them.  Measured with an fp32
// output, SiLU is off by 3.5 steps of 2^-24 from z = -1 up, 9 at -10, 18 at -20 and 65 at -87; GELU's tanh form, whose argument is a
// polynomial, by 5 from -1 up, 47 at -5 and 255 at -10.  All of it is far inside a 16-bit rounding (2^-11 and 2^-8).  Below
// v = -87.3 the divisor is past 2^126 and the quotient 0 instead of less than 2^-126: SiLU is -0 there where up to -1e-36 is meant.
__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

// The normal distribution's mass beyond |z|, 1 - Phi(|z|), over exp(-z^2 / 2): u P(u) with u = 1 / (1 + 0.28 |z|), where P is a
// polynomial fitted to it (relative error at most 1.8e-7 for all z, by reweighted least squares), so that the mass keeps
// its digits however small it is.  GELU and its derivative need that exponential anyway: with the library's erfc on top of
// it 8192 x 2048 -> 7168 took 233 us, 260 with the slope, 163 without an activation.
template <int kCount>
__device__ __forceinline__ void gelu_tail(const float (&z)[kCount], float (&out)[kCount]) {
  constexpr float kP[9] = {0.11170385777950287f, 0.11169980466365814f,   0.10308467596769333f, 0.08363071829f, 0.07277529686689377f,
                           -0.006449869368225336f, 0.0924290269613266f, -0.09359373897314072f, 0.024720141664147377f};
#pragma unroll
  for (int i = 0; i < kCount; i += 2) {
    const float a = __fdividef(1.f, fmaf(0.28f, fabsf(z[i]), 1.f)), b = __fdividef(1.f, fmaf(0.28f, fabsf(z[i + 1]), 1.f));
    const uint64_t u = pack_f32x2(__float_as_uint(a), __float_as_uint(b));
    uint64_t p = pack_f32x2(__float_as_uint(kP[8]), __float_as_uint(kP[8]));
#pragma unroll
    for (int k = 7; k >= 0; --k) {
      uint64_t next = pack_f32x2(__float_as_uint(kP[k]), __float_as_uint(kP[k]));
      fma_f32x2(next, p, u);
      p = next;
    }
    unpack_f32x2(p, out[i], out[i + 1]);
    out[i] *= a;
    out[i + 1] *= b;
  }
}

// act(z) in place, and with kSlope act'(z), for values that have nothing to do with one another.  Both stay finite
// wherever z is; NaN stays NaN in act(z).
template <bool kSlope, int kCount>
__device__ __forceinline__ void activate(int act, float (&z)[kCount], float (&slope)[kCount]) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        if (kSlope) slope[i] = z[i] > 0.f ? 1.f : 0.f;
        z[i] = z[i] < 0.f ? 0.f : z[i];
      }
      break;
    case kActSilu:
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const float s = sigmoid(z[i]);
        if (kSlope) slope[i] = s * (1.f + z[i] * (1.f - s));
        z[i] *= s;
      }
      break;
    case kActGelu: {
      float tail[kCount];
      gelu_tail(z, tail);
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const float e = __expf(-0.5f * z[i] * z[i]);
        const float q = tail[i] * e;
        const float c = z[i] > 0.f ? 1.f - q : q;
        if (kSlope) slope[i] = c + z[i] * (e * 0.39894228040143268f);
        z[i] *= c;
      }
      break;
    }
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        // (1 + tanh u) / 2 = sigmoid(2u); past |z| = 30 it is 0 or 1 in fp32, and z^3 stays finite
        const float t = fminf(fmaxf(z[i], -30.f), 30.f);
        const float c = sigmoid(1.5957691216057307f * (t + 0.044715f * t * t * t));
        if (kSlope) slope[i] = c + t * c * (1.f - c) * (1.5957691216057307f * (1.f + 0.134145f * t * t));
        z[i] *= c;
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < kCount; ++i) slope[i] = 1.f;
  }
}

// The memory that a call writes must be apart from all other memory it is given: a kernel reads its inputs while it writes.
struct Span {
  const char* name;
  uintptr_t begin, end;  // empty where there is no tensor
};
inline Span span_of(const char* name, const void* p, int64_t rows, int64_t pitch, int64_t cols, int64_t bytes) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  return {name, at, p == nullptr || rows <= 0 ? at : at + uintptr_t(((rows - 1) * pitch + cols) * bytes)};
}
inline int check_apart(const char* what, std::initializer_list<Span> written, std::initializer_list<Span> read) {
  auto check = [what](const Span& a, const Span& b) -> int {
    MB200_REQUIRE(a.begin >= b.end || b.begin >= a.end || a.begin == a.end || b.begin == b.end, kInvalidArgument,
                  "%s: %s and %s share memory", what, a.name, b.name);
    return kOk;
  };
  int rc;
  for (const Span* w = written.begin(); w != written.end(); ++w) {
    for (const Span& r : read)
      if ((rc = check(*w, r))) return rc;
    for (const Span* v = w + 1; v != written.end(); ++v)
      if ((rc = check(*w, *v))) return rc;
  }
  return kOk;
}

// layer_norm.cu
// out[i] = sum over k of parts[k][i], i < columns, in a fixed order; what lies from `first` on goes to `rest` instead.
// Either may be null: its columns are left out.
int launch_column_sums(const float* parts, int count, int64_t columns, float* out, int64_t first, float* rest, cudaStream_t stream);

// few_rows.cu: the dense forward product of at most kFewRows rows
constexpr int kFewRows = 16;
int launch_few_rows(const ProductArgs& args, int device, cudaStream_t stream);

// products.cu
// status word of the products on the current device
int product_status(int* status_out, int clear, cudaStream_t stream);
int launch_product(ProductKind kind, const ProductArgs& args, int device, cudaStream_t stream);
// The gradients of a forward product that are wanted (dx or dw may be null): `args` says the rest, b = dz among it.
int launch_gradients(const ProductArgs& args, void* dx, void* dw, int dw_fp32, const void* w, int64_t w_pitch, int64_t w_group,
                     const void* x, int64_t x_pitch, int device, cudaStream_t stream);

}  // namespace mb200
