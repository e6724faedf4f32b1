// Layer norm over the last dimension and its gradients.
//
//   mean = sum(x) / hidden, rstd = 1 / sqrt(sum((x - mean)^2) / hidden + eps), y = (x - mean) rstd w + b
//   h = (x - mean) rstd, g = dy w:  dx = rstd (g - mean(g) - h mean(g h)),  dw = sum dy h,  db = sum dy
//
// Statistics, gradients of the parameters and everything in between are fp32; y and dx are rounded once.
//
// Bound by HBM: bf16 rows of 7168 run at 5.7 TB/s forward (32768 of them 165 us, 143 at the copy rate) and at 5.1 backward (16384
// of them 139 us, 108 at the copy rate); what is missing is the exchange within a row, which has 14 warps on an SM to hide
// behind.  8 rows take 3.7 us forward and 7.8 backward, half of that the second kernel.

#include <algorithm>
#include <atomic>

#include "../../include/moe_bench_b200.h"
#include "linear.cuh"

namespace mb200 {

namespace {

struct NormArgs {
  const void* x;
  const void* dy;       // backward
  int64_t x_pitch, dy_pitch;
  int64_t rows, hidden;
  const void* weight;   // null: 1
  const void* bias;     // null: 0
  int params_fp32;
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

// ---- rows that fit the registers of a block ---------------------------------------------------------
// A row is kPer vectors of kVec elements in each of blockDim.x threads; blockDim.y rows per block (more than one only
// where a row takes a single warp).  x (and dy) are read once, the next row's while this one is reduced; a thread has
// the same columns of every row, so its parameters stay in registers.  HBM is the bound, but 16-bit rows come close to
// the issue slots (two elements per 32-bit word to take apart and put together), so all arithmetic is on pairs of
// fp32 (f32x2) and every element is taken apart once: 951 instructions per warp and row of 7168 (bf16, forward) became 430.

// kVec elements side by side, as one access (16 bytes) or one element
template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Vec {
  T v[kVec];
};
template <typename T, int kVec>
__device__ __forceinline__ Vec<T, kVec> load_once(const T* p) {
  Vec<T, kVec> r;
  if constexpr (sizeof(T) * kVec == 16) {
    *reinterpret_cast<uint4*>(&r) = __ldcs(reinterpret_cast<const uint4*>(p));
  } else if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint16_t*>(&r) = __ldcs(reinterpret_cast<const unsigned short*>(p));
  } else {
    *reinterpret_cast<float*>(&r) = __ldcs(reinterpret_cast<const float*>(p));
  }
  return r;
}

// Two fp32 values that an instruction works on together; each is rounded as it would be alone.
using Pair = uint64_t;
__device__ __forceinline__ Pair pair_of(float a, float b) { return pack_f32x2(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float sum_of(Pair p) {
  float a, b;
  unpack_f32x2(p, a, b);
  return a + b;
}

// A thread's kPer vectors as pairs.
template <typename T, int kVec, int kPer>
__device__ __forceinline__ void take_apart(const Vec<T, kVec> (&v)[kPer], Pair (&out)[kVec * kPer / 2]) {
  if constexpr (kVec == 1) {
#pragma unroll
    for (int k = 0; k < kPer; k += 2) out[k / 2] = pair_of(to_float(v[k].v[0]), to_float(v[k + 1].v[0]));
  } else if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&v[k]);
#pragma unroll
      for (int i = 0; i < kVec / 2; ++i) {
        if constexpr (sizeof(T) == 2 && __is_same(T, __half)) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + i));
          out[k * kVec / 2 + i] = pair_of(f.x, f.y);
        } else {
          out[k * kVec / 2 + i] = pack_f32x2(w[i] << 16, w[i] & 0xffff0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
#pragma unroll
      for (int i = 0; i < kVec / 2; ++i) out[k * kVec / 2 + i] = pair_of(v[k].v[2 * i], v[k].v[2 * i + 1]);
  }
}

// `to`: this thread's first vector of the output row
template <typename T, int kVec, int kPer>
__device__ __forceinline__ void store_row(T* to, uint32_t mask, const Pair (&p)[kVec * kPer / 2]) {
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (mask >> k & 1) {
      Vec<T, kVec> o;
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const int e = k * kVec + i;
        float f[2];
        unpack_f32x2(p[e / 2], f[0], f[1]);
        if constexpr (sizeof(T) == 2 && kVec > 1) {
          if (i % 2 == 0) reinterpret_cast<uint32_t*>(&o)[i / 2] = pack_h16x2(f[0], f[1], __is_same(T, __half));
        } else {
          o.v[i] = from_float<T>(f[e & 1]);
        }
      }
      *reinterpret_cast<Vec<T, kVec>*>(to + k * int(blockDim.x) * kVec) = o;
    }
  }
}

// Parameters of this thread's columns, of T or fp32; `other` where there are none and past the row's end.
template <typename T, int kVec, int kPer>
__device__ __forceinline__ void load_params(const void* p, int fp32, int64_t hidden, float other, Pair (&out)[kVec * kPer / 2]) {
  float f[kVec * kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int64_t at = int64_t(threadIdx.x + k * blockDim.x) * kVec;
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[k * kVec + i] = other;
    if (p == nullptr || at >= hidden) continue;
    if (fp32) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) f[k * kVec + i] = __ldg(reinterpret_cast<const float*>(p) + at + i);
    } else {
      const Vec<T, kVec> r = *reinterpret_cast<const Vec<T, kVec>*>(reinterpret_cast<const T*>(p) + at);
#pragma unroll
      for (int i = 0; i < kVec; ++i) f[k * kVec + i] = to_float(r.v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kVec * kPer / 2; ++i) out[i] = pair_of(f[2 * i], f[2 * i + 1]);
}

// Sums of kCount values over a row's threads, the same in all of them.  The calls of a block take the two halves of
// `part` in turn, so that one barrier is enough: of the row's own threads, where a block takes several rows side by side.
template <int kCount>
__device__ __forceinline__ void row_sums(float (&v)[kCount], float (*part)[32][2], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int c = 0; c < kCount; ++c) v[c] += __shfl_xor_sync(0xffffffffu, v[c], o);
  if (blockDim.x == 32) return;
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0)
#pragma unroll
    for (int c = 0; c < kCount; ++c) part[turn][threadIdx.x >> 5][c] = v[c];
  __syncwarp();  // the barrier is reached by whole warps
  asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.y + 1), "r"(blockDim.x) : "memory");
#pragma unroll
  for (int c = 0; c < kCount; ++c) v[c] = lane < warps ? part[turn][lane][c] : 0.f;
  turn ^= 1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int c = 0; c < kCount; ++c) v[c] += __shfl_xor_sync(0xffffffffu, v[c], o);
}

// The rows of a thread on their way: kStages rows ahead in shared memory by cp.async, every thread its own vectors (so
// that nothing but its own wait stands between copy and use), or where single elements are copied the next row in registers.
// Columns past the row's end and rows past the last read as zero.
constexpr int kStages = 2;  // three: 1 to 2 % slower
template <typename T, int kVec, int kPer, int kTensors>
struct RowStream {
  static constexpr bool kShared = kVec > 1;
  static constexpr int kAhead = kShared ? kStages : 1;
  const T* next[kTensors];     // this thread's first vector of the next row to ask for
  int64_t row_step[kTensors];  // elements to the one after it
  int rows_left;               // rows that this thread's group has still to ask for
  uint32_t mask;               // which of its vectors lie inside the row
  uint32_t slot, vec_bytes;    // its first vector of stage 0, bytes from one to the next
  Vec<T, kVec> ahead[kShared ? 1 : kTensors][kPer];

  __device__ __forceinline__ RowStream(const void* p0, int64_t pitch0, const void* p1, int64_t pitch1, int64_t first_row, int64_t step,
                                       int64_t rows, uint32_t mask_, uint32_t smem)
      : mask(mask_) {
    rows_left = first_row < rows ? int((rows - first_row + step - 1) / step) : 0;
    const int64_t row = rows_left > 0 ? first_row : 0;
    next[0] = reinterpret_cast<const T*>(p0) + row * pitch0 + int(threadIdx.x) * kVec;
    row_step[0] = step * pitch0;
    if constexpr (kTensors > 1) {
      next[1] = reinterpret_cast<const T*>(p1) + row * pitch1 + int(threadIdx.x) * kVec;
      row_step[1] = step * pitch1;
    }
    vec_bytes = blockDim.x * blockDim.y * 16;
    slot = smem + (threadIdx.y * blockDim.x + threadIdx.x) * 16;
  }
  __device__ __forceinline__ void request(int stage) {
    const uint32_t here = rows_left > 0 ? mask : 0u;
#pragma unroll
    for (int n = 0; n < kTensors; ++n)
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const bool inside = here >> k & 1;
        const T* from = next[n] + k * int(blockDim.x) * kVec;
        if constexpr (kShared) {
          const uint32_t to = slot + ((stage * kTensors + n) * kPer + k) * vec_bytes;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(inside ? from : next[n]), "r"(inside ? 16 : 0)
                       : "memory");
        } else {
          ahead[n][k] = Vec<T, kVec>{};
          if (inside) ahead[n][k] = load_once<T, kVec>(from);
        }
      }
    if constexpr (kShared) asm volatile("cp.async.commit_group;" ::: "memory");
    --rows_left;
#pragma unroll
    for (int n = 0; n < kTensors; ++n) next[n] += rows_left > 0 ? row_step[n] : 0;
  }
  __device__ __forceinline__ void wait() {
    if constexpr (kShared) asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
  }
  __device__ __forceinline__ void take(int n, int stage, Pair (&out)[kVec * kPer / 2]) {
    if constexpr (kShared) {
      Vec<T, kVec> v[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&v[k]);
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(slot + ((stage * kTensors + n) * kPer + k) * vec_bytes)
                     : "memory");
      }
      take_apart<T, kVec, kPer>(v, out);
    } else {
      take_apart<T, kVec, kPer>(ahead[n], out);
    }
  }
};

// Which of a thread's vectors lie inside the row, and how many elements its warp and the warp with the number of its lane
// have; the same for every row.
template <int kVec, int kPer>
struct RowShare {
  uint32_t mask = 0;
  float own_inv, there, there_inv;
  static __device__ __forceinline__ float count(int warp, int64_t hidden) {
    int64_t n = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int64_t left = hidden - int64_t(warp * 32 + k * blockDim.x) * kVec;
      n += left <= 0 ? 0 : left < 32 * kVec ? left : 32 * kVec;
    }
    return float(n);
  }
  __device__ __forceinline__ explicit RowShare(int64_t hidden) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (int64_t(threadIdx.x + k * blockDim.x) * kVec < hidden) mask |= 1u << k;
    const float own = count(threadIdx.x >> 5, hidden);
    own_inv = own > 0.f ? 1.f / own : 0.f;
    there = int(threadIdx.x & 31) < int(blockDim.x >> 5) ? count(threadIdx.x & 31, hidden) : 0.f;
    there_inv = there > 0.f ? 1.f / there : 0.f;
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Mean of a row and sum of the squares about it, with one exchange between its warps: each warp takes the squares about
// its own mean, which are then moved to the common one, sum (x - m)^2 = sum over the warps of sum (x - m_w)^2 +
// n_w (m_w - m)^2: terms that do not cancel, however far the row is from 0.
template <int kVec, int kPer>
__device__ __forceinline__ void row_moments(const Pair (&x)[kVec * kPer / 2], const RowShare<kVec, kPer>& share, float inv,
                                            float (*part)[32][2], int& turn, float& mean, float& squares) {
  constexpr int kPairs = kVec * kPer / 2;
  Pair s2 = 0;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) s2 = add2(s2, x[i]);
  const float s = warp_sum(sum_of(s2));
  const float m = s * share.own_inv;
  const Pair m2 = pair_of(-m, -m);
  s2 = 0;
  if constexpr (kVec == 1) {
#pragma unroll
    for (int k = 0; k < kPer; k += 2) {
      float a, b;
      unpack_f32x2(add2(x[k / 2], m2), a, b);
      const Pair d = pair_of(share.mask >> k & 1 ? a : 0.f, share.mask >> (k + 1) & 1 ? b : 0.f);
      s2 = fma2(d, d, s2);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (share.mask >> k & 1)
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
          const Pair d = add2(x[k * kVec / 2 + i], m2);
          s2 = fma2(d, d, s2);
        }
  }
  const float q = warp_sum(sum_of(s2));
  mean = m;
  squares = q;
  if (blockDim.x == 32) return;
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) {
    part[turn][threadIdx.x >> 5][0] = s;
    part[turn][threadIdx.x >> 5][1] = q;
  }
  __syncthreads();
  const float ws = lane < warps ? part[turn][lane][0] : 0.f;
  const float wq = lane < warps ? part[turn][lane][1] : 0.f;
  turn ^= 1;
  mean = warp_sum(ws) * inv;
  const float off = ws * share.there_inv - mean;
  squares = warp_sum(fmaf(share.there * off, off, wq));
}

template <typename T, int kVec, int kPer, int kMaxThreads, int kBlocks>
__global__ void __launch_bounds__(kMaxThreads, kBlocks) norm_kernel(const NormArgs p) {
  constexpr int kPairs = kVec * kPer / 2;
  extern __shared__ __align__(16) uint8_t rows_smem[];
  __shared__ float part[2][32][2];
  int turn = 0, stage = 0;
  const int64_t step = int64_t(gridDim.x) * blockDim.y;
  const float inv = 1.f / float(p.hidden);
  int64_t r = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  using Stream = RowStream<T, kVec, kPer, 1>;
  constexpr int kAhead = Stream::kAhead;
  const RowShare<kVec, kPer> share(p.hidden);
  Stream x(p.x, p.x_pitch, nullptr, 0, r, step, p.rows, share.mask, smem_u32(rows_smem));
  T* to = reinterpret_cast<T*>(p.out) + r * p.hidden + int(threadIdx.x) * kVec;
  for (int i = 0; i < kAhead; ++i) x.request(i);
  Pair w[kPairs], b[kPairs];
  load_params<T, kVec, kPer>(p.weight, p.params_fp32, p.hidden, 1.f, w);
  load_params<T, kVec, kPer>(p.bias, p.params_fp32, p.hidden, 0.f, b);
  // all rows of a block take the same number of turns: its threads meet at the barriers
  for (int64_t first = int64_t(blockIdx.x) * blockDim.y; first < p.rows; first += step, r += step) {
    Pair v[kPairs];
    x.wait();
    x.take(0, stage, v);
    x.request(stage);
    stage = stage + 1 == kAhead ? 0 : stage + 1;
    float mean, squares;
    row_moments<kVec, kPer>(v, share, inv, part, turn, mean, squares);
    const float rstd = 1.f / sqrtf(squares * inv + p.eps);
    if (r < p.rows) {
      const Pair m2 = pair_of(-mean, -mean), r2 = pair_of(rstd, rstd);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) v[i] = fma2(mul2(add2(v[i], m2), r2), w[i], b[i]);
      store_row<T, kVec, kPer>(to, share.mask, v);
      to += step * p.hidden;
      if (threadIdx.x == 0) {
        p.mean[r] = mean;
        p.rstd[r] = rstd;
      }
    }
  }
}

constexpr int kMostRows = 8;  // rows that a block takes side by side at most

template <int kCount>
__device__ __forceinline__ void store_floats(float* to, const float (&f)[kCount]) {
  if constexpr (kCount % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kCount; i += 4) *reinterpret_cast<float4*>(to + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < kCount; ++i) to[i] = f[i];
  }
}

// Every thread keeps the sums of its columns over the rows it sees, and leaves them in `sums` at the end.  Columns past
// the row's end have dy = 0, so they add nothing to any sum.
template <typename T, int kVec, int kPer, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) norm_grad_kernel(const NormArgs p) {
  constexpr int kPairs = kVec * kPer / 2;
  extern __shared__ __align__(16) uint8_t rows_smem[];
  __shared__ float parts[kMostRows][2][32][2];
  float (*part)[32][2] = parts[threadIdx.y];
  int turn = 0, stage = 0;
  const int64_t step = int64_t(gridDim.x) * blockDim.y;
  const float inv = 1.f / float(p.hidden);
  int64_t r = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  using Stream = RowStream<T, kVec, kPer, 2>;
  constexpr int kAhead = Stream::kAhead;
  uint32_t mask = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k)
    if (int64_t(threadIdx.x + k * blockDim.x) * kVec < p.hidden) mask |= 1u << k;
  Stream stream(p.x, p.x_pitch, p.dy, p.dy_pitch, r, step, p.rows, mask, smem_u32(rows_smem));
  T* to = reinterpret_cast<T*>(p.out) + r * p.hidden + int(threadIdx.x) * kVec;
  for (int i = 0; i < kAhead; ++i) stream.request(i);
  float mean = r < p.rows ? __ldg(p.mean + r) : 0.f, rstd = r < p.rows ? __ldg(p.rstd + r) : 0.f;
  Pair w[kPairs], dw[kPairs] = {}, db[kPairs] = {};
  load_params<T, kVec, kPer>(p.weight, p.params_fp32, p.hidden, 1.f, w);
  for (int64_t first = int64_t(blockIdx.x) * blockDim.y; first < p.rows; first += step, r += step) {
    Pair h[kPairs], g[kPairs];
    stream.wait();
    stream.take(0, stage, h);
    stream.take(1, stage, g);
    stream.request(stage);
    stage = stage + 1 == kAhead ? 0 : stage + 1;
    const Pair m2 = pair_of(-mean, -mean), r2 = pair_of(rstd, rstd);
    const bool here = r < p.rows;
    const bool more = r + step < p.rows;
    mean = more ? __ldg(p.mean + r + step) : 0.f;
    rstd = more ? __ldg(p.rstd + r + step) : 0.f;
    Pair sg = 0, sgh = 0;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      h[i] = mul2(add2(h[i], m2), r2);
      dw[i] = fma2(g[i], h[i], dw[i]);
      db[i] = add2(db[i], g[i]);
      g[i] = mul2(g[i], w[i]);
      sg = add2(sg, g[i]);
      sgh = fma2(g[i], h[i], sgh);
    }
    if (p.out) {
      float s[2] = {sum_of(sg), sum_of(sgh)};
      row_sums(s, part, turn);
      if (here) {
        const Pair a2 = pair_of(-s[0] * inv, -s[0] * inv), b2 = pair_of(-s[1] * inv, -s[1] * inv);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) g[i] = mul2(r2, fma2(h[i], b2, add2(g[i], a2)));
        store_row<T, kVec, kPer>(to, mask, g);
        to += step * p.hidden;
      }
    }
  }
  if (p.sums == nullptr) return;
  // a block's sums of dy*h, then of dy; the rows that it takes side by side are added first, in order
  float* sums = p.sums + int64_t(blockIdx.x) * 2 * p.hidden;
  float* to_smem = reinterpret_cast<float*>(rows_smem) + threadIdx.y * 2 * kPer * kVec * blockDim.x;
  if (blockDim.y > 1) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int at = int(threadIdx.x + k * blockDim.x) * kVec;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float f[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        float both[2];
        unpack_f32x2(which ? db[(k * kVec + i) / 2] : dw[(k * kVec + i) / 2], both[0], both[1]);
        f[i] = both[(k * kVec + i) & 1];
      }
      if (blockDim.y > 1) store_floats(to_smem + which * kPer * kVec * blockDim.x + at, f);
      else if (at < p.hidden) store_floats(sums + which * p.hidden + at, f);
    }
  }
  if (blockDim.y == 1) return;
  __syncthreads();
  const int padded = kPer * kVec * blockDim.x;
  for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < 2 * padded; c += blockDim.x * blockDim.y) {
    const int which = c >= padded, at = c - which * padded;
    if (at >= p.hidden) continue;
    float t = 0.f;
    for (int y = 0; y < int(blockDim.y); ++y) t += reinterpret_cast<const float*>(rows_smem)[y * 2 * padded + c];
    sums[which * p.hidden + at] = t;
  }
}

// ---- rows of any length ------------------------------------------------------------------------------
constexpr int kLongThreads = 512;

template <typename T>
__device__ __forceinline__ float param(const void* p, int fp32, int64_t i, float other) {
  if (p == nullptr) return other;
  return fp32 ? __ldg(reinterpret_cast<const float*>(p) + i) : to_float(reinterpret_cast<const T*>(p)[i]);
}

// A block per row, the row read once per pass.
template <typename T>
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
      y[i] = from_float<T>(fmaf((to_float(x[i]) - mean) * rstd, param<T>(p.weight, p.params_fp32, i, 1.f),
                                param<T>(p.bias, p.params_fp32, i, 0.f)));
    }
    if (threadIdx.x == 0) {
      p.mean[r] = mean;
      p.rstd[r] = rstd;
    }
  }
}

template <typename T>
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
      const float g = d * param<T>(p.weight, p.params_fp32, i, 1.f);
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
      const float g = d * param<T>(p.weight, p.params_fp32, i, 1.f);
      if (dx) dx[i] = from_float<T>(rstd * (g - sg - h * sgh));
      if (sums) {  // this thread's own column of this block's own sums
        const bool first = r == blockIdx.x;
        sums[i] = first ? d * h : fmaf(d, h, sums[i]);
        sums[p.hidden + i] = first ? d : sums[p.hidden + i] + d;
      }
    }
  }
}

// Parts added in a fixed order, 32 kWidth columns x 32 lanes per block: lane k takes parts k, k + 32, ..., then the lanes' sums by
// a tree.  Bound by the second launch and by the latency of its loads: 148 parts of 14336 columns (8.5 MB, which lie in L2)
// 5 us after the kernel before, 6 with one column per thread.
constexpr int kSumLanes = 32;
template <int kWidth>
__global__ void __launch_bounds__(32 * kSumLanes) column_sums_kernel(const float* parts, int count, int64_t columns, float* out,
                                                                     int64_t first, float* rest) {
  __shared__ Vec<float, kWidth> lanes[kSumLanes][33];
  const int c = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const int64_t i = (int64_t(blockIdx.x) * 32 + c) * kWidth;
  Vec<float, kWidth> s{};
  if (i < columns)
#pragma unroll 4
    for (int k = lane; k < count; k += kSumLanes) {
      const Vec<float, kWidth> v = *reinterpret_cast<const Vec<float, kWidth>*>(parts + k * columns + i);
#pragma unroll
      for (int e = 0; e < kWidth; ++e) s.v[e] += v.v[e];
    }
  lanes[lane][c] = s;
  __syncthreads();
  s = lanes[c][lane];  // this warp's columns, one lane's sums per thread
#pragma unroll
  for (int e = 0; e < kWidth; ++e) s.v[e] = warp_sum(s.v[e]);
  const int64_t at = (int64_t(blockIdx.x) * 32 + lane) * kWidth + c;
  if (c >= kWidth || at >= columns) return;
  float mine = s.v[0];
#pragma unroll
  for (int e = 1; e < kWidth; ++e) mine = c == e ? s.v[e] : mine;
  if (at < first) {
    if (out) out[at] = mine;
  } else if (rest) {
    rest[at - first] = mine;
  }
}

// How a call runs: which kernel, its block and its grid.
struct Plan {
  int vec;      // elements per access, 0: the kernel for rows of any length
  int per;      // vectors per thread
  int most;     // threads the kernel is built for
  dim3 block;
  int blocks;
  int parts;    // sums per column that the blocks of the backward kernel leave
};

// The register kernels: vectors (or single elements) per thread, threads at most, blocks that an SM's registers hold
// for each thread of a block (65536 / registers).
struct Shape {
  int per, most, threads_per_sm;
};
// In 64 registers the 16-bit kernel of up to 1024 elements keeps 14 words in local memory (20000 x 1024: 22.8 us, 13 of them at
// the copy rate).
constexpr Shape kForwardVec[] = {{2, 64, 1024}, {4, 256, 512}, {4, 512, 512}};
constexpr Shape kForwardVecFew[] = {{1, 1024, 1024}, {4, 512, 512}};
// single elements, 1777 rows of 1031: 7.7 us with four per thread, 14.2 with sixteen; past 2048 it is the other way (20000 rows
// of 2049: 83 against 112), although sixteen leave 66 words of a thread in local memory, and 26 to 30 backward
constexpr Shape kForwardOne[] = {{4, 512, 1024}, {16, 1024, 1024}};
constexpr Shape kForwardOneFew[] = {{4, 1024, 1024}, {16, 1024, 1024}};
// 16-bit rows of 16384 elements keep part of their column sums in local memory: 172 us for 4096 of them, where the kernel for
// rows of any length takes 571
constexpr Shape kBackwardVec[] = {{2, 512, 512}, {4, 512, 512}};
constexpr Shape kBackwardVecFew[] = {{1, 1024, 1024}, {2, 512, 512}, {4, 512, 512}};
constexpr Shape kBackwardOne[] = {{4, 512, 1024}, {16, 512, 512}};
constexpr Shape kBackwardOneFew[] = {{4, 1024, 1024}, {16, 512, 512}};

template <size_t kCount>
bool pick(const Shape (&shapes)[kCount], int64_t vecs, Shape& out) {
  for (const Shape& s : shapes)
    if (vecs <= int64_t(s.per) * s.most) {
      out = s;
      return true;
    }
  return false;
}

// Few rows (each SM gets one at most): as many threads as there are, for latency; many: few threads that keep
// several loads each in flight.
Plan make_plan(bool backward, int elem_bytes, bool aligned, int64_t rows, int64_t hidden, int device) {
  const int sms = device_sm_count(device) > 0 ? device_sm_count(device) : 1;
  Plan l{};
  l.vec = aligned ? 16 / elem_bytes : 1;
  const int64_t vecs = (hidden + l.vec - 1) / l.vec;
  Shape s;
  const bool few = rows <= sms;
  const bool found = backward ? (aligned ? (few ? pick(kBackwardVecFew, vecs, s) : pick(kBackwardVec, vecs, s))
                                         : (few ? pick(kBackwardOneFew, vecs, s) : pick(kBackwardOne, vecs, s)))
                              : (aligned ? (few ? pick(kForwardVecFew, vecs, s) : pick(kForwardVec, vecs, s))
                                         : (few ? pick(kForwardOneFew, vecs, s) : pick(kForwardOne, vecs, s)));
  if (!found) {
    l.vec = 0;
    l.block = dim3(kLongThreads);
    l.blocks = int(rows < 2 * sms ? rows : 2 * sms);
    l.parts = l.blocks;
    return l;
  }
  l.per = s.per;
  l.most = s.most;
  const int tpr = int((vecs + l.per - 1) / l.per + 31) / 32 * 32;
  // Rows of one warp go side by side, as many as the shape has threads for, up to eight (forward two with many rows, whose blocks
  // have 64 threads; eight with few); backward, where a block leaves sums for a second kernel to add, also rows of up to four
  // warps, side by side (10000 rows of 1536: 31 -> 21 us, 3000 of 1024 13.7 -> 9.5; of eight warps 19.6 -> 21.1, so not there)
  const bool side_by_side = tpr == 32 || (backward && !few && tpr <= 128);
  l.block = dim3(tpr, side_by_side ? std::min(kMostRows, s.most / tpr) : 1);
  const int threads = tpr * int(l.block.y);
  int resident = s.threads_per_sm / threads;
  resident = resident < 1 ? 1 : resident;
  const int64_t wanted = (rows + l.block.y - 1) / l.block.y;
  l.blocks = int(wanted < int64_t(sms) * resident ? wanted : int64_t(sms) * resident);
  l.parts = l.blocks;
  return l;
}

using KernelFn = void (*)(const NormArgs);
template <typename T>
KernelFn forward_kernel(const Plan& l) {
  constexpr int kV = 16 / sizeof(T);
  if (l.vec == 0) return norm_long_kernel<T>;
  if (l.vec == 1) return l.per == 4 ? norm_kernel<T, 1, 4, 1024, 1> : norm_kernel<T, 1, 16, 1024, 1>;
  if (l.per == 1) return norm_kernel<T, kV, 1, 1024, 1>;
  return l.per == 2 ? norm_kernel<T, kV, 2, 64, 16> : norm_kernel<T, kV, 4, 512, 1>;
}
template <typename T>
KernelFn backward_kernel(const Plan& l) {
  constexpr int kV = 16 / sizeof(T);
  if (l.vec == 0) return norm_grad_long_kernel<T>;
  if (l.vec == 1) return l.per == 4 ? norm_grad_kernel<T, 1, 4, 1024> : norm_grad_kernel<T, 1, 16, 512>;
  if (l.per == 1) return norm_grad_kernel<T, kV, 1, 1024>;
  return l.per == 2 ? norm_grad_kernel<T, kV, 2, 512> : norm_grad_kernel<T, kV, 4, 512>;
}

int launch(bool backward, int precision, const NormArgs& a, const Plan& l, int device, cudaStream_t stream) {
  const int type = precision == MB200_PRECISION_FP32 ? 0 : precision == MB200_PRECISION_FP16 ? 1 : 2;
  const KernelFn kernel = type == 0   ? (backward ? backward_kernel<float>(l) : forward_kernel<float>(l))
                          : type == 1 ? (backward ? backward_kernel<__half>(l) : forward_kernel<__half>(l))
                                      : (backward ? backward_kernel<__nv_bfloat16>(l) : forward_kernel<__nv_bfloat16>(l));
  size_t smem = l.vec > 1 ? size_t(kStages) * l.block.x * l.block.y * l.per * 16 * (backward ? 2 : 1) : 0;
  if (backward && a.sums && l.block.y > 1) smem = std::max(smem, size_t(l.block.x) * l.block.y * l.per * l.vec * 2 * 4);
  if (smem > 40 * 1024) {  // with the static share past the 48 KiB that need no asking
    // the most any plan takes, once per device and kernel; a second thread that sets it again does no harm
    static std::atomic<bool> configured[kMaxDevices][2][3][5];
    std::atomic<bool>* done = device >= 0 && device < kMaxDevices ? &configured[device][backward][type][l.per] : nullptr;
    if (!done || !done->load(std::memory_order_acquire)) {
      MB200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
      if (done) done->store(true, std::memory_order_release);
    }
  }
  kernel<<<l.blocks, l.block, smem, stream>>>(a);
  MB200_CHECK_CUDA(cudaGetLastError());
  return kOk;
}

// Whether every row of every tensor starts on a 16-byte boundary.
bool rows_aligned(const NormArgs& a, int elem_bytes) {
  auto at = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const int64_t v = 16 / elem_bytes;
  return a.hidden % v == 0 && a.x_pitch % v == 0 && (!a.dy || a.dy_pitch % v == 0) && at(a.x) && at(a.dy) && at(a.weight) &&
         at(a.bias) && at(a.out);
}

int check_norm(int precision, int64_t rows, int64_t hidden, const char* what) {
  MB200_REQUIRE(precision == MB200_PRECISION_BF16 || precision == MB200_PRECISION_FP16 || precision == MB200_PRECISION_FP32,
                kInvalidArgument, "%s: precision %d (bf16, fp16 or fp32)", what, precision);
  MB200_REQUIRE(rows >= 0 && hidden >= 1, kInvalidArgument, "%s: rows=%lld hidden=%lld", what, (long long)rows,
                (long long)hidden);
  MB200_REQUIRE(hidden <= (int64_t(1) << 30), kUnsupportedShape, "%s: hidden=%lld", what, (long long)hidden);
  return kOk;
}

}  // namespace

// Four columns per thread as soon as half of the SMs get a block.
constexpr int kWide = 64;
int launch_column_sums(const float* parts, int count, int64_t columns, float* out, int64_t first, float* rest, cudaStream_t stream) {
  if (columns % 4 == 0 && columns >= 128 * kWide && (reinterpret_cast<uintptr_t>(parts) & 15) == 0)
    column_sums_kernel<4><<<unsigned((columns + 127) / 128), 32 * kSumLanes, 0, stream>>>(parts, count, columns, out, first, rest);
  else
    column_sums_kernel<1><<<unsigned((columns + 31) / 32), 32 * kSumLanes, 0, stream>>>(parts, count, columns, out, first, rest);
  MB200_CHECK_CUDA(cudaGetLastError());
  return kOk;
}

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
  const int size = precision == MB200_PRECISION_FP32 ? 4 : 2, param_size = params_fp32 ? 4 : size;
  // y = x is fine: a row is written by the threads that have read it, and no other row reads it
  const bool in_place = y == x && (x_pitch == hidden || rows == 1);
  if ((rc = check_apart("layer_norm",
                        {span_of("y", y, rows, hidden, hidden, size), span_of("mean", mean, 1, rows, rows, 4), span_of("rstd", rstd, 1, rows, rows, 4)},
                        {span_of("x", in_place ? nullptr : x, rows, x_pitch, hidden, size),
                         span_of("weight", weight, 1, hidden, hidden, param_size), span_of("bias", bias, 1, hidden, hidden, param_size)})))
    return rc;
  NormArgs a{};
  a.x = x;
  a.x_pitch = x_pitch;
  a.rows = rows;
  a.hidden = hidden;
  a.weight = weight;
  a.bias = bias;
  a.params_fp32 = params_fp32 != 0;
  a.eps = eps;
  a.out = y;
  a.mean = mean;
  a.rstd = rstd;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Plan l = make_plan(false, size, rows_aligned(a, size), rows, hidden, device);
  return launch(false, precision, a, l, device, s);
}

int64_t mb200_layer_norm_backward_workspace_bytes(int64_t rows, int64_t hidden, int device) {
  if (check_norm(MB200_PRECISION_FP32, rows, hidden, "layer_norm_backward_workspace_bytes")) return -1;
  // the most that any type and alignment needs
  int parts = 0;
  for (const int size : {2, 4})
    for (const bool aligned : {false, true}) parts = std::max(parts, make_plan(true, size, aligned, rows, hidden, device).parts);
  return int64_t(parts) * 2 * hidden * 4;
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
  NormArgs a{};
  a.x = x;
  a.dy = dy;
  a.x_pitch = x_pitch;
  a.dy_pitch = dy_pitch;
  a.rows = rows;
  a.hidden = hidden;
  a.weight = weight;
  a.params_fp32 = params_fp32 != 0;
  a.out = dx;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  const int size = precision == MB200_PRECISION_FP32 ? 4 : 2;
  const Plan l = make_plan(true, size, rows_aligned(a, size), rows, hidden, device);
  if (dweight || dbias) {
    const int64_t need = int64_t(l.parts) * 2 * hidden * 4;
    MB200_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, kInvalidArgument,
                  "layer_norm_backward: needs a 16-byte aligned workspace");
    MB200_REQUIRE(workspace_bytes >= need, kWorkspaceTooSmall, "layer_norm_backward: workspace %lld < %lld bytes",
                  (long long)workspace_bytes, (long long)need);
    a.sums = reinterpret_cast<float*>(workspace);
  }
  if ((rc = check_apart("layer_norm_backward",
                        {span_of("dx", dx, rows, hidden, hidden, size), span_of("dweight", dweight, 1, hidden, hidden, 4),
                         span_of("dbias", dbias, 1, hidden, hidden, 4),
                         span_of("workspace", a.sums, int64_t(l.parts) * 2, hidden, hidden, 4)},
                        {span_of("dy", dy, rows, dy_pitch, hidden, size), span_of("x", x, rows, x_pitch, hidden, size),
                         span_of("mean", mean, 1, rows, rows, 4), span_of("rstd", rstd, 1, rows, rows, 4),
                         span_of("weight", weight, 1, hidden, hidden, params_fp32 ? 4 : size)})))
    return rc;
  if ((rc = launch(true, precision, a, l, device, s))) return rc;
  if (a.sums) return launch_column_sums(a.sums, l.parts, 2 * hidden, dweight, hidden, dbias, s);
  return kOk;
}

}  // extern "C"
