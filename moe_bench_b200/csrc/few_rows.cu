// The dense forward product for few rows: y = act(x w^T + b) + r where the weights' stream is all that counts.
//
// A block takes 16 features (a cluster of up to 8 blocks shares them, each with a part of the sum), its 8 warps
// a part of the sum each.  The weights go straight from HBM into the operand registers of the matrix instruction
// m16n8k16: the order of the terms of a sum is free, so a lane's 16 bytes of a row are 8 neighbouring terms where
// the instruction would have pairs, on both sides alike, and no shared memory, barrier or tensor memory
// stands between load and product.  Parts are added in a fixed order: warps through shared memory, then blocks through
// the first block's view of the others'.  The tensor pipe is idle most of the time on either path.
//
// Bound by HBM and, where there is little to load, by one load's latency and the launch: one row on 7168 x 256 takes 5.3 us
// (launch to launch, weights from HBM), 8 rows on 7168 x 2048 9.8 us of 4.5 at the copy rate; the tiled kernel with its
// join 11.1 and 14.8 us.  Past 16 rows x is read too often (7168 x 2048: 32 rows 22.8 against 15.1 us).

#include "linear.cuh"

namespace mb200 {

namespace {

constexpr int kWarps = 8;
constexpr int kFeatures = 16;
constexpr int kChunk = 32;   // terms of a sum that a warp takes at once: 8 in each of 4 lanes
constexpr int kUnroll = 4;   // chunks requested together

__device__ __forceinline__ uint4 load_stream(const void* p, int64_t elem) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(reinterpret_cast<const uint16_t*>(p) + elem));
  return v;
}

// d += a b: a 16 features x 16 terms, b 16 terms x 8 rows
__device__ __forceinline__ void mma_h16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                        int fp16) {
  if (fp16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The epilogue of four neighbouring features of a row; `vec`: every tensor takes them as one access (then m is a multiple of 4).
// The residual may be the output's buffer: its loads promise nothing, and come before the row's stores.
__device__ __forceinline__ void store4(void* out, int fp32, int fp16, int m, int64_t row, int f, const float (&v)[4], int vec) {
  const int64_t at = row * m + f;
  if (vec) {
    if (fp32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + at) =
        make_uint2(pack_h16x2(v[0], v[1], fp16), pack_h16x2(v[2], v[3], fp16));
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (f + k < m) {
      if (fp32) reinterpret_cast<float*>(out)[at + k] = v[k];
      else reinterpret_cast<uint16_t*>(out)[at + k] = to_h16(v[k], fp16);
    }
}
__device__ __forceinline__ void finish4(const Epilogue& e, int m, int64_t row, int f, float (&z)[4], int vec) {
  if (e.bias)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f + i < m) z[i] += e.bias_fp32 ? __ldg(reinterpret_cast<const float*>(e.bias) + f + i) : load_h16(e.bias, f + i, e.fp16);
  float residual[4] = {};
  if (e.residual) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(e.residual) + row * e.residual_pitch + f;
    if (vec) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) residual[i] = load_h16(&v, i, e.fp16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (f + i < m) residual[i] = load_h16(p, i, e.fp16);
    }
  }
  float slope[4];
  if (e.slope) {
    activate<true>(e.act, z, slope);
    store4(e.slope, 0, e.fp16, m, row, f, slope, vec);
  } else if (e.act) {
    activate<false>(e.act, z, slope);
  }
  if (e.residual)
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] += residual[i];
  store4(e.out, e.out_fp32, e.fp16, m, row, f, z, vec);
}
int epilogue_vec(const Epilogue& e, int m) {
  auto at = [](const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
  return m % 4 == 0 && at(e.out, e.out_fp32 ? 16 : 8) && at(e.slope, 8) && (!e.residual || (at(e.residual, 8) && e.residual_pitch % 4 == 0));
}

// kOctets: groups of 8 rows
template <int kOctets>
__global__ void __launch_bounds__(kWarps * 32) few_rows_kernel(const ProductArgs p, int parts, int vec) {
  constexpr int kRows = 8 * kOctets;
  __shared__ float sums[kWarps][kRows][kFeatures];
  __shared__ __align__(16) float block_sum[kRows][kFeatures];  // read four at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int part = int(blockIdx.x) % parts;  // consecutive blocks form a cluster
  const int f0 = int(blockIdx.x) / parts * kFeatures;
  const int chunks = (p.k + kChunk - 1) / kChunk;
  const int begin = int(int64_t(chunks) * part / parts), end = int(int64_t(chunks) * (part + 1) / parts);

  // features and rows past the end read the last one again; their results are dropped
  const int64_t w_lo = int64_t(min(f0 + g, p.m - 1)) * p.a_pitch + q * 8;
  const int64_t w_hi = int64_t(min(f0 + g + 8, p.m - 1)) * p.a_pitch + q * 8;
  int64_t x_at[kOctets];
#pragma unroll
  for (int o = 0; o < kOctets; ++o) x_at[o] = int64_t(min(8 * o + g, p.rows - 1)) * p.b_pitch + q * 8;

  float acc[kOctets][4] = {};
  for (int c0 = begin + warp * kUnroll; c0 < end; c0 += kWarps * kUnroll) {
    uint4 a[kUnroll][2], b[kUnroll][kOctets];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = (c0 + u) * kChunk;
      const bool inside = c0 + u < end && k + q * 8 < p.k;
      a[u][0] = inside ? load_stream(p.a, w_lo + k) : make_uint4(0, 0, 0, 0);
      a[u][1] = inside ? load_stream(p.a, w_hi + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int o = 0; o < kOctets; ++o)
        b[u][o] = inside ? __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.b) + x_at[o] + k))
                         : make_uint4(0, 0, 0, 0);
    }
    __syncwarp();  // in the sum's last chunk not every lane has terms; the products are the whole warp's
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int o = 0; o < kOctets; ++o) {
        mma_h16(acc[o], a[u][0].x, a[u][1].x, a[u][0].y, a[u][1].y, b[u][o].x, b[u][o].y, p.epi.fp16);
        mma_h16(acc[o], a[u][0].z, a[u][1].z, a[u][0].w, a[u][1].w, b[u][o].z, b[u][o].w, p.epi.fp16);
      }
  }
#pragma unroll
  for (int o = 0; o < kOctets; ++o) {
    sums[warp][8 * o + 2 * q][g] = acc[o][0];
    sums[warp][8 * o + 2 * q + 1][g] = acc[o][1];
    sums[warp][8 * o + 2 * q][g + 8] = acc[o][2];
    sums[warp][8 * o + 2 * q + 1][g + 8] = acc[o][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * kFeatures; i += kWarps * 32) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += (&sums[w][0][0])[i];
    (&block_sum[0][0])[i] = s;
  }
  if (parts > 1) cluster_sync();
  else __syncthreads();
  if (part == 0) {
    for (int i = threadIdx.x; i < kRows * kFeatures / 4; i += kWarps * 32) {
      const int row = i >> 2, f = (i & 3) * 4;
      if (row >= p.rows || f0 + f >= p.m) continue;
      float z[4] = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < parts; ++k) {
        const uint32_t at = map_to_cta(smem_u32(&block_sum[row][f]), k);
        float v[4];
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at) : "memory");
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] += v[e];
      }
      finish4(p.epi, p.m, row, f0 + f, z, vec);
    }
  }
  if (parts > 1) cluster_sync();  // the other blocks' sums have been read
}

}  // namespace

int launch_few_rows(const ProductArgs& args, int device, cudaStream_t stream) {
  const int sms = device_sm_count(device);
  MB200_REQUIRE(sms > 0, kCudaError, "linear: cannot read the SM count of device %d", device);
  const int groups = (args.m + kFeatures - 1) / kFeatures, chunks = (args.k + kChunk - 1) / kChunk;
  // up to four blocks per SM, as long as each warp has a chunk (8 rows of 7168 x 2048: 12.8 us with two, 9.8 with four, 13.9
  // with eight, whose clusters are twice the size)
  int parts = 8;
  while (parts > 1 && (int64_t(groups) * parts > 4 * sms || chunks < parts * kWarps)) parts /= 2;
  const int vec = epilogue_vec(args.epi, args.m);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(parts);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(groups) * parts);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  const auto kernel = args.rows <= 8 ? few_rows_kernel<1> : few_rows_kernel<2>;
  MB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, args, parts, vec));
  return kOk;
}

}  // namespace mb200
