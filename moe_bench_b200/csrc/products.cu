// The products around the expert FFN (linear.cuh) on the sm_100a tensor cores: forward, input gradient
// and weight gradient, dense or over ragged row segments.
//
// out[j][f] = sum over c of A(f, c) B(j, c): the features f, which lie side by side in the output, sit on the
// accumulator's rows (tensor-memory lanes), the output rows j on its columns.  A pair of CTAs computes a tile of
// 256 features x up to 256 output rows (any multiple of 32): each CTA holds 128 features and half of the output
// rows of every 64-deep step, 32 KiB for 512 cycles of products, where a single CTA with the same
// accumulator needs 48.  Row segments therefore cost what they hold, rounded up to 32.
//
// Operands come in as they lie in memory, no transposed copies: 128-byte-swizzled TMA boxes of 64 terms of the
// sum x 16..128 rows where the terms lie side by side (w and x of the forward, dz of the input gradient), of 64
// features x 64 terms where the features do (w of the input gradient, x and dz of the weight gradient).  Terms past
// the end of a dense sum are the copy's zero fill.  A segment's last step in the weight gradient would read the next
// segment's rows: those are overwritten with zeros in shared memory before the products read them, in both
// operands, so that NaN and infinities there reach nothing.
//
// 384 threads: warp 0 loads, warp 1 of the pair's first CTA issues the products, warp 2 clears those tails,
// warps 4-11 drain the accumulators (two sets, so that the next tile's products run meanwhile).  A lane holds one
// feature of many output rows, memory wants many features of one row: where outputs are of 16 bits and start on 16 bytes, 32
// features x 32 output rows at a time are read as fragments, finished, rounded and transposed by stmatrix; else a warp
// stores its lanes' features row by row.  Every wait is bounded.
//
// Few tiles leave pairs idle, so up to eight pairs form a cluster and share a tile, each with a part of its sums; the parts
// meet in shared memory and are added in the pairs' order (join_parts).

#include <algorithm>
#include <atomic>

#include "linear.cuh"

namespace mb200 {

namespace {

constexpr int kThreads = 384;
constexpr int kEpilogueWarps = 8;
constexpr int kFirstEpilogueWarp = 4;
constexpr int kMaxStages = 10;
constexpr int kStep = 64;                 // terms of the sum per step
constexpr int kABytes = 128 * 128;        // a CTA's 128 features of a step
constexpr int kTileRows = 256;            // output rows of a tile at most
constexpr int kTileFeatures = 256;
constexpr int kBoxes = 4;                 // row boxes of 16, 32, 64, 128
constexpr int kTmemCols = 512;
constexpr int kBand = 8;                  // tiles that run side by side share 8 row blocks and as many feature blocks

struct SmemTail {
  alignas(16) float turn[kEpilogueWarps][16 * 32];
  uint64_t full[kMaxStages];    // of the pair's first CTA: a step of both CTAs has landed
  uint64_t empty[kMaxStages];   // the products have read the stage
  uint64_t raw[kMaxStages];     // weight gradient: this CTA's part of a segment's last step has landed
  uint64_t acc_full[2];
  uint64_t acc_empty[2];        // of the pair's first CTA
  uint32_t tmem_base;
  int abort_flag;
  int max_len;                  // longest segment
  int begin[kMaxExperts];
  int len[kMaxExperts];
  int blocks[kMaxExperts + 1];  // row blocks before each group
};

constexpr size_t kSmemLimit = 227 * 1024;
constexpr size_t kRingBytes = (kSmemLimit - 1024 - sizeof(SmemTail)) / 1024 * 1024;
constexpr size_t kSmemBytes = 1024 + kRingBytes + sizeof(SmemTail);
static_assert(kRingBytes >= 6 * (kABytes + 128 * 128), "full tiles want six stages");

struct Maps {
  CUtensorMap a;
  CUtensorMap a2;  // both gradients: x
  CUtensorMap b[kBoxes];
};

struct TileShape {
  int f_tiles;      // feature blocks
  int row_blocks;   // weight gradient: blocks of output rows per group
  int splits;       // pairs of CTAs that share a tile, each with a part of its sums; they form a cluster
  int vec8;         // the output is of 16 bits, and every tensor takes eight features as one access
  int vec8_2;       // the same for the weight gradient where both gradients are computed
  int rounds, lead; // dense gradients in one launch: see Walk; rounds -1: one tile after the other
};

__device__ int g_status[1];  // first failure of a wait

struct Tile {
  int weight;         // a tile of the weight gradient
  int group, f0;
  int64_t out_row;    // first output row
  int b_row;          // its row coordinate in b (weight gradient: its column)
  int cols, valid;    // output rows computed, and stored
  int c_begin;        // weight gradient: first row of the segment
  int depth;          // terms of the whole sum
  int step0, step1;   // steps of this pair's part
};

template <int kKind>
__device__ __forceinline__ Tile locate_tile(int tile, int part, const ProductArgs& p, const TileShape& s, const SmemTail* t) {
  Tile r;
  r.weight = kKind == kWeightGrad;
  int blocks, local;
  if (kKind == kWeightGrad) {
    blocks = s.row_blocks;
    const int per_group = blocks * s.f_tiles;
    r.group = p.groups == 1 ? 0 : tile / per_group;
    local = tile - r.group * per_group;
  } else {
    // the last group whose first tile is not past `tile`: 32 coarse probes, then one per group
    int lo = 0;
    if (p.groups > 1) {
      const int lane = threadIdx.x & 31;
      const int step = (p.groups + 31) / 32;
      const int coarse = lane * step;
      lo = (__popc(__ballot_sync(0xffffffffu, coarse < p.groups && t->blocks[coarse] * s.f_tiles <= tile)) - 1) * step;
      const int fine = lo + lane;
      lo += __popc(__ballot_sync(0xffffffffu, lane < step && fine < p.groups && t->blocks[fine] * s.f_tiles <= tile)) - 1;
    }
    r.group = lo;
    blocks = t->blocks[lo + 1] - t->blocks[lo];
    local = tile - t->blocks[lo] * s.f_tiles;
  }
  int band = local / (kBand * s.f_tiles);
  local -= band * kBand * s.f_tiles;
  const int in_band = min(kBand, blocks - band * kBand);
  const int f = local / in_band;
  const int j = band * kBand + local - f * in_band;
  r.f0 = f * kTileFeatures;
  if (kKind == kWeightGrad) {
    int begin, end;
    segment_of(p, r.group, begin, end);
    r.b_row = j * kTileRows;
    const int left = p.n - r.b_row;
    r.cols = left > 128 ? 256 : 128;  // whole 64-column boxes in each CTA
    r.valid = min(left, r.cols);
    r.out_row = int64_t(r.group) * p.n + r.b_row;
    r.c_begin = begin;
    r.depth = end - begin;
  } else {
    const int len = t->len[r.group];
    const int per = ((len + blocks - 1) / blocks + 31) / 32 * 32;  // balanced parts
    const int start = j * per;
    r.b_row = t->begin[r.group] + start;
    r.valid = max(min(per, len - start), 0);
    r.cols = max((r.valid + 31) / 32 * 32, 32);
    r.out_row = r.b_row;
    r.c_begin = 0;
    r.depth = p.k;
  }
  const int steps = (r.depth + kStep - 1) / kStep;
  r.step0 = s.splits > 1 ? int(int64_t(steps) * part / s.splits) : 0;
  r.step1 = s.splits > 1 ? int(int64_t(steps) * (part + 1) / s.splits) : steps;
  return r;
}

// Both gradients: the input gradient's tiles have the first numbers, then come the weight gradient's.
template <int kKind>
__device__ __forceinline__ Tile locate(int tile, int first_tiles, int part, const ProductArgs& p, const TileShape& s, const SmemTail* t) {
  if constexpr (kKind != kBothGrads) return locate_tile<kKind>(tile, part, p, s, t);
  else if (tile < first_tiles) return locate_tile<kInputGrad>(tile, part, p, s, t);
  else return locate_tile<kWeightGrad>(tile - first_tiles, part, p, s, t);
}

// 32 features x 16 output rows, a feature per lane, turned round: 4 neighbouring features of rows (lane / 8) + 4 i per thread.
__device__ __forceinline__ void turn_chunk(float* block, const uint32_t (&v)[16], bool summed, float (&z)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 16; ++i) block[i * 32 + lane] = summed ? __uint_as_float(v[i]) : 0.f;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(z + 4 * i) =
      *reinterpret_cast<const float4*>(block + ((lane >> 3) + 4 * i) * 32 + 4 * (lane & 7));
  __syncwarp();
}

// The tiles of a pair (or, with shared tiles, of a cluster: its only one), in turn.  Dense gradients: first tiles of the input
// gradient, then of the weight gradient, whose sums may be long.  Where the latter do not come out even, the first `lead` pairs have one
// more of them, and of the former only `rounds`; the others go on alone (9000 x 7168 -> 256, 28 tiles of 141 steps after 1008 of 4: 95
// us in order, 76 so).
template <int kKind>
struct Walk {
  int tile;  // from `total` on there is none
  int first, total, worker, workers, lead, rounds, round;
  __device__ __forceinline__ Walk(int first_, int total_, int worker_, int workers_, const TileShape& s)
      : tile(worker_), first(first_), total(total_), worker(worker_), workers(workers_), lead(s.lead), rounds(s.rounds), round(0) {
    if (kKind == kBothGrads && rounds >= 0) at_round();
  }
  __device__ __forceinline__ void at_round() {
    // tile numbers stay below 2^30, and no round starts far behind the last
    const int t = round < rounds ? round * workers + worker : rounds * workers + (round - rounds) * (workers - lead) + worker - lead;
    tile = t < first && (worker >= lead || round < rounds) ? t : first + worker;
  }
  __device__ __forceinline__ void next() {
    if (kKind != kBothGrads || rounds < 0 || tile >= first) {
      tile += workers;
    } else {
      ++round;
      at_round();
    }
  }
};

struct Output {
  void* ptr;
  int fp32, vec8;
};
__device__ __forceinline__ Output output_of(const ProductArgs& p, const TileShape& s, int both_and_weight) {
  return both_and_weight ? Output{p.out2, p.out2_fp32, s.vec8_2} : Output{p.epi.out, p.epi.out_fp32, s.vec8};
}

// fp32 outputs, rows that do not start on vectors and joined parts: one feature of 16 output rows per lane, as tensor memory has
// them, so that a warp's 32 single elements lie side by side in a row.  The issue slots are the bound: types are told apart
// once per chunk, addresses run (7619 x 72 -> 515, bf16: 11.8 us; 20.8 with four features of a row per lane).
struct ColumnResidual {
  uint32_t v[8];
};
__device__ __forceinline__ ColumnResidual load_residual_column(const Epilogue& e, int m, const Tile& c, int chunk, int f) {
  ColumnResidual r{};
  if (e.residual && f < m) {
    const int rows = c.valid - chunk * 16;
    const uint16_t* at = reinterpret_cast<const uint16_t*>(e.residual) + (c.out_row + chunk * 16) * e.residual_pitch + f;
#pragma unroll
    for (int i = 0; i < 16; ++i, at += e.residual_pitch)
      if (i < rows) r.v[i / 2] |= uint32_t(*at) << 16 * (i & 1);
  }
  return r;
}
__device__ __forceinline__ void store_column(void* out, int fp32, int fp16, int64_t at, int m, int rows, const float (&z)[16]) {
  if (fp32) {
    float* to = reinterpret_cast<float*>(out) + at;
#pragma unroll
    for (int i = 0; i < 16; ++i, to += m)
      if (i < rows) *to = z[i];
  } else {
    uint16_t* to = reinterpret_cast<uint16_t*>(out) + at;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const uint32_t h = pack_h16x2(z[i], z[i + 1], fp16);
      if (i < rows) *to = uint16_t(h);
      to += m;
      if (i + 1 < rows) *to = uint16_t(h >> 16);
      to += m;
    }
  }
}
template <bool kFinish>
__device__ __forceinline__ void emit_column(const ProductArgs& p, const Output& out, const Tile& c, int chunk, int f, float (&z)[16],
                                            float bias, const ColumnResidual& res) {
  const Epilogue& e = p.epi;
  if (f >= p.m) return;
  const int rows = c.valid - chunk * 16;
  const int64_t at = (c.out_row + chunk * 16) * p.m + f;
  if (kFinish) {
    float slope[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] += bias;
    if (e.slope) {
      activate<true>(e.act, z, slope);
      store_column(e.slope, 0, e.fp16, at, p.m, rows, slope);
    } else if (e.act) {
      activate<false>(e.act, z, slope);
    }
    if (e.residual)
#pragma unroll
      for (int i = 0; i < 16; ++i) z[i] += load_h16(&res.v[i / 2], i & 1, e.fp16);
  }
  store_column(out.ptr, out.fp32, e.fp16, at, p.m, rows, z);
}
__device__ __forceinline__ float load_bias(const Epilogue& e, int m, int f) {
  if (e.bias == nullptr || f >= m) return 0.f;
  return e.bias_fp32 ? __ldg(reinterpret_cast<const float*>(e.bias) + f) : load_h16(e.bias, f, e.fp16);
}

// The pairs of a cluster have a part of the same tile's sums each, in tensor memory.  Pair k finishes the chunks
// k, k + splits, ...: it gets the other pairs' parts of them pushed into its ring, which nothing uses any more, and adds them in
// the pairs' order.  Called by all threads of the cluster; a cluster has one tile at most.
template <int kKind, bool kFinish>
__device__ __forceinline__ void join_parts(const ProductArgs& p, const TileShape& shape, SmemTail* t, uint32_t ring, uint32_t tmem,
                                           int worker, int part, uint32_t cta, int total_tiles, int first_tiles, WaitCtx& ctx) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3, group = (warp - kFirstEpilogueWarp) >> 2;
  const bool mine = warp >= kFirstEpilogueWarp && worker < total_tiles;
  const int splits = shape.splits;
  Tile c{};
  bool ok = false;
  if (mine) {
    c = locate<kKind>(worker, first_tiles, part, p, shape, t);
    ok = mbar_wait(smem_u32(&t->acc_full[0]), 0, ctx, 26);
    tc_fence_after();
  }
  cluster_sync_relaxed();  // every pair's products have read their stages
  const bool summed = c.step1 > c.step0;
  const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
  const int chunks = (c.valid + 15) >> 4;
  // block of [16 rows][32 features] for chunk k of pair `from`, in the ring of the pair that finishes it
  auto block_of = [&](int k, int from) { return uint32_t(((k / splits * splits + from) * 4 + quarter) * 2048); };
  if (ok) {
    for (int k = group; k < chunks; k += 2) {
      if (k % splits == part) continue;
      uint32_t v[16];
      tmem_ld16(lanes + k * 16, v);
      tmem_ld_wait16(v);
      float z[16];
      turn_chunk(t->turn[warp - kFirstEpilogueWarp], v, summed, z);
      const uint32_t to = map_to_cta(ring + block_of(k, part), uint32_t(k % splits) * 2 + (cta & 1)) + (lane >> 3) * 128 + (lane & 7) * 16;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + i * 512), "f"(z[4 * i]), "f"(z[4 * i + 1]),
                     "f"(z[4 * i + 2]), "f"(z[4 * i + 3])
                     : "memory");
    }
  }
  cluster_sync();
  if (!ok) return;
  const Output out = output_of(p, shape, kKind == kBothGrads && c.weight);
  const int f = c.f0 + int(cta & 1) * 128 + quarter * 32 + lane;
  const float bias = kFinish ? load_bias(p.epi, p.m, f) : 0.f;
  for (int k = part + group * splits; k < chunks; k += 2 * splits) {
    ColumnResidual res{};
    if (kFinish) res = load_residual_column(p.epi, p.m, c, k, f);
    uint32_t v[16];
    __syncwarp();  // a lane without a feature has not loaded; tensor memory is read by whole warps
    tmem_ld16(lanes + k * 16, v);
    tmem_ld_wait16(v);
    float z[16] = {};
    for (int from = 0; from < splits; ++from) {
      const uint32_t at = ring + block_of(k, from) + lane * 4;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float q;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(q) : "r"(at + i * 128) : "memory");
        z[i] += from != part ? q : summed ? __uint_as_float(v[i]) : 0.f;
      }
    }
    emit_column<kFinish>(p, out, c, k, f, z, bias, res);
  }
}

// kFinish: the output is more than the rounded sum (bias, activation, residual or slope)
template <int kKind, bool kFinish>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ Maps maps, const ProductArgs p, const TileShape shape) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw_addr & 1023u)) & 1023u;
  const uint32_t ring = raw_addr + pad;
  SmemTail* t = reinterpret_cast<SmemTail*>(smem_raw + pad + kRingBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a cluster is `splits` pairs of CTAs: this CTA's place in its pair, the pair's place, the pair's first CTA
  const uint32_t cta = cluster_rank(), rank = cta & 1, first_cta = cta & ~1u;
  const int part = int(cta >> 1);
  const int worker = int(blockIdx.x) / (2 * shape.splits), workers = int(gridDim.x) / (2 * shape.splits);
  const uint16_t pair_mask = uint16_t(3u << first_cta);

  if (warp == 0) {
    if (lane < kMaxStages) {
      mbar_init(smem_u32(&t->full[lane]), kKind >= kWeightGrad ? 2 : 1);
      mbar_init(smem_u32(&t->empty[lane]), 1);
      mbar_init(smem_u32(&t->raw[lane]), 1);
    }
    if (lane < 2) {
      mbar_init(smem_u32(&t->acc_full[lane]), 1);
      mbar_init(smem_u32(&t->acc_empty[lane]), 2 * kEpilogueWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  } else if (warp == 1) {
    if (lane == 0) {
      prefetch_tmap(&maps.a);
      if (kKind == kBothGrads) prefetch_tmap(&maps.a2);
      t->abort_flag = 0;
      t->max_len = 0;
      if (p.offsets == nullptr) {
        t->begin[0] = 0;
        t->len[0] = p.rows;
        t->blocks[0] = 0;
        t->blocks[1] = (p.rows + kTileRows - 1) / kTileRows;
      }
    } else if (kKind == kWeightGrad ? lane == 3 : lane <= kBoxes) {
      prefetch_tmap(&maps.b[lane - 1]);
    }
  } else if (warp == 3) {
    tmem_alloc_pair(smem_u32(&t->tmem_base), kTmemCols);
  }

  int total_tiles;
  int half_rows = 128;  // rows of b that a CTA loads for a step at most
  if (kKind == kWeightGrad) {
    total_tiles = p.groups * shape.row_blocks * shape.f_tiles;
    if (p.n <= 128) half_rows = 64;
  } else if (p.offsets == nullptr) {
    total_tiles = (p.rows + kTileRows - 1) / kTileRows * shape.f_tiles;
    half_rows = min(128, (p.rows + 31) / 32 * 16);
  } else {
    __syncthreads();  // max_len is 0
    int longest = 0;
    for (int g = threadIdx.x; g < p.groups; g += kThreads) {
      int begin, end;
      segment_of(p, g, begin, end);
      t->begin[g] = begin;
      t->len[g] = end - begin;
      longest = max(longest, end - begin);
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0 && longest > 0) atomicMax(&t->max_len, longest);
    __syncthreads();
    if (warp == 0) {  // row blocks before each group: every lane adds up a run of groups
      const int per = (p.groups + 31) / 32;
      const int lo = min(lane * per, p.groups), hi = min(lo + per, p.groups);
      int sum = 0;
      for (int g = lo; g < hi; ++g) sum += (t->len[g] + kTileRows - 1) / kTileRows;
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      int run = incl - sum;
      for (int g = lo; g < hi; ++g) {
        t->blocks[g] = run;
        run += (t->len[g] + kTileRows - 1) / kTileRows;
      }
      if (lane == 31) t->blocks[p.groups] = incl;
    }
    __syncthreads();
    total_tiles = t->blocks[p.groups] * shape.f_tiles;
    half_rows = min(128, (t->max_len + 31) / 32 * 16);
  }
  const int first_tiles = total_tiles;
  if (kKind == kBothGrads) {
    total_tiles += p.groups * shape.row_blocks * shape.f_tiles;
    half_rows = max(half_rows, p.n <= 128 ? 64 : 128);
  }
  // a cluster that joins parts has one tile at most; only offsets that do not ascend could ask for more
  if (shape.splits > 1) total_tiles = min(total_tiles, workers);
  const int stage_bytes = kABytes + max(half_rows, 16) * 128;
  const int stages = min(kMaxStages, int(kRingBytes) / stage_bytes);
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers exist
  tc_fence_after();
  const uint32_t tmem = t->tmem_base;
  WaitCtx ctx{&t->abort_flag, g_status, kDefaultWaitLimitNs};

  const int quarter = warp & 3;                              // tensor-memory lanes 32*quarter .. +31 of an epilogue warp
  const int first_chunk = (warp - kFirstEpilogueWarp) >> 2;  // its chunks of 16 output rows: every other one

  if (warp == 0) {
    // ---------------- loads ----------------
    // One thread runs the steps of a tile (a wait by the whole warp, with its vote and election, took 230 cycles of a
    // step's 520).  The ring's first round finds every stage empty.
    int stage = 0, round = 0;
    bool ok = true;
    for (Walk<kKind> walk(first_tiles, total_tiles, worker, workers, shape); ok && walk.tile < total_tiles; walk.next()) {
      const Tile c = locate<kKind>(walk.tile, first_tiles, part, p, shape, t);
      const int steps = c.step1 - c.step0;
      if (elect_one()) {
        const int half = c.cols >> 1;
        const int f = c.f0 + int(rank) * 128, j = c.b_row + int(rank) * half;
        const uint32_t bytes = kABytes + half * 128;
        const bool weight = kKind == kWeightGrad || (kKind == kBothGrads && c.weight);
        const bool ragged = weight && c.depth % kStep != 0;
        const CUtensorMap* map_a = kKind == kBothGrads && weight ? &maps.a2 : &maps.a;
        int at = stage, lap = round;
        for (int kb = c.step0; kb < c.step1; ++kb) {
          if (lap > 0 && !mbar_wait_lane(smem_u32(&t->empty[at]), (lap & 1) ^ 1, ctx, 21)) {
            ok = false;
            break;
          }
          const bool tail = ragged && kb == c.depth / kStep;
          const uint32_t own_bar = smem_u32(tail ? &t->raw[at] : &t->full[at]);
          const uint32_t bar = map_to_cta(own_bar, tail ? cta : first_cta);
          if (tail) {
            mbar_expect_tx(own_bar, bytes);
          } else if (rank == 0) {
            mbar_expect_tx(own_bar, 2 * bytes);
            if (kKind >= kWeightGrad) mbar_arrive(own_bar);
          }
          const uint32_t a_dst = ring + at * stage_bytes, b_dst = a_dst + kABytes;
          const int k0 = kb * kStep;
          if (kKind == kForward) {
            tma_load_3d_pair(a_dst, map_a, k0, f, c.group, bar);
          } else {
            const int c1 = weight ? c.c_begin + k0 : k0, c2 = weight ? 0 : c.group;
            tma_load_3d_pair(a_dst, map_a, f, c1, c2, bar);
            tma_load_3d_pair(a_dst + 8192, map_a, f + 64, c1, c2, bar);
          }
          if (weight) {
            tma_load_3d_pair(b_dst, &maps.b[2], j, c.c_begin + k0, 0, bar);
            if (half == 128) tma_load_3d_pair(b_dst + 8192, &maps.b[2], j + 64, c.c_begin + k0, 0, bar);
          } else {
            int r = 0;
#pragma unroll
            for (int b = kBoxes - 1; b >= 0; --b)
              if (half & (16 << b)) {
                tma_load_3d_pair(b_dst + r * 128, &maps.b[b], k0, j + r, 0, bar);
                r += 16 << b;
              }
          }
          if (++at == stages) { at = 0; ++lap; }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      round += (stage + steps) / stages;
      stage = (stage + steps) % stages;
    }
    // the products' last arrivals come from the pair's first CTA: this one is not gone before they are here
    for (int i = 0; ok && i < stages; ++i) {
      if (round > 0) ok = mbar_wait(smem_u32(&t->empty[stage]), (round & 1) ^ 1, ctx, 21);
      if (++stage == stages) { stage = 0; ++round; }
    }
  } else if (warp == 1) {
    // ---------------- products (the pair's first CTA) ----------------
    // One thread again; it asks for the next step while this one's products are issued.
    int stage = 0, round = 0;
    uint32_t it = 0;
    bool ok = true;
    const uint32_t fmt = p.epi.fp16 ? 0u : 1u;
    for (Walk<kKind> walk(first_tiles, total_tiles, worker, workers, shape); rank == 0 && ok && walk.tile < total_tiles; walk.next(), ++it) {
      const Tile c = locate<kKind>(walk.tile, first_tiles, part, p, shape, t);
      const int steps = c.step1 - c.step0;
      if (elect_one()) {
        const uint32_t buf = it & 1, use = it >> 1;
        ok = mbar_wait_cluster_lane(smem_u32(&t->acc_empty[buf]), (use & 1) ^ 1, ctx, 22);
        tc_fence_after();
        const uint32_t d = tmem + buf * 256;
        const bool weight = kKind == kWeightGrad || (kKind == kBothGrads && c.weight);
        const uint32_t idesc = make_idesc(fmt, fmt, 256, uint32_t(c.cols)) | (kKind != kForward ? 1u << 15 : 0u) |
                               (weight ? 1u << 16 : 0u);
        const int b_step = weight ? 128 : 2;
        int at = stage, lap = round;
        uint32_t ready = steps > 0 ? mbar_peek_cluster(smem_u32(&t->full[at]), lap & 1) : 0;
        for (int kb = c.step0; ok && kb < c.step1; ++kb) {
          if (!ready && !mbar_wait_cluster_lane(smem_u32(&t->full[at]), lap & 1, ctx, 23)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = ring + at * stage_bytes;
          const uint64_t a_desc = kKind == kForward ? make_kmajor_sw128_desc(a_addr) : make_mnmajor_sw128_desc(a_addr);
          const uint64_t b_desc = weight ? make_mnmajor_sw128_desc(a_addr + kABytes)
                                                       : make_kmajor_sw128_desc(a_addr + kABytes);
          constexpr int kAStep = kKind == kForward ? 2 : 128;
          const int parts = min(4, (c.depth - kb * kStep + 15) / 16);
          const uint32_t empty_bar = smem_u32(&t->empty[at]);
          if (++at == stages) { at = 0; ++lap; }
          ready = kb + 1 < c.step1 ? mbar_peek_cluster(smem_u32(&t->full[at]), lap & 1) : 0;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < parts)
              umma_h16_pair(d, a_desc + kAStep * k, b_desc + b_step * k, idesc, kb > c.step0 || k > 0);
          tc_commit_pair(empty_bar, pair_mask);
        }
        if (ok) tc_commit_pair(smem_u32(&t->acc_full[buf]), pair_mask);
      }
      ok = __all_sync(0xffffffffu, ok);
      round += (stage + steps) / stages;
      stage = (stage + steps) % stages;
    }
    // nor before the other CTA's last arrivals on its accumulators (none where parts are joined)
    if (rank == 0 && ok && shape.splits == 1 && elect_one())
      for (uint32_t b = 0; b < 2 && b < it; ++b)
        mbar_wait_cluster_lane(smem_u32(&t->acc_empty[b]), ((it - 1 - b) >> 1) & 1, ctx, 22);
    __syncwarp();
  } else if (warp == 2) {
    // ---------------- weight gradient: rows past the segment's end become zeros ----------------
    int stage = 0;
    uint32_t phases = 0;  // parity of raw[stage], one bit each
    bool ok = true;
    for (Walk<kKind> walk(first_tiles, total_tiles, worker, workers, shape); kKind >= kWeightGrad && ok && walk.tile < total_tiles; walk.next()) {
      const Tile c = locate<kKind>(walk.tile, first_tiles, part, p, shape, t);
      const int last = c.depth / kStep;
      if ((kKind == kWeightGrad || c.weight) && c.depth % kStep != 0 && last >= c.step0 && last < c.step1) {
        const int at = (stage + last - c.step0) % stages;
        ok = mbar_wait(smem_u32(&t->raw[at]), (phases >> at) & 1, ctx, 24);
        if (!ok) break;
        phases ^= 1u << at;
        // a row is 128 bytes of each 64-element box; the products read whole groups of 16 rows
        const int from = c.depth - last * kStep, to = (from + 15) / 16 * 16;
        const int boxes = 2 + (c.cols >> 7);
        const uint32_t base = ring + at * stage_bytes + (lane & 7) * 16;
        for (int r = from + (lane >> 3); r < to; r += 4)
#pragma unroll
          for (int box = 0; box < 4; ++box)
            if (box < boxes)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + box * 8192 + r * 128), "r"(0) : "memory");
        fence_proxy_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&t->full[at]), first_cta));
        __syncwarp();
      }
      stage = (stage + c.step1 - c.step0) % stages;
    }
  } else if (warp >= kFirstEpilogueWarp && shape.splits == 1) {
    // ---------------- epilogue: each warp on 32 features ----------------
    float* turn_block = t->turn[warp - kFirstEpilogueWarp];
    uint32_t it = 0;
    for (Walk<kKind> walk(first_tiles, total_tiles, worker, workers, shape); walk.tile < total_tiles; walk.next(), ++it) {
      const Tile c = locate<kKind>(walk.tile, first_tiles, part, p, shape, t);
      const Output out = output_of(p, shape, kKind == kBothGrads && c.weight);
      const uint32_t buf = it & 1, use = it >> 1;
      const bool summed = c.step1 > c.step0;
      const uint32_t lanes = tmem + buf * 256 + (uint32_t(quarter * 32) << 16);
      const int chunks = (c.valid + 15) >> 4;
      bool released = false;
      auto release = [&]() {  // this warp's share is in registers: the accumulator may be overwritten
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(&t->acc_empty[buf]), first_cta));
        released = true;
      };
      if (out.vec8 && summed) {
        // 16-bit outputs: two chunks at a time, read as fragments of 8x8 matrices (a lane has features 8m + lane / 4 of
        // two neighbouring output rows), finished in that layout, rounded two rows per instruction, transposed by stmatrix
        // into 1 KiB each ([row][32 features], the 16-byte pieces of a row XOR-swizzled) and stored 8 features per
        // thread.  The residual comes in the same way backwards, a pair of chunks ahead.
        uint16_t* block = reinterpret_cast<uint16_t*>(turn_block);
        const uint32_t st_addr = smem_u32(block) + uint32_t(lane & 7) * 64 + (uint32_t(lane >> 3) ^ ((lane >> 1) & 3u)) * 16;
        const int f8 = c.f0 + int(rank) * 128 + quarter * 32 + (lane & 3) * 8;
        // 16-byte piece i of this lane's four in a pair of chunks: its row and its place in `block`
        auto row_of = [&](int k, int i) { return (k + 2 * (i >> 1)) * 16 + 8 * (i & 1) + (lane >> 2); };
        auto place_of = [&](int i) {
          const int piece = lane + 32 * (i & 1);
          return reinterpret_cast<uint4*>(block + (i >> 1) * 512 + (piece >> 2) * 32 + ((piece & 3) ^ ((piece >> 3) & 3)) * 8);
        };
        uint4 res[4] = {};
        auto request = [&](int k) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row_of(k, i) < c.valid && f8 < p.m)
              res[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.epi.residual) +
                                                       (c.out_row + row_of(k, i)) * p.epi.residual_pitch + f8);
        };
        auto store = [&](void* to, int k) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 q = *place_of(i);
            if (row_of(k, i) < c.valid && f8 < p.m)
              *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(to) + (c.out_row + row_of(k, i)) * p.m + f8) = q;
          }
          __syncwarp();
        };
        // h[2m + r]: features 8m .., rows 8r .. of chunk u of the pair, of values in fragment order
        auto place = [&](int u, const float (&z)[16]) {
          uint32_t h[8];
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int i = (m >> 1) * 8 + r * 4 + (m & 1) * 2;
              h[2 * m + r] = pack_h16x2(z[i], z[i + 1], p.epi.fp16);
            }
          stmatrix_x4_trans(st_addr + u * 1024, h[0], h[2], h[4], h[6]);
          stmatrix_x4_trans(st_addr + u * 1024 + 8 * 64, h[1], h[3], h[5], h[7]);
        };
        float bias_m[4] = {};
        if (kFinish) {
          if (p.epi.bias)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              const int fm = f8 - (lane & 3) * 8 + 8 * m + (lane >> 2);
              if (fm < p.m) bias_m[m] = p.epi.bias_fp32 ? __ldg(reinterpret_cast<const float*>(p.epi.bias) + fm) : load_h16(p.epi.bias, fm, p.epi.fp16);
            }
          if (p.epi.residual) request(first_chunk);
        }
        if (!mbar_wait(smem_u32(&t->acc_full[buf]), use & 1, ctx, 25)) break;
        __syncwarp();  // the loads above are some lanes'; tensor memory is read by whole warps
        tc_fence_after();
        for (int k = first_chunk; k < chunks; k += 4) {
          uint32_t v[2][16];
#pragma unroll
          for (int u = 0; u < 2; ++u)
            if (k + 2 * u < chunks) {
              tmem_ld_frag16(lanes + (k + 2 * u) * 16, v[u]);
              tmem_ld_frag16(lanes + (k + 2 * u) * 16 + (16u << 16), v[u] + 8);
            }
          tmem_ld_wait16x2(v);
          if (k + 4 >= chunks) release();
          if (!kFinish) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float z[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) z[i] = __uint_as_float(v[u][i]);
              place(u, z);
            }
            store(out.ptr, k);
            continue;
          }
          float z[2][16];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) z[u][i] = __uint_as_float(v[u][i]) + bias_m[(i >> 3) * 2 + ((i >> 1) & 1)];
          if (p.epi.slope) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float slope[16];
              activate<true>(p.epi.act, z[u], slope);
              place(u, slope);
            }
            store(p.epi.slope, k);
          } else if (p.epi.act) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float slope[16];
              activate<false>(p.epi.act, z[u], slope);
            }
          }
          if (p.epi.residual) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *place_of(i) = res[i];
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              uint32_t h[8];
              ldmatrix_x4_trans(st_addr + u * 1024, h[0], h[2], h[4], h[6]);
              ldmatrix_x4_trans(st_addr + u * 1024 + 8 * 64, h[1], h[3], h[5], h[7]);
#pragma unroll
              for (int i = 0; i < 16; ++i) z[u][i] += load_h16(&h[((i >> 3) * 2 + ((i >> 1) & 1)) * 2 + ((i >> 2) & 1)], i & 1, p.epi.fp16);
            }
            if (k + 4 < chunks) request(k + 4);
            __syncwarp();
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) place(u, z[u]);
          store(out.ptr, k);
        }
      } else if (!kFinish && out.vec8) {
        // a weight gradient without rows is 0
        if (!mbar_wait(smem_u32(&t->acc_full[buf]), use & 1, ctx, 25)) break;
        tc_fence_after();
        release();
        const int f8 = c.f0 + int(rank) * 128 + quarter * 32 + (lane & 3) * 8;
        for (int r = first_chunk * 8 + (lane >> 2); r < c.valid; r += 16)
          if (f8 < p.m)
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out.ptr) + (c.out_row + r) * p.m + f8) = make_uint4(0, 0, 0, 0);
      } else {
        const int f = c.f0 + int(rank) * 128 + quarter * 32 + lane;
        const float bias = kFinish ? load_bias(p.epi, p.m, f) : 0.f;
        ColumnResidual res{};  // a chunk ahead
        if (kFinish) res = load_residual_column(p.epi, p.m, c, first_chunk, f);
        if (!mbar_wait(smem_u32(&t->acc_full[buf]), use & 1, ctx, 25)) break;
        tc_fence_after();
        for (int k = first_chunk; k < chunks; k += 2) {
          uint32_t v[16];
          __syncwarp();  // lanes without a feature have neither loaded nor stored
          tmem_ld16(lanes + k * 16, v);
          ColumnResidual next{};
          if (kFinish) next = load_residual_column(p.epi, p.m, c, k + 2, f);
          __syncwarp();
          tmem_ld_wait16(v);
          if (k + 2 >= chunks) release();
          float z[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) z[i] = summed ? __uint_as_float(v[i]) : 0.f;
          emit_column<kFinish>(p, out, c, k, f, z, bias, res);
          res = next;
        }
      }
      if (!released) release();
    }
  }

  if (shape.splits > 1) join_parts<kKind, kFinish>(p, shape, t, ring, tmem, worker, part, cta, total_tiles, first_tiles, ctx);

  // ---------------- teardown ----------------
  __syncwarp();
  tc_fence_before();
  // a wait was abandoned: copies and products still in flight get time to land (another warp may raise the flag while the
  // lanes read it)
  if (__any_sync(0xffffffffu, t->abort_flag)) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  cluster_sync_relaxed();  // the other CTA arrives on this one's barriers no more
  tc_fence_after();
  if (warp == 3) tmem_dealloc_pair(tmem, kTmemCols);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int kMaxSplits = 8;  // clusters of 16 CTAs

cudaLaunchConfig_t cluster_config(int clusters, int splits, cudaStream_t stream, cudaLaunchAttribute* attr) {
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = unsigned(2 * splits);
  attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(clusters) * 2 * splits);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// Clusters of `splits` pairs that run at the same time; it depends on how many SMs the parts of this GPU have (74, 33, 22,
// 15, 11, 7, 7 and 7 on one B200).  Read once per device; a second thread that reads it again does no harm.
int active_clusters(const void* kernel, int splits, int device) {
  static std::atomic<int> cached[kMaxDevices][kMaxSplits + 1];
  std::atomic<int>* slot = device >= 0 && device < kMaxDevices ? &cached[device][splits] : nullptr;
  int n = slot ? slot->load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = cluster_config(1, splits, nullptr, attr);
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (slot && n > 0) slot->store(n, std::memory_order_relaxed);
  return n;
}

// Few tiles leave most pairs of CTAs idle: some share a tile then, as long as all clusters run at the same time.  The join
// costs as much as 12 steps, whatever the number of pairs; with four (200 x 512 features: 24 steps 9.9 us instead of 11.5, two pairs
// 11.4; 16 steps 9.5 and 9.6; 8 steps 9.0 and 7.6), more where each then still has 12 (64 steps 12.0 with five, 12.5 with four).
// `tiles`: as many as there can be.
constexpr int kJoinSteps = 12;
int split_count(const void* kernel, int64_t tiles, int64_t steps, int device) {
  if (tiles * 2 > device_sm_count(device) / 2) return 1;  // the launch need not ask
  int s = int(std::min(int64_t(kMaxSplits), std::max(steps / kJoinSteps, int64_t(4))));
  while (s > 1 && steps - steps / s >= kJoinSteps && tiles > active_clusters(kernel, s, device)) --s;
  return steps - steps / s >= kJoinSteps ? s : 1;
}

// Tiled view of 16-bit elements: c0 side by side, c1 `pitch` elements apart, c2 `group` elements apart.
int make_map(CUtensorMap* map, const void* base, int64_t c0, int64_t c1, int64_t c2, int64_t pitch, int64_t group,
             uint32_t box1, int fp16) {
  return make_tensor_map_3d(map, base, uint64_t(c0), uint64_t(c1), uint64_t(c2), uint64_t(pitch) * 2,
                            uint64_t(group) * 2, box1, fp16);
}

bool aligned_to(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

using KernelFn = void (*)(const Maps, const ProductArgs, const TileShape);
KernelFn kernel_of(ProductKind kind, bool finish) {
  switch (kind) {
    case kForward: return finish ? product_kernel<kForward, true> : product_kernel<kForward, false>;
    case kInputGrad: return product_kernel<kInputGrad, false>;
    case kWeightGrad: return product_kernel<kWeightGrad, false>;
    default: return product_kernel<kBothGrads, false>;
  }
}

int configure(ProductKind kind, bool finish, int device) {
  const KernelFn kernel = kernel_of(kind, finish);
  const int variant = kind == kForward ? (finish ? 1 : 0) : kind + 1;
  static std::atomic<bool> configured[kMaxDevices][5];
  if (device < 0 || device >= kMaxDevices || !configured[device][variant].load(std::memory_order_acquire)) {
    MB200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes)));
    MB200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (device >= 0 && device < kMaxDevices) configured[device][variant].store(true, std::memory_order_release);
  }
  return kOk;
}

// Tiles that there can be.
int64_t most_tiles(ProductKind kind, const ProductArgs& p) {
  const int64_t f_tiles = ceil_div(p.m, kTileFeatures);
  if (kind == kWeightGrad) return p.groups * ceil_div(p.n, kTileRows) * f_tiles;
  // a segment's last block may be short: at most one more per segment than the rows fill
  return (p.offsets ? int64_t(p.rows) / kTileRows + std::min(p.groups, p.rows) : ceil_div(p.rows, kTileRows)) * f_tiles;
}

// Steps of a tile's sum; of ragged segments in the weight gradient those of an average one.
int64_t steps_of(ProductKind kind, const ProductArgs& p) { return ceil_div(kind == kWeightGrad ? p.rows / p.groups : p.k, kStep); }

// Time of a launch in steps (0.27 us), start, epilogue of the last tile and launch being about 30: a tile takes its sums' steps, or
// the 9 that its epilogue takes; t1 tiles of s1 steps and then t2 of s2 (Walk).
constexpr int kLaunchSteps = 30;
constexpr int kDrainSteps = 9;
struct LaunchPlan {
  int64_t steps;
  int splits, rounds, lead;
};
LaunchPlan plan_launch(int64_t t1, int64_t s1, int64_t t2, int64_t s2, const void* kernel, int device) {
  const int64_t pairs = std::max(device_sm_count(device) / 2, 1), tiles = t1 + t2;
  const int64_t longest = std::max(t1 ? s1 : 0, t2 ? s2 : 0);
  LaunchPlan best{};
  best.splits = split_count(kernel, tiles, longest, device);
  best.rounds = -1;
  if (best.splits > 1) {
    best.steps = kLaunchSteps + kJoinSteps + ceil_div(longest, best.splits);
    return best;
  }
  const int64_t workers = std::min(tiles, pairs), lead = t2 % workers, others = workers - lead;
  const int64_t c1 = std::max<int64_t>(s1, kDrainSteps), c2 = std::max<int64_t>(s2, kDrainSteps);
  best.lead = int(lead);
  // the others' rounds alone: as many as the leading pairs' tiles take, or one or two fewer
  const int64_t most = lead ? std::min(ceil_div(c2, c1) + 1, ceil_div(t1, others)) : 0;
  for (int64_t alone = most; alone >= std::max<int64_t>(most - 2, 0); --alone) {
    const int64_t rounds = ceil_div(std::max<int64_t>(t1 - alone * others, 0), workers);
    const int64_t steps = kLaunchSteps + t2 / workers * c2 + std::max(alone * c1, lead ? c2 : 0) + rounds * c1;
    if (best.rounds < 0 || steps < best.steps) {
      best.steps = steps;
      best.rounds = int(rounds);
    }
  }
  return best;
}

// Whether both gradients take less time in one launch.  1000 x 2048 -> 1024: 12 us with one launch, 26 with two.
bool one_launch(const ProductArgs& p, int device) {
  const int64_t t1 = most_tiles(kInputGrad, p), s1 = steps_of(kInputGrad, p), t2 = most_tiles(kWeightGrad, p), s2 = steps_of(kWeightGrad, p);
  const void* kernel = reinterpret_cast<const void*>(kernel_of(kBothGrads, false));
  return plan_launch(t1, s1, t2, s2, kernel, device).steps <=
         plan_launch(t1, s1, 0, 0, kernel, device).steps + plan_launch(0, 0, t2, s2, kernel, device).steps;
}

}  // namespace

int product_status(int* status_out, int clear, cudaStream_t stream) {
  MB200_CHECK_CUDA(cudaStreamSynchronize(stream));
  MB200_CHECK_CUDA(cudaMemcpyFromSymbol(status_out, g_status, sizeof(int)));
  const int zero = 0;
  if (clear) MB200_CHECK_CUDA(cudaMemcpyToSymbol(g_status, &zero, sizeof(int)));
  return kOk;
}

int launch_product(ProductKind kind, const ProductArgs& args, int device, cudaStream_t stream) {
  const int sms = device_sm_count(device);
  MB200_REQUIRE(sms > 1, kCudaError, "product: cannot read the SM count of device %d", device);
  const bool weight = kind == kWeightGrad, both = kind == kBothGrads;
  TileShape s{};
  s.f_tiles = int(ceil_div(args.m, kTileFeatures));
  s.row_blocks = weight || both ? int(ceil_div(args.n, kTileRows)) : 0;
  const int64_t tiles = most_tiles(both ? kInputGrad : kind, args) + (both ? most_tiles(kWeightGrad, args) : 0);
  MB200_REQUIRE(tiles < (int64_t(1) << 30), kUnsupportedShape, "product: %lld tiles do not fit 32-bit tile numbers",
                (long long)tiles);
  const Epilogue& e = args.epi;
  const bool finish = e.bias || e.act || e.residual || e.slope;
  s.vec8 = !e.out_fp32 && args.m % 8 == 0 && aligned_to(e.out, 16) && aligned_to(e.slope, 16) &&
           (!e.residual || (aligned_to(e.residual, 16) && e.residual_pitch % 8 == 0));
  s.vec8_2 = !args.out2_fp32 && args.m % 8 == 0 && aligned_to(args.out2, 16);

  Maps maps{};
  int rc;
  const int fp16 = e.fp16;
  if (kind == kForward) rc = make_map(&maps.a, args.a, args.k, args.m, args.groups, args.a_pitch, args.a_group, 128, fp16);
  else if (!weight) rc = make_map(&maps.a, args.a, args.m, args.k, args.groups, args.a_pitch, args.a_group, 64, fp16);
  else rc = make_map(&maps.a, args.a, args.m, args.rows, 1, args.a_pitch, 0, 64, fp16);
  if (!rc && both) rc = make_map(&maps.a2, args.a2, args.m, args.rows, 1, args.a2_pitch, 0, 64, fp16);
  if (rc) return rc;
  // boxes of 64 columns of b; the weight gradient takes those of 64 rows
  for (int i = weight ? 2 : 0; i < (weight ? 3 : kBoxes); ++i)
    if ((rc = make_map(&maps.b[i], args.b, weight ? args.n : args.k, args.rows, 1, args.b_pitch, 0, 16u << i, fp16))) return rc;

  const KernelFn kernel = kernel_of(kind, finish);
  if ((rc = configure(kind, finish, device))) return rc;
  const LaunchPlan plan = plan_launch(weight ? 0 : most_tiles(kInputGrad, args), steps_of(kInputGrad, args),
                                    weight || both ? most_tiles(kWeightGrad, args) : 0, steps_of(kWeightGrad, args),
                                    reinterpret_cast<const void*>(kernel), device);
  s.splits = plan.splits;
  s.rounds = args.offsets ? -1 : plan.rounds;  // the number of ragged tiles is only a bound here
  s.lead = plan.lead;
  cudaLaunchAttribute attr[1];
  const cudaLaunchConfig_t cfg = cluster_config(int(std::min(tiles, int64_t(sms / 2))), s.splits, stream, attr);
  MB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, maps, args, s));
  return kOk;
}

int launch_gradients(const ProductArgs& args, void* dx, void* dw, int dw_fp32, const void* w, int64_t w_pitch, int64_t w_group,
                     const void* x, int64_t x_pitch, int device, cudaStream_t stream) {
  ProductArgs p = args;
  p.a = w;
  p.a_pitch = w_pitch;
  p.a_group = w_group;
  p.epi.out = dx;
  // One launch for both saves a last wave of tiles (dense, 4096 x 7168 -> 2048: 208 us, 231 with two) or all of a launch, unless
  // the weights are so many that reading them and writing their gradients at once takes longer than one after the other (32
  // experts of 2048 x 7168, 16384 rows: 1040 us, 920 with two; 256 of 2048 x 768, 8192 rows: the same; 16 of 7168 x 2048, 8192
  // rows: 495, 530 with two).
  int rc;
  bool together = dx && dw && int64_t(p.groups) * p.n * p.m < int64_t(1) << 28;
  if (together) {
    if ((rc = configure(kBothGrads, false, device))) return rc;
    together = one_launch(p, device);
  }
  if (together) {
    p.a2 = x;
    p.a2_pitch = x_pitch;
    p.out2 = dw;
    p.out2_fp32 = dw_fp32;
    return launch_product(kBothGrads, p, device, stream);
  }
  if (dx && (rc = launch_product(kInputGrad, p, device, stream))) return rc;
  if (!dw) return kOk;
  p.a = x;
  p.a_pitch = x_pitch;
  p.epi.out = dw;
  p.epi.out_fp32 = dw_fp32;
  return launch_product(kWeightGrad, p, device, stream);
}

}  // namespace mb200
