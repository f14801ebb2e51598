// Eviction from the 8-bit cache: the tokens with the largest sums of weights, head by head, into new pages.
//
// First launch (select): a CTA, or a cluster of them, for each sequence and head finds the value of the last token that stays by its digits (11, 11 and
// 10 bits of the sums as ordered integers, kept in shared memory: a histogram in each CTA, looked through over the cluster), then writes the kept
// indices in order.  A token is kept if its sum is above that value, or equal to it and among the first so many that are: ties go to the lowest
// index.  Second launch (move): a warp for each new page and head copies 16 tokens, rounding their codes again under the largest of their scales.
// Bound by HBM: 4 bytes a token and head for the sums, 2 D read and 2 D written for a kept one.  The new pages are others than the old ones:
// the order in which CTAs run does not matter, and pages that sequences share stay as they are.
// Measured, int8, 8 heads of 128: 32 sequences of 1024 to 8192 tokens to 2048 in 65.7 us, of which the move takes 45 for 268 MB (6.0 TB/s); one of 131071 to 16384
// (e4m3) in 40.8, 22 of them the choice, whose steps wait for one another (the sums are read once; digits counted from global memory again took 60).
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace cg = cooperative_groups;

namespace fa {
namespace kv8 {
namespace {

constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kMostRoom = 40960;      // keys of a CTA's shared memory

// Sums as integers in their order: NaN above all, -0 beside 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  x = __fadd_rn(x, 0.f);
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// The sum back from its key (a NaN as one of them).
__device__ __forceinline__ float sum_of(uint32_t k) { return __uint_as_float(k == 0xffffffffu ? 0x7fffffffu : k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

struct Row {
  const float* mass;
  int len;
};
__device__ __forceinline__ Row row_of(const EvictArgs& a, int b, int h) {
  const int at = a.mass_index != nullptr ? a.mass_index[b] : b;
  Row r;
  r.len = max(0, min(a.lens[b], min(a.c.max_pages * kPage, a.mass_cap)));
  if (at < 0 || at >= a.mass_rows) {
    r.len = 0;
    if (threadIdx.x == 0) atomicOr(a.c.status, kStatusBadPageId);
  }
  r.mass = a.mass + ((int64_t)max(0, min(at, a.mass_rows - 1)) * a.c.heads + h) * a.mass_cap;
  return r;
}

// Where the bins, counted from the top, reach `want`: the bin, and how many of it are wanted.  By one warp: 64 groups of 32 bins first, each summed over the
// cluster, then the 32 bins of the one in question, so that two reads from other SMs are all that is waited for.  at(r): bins and groups of CTA r.
struct Found {
  uint32_t bin, want;
};
struct Bins {
  const uint32_t *fine, *group;
};
template <int MOST, class At>
__device__ __forceinline__ Found find_bin(uint32_t want, int C, At at) {
  const int lane = threadIdx.x & 31;
  const auto running = [&](uint32_t x) {      // inclusive, over lanes
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    return x;
  };
  uint32_t hi[MOST], lo[MOST], n0 = 0, n1 = 0;      // groups 63 - 2 lane and 62 - 2 lane
#pragma unroll
  for (int r = 0; r < MOST; ++r)
    if (r < C) {
      const uint2 v = *reinterpret_cast<const uint2*>(at(r).group + 62 - 2 * lane);
      lo[r] = v.x;
      hi[r] = v.y;
    }
#pragma unroll
  for (int r = 0; r < MOST; ++r)
    if (r < C) {
      n0 += hi[r];
      n1 += lo[r];
    }
  const uint32_t upto = running(n0 + n1), before = upto - n0 - n1;
  const int who = __ffs(__ballot_sync(0xffffffffu, upto >= want)) - 1;
  const bool first = before + n0 >= want;
  const int group = __shfl_sync(0xffffffffu, 63 - 2 * lane - (first ? 0 : 1), who);
  want -= __shfl_sync(0xffffffffu, before + (first ? 0u : n0), who);
  uint32_t n = 0;
#pragma unroll
  for (int r = 0; r < MOST; ++r)
    if (r < C) hi[r] = at(r).fine[group * 32 + 31 - lane];
#pragma unroll
  for (int r = 0; r < MOST; ++r)
    if (r < C) n += hi[r];
  const uint32_t sum = running(n);
  const int bin = __ffs(__ballot_sync(0xffffffffu, sum >= want)) - 1;
  return {(uint32_t)(group * 32 + 31 - bin), want - __shfl_sync(0xffffffffu, sum - n, bin)};
}

// MOST: CTAs of a cluster at most.  STAGED: each CTA keeps the keys of its stretch of the row in shared memory; else they are read again for every pass.
template <int MOST, bool STAGED, int kThreads>
__global__ void __launch_bounds__(kThreads) select_kernel(const EvictArgs a) {
  constexpr int kWarps = kThreads / 32, kEach = kBins / kThreads;      // bins of a thread
  cg::cluster_group cluster = cg::this_cluster();
  const int C = MOST > 1 ? (int)cluster.num_blocks() : 1, rank = MOST > 1 ? (int)cluster.block_rank() : 0;
  const int pair = blockIdx.x / C, b = pair / a.c.heads, h = pair - b * a.c.heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  extern __shared__ uint32_t staged[];
  __shared__ __align__(16) uint32_t hist[3][kBins];
  __shared__ __align__(16) uint32_t group[3][kBins / 32];
  __shared__ uint2 counts[kWarps];
  __shared__ Found found;
  const auto sync = [&] {
    if constexpr (MOST > 1) cluster.sync(); else __syncthreads();
  };
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Row row = row_of(a, b, h);
  int* kept = a.kept + (int64_t)pair * a.budget;
  float* new_mass = a.new_mass + (int64_t)pair * a.budget;
  const int len = row.len;
  if (h == 0 && rank == 0 && tid == 0) a.new_lens[b] = min(len, a.budget);
  if (len <= a.budget) {                      // (all CTAs of the cluster)
    for (int i = rank * kThreads + tid; i < a.budget; i += C * kThreads) {
      kept[i] = i < len ? i : -1;
      new_mass[i] = i < len ? row.mass[i] : 0.f;
    }
    return;
  }
  const int lo = a.sink, hi = len - a.recent;      // the tokens that are chosen from
  const int times = (len + C * kThreads - 1) / (C * kThreads);      // of 32 tokens, for each warp
  const int begin = rank * times * kThreads, end = min(len, begin + times * kThreads);      // the CTA's stretch
  const auto key_at = [&](int i) {
    if constexpr (STAGED) return staged[i - begin];
    return key_of(row.mass[i]);
  };
  for (int i = tid; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(&hist[0][0])[i] = make_uint4(0, 0, 0, 0);
  if constexpr (STAGED) {
#pragma unroll 8
    for (int i = begin + tid; i < end; i += kThreads) staged[i - begin] = key_of(row.mass[i]);
  }
  __syncthreads();
  uint32_t want = (uint32_t)(a.budget - a.sink - a.recent);      // of those whose leading digits are `value`'s, so many are still wanted
  uint32_t value = 0xffffffffu;
  const bool none = want == 0;
  if (!none) {
    value = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      const uint32_t mask = pass == 0 ? 0u : (0xffffffffu << (shift + bits)), digit = (1u << bits) - 1;
      uint32_t* bins = hist[pass];
      const int last = min(hi, end);
      for (int i0 = max(lo, begin) + tid; i0 < last; i0 += 4 * kThreads) {
        uint32_t k[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) k[e] = i0 + e * kThreads < last ? key_at(i0 + e * kThreads) : 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i0 + e * kThreads < last && (k[e] & mask) == value) atomicAdd(bins + ((k[e] >> shift) & digit), 1u);
      }
      __syncthreads();
      uint32_t sum = 0;                       // of 32 bins, by 32 / kEach threads
#pragma unroll
      for (int e = 0; e < kEach; ++e) sum += bins[tid * kEach + e];
#pragma unroll
      for (int d = 1; d < 32 / kEach; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (tid % (32 / kEach) == 0) group[pass][tid / (32 / kEach)] = sum;
      sync();
      if (warp == 0) {
        const Found f = find_bin<MOST>(want, C, [&](int r) -> Bins {
          if constexpr (MOST > 1) return {cluster.map_shared_rank(bins, r), cluster.map_shared_rank(group[pass], r)};
          return {bins, group[pass]};
        });
        if (lane == 0) found = f;
      }
      __syncthreads();
      value |= found.bin << shift;
      want = found.want;
    }
  }
  // A token is kept for certain, or equal to the last value: running counts over lanes, warps and CTAs, each warp on a stretch of its own.  (With nothing
  // wanted the last value is above every sum's, and of NaNs none are taken.)
  constexpr int kBatch = 4;                   // keys under way at once
  const int mine = begin + warp * times * 32 + lane;
  const auto keys_from = [&](int k0, uint32_t (&x)[kBatch]) {
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      const int i = mine + (k0 + e) * 32;
      x[e] = 0;
      if (k0 + e < times && i < len) x[e] = key_at(i);
    }
  };
  const auto certain = [&](int i, uint32_t k) { return (i < len) & ((i < lo) | (i >= hi) | (k > value)); };
  const auto equal = [&](int i, uint32_t k) { return (i >= lo) & (i < hi) & (k == value); };
  uint32_t sure = 0, same = 0;
  for (int k0 = 0; k0 < times; k0 += kBatch) {
    uint32_t x[kBatch];
    keys_from(k0, x);
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      const int i = k0 + e < times ? mine + (k0 + e) * 32 : len;
      sure += certain(i, x[e]);
      same += equal(i, x[e]);
    }
  }
  sure = __reduce_add_sync(0xffffffffu, sure);
  same = __reduce_add_sync(0xffffffffu, same);
  if (lane == 0) counts[warp] = make_uint2(sure, same);
  sync();
  sure = same = 0;
  for (int x = lane; x < rank * kWarps + warp; x += 32) {      // the warps before this one
    const uint2* from = counts;
    if constexpr (MOST > 1) from = cluster.map_shared_rank(counts, x / kWarps);
    const uint2 v = from[x % kWarps];
    sure += v.x;
    same += v.y;
  }
  sure = __reduce_add_sync(0xffffffffu, sure);
  same = __reduce_add_sync(0xffffffffu, same);
  if constexpr (MOST > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
  const uint32_t below = (1u << lane) - 1;
  for (int k0 = 0; k0 < times; k0 += kBatch) {
    uint32_t x[kBatch], cs[kBatch], es[kBatch];
    keys_from(k0, x);
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      const int i = k0 + e < times ? mine + (k0 + e) * 32 : len;
      cs[e] = __ballot_sync(0xffffffffu, certain(i, x[e]));
      es[e] = __ballot_sync(0xffffffffu, equal(i, x[e]));
    }
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      const uint32_t q = same + __popc(es[e] & below), at = sure + __popc(cs[e] & below) + min(q, want);
      const bool takes = ((cs[e] >> lane) & 1u) | (((es[e] >> lane) & 1u) & (q < want));
      if (takes && at < (uint32_t)a.budget) {
        kept[at] = mine + (k0 + e) * 32;
        new_mass[at] = sum_of(x[e]);
      }
      sure += __popc(cs[e]);
      same += __popc(es[e]);
    }
  }
  if constexpr (MOST > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // nobody leaves while its shared memory is read
}

constexpr int kMoveWarps = 4;

template <int D, bool E4M3>
__global__ void __launch_bounds__(kMoveWarps * 32) move_kernel(const EvictArgs a, int new_pages) {
  constexpr int kLanes = D / 16;             // lanes of a row, 16 bytes each
  constexpr int kRows = 32 / kLanes;
  constexpr int kLoads = kPage / kRows;
  const int lane = threadIdx.x & 31;
  const int64_t job = (int64_t)blockIdx.x * kMoveWarps + (threadIdx.x >> 5);
  const int h = (int)(job % a.c.heads);
  const int p = (int)(job / a.c.heads % new_pages);
  const int64_t b = job / a.c.heads / new_pages;
  if (b >= a.batch) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n = min(kPage, a.new_lens[b] - p * kPage);
  if (n <= 0) return;
  const int to = a.new_table[b * a.new_width + p];
  if (!page_ok(a.c, to)) {
    if (lane == 0) atomicOr(a.c.status, kStatusBadPageId);
    return;
  }
  // lane i < n: token i of the new page
  int64_t src = -1;                            // its row among all pages' rows
  uint32_t scale[2] = {0, 0};                  // (from 0 up: their bits are in their order)
  if (lane < n) {
    const int tok = a.kept[(b * a.c.heads + h) * a.budget + p * kPage + lane];
    const int id = a.c.table[b * a.c.width + (tok >> 4)];
    if (page_ok(a.c, id)) {
      const int64_t at = (int64_t)id * a.c.heads + h;
      const uint2 s = *reinterpret_cast<const uint2*>(a.c.scale + at * 2);
      scale[0] = s.x;
      scale[1] = s.y;
      src = at * kPage + (tok & (kPage - 1));
    } else {
      atomicOr(a.c.status, kStatusBadPageId);
    }
  }
  const int r0 = lane / kLanes, col = lane % kLanes;
  const int64_t dst = ((int64_t)to * a.c.heads + h) * kPage;
  uint4 x[2][kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int64_t from = __shfl_sync(0xffffffffu, src, i * kRows + r0);
    x[0][i] = x[1][i] = make_uint4(0, 0, 0, 0);
    if (from >= 0) {
      x[0][i] = load_stream16(a.c.k + from * D + col * 16);
      x[1][i] = load_stream16(a.c.v + from * D + col * 16);
    }
  }
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, scale[kind]);
    const float ratio = scale[kind] == best ? 1.f : __fdiv_rn(__uint_as_float(scale[kind]), __uint_as_float(best));
    uint8_t* codes = kind ? a.c.v : a.c.k;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * kRows + r0;
      const float f = __shfl_sync(0xffffffffu, ratio, r);
      uint32_t w[4] = {x[kind][i].x, x[kind][i].y, x[kind][i].z, x[kind][i].w};
      if (f != 1.f) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = recode4<E4M3>(w[j], f);
      }
      if (r < n) *reinterpret_cast<uint4*>(codes + (dst + r) * D + col * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (lane == 0) a.c.scale[((int64_t)to * a.c.heads + h) * 2 + kind] = __uint_as_float(best);
  }
}

template <int D>
cudaError_t launch_move(const EvictArgs& a, bool e4m3, cudaStream_t s) {
  const int new_pages = (a.budget + kPage - 1) / kPage;
  const unsigned grid = (unsigned)(((int64_t)a.batch * a.c.heads * new_pages + kMoveWarps - 1) / kMoveWarps);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kMoveWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // (its blocks wait for the end of the choice)
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return e4m3 ? cudaLaunchKernelEx(&cfg, move_kernel<D, true>, a, new_pages) : cudaLaunchKernelEx(&cfg, move_kernel<D, false>, a, new_pages);
}

template <int MOST, bool STAGED, int THREADS>
cudaError_t launch_select(cudaLaunchConfig_t cfg, const EvictArgs& a, int64_t stretch) {
  static SharedMemoryLimit limit;
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = STAGED ? (size_t)stretch * 4 : 0;
  const cudaError_t e = limit.raise(reinterpret_cast<const void*>(select_kernel<MOST, STAGED, THREADS>), (int)cfg.dynamicSmemBytes);
  return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, select_kernel<MOST, STAGED, THREADS>, a);
}

}  // namespace

cudaError_t launch_evict(const EvictArgs& a, bool e4m3, int sms, cudaStream_t s) {
  // A CTA of 512 threads for each sequence and head; a cluster of up to 8 of 1024 where those leave SMs idle and rows are long enough to share, or where a
  // row's keys do not fit in the shared memory of one.
  const int pairs = a.batch * a.c.heads;
  int64_t longest = (int64_t)a.c.max_pages * kPage;
  if (a.mass_cap < longest) longest = a.mass_cap;
  int cluster = 1;
  while (cluster < kMaxCluster && (((int64_t)pairs * cluster < sms && longest / (cluster * 2) >= 2048) || longest / cluster > kMostRoom)) cluster *= 2;
  const int threads = cluster == 1 ? 512 : 1024;
  const int64_t stretch = (longest + (int64_t)cluster * threads - 1) / ((int64_t)cluster * threads) * threads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pairs * cluster));
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 2;
  cudaError_t e = cluster == 1 ? launch_select<1, true, 512>(cfg, a, stretch) : stretch <= kMostRoom ? launch_select<kMaxCluster, true, 1024>(cfg, a, stretch)
                                                                                                     : launch_select<kMaxCluster, false, 1024>(cfg, a, stretch);
  if (e != cudaSuccess) return e;
  switch (a.c.dim) {
    case 64: return launch_move<64>(a, e4m3, s);
    case 128: return launch_move<128>(a, e4m3, s);
    default: return launch_move<256>(a, e4m3, s);
  }
}

}  // namespace kv8
}  // namespace fa
