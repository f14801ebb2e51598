// Eviction from the 8-bit cache: the tokens with the largest sums of weights, head by head, into new pages.
//
// First launch (select): a cluster of CTAs for each sequence and head finds the value of the last token that stays by its digits (11, 11 and
// 10 bits of the sums as ordered integers: a histogram in shared memory for each, added up over the cluster), then writes the kept indices
// in order.  A token is kept if its sum is above that value, or equal to it and among the first so many that are: ties go to the lowest
// index.  Second launch (move): a warp for each new page and head copies 16 tokens, rounding their codes again under the largest of their scales.
// Bound by HBM: 4 bytes a token and head for the sums, 2 D read and 2 D written for a kept one.  The new pages are others than the old ones:
// the order in which CTAs run does not matter, and pages that sequences share stay as they are.
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace cg = cooperative_groups;

namespace fa {
namespace kv8 {
namespace {

constexpr int kThreads = 512;
constexpr int kBins = 2048;

// Sums as integers in their order: NaN above all, -0 beside 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  x = __fadd_rn(x, 0.f);
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xffffffffu;
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

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

// Exclusive running sum over the block; *total: the whole sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    const uint32_t s = warp_sums[i];
    if (i < w) before += s;
    all += s;
  }
  *total = all;
  return before + x - v;
}

__global__ void __launch_bounds__(kThreads) select_kernel(const EvictArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int pair = blockIdx.x / C, b = pair / a.c.heads, h = pair % a.c.heads;
  const int tid = threadIdx.x;
  __shared__ uint32_t hist[3][kBins];
  __shared__ uint32_t warp_sums[kThreads / 32];
  __shared__ uint32_t found[2];
  __shared__ uint32_t counts[2];
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
  const int slice = (len + C - 1) / C;
  const int begin = min(len, rank * slice), end = min(len, begin + slice);
  uint32_t want = (uint32_t)(a.budget - a.sink - a.recent);      // of those whose leading digits are `value`'s, so many are still wanted
  uint32_t value = 0xffffffffu;
  bool none = want == 0;
  if (!none) {
    for (int i = tid; i < 3 * kBins; i += kThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    value = 0;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      const uint32_t mask = pass == 0 ? 0u : (0xffffffffu << (shift + bits));
      for (int i = max(lo, begin) + tid; i < min(hi, end); i += kThreads) {
        const uint32_t k = key_of(row.mass[i]);
        if ((k & mask) == value) atomicAdd(&hist[pass][(k >> shift) & ((1u << bits) - 1)], 1u);
      }
      cluster.sync();
      // bins from the top, four for each thread
      constexpr int kEach = kBins / kThreads;
      const int top = kBins - 1 - tid * kEach;
      uint32_t n[kEach], sum = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        n[e] = 0;
        for (int r = 0; r < C; ++r) n[e] += *cluster.map_shared_rank(&hist[pass][top - e], r);
        sum += n[e];
      }
      uint32_t total;
      uint32_t above = block_scan(sum, warp_sums, &total);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (above < want && above + n[e] >= want) {
          found[0] = (uint32_t)(top - e);
          found[1] = want - above;
        }
        above += n[e];
      }
      __syncthreads();
      value |= found[0] << shift;
      want = found[1];
      __syncthreads();
    }
  }
  // How many of the slice are kept for certain, and how many are equal to the last value.
  const auto kind = [&](int i) -> uint32_t {      // 1: kept, 1 << 16: equal
    if (i < lo || i >= hi) return 1u;
    if (none) return 0u;
    const uint32_t k = key_of(row.mass[i]);
    return k > value ? 1u : k == value ? 1u << 16 : 0u;
  };
  if (tid < 2) counts[tid] = 0;
  __syncthreads();
  uint32_t sure = 0, equal = 0;
  for (int i = begin + tid; i < end; i += kThreads) {
    const uint32_t k = kind(i);
    sure += k & 1u;
    equal += k >> 16;
  }
  sure = __reduce_add_sync(0xffffffffu, sure);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if ((tid & 31) == 0) {
    atomicAdd(&counts[0], sure);
    atomicAdd(&counts[1], equal);
  }
  cluster.sync();
  sure = equal = 0;
  for (int r = 0; r < rank; ++r) {
    sure += *cluster.map_shared_rank(&counts[0], r);
    equal += *cluster.map_shared_rank(&counts[1], r);
  }
  cluster.sync();                             // nobody leaves while its shared memory is read
  constexpr int kEach = 4;
  for (int i0 = begin; i0 < end; i0 += kThreads * kEach) {
    uint32_t k[kEach], mine = 0, total;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = i0 + tid * kEach + e;
      k[e] = i < end ? kind(i) : 0u;
      mine += k[e];
    }
    const uint32_t before = block_scan(mine, warp_sums, &total);
    uint32_t s = sure + (before & 0xffffu), q = equal + (before >> 16);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = i0 + tid * kEach + e;
      if (k[e] == 1u || (k[e] != 0 && q < want)) {
        const uint32_t at = s + min(q, want);
        if (at < (uint32_t)a.budget) {
          kept[at] = i;
          new_mass[at] = row.mass[i];
        }
      }
      s += k[e] & 1u;
      q += k[e] >> 16;
    }
    sure += total & 0xffffu;
    equal += total >> 16;
  }
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
  if (e4m3) move_kernel<D, true><<<grid, kMoveWarps * 32, 0, s>>>(a, new_pages);
  else move_kernel<D, false><<<grid, kMoveWarps * 32, 0, s>>>(a, new_pages);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_evict(const EvictArgs& a, bool e4m3, int sms, cudaStream_t s) {
  // A cluster of up to 8 CTAs where the sequences and heads alone leave SMs idle and rows are long enough to share.
  const int pairs = a.batch * a.c.heads;
  int64_t longest = (int64_t)a.c.max_pages * kPage;
  if (a.mass_cap < longest) longest = a.mass_cap;
  int cluster = 1;
  while (cluster < 8 && pairs * cluster < sms && longest / (cluster * 2) >= 4 * kThreads) cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pairs * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, select_kernel, a);
  if (e != cudaSuccess) return e;
  switch (a.c.dim) {
    case 64: return launch_move<64>(a, e4m3, s);
    case 128: return launch_move<128>(a, e4m3, s);
    default: return launch_move<256>(a, e4m3, s);
  }
}

}  // namespace kv8
}  // namespace fa
