// New keys and values into the pages of the 8-bit cache.
//
// For each page, head and kind that gets rows: a = max |x| of the new rows, scale' = max(a / top, 2^-100, the scale before if the page has
// rows already), code = round(x / scale').  Bound by HBM: a prompt's row of D values is read as 2 D bytes and written as D.  One warp takes a page of one head
// and kind whole into registers (D bytes a lane), so the rows are read once; the largest magnitude is found on the 16-bit patterns two at a
// time, where NaN is above infinity.  Measured: 16 prompts of 128 to 4096 tokens, 8 heads of 128, bf16 to e4m3: 37.6 us for 208 MB, 5.5 TB/s (44 with a
// warp a kind and 64-bit divisions to find its place; six CTAs an SM: with four 4 % more, with eight the same); one new token of 64 sequences 3.1.
#include "kv8.cuh"

namespace fa {
namespace kv8 {
namespace {

template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
  if constexpr (BF16) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w));
    a = f.x;
    b = f.y;
  }
}

// `n` rows from `row` on (stride in elements) into the slots from `slot` on of one page.
template <int D, bool E4M3, bool BF16>
__device__ __forceinline__ void append_page(const AppendArgs& a, const uint16_t* row, int64_t stride, uint8_t* codes, float* scale, int slot, int n, int lane) {
  constexpr int kLanes = D / 8;              // lanes of a row, 16 bytes each
  constexpr int kRows = 32 / kLanes;         // rows of one load
  constexpr int kLoads = kPage / kRows;
  const int r0 = lane / kLanes, col = lane % kLanes;
  uint4 x[kLoads];
  uint32_t most = 0;
  const uint16_t* from = row + r0 * stride + col * 8;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    x[i] = make_uint4(0, 0, 0, 0);
    if (i * kRows + r0 < n) x[i] = load_stream16(from);
    from += kRows * stride;
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) most = __vmaxu2(most, w[j] & 0x7fff7fffu);
  }
  most = max(most & 0xffffu, most >> 16);
  most = __reduce_max_sync(0xffffffffu, most);
  float m, unused;
  unpack2<BF16>(most, m, unused);
  if (!(m <= 3.4028235e38f)) m = __int_as_float(0x7f800000);
  const float before = slot > 0 ? *scale : 0.f;
  const float made = fmaxf(fmaxf(__fmul_rn(m, (float)(1.0 / top_of(E4M3))), kLeastScale), before);
  if (slot > 0 && made > before) {           // the page's earlier rows, again
    const float ratio = __fdiv_rn(before, made);
    uint32_t* old = reinterpret_cast<uint32_t*>(codes);
    for (int i = lane; i < slot * (D / 4); i += 32) old[i] = recode4<E4M3>(old[i], ratio);
  }
  __syncwarp();
  if (lane == 0) *scale = made;
  const uint32_t finite = made <= 3.4028235e38f ? 0xffffffffu : 0u;
  const float inv = __frcp_rn(made);
  uint8_t* to = codes + (slot + r0) * D + col * 8;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    uint32_t out[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float f[4];
      unpack2<BF16>(w[2 * j], f[0], f[1]);
      unpack2<BF16>(w[2 * j + 1], f[2], f[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = __fmul_rn(f[e], inv);
      out[j] = encode4<E4M3>(f) & finite;
    }
    if (i * kRows + r0 < n) *reinterpret_cast<uint2*>(to + i * kRows * D) = make_uint2(out[0], out[1]);
  }
}

// The sequence of packed token t: the last one with cu[b] <= t that is not empty.
__device__ __forceinline__ int sequence_of(const int* cu, int batch, int t) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

constexpr int kWarps = 4;

// A warp per window of tokens (packed prompts: 16, a decode step: 1) and head: it takes the pages that begin, for this call, in the window, their keys and
// then their values.  SPLIT: a warp for each kind.
template <int D, bool E4M3, bool BF16, bool SPLIT>
__global__ void __launch_bounds__(kWarps * 32, D == 256 ? 3 : 6) append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int window = a.cu != nullptr ? kPage : 1;
  const int h = blockIdx.y;
  const uint32_t job = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int64_t first = (int64_t)(SPLIT ? job >> 1 : job) * window;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (first >= a.total) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // lane i < window: token first + i, and whether it is the first of a page's new rows
  const int t = (int)first + lane, total = (int)a.total;
  int page = 0, slot = 0, n = 0;
  bool leads = false;
  if (lane < window && t < total) {
    int b = t, begin = t, end = t + 1;
    if (a.cu != nullptr) {
      b = sequence_of(a.cu, a.batch, t);
      begin = a.cu[b];
      end = min(a.cu[b + 1], total);
    }
    const int start = a.positions != nullptr ? a.positions[b] : 0;      // (negative: a row of a padded batch)
    if (t >= begin && t < end && begin >= 0 && start >= 0) {
      const int64_t pos = (int64_t)start + (t - begin);
      slot = (int)pos & (kPage - 1);
      leads = t == begin || slot == 0;
      n = min(kPage - slot, end - t);
      const int64_t index = pos >> 4;
      page = -1;
      if (leads && index < a.c.max_pages) page = a.c.table[(int64_t)b * a.c.width + index];
      if (leads && !page_ok(a.c, page)) {
        atomicOr(a.c.status, kStatusBadPageId);
        leads = false;
      }
    }
  }
  for (uint32_t todo = __ballot_sync(0xffffffffu, leads); todo; todo &= todo - 1) {
    const int i = __ffs(todo) - 1;
    const int s = __shfl_sync(0xffffffffu, slot, i), count = __shfl_sync(0xffffffffu, n, i);
    const int64_t at = (int64_t)__shfl_sync(0xffffffffu, page, i) * a.c.heads + h;
#pragma unroll 1
    for (int kind = SPLIT ? (int)(job & 1) : 0; kind < (SPLIT ? (int)(job & 1) + 1 : 2); ++kind) {
      const int64_t stride = kind ? a.v_stride : a.k_stride;
      append_page<D, E4M3, BF16>(a, static_cast<const uint16_t*>(kind ? a.v : a.k) + (int64_t)h * D + (first + i) * stride, stride,
                                 (kind ? a.c.v : a.c.k) + at * kPage * D, a.c.scale + at * 2 + kind, s, count, lane);
    }
  }
}

template <int D, bool E4M3>
cudaError_t launch_append_d(const AppendArgs& a, bool bf16, cudaStream_t s) {
  // A decode step has a page for each sequence and head: a warp for each kind.  Prompts have enough pages, and a warp looks the places up once for both.
  const bool split = a.cu == nullptr;
  const int64_t windows = split ? 2 * a.total : (a.total + kPage - 1) / kPage;
  const dim3 grid((unsigned)((windows + kWarps - 1) / kWarps), (unsigned)a.c.heads);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // (its blocks wait for the end of the launch in front)
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (split) return bf16 ? cudaLaunchKernelEx(&cfg, append_kernel<D, E4M3, true, true>, a) : cudaLaunchKernelEx(&cfg, append_kernel<D, E4M3, false, true>, a);
  return bf16 ? cudaLaunchKernelEx(&cfg, append_kernel<D, E4M3, true, false>, a) : cudaLaunchKernelEx(&cfg, append_kernel<D, E4M3, false, false>, a);
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, bool e4m3, bool bf16, cudaStream_t s) {
  switch (a.c.dim) {
    case 64: return e4m3 ? launch_append_d<64, true>(a, bf16, s) : launch_append_d<64, false>(a, bf16, s);
    case 128: return e4m3 ? launch_append_d<128, true>(a, bf16, s) : launch_append_d<128, false>(a, bf16, s);
    default: return e4m3 ? launch_append_d<256, true>(a, bf16, s) : launch_append_d<256, false>(a, bf16, s);
  }
}

}  // namespace kv8
}  // namespace fa
