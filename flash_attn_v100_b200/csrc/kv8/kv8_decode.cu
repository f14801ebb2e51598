// Attention of each sequence's newest tokens on the paged 8-bit cache.
//
//   s_rj = f(q_r . k_j ks_j),  p_rj = 2^(s_rj - m_r),  o_r = sum_j p_rj vs_j v_j / sum_j p_rj
//
// with one scale ks, vs for the 16 tokens of a page and head.  Bound by HBM (2 D bytes a token and KV head against 4 D flop a row), so the
// rows of a KV head (its query heads times the new tokens) share every code that is read, in blocks of 8 or 16.  Keys, and then output dimensions,
// are the 16 rows of mma.sync.m16n8k16 and the query rows its 8 columns: S^T = K Q^T, O^T = V^T P^T.
// A warp copies pages to a ring of its own in shared memory (cp.async, 16 bytes a lane, the pieces of a row placed so that the reads meet no bank twice) and
// runs ahead of its own reads from one piece into the next.  A lane's 16 bytes of a key row are four steps of the (permuted) contraction, and its 16
// bytes of four tokens' values the rows of eight tiles of O^T.  They become fp16 in registers, exactly.
// K's scale multiplies the finished scores.  V's scale goes into the exponent: with m the running maximum of s + log2 vs, less 25, the weight that meets the
// codes is 2^(s - m) vs / 2^10 <= 2^15, so fp16 keeps 11 bits of the products down to 2^-29 of the largest (with 1 as the largest weight all below 2^-25 were
// lost, of many tokens behind a strong one a visible part); the sum of weights takes 2^(s - m) in fp32, which has room for every scale that an append makes:
// it is 2^-96 at 2^121 and at most 2^100 at 2^-100, where log2 vs counts as -75 and the weights reach 2^-10.
// The pages of all sequences and heads are cut evenly over the warps; where there are fewer segments than half the CTAs each is cut into equal
// parts, at least kLeastPart pages, that the warps of a CTA share.  Parts of a cut segment go through global memory to a second launch, which, like the
// first, is on its way before the launch in front of it has ended.
// Measured, int8, 32 heads on 8 of 128: 64 sequences of 512 to 8192 tokens 109.9 us for 573 MB (5.2 TB/s), one of 131071 (e4m3) 51.0 us for 269 MB; four of up to
// 101 tokens 5.8 us.  Two CTAs of four warps an SM, 16 KB of ring each: with three the first takes as long, the second 57 us (bytes on their way are enough
// with eight warps, and more wait longer for theirs).  Of the first case 4 us pass before the memory is busy and 5 behind the last code; between them it
// delivers 7.3 TB/s until the first SMs are through, and the last are a sixth later: some get their bytes slower than others.  Looked at and left: loads
// straight to registers (117), L2 prefetches 2 to 6 steps ahead (slower by 5 to 14 %), a quarter of the pages in small ranges for warps that are through
// early, as CTAs of their own, taken over by running ones or counted out by an atomic (116 to 150: a new piece waits for its page numbers, its rows of q
// and its codes in turn behind all bytes on their way), more CTAs than fit at once (12 us a wave), keys as they are in three products with whole-numbered
// parts of q (mma.s8: no conversion, the same time; 37 instead of 32 us for 20 rows of 16 sequences).  Of a step's 2600 cycles 50 are waits for codes and 880
// the issue of the next copies, which is where a full memory system makes itself felt.
#include <limits.h>
#include <math_constants.h>

#include "kv8.cuh"

namespace fa {
namespace kv8 {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kLeastPart = 8;
constexpr int kOpening = 4;
constexpr float kUnit = 1024.f, kTop = 25.f;      // a weight times V's scale is at most kUnit * 2^15: fp16 ends at 2^16
constexpr float kLeastLog = -75.f;                // of V's scale

__device__ __forceinline__ float log2_of(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A score x in base 2 under its cap, both ways to 2^-19 of the result: from a quarter of the cap on cap tanh(x / cap) = cap (1 - 2 / (e^(2x / cap) + 1)), off by
// less than 2^-21 cap, and below x (1 - u^2/3 + 2 u^4/15 - 17 u^6/315), u = x / cap, whose next term is 2^-21 of x.  (The first alone loses the scores
// of large caps: 1 % of the weights at 1e5, all at 1e8.)
__device__ __forceinline__ float capped_far(float x, const DecodeArgs& a) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(fast_exp2(x * a.cap_exp) + 1.f));
  return fmaf(-2.f * a.cap, r, a.cap);
}
__device__ __forceinline__ float capped_near(float x, const DecodeArgs& a) {
  const float u = x * a.inv_cap, u2 = u * u;
  return fmaf(x * u2, fmaf(u2, fmaf(u2, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), x);
}
// The root of 2^(m - top): a sum of weights goes from m to top in two steps, as it may be large where the factor is below fp32's range.
__device__ __forceinline__ float half_step(float m, float top) { return fast_exp2(0.5f * (m - top)); }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// int8 codes become fp16 as 1152 + code (0x6400 | (byte ^ 0x80)) less 1152, exactly.  (Left in the keys, and its multiple of the query row's sum taken off the score,
// the 1152 cost the score seven bits: the weights' sums were off by up to 2e-5, where fp32 has 1e-6.)
constexpr uint32_t kMagic = 0x64646464u, kBias2 = 0x64806480u;

// Four codes of a key row as the two halves of a step's contraction.
template <bool E4M3>
__device__ __forceinline__ void key_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    w ^= 0x80808080u;
    lo = sub2(__byte_perm(w, kMagic, 0x4140), kBias2);
    hi = sub2(__byte_perm(w, kMagic, 0x4342), kBias2);
  }
}
// Bytes 0, 1 (high: 2, 3) of two tokens' words as fp16 pairs (token, next token).
template <bool E4M3>
__device__ __forceinline__ void value_pairs(uint32_t t0, uint32_t t1, bool high, uint32_t& d0, uint32_t& d1) {
  uint32_t x = __byte_perm(t0, t1, high ? 0x7362 : 0x5140);
  if constexpr (E4M3) {
    asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(d0), "=r"(d1) : "r"(x));
  } else {
    x ^= 0x80808080u;
    d0 = sub2(__byte_perm(x, kMagic, 0x4140), kBias2);
    d1 = sub2(__byte_perm(x, kMagic, 0x4342), kBias2);
  }
}

__device__ __forceinline__ int pages_of(const DecodeArgs& a, int b) {
  return min((max(a.lens[b], 0) + kPage - 1) / kPage, a.c.max_pages);
}
__device__ __forceinline__ int len_of(const DecodeArgs& a, int b) { return min(max(a.lens[b], 0), a.c.max_pages * kPage); }

// How the pages are cut.  even: unit u (a warp) takes `per` of all segments' places in order, from u * per on; a segment has kOpening places that stand for what a piece costs apart from its pages, then one for each page.  else: every
// segment of sequence b has ceil(pages / per) parts, and unit u (a CTA) takes one.  first[b]: places (parts) of a KV head and row block before sequence b.
struct Plan {
  int per;
};

// Running sums of f(b) in first[0 .. batch], by the whole block; returns their total.
template <class F>
__device__ __forceinline__ int running_sum(int batch, int* first, int* warp_sums, F f) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int each = (batch + kThreads - 1) / kThreads, b0 = min(batch, (int)threadIdx.x * each), b1 = min(batch, b0 + each);
  int sum = 0;
  for (int b = b0; b < b1; ++b) sum += f(b);
  int x = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  int at = x - sum, total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < w) at += warp_sums[i];
    total += warp_sums[i];
  }
  for (int b = b0; b < b1; ++b) {
    first[b] = at;
    at += f(b);
  }
  if (threadIdx.x == 0) first[batch] = total;
  __syncthreads();
  return total;
}

// The same by each warp for itself, f(b, the running sum before b) once it is known: all warps write the same, and none waits for another.
template <class F, class G>
__device__ __forceinline__ int running_sum_of_warp(int batch, F f, G g) {
  const int lane = threadIdx.x & 31;
  int total = 0;
  for (int b0 = 0; b0 < batch; b0 += 32) {
    const int v = b0 + lane < batch ? f(b0 + lane) : 0;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (b0 + lane < batch) g(b0 + lane, total + x - v);
    total += __shfl_sync(0xffffffffu, x, 31);
  }
  return total;
}

constexpr int kFewSequences = 128;      // up to which a warp is as fast alone as the block with its waits (64: 0.4 and 1.5 us)

__device__ __forceinline__ Plan make_plan(const DecodeArgs& a, int* first, int* lens, int* warp_sums) {
  Plan p = {1};
  const int lanes = a.c.heads * a.blocks, segments = a.batch * lanes, most = a.c.max_pages * kPage;
  const bool few = a.batch <= kFewSequences;
  const auto places = [&](int len) { return len == 0 ? 0 : (len + kPage - 1) / kPage + (a.even ? kOpening : 0); };
  const auto parts = [&](int b) { return ((lens[b] + kPage - 1) / kPage + p.per - 1) / p.per; };
  int units;
  if (few) {
    units = running_sum_of_warp(a.batch, [&](int b) {
      const int len = min(max(a.lens[b], 0), most);
      lens[b] = len;
      return places(len);
    }, [&](int b, int before) { if (a.even) first[b] = before; });
    if (a.even) first[a.batch] = units;
  } else {
    for (int b = threadIdx.x; b < a.batch; b += kThreads) lens[b] = min(max(a.lens[b], 0), most);
    __syncthreads();
    units = running_sum(a.batch, first, warp_sums, [&](int b) { return places(lens[b]); });
  }
  units *= lanes;
  if (a.even) {
    const int warps = a.n_cta * kWarps;
    p.per = max(1, (units + warps - 1) / warps);
  } else {
    // no more parts than CTAs: sum of ceil(pages / per) <= units / per + segments
    p.per = max(kLeastPart, (units + a.n_cta - segments - 1) / (a.n_cta - segments));
    if (few) {
      __syncwarp();
      const int total = running_sum_of_warp(a.batch, parts, [&](int b, int before) { first[b] = before; });
      first[a.batch] = total;
    } else {
      running_sum(a.batch, first, warp_sums + kWarps, parts);
    }
  }
  __syncwarp();
  return p;
}

// What the second launch needs to know of a row: reference and sum of a part, or the logarithm of a whole row's sum for its keys' weights.
__device__ __forceinline__ void leave_sums(const DecodeArgs& a, bool whole, int64_t slot, int64_t head, int row, int r, int row_block, float m, float l) {
  if (!whole) *reinterpret_cast<float2*>(a.part_ml + (slot * row_block + r) * 2) = make_float2(m, l);
  else if (a.lse != nullptr) a.lse[head * a.rows + row] = l == 0.f ? CUDART_INF_F : m + log2f(l);
}

// The last b with first[b] * lanes <= x that is not empty (there is one).
__device__ __forceinline__ int find(const int* first, int batch, int x, int lanes) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] * lanes <= x) lo = mid; else hi = mid;
  }
  return lo;
}

template <int D, int NT>
struct Shape {
  static constexpr int kTile = D == 256 || (D == 128 && NT == 2) ? 1 : 2;      // pages of a warp's step
  static constexpr int kSlots = D == 128 && NT == 1 ? 2 : 3;     // steps whose codes are under way or in use
  static constexpr int kChunks = D / 64;       // 16-byte pieces of a key row that a lane takes
  static constexpr int kSteps = D / 16;        // of the contraction, and tiles of O^T
  static constexpr int kRows = NT * 8;
  static constexpr int kCtas = D == 64 ? (NT == 2 ? 3 : 4) : 2;
  static constexpr int kRing = kSlots * kTile * (2 * kPage * D + 8);      // bytes of a warp
  static constexpr int kMerge = kRows * (D + 4 + 2) * 4;            // what a warp hands over at the end of a shared piece, in the same place
  static constexpr int kWarpBytes = ((kRing > kMerge ? kRing : kMerge) + 127) / 128 * 128;
};

// Where 16-byte piece `chunk` of a row lies in a page's tile of shared memory, so that the eight lanes of a phase meet eight banks' groups: keys are read by rows
// g, g + 1 and pieces 0 to 3, values by rows 0, 2, 4, 6 (+ 1) and two pieces (D = 64: halves of one).
template <int D>
__device__ __forceinline__ int key_at(int row, int chunk) {
  return row * D + ((D >= 128 ? chunk ^ ((row & 1) << 2) : chunk) << 4);
}
template <int D>
__device__ __forceinline__ int value_at(int row, int chunk) {
  if constexpr (D == 64) return (row >> 1) * 128 + ((((row & 1) << 2 | chunk) ^ (row & 6)) << 4);
  if constexpr (D == 128) return row * D + ((chunk ^ (row & 6)) << 4);
  return row * D + ((chunk ^ ((row >> 1 & 1) | (row & 4))) << 4);
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
__device__ __forceinline__ uint2 lds8(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at));
  return r;
}
// Codes are read once: the hint lets what is read again, scores and parts, stay in L2 (a decode with sums 73.5 -> 71.2 us, others 1 to 2 %).
__device__ __forceinline__ void copy16(uint32_t to, const void* from, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "l"(policy) : "memory");
}

template <int D, int NT, bool E4M3>
__global__ void __launch_bounds__(kThreads, Shape<D, NT>::kCtas) decode_kernel(const DecodeArgs a) {
  using S = Shape<D, NT>;
  constexpr int kTile = S::kTile, kSlots = S::kSlots, kChunks = S::kChunks, kSteps = S::kSteps, kRows = S::kRows;
  extern __shared__ __align__(128) int smem[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(smem);               // [kWarps][kWarpBytes]
  int* first = smem + kWarps * S::kWarpBytes / 4;                 // [batch + 1]
  int* lens = first + a.batch + 1;                                // [batch]
  const auto sm_o = [&](int w) { return reinterpret_cast<float*>(ring + w * S::kWarpBytes); };      // [kRows][D + 4]
  const auto sm_ml = [&](int w) { return sm_o(w) + kRows * (D + 4); };                              // [kRows][2]
  __shared__ int warp_sums[2 * kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int lanes = a.c.heads * a.blocks;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Plan plan = make_plan(a, first, lens, warp_sums);
  // even: every warp has a range of its own.  else: the warps of a CTA share its part.
  const int unit = a.even ? blockIdx.x * kWarps + warp : blockIdx.x;
  const int share = a.even ? 1 : kWarps, turn = a.even ? 0 : warp;
  const int total = first[a.batch] * lanes, range0 = a.even ? unit * plan.per : unit;
  const int end = min(total, a.even ? range0 + plan.per : unit + 1);

  // A piece: the pages [p0, p1) of one sequence, KV head and row block.  The warp takes it in steps: pages p0 + (turn + share * i) * kTile + {0 .. kTile - 1}.
  struct Piece {
    int b, h, rb, p0, p1, pages, next, steps;
  };
  const auto locate = [&](int at) {
    Piece x;
    x.b = find(first, a.batch, at, lanes);
    x.pages = (lens[x.b] + kPage - 1) / kPage;
    const int in = at - first[x.b] * lanes;
    if (a.even) {
      const int places = x.pages + kOpening, seg = in / places, before = in - seg * places;
      x.h = a.blocks == 1 ? seg : seg / a.blocks;
      x.rb = seg - x.h * a.blocks;
      x.next = min(end, at + places - before);
      x.p0 = max(0, before - kOpening);
      x.p1 = before + x.next - at - kOpening;      // (<= p0: the range ends before the first page)
    } else {
      const int parts = first[x.b + 1] - first[x.b], i = a.blocks == 1 ? in : in / a.blocks;
      x.rb = in - i * a.blocks;
      x.h = i / parts;
      const int part = i - x.h * parts;
      x.p0 = (int)((int64_t)x.pages * part / parts);
      x.p1 = (int)((int64_t)x.pages * (part + 1) / parts);
      x.next = end;
    }
    x.steps = (max(0, x.p1 - x.p0 + kTile - 1) / kTile - turn + share - 1) / share;
    return x;
  };

  // The ring: slot s has the keys of kTile pages, their values and, behind all slots, their scales.  What fills it runs kSlots steps ahead of what reads it, from one
  // piece into the next.  A lane copies 16 bytes of every 512, and holds the number of one of the next 32 pages.
  constexpr int kAhead = 32 / kTile;
  constexpr int kPageBytes = kPage * D, kCopies = kPageBytes / 512, kLanesRow = D / 16;
  const int64_t page_bytes = (int64_t)a.c.heads * kPageBytes;
  const uint32_t mine_at = smem_u32(ring + warp * S::kWarpBytes), scales_at = mine_at + kSlots * 2 * kTile * kPageBytes;
  Piece f;                                      // the piece that is being copied
  int f_i = 0, f_at = range0, f_id = 0, f_id_next = 0, pg[kTile];
  const int* f_table = nullptr;
  f.steps = 0;
  const auto page_numbers = [&](int i0) {       // of the steps i0 .. i0 + kAhead - 1
    const int p = f.p0 + (turn + share * (i0 + lane / kTile)) * kTile + lane % kTile;
    return p < f.p1 ? f_table[p] : 0;
  };
  const auto adopt = [&](int id) {              // -1: none of the cache's, which is recorded and spoils what sees the page
    if (!page_ok(a.c, id)) {
      atomicOr(a.c.status, kStatusBadPageId);
      id = -1;
    }
    return id;
  };
  const auto open = [&] {                       // (only the last piece of a range can be without pages: it then ends the range)
    f = locate(f_at);
    f_at = f.next;
    f_i = 0;
    if (f.steps <= 0) return;
    f_table = a.c.table + (int64_t)f.b * a.c.width;
    f_id = page_numbers(0);
    if (f.steps > kAhead) f_id_next = page_numbers(kAhead);
    const int64_t q0 = (((int64_t)f.b * a.c.heads + f.h) * a.rows + f.rb * kRows) * D;      // (the rows of a KV head, in lines of 64 elements)
    if (lane < min(kRows, a.rows - f.rb * kRows) * (D / 64))
      asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint16_t*>(a.q) + q0 + lane * 64));
  };
  // Where a lane's pieces of rows go: the places repeat after kKinds copies, 512 bytes each.
  const uint64_t policy = l2_policy_evict_first();
  constexpr int kKinds = D == 256 ? 4 : 2;
  uint32_t key_to[kKinds], value_to[kKinds];
#pragma unroll
  for (int c = 0; c < kKinds; ++c) {
    key_to[c] = mine_at + key_at<D>(c * (32 / kLanesRow) + lane / kLanesRow, lane % kLanesRow);
    value_to[c] = mine_at + kTile * kPageBytes + value_at<D>(c * (32 / kLanesRow) + lane / kLanesRow, lane % kLanesRow);
  }
  const auto copy_page = [&](const uint32_t (&to)[kKinds], int slot, int u, const uint8_t* from) {
#pragma unroll
    for (int c = 0; c < kCopies; ++c) copy16(to[c % kKinds] + slot * (2 * kTile * kPageBytes) + u * kPageBytes + c / kKinds * (kKinds * 512), from + c * 512, policy);
  };
  const auto copy_keys = [&](int slot) {
    if (f_i < f.steps) {
      const int base = f.p0 + (turn + share * f_i) * kTile, j = f_i % kAhead * kTile;
      if (j == 0) f_id = adopt(f_id);
      const int64_t head_at = (int64_t)f.h * kPageBytes + lane * 16;
      const int own = __shfl_sync(0xffffffffu, f_id, j + lane % kTile);
#pragma unroll
      for (int u = 0; u < kTile; ++u) {
        pg[u] = max(0, __shfl_sync(0xffffffffu, f_id, j + u));
        if (base + u < f.p1) copy_page(key_to, slot, u, a.c.k + pg[u] * page_bytes + head_at);
      }
      if (lane < kTile && base + lane < f.p1) {
        const uint32_t to = scales_at + (slot * kTile + lane) * 8;
        if (own >= 0) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(a.c.scale + ((int64_t)own * a.c.heads + f.h) * 2) : "memory");
        else asm volatile("st.shared.v2.f32 [%0], {%1, %1};" ::"r"(to), "f"(CUDART_NAN_F) : "memory");
      }
    }
    cp_async_commit();
  };
  const auto copy_values = [&](int slot) {
    if (f_i < f.steps) {
      const int base = f.p0 + (turn + share * f_i) * kTile;
      const int64_t head_at = (int64_t)f.h * kPageBytes + lane * 16;
#pragma unroll
      for (int u = 0; u < kTile; ++u)
        if (base + u < f.p1) copy_page(value_to, slot, u, a.c.v + pg[u] * page_bytes + head_at);
      ++f_i;
      if (f_i == f.steps) {
        if (f_at < end) open();
      } else if (f_i % kAhead == 0) {
        f_id = f_id_next;
        if (f_i + kAhead < f.steps) f_id_next = page_numbers(f_i + kAhead);
      }
    }
    cp_async_commit();
  };
  // Query rows of a piece as they are, a lane's 16 columns of 64 of row g (and g + 8).
  uint4 raw_q[NT][kChunks][2];
  const auto load_q = [&](const Piece& x) {
    const int r0 = x.rb * kRows, last = min(kRows, a.rows - r0) - 1;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint16_t* q = static_cast<const uint16_t*>(a.q) + (((int64_t)x.b * a.c.heads + x.h) * a.rows + r0 + min(n * 8 + g, last)) * D;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) raw_q[n][c][i] = *reinterpret_cast<const uint4*>(q + (c * 4 + t) * 16 + i * 8);
    }
  };
  Piece x;
  int at = range0;
  if (at < end) {
    open();
    x = f;
    load_q(x);
#pragma unroll 1                                // (a longer program starts later)
    for (int i = 0; i < kSlots; ++i) {
      copy_keys(i);
      copy_values(i);
    }
  }
  if (blockIdx.x == 0) {
    for (int i = tid; i <= a.batch; i += kThreads) a.plan[kPlanHead + i] = first[i];
    if (tid == 0) a.plan[0] = plan.per;
  }
  // Sequences without keys, while the first codes are on their way.
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (lens[b] != 0) continue;
    const int64_t n = (int64_t)a.c.heads * a.rows * D;
    uint16_t* o = static_cast<uint16_t*>(a.out) + b * n;
    for (int64_t i = tid; i < n; i += kThreads) o[i] = 0;
  }
  int at_slot = 0;
  while (at < end) {
    const int b = x.b, h = x.h, rb = x.rb, p0 = x.p0, p1 = x.p1, len = lens[b];
    const int64_t slot = a.even ? 2 * unit + (at == range0 ? 0 : 1) : unit;
    at = x.next;
    if (a.even && p1 <= p0) break;
    const bool whole = p0 == 0 && p1 == x.pages;
    const int r0 = rb * kRows, rows = min(kRows, a.rows - r0);
    const int64_t head = (int64_t)b * a.c.heads + h;
    // ---- query rows as the second operand, fp16; bf16 rows are brought into its range by a power of two
    uint32_t qf[NT][kSteps][2];
    float factor[NT][2];                        // of the lane's columns 2t and 2t + 1
    int limit[NT][2];                           // keys that they see
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float up = 1.f;
      uint32_t raw[kSteps][2];
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          raw[c * 4 + i * 2][0] = raw_q[n][c][i].x; raw[c * 4 + i * 2][1] = raw_q[n][c][i].y;
          raw[c * 4 + i * 2 + 1][0] = raw_q[n][c][i].z; raw[c * 4 + i * 2 + 1][1] = raw_q[n][c][i].w;
        }
      if (a.bf16) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) most = __vmaxu2(most, __vmaxu2(raw[i][0] & 0x7fff7fffu, raw[i][1] & 0x7fff7fffu));
        most = max(most & 0xffffu, most >> 16);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // The largest magnitude, of exponent e, goes to between 2^14 and 2^15: elements down to 2^-30 of it keep all their bits, smaller ones are off by at
        // most 2^-39 of it.
        const int e = min(max((int)(most >> 7) - 127, -112), 127);
        const float down = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        up = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            raw[i][j] = pack_half2(__uint_as_float(raw[i][j] << 16) * down, __uint_as_float(raw[i][j] & 0xffff0000u) * down);
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        qf[n][i][0] = raw[i][0];
        qf[n][i][1] = raw[i][1];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = n * 8 + 2 * t + c;
        factor[n][c] = a.scale * __shfl_sync(0xffffffffu, up, (2 * t + c) * 4);
        limit[n][c] = col < rows ? len - a.tokens + 1 + (r0 + col) % a.tokens : 0;
      }
    }
    const int free_keys = len - a.tokens + 1;    // these every row sees

    float o[NT][kSteps][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][j][i] = 0.f;
      m[n][0] = m[n][1] = -CUDART_INF_F;
      l[n][0] = l[n][1] = 0.f;
    }

    int spoiled = INT_MAX;                      // first key of the first page whose V scale is not finite
    for (int i = 0; i < x.steps; ++i) {
      const int base = p0 + (turn + share * i) * kTile;
      cp_async_wait<2 * kSlots - 1>();
      __syncwarp();
      float ks[kTile], vs[kTile];
#pragma unroll
      for (int u = 0; u < kTile; ++u) {
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(ks[u]), "=f"(vs[u]) : "r"(scales_at + (at_slot * kTile + u) * 8));
        if (!(fabsf(ks[u]) <= 3.4028235e38f)) ks[u] = CUDART_NAN_F;      // a scale that is not finite spoils what sees the page, whatever the codes
        if (base + u >= p1) vs[u] = 0.f;
        // So does V's, but 0 times it would also spoil what does not see the page: the page adds nothing, and the rows that see it are marked at the end.
        if (!(fabsf(vs[u]) <= 3.4028235e38f)) {
          spoiled = min(spoiled, (base + u) * kPage);
          vs[u] = 0.f;
        }
      }
      // ---- S^T = K Q^T
      float s[kTile][NT][4];
#pragma unroll
      for (int u = 0; u < kTile; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
      const uint32_t keys = mine_at + at_slot * 2 * kTile * kPageBytes, vals = keys + kTile * kPageBytes;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int u = 0; u < kTile; ++u) {
          const uint4 x0 = lds16(keys + u * kPageBytes + key_at<D>(g, c * 4 + t)), x1 = lds16(keys + u * kPageBytes + key_at<D>(g + 8, c * 4 + t));
          const uint32_t k0[4] = {x0.x, x0.y, x0.z, x0.w}, k1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t f[4];
            key_pairs<E4M3>(k0[w], f[0], f[2]);
            key_pairs<E4M3>(k1[w], f[1], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16_16816(s[u][n], f, qf[n][c * 4 + w][0], qf[n][c * 4 + w][1]);
          }
        }
      __syncwarp();
      copy_keys(at_slot);
      // ---- scores in base 2
      const int key0 = base * kPage;
#pragma unroll
      for (int u = 0; u < kTile; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][n][e] *= factor[n][e & 1] * ks[u];
      if (a.capped) {
        bool far = false;
#pragma unroll
        for (int u = 0; u < kTile; ++u)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) far |= fabsf(s[u][n][e]) >= a.near;
        if (__any_sync(0xffffffffu, far)) {
#pragma unroll
          for (int u = 0; u < kTile; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float x = s[u][n][e], y = capped_near(x, a), z = capped_far(x, a);
                s[u][n][e] = fabsf(x) >= a.near ? z : y;
              }
        } else {
#pragma unroll
          for (int u = 0; u < kTile; ++u)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[u][n][e] = capped_near(s[u][n][e], a);
        }
      }
      const bool masked = key0 + kTile * kPage > free_keys || base + kTile > p1;
      if (masked) {
#pragma unroll
        for (int u = 0; u < kTile; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + u * kPage + g + (e >> 1) * 8;
#pragma unroll
            for (int n = 0; n < NT; ++n)
              if (key >= limit[n][e & 1] || base + u >= p1) s[u][n][e] = -CUDART_INF_F;
          }
      }
      if (a.scores != nullptr) {
        const int cols = a.score_cols;
        float* to = a.scores + ((head * a.blocks + rb) * a.c.max_pages + base) * kPage * cols;
#pragma unroll
        for (int u = 0; u < kTile; ++u)
          if (base + u < p1)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int half = 0; half < 2; ++half)
                if (n * 8 + 2 * t < cols)
                  *reinterpret_cast<float2*>(to + (u * kPage + g + half * 8) * cols + n * 8 + 2 * t) = make_float2(s[u][n][half * 2], s[u][n][half * 2 + 1]);
      }
      // ---- running maximum of s + log2 vs, less 25
      uint32_t pf[kTile][NT][2];
      bool moved = false;
      float top[NT][2], lv[kTile];
#pragma unroll
      for (int u = 0; u < kTile; ++u) {
        lv[u] = fmaxf(log2_of(vs[u]), kLeastLog) - kTop;
        vs[u] *= 1.f / kUnit;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float y = -CUDART_INF_F;
#pragma unroll
          for (int u = 0; u < kTile; ++u) y = fmaxf(y, fmaxf(s[u][n][c], s[u][n][c + 2]) + lv[u]);
          top[n][c] = y;
        }
#pragma unroll
      for (int d = 4; d < 32; d *= 2)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) top[n][c] = fmaxf(top[n][c], __shfl_xor_sync(0xffffffffu, top[n][c], d));
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) moved |= top[n][c] > m[n][c];
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float shrink[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            top[n][c] = fmaxf(m[n][c], top[n][c]);
            const float half = top[n][c] == -CUDART_INF_F ? 1.f : half_step(m[n][c], top[n][c]);
            m[n][c] = top[n][c];
            l[n][c] = l[n][c] * half * half;
            shrink[c] = half * half;
          }
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][k][e] *= shrink[e & 1];
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float ref[2] = {m[n][0] == -CUDART_INF_F ? 0.f : m[n][0], m[n][1] == -CUDART_INF_F ? 0.f : m[n][1]};
#pragma unroll
        for (int u = 0; u < kTile; ++u) {
          float p[4];                             // (at most 2^100, and times vs at most 2^15)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = fast_exp2(s[u][n][e] - ref[e & 1]);
            l[n][e & 1] += p[e];
          }
          pf[u][n][0] = transpose8x8(pack_half2(p[0] * vs[u], p[1] * vs[u]));
          pf[u][n][1] = transpose8x8(pack_half2(p[2] * vs[u], p[3] * vs[u]));
        }
      }
      // ---- O^T += V^T P^T
      cp_async_wait<2 * kSlots - 1>();
      __syncwarp();
#pragma unroll
      for (int u = 0; u < kTile; ++u) {
        uint32_t vr[4][D / 32];                 // rows 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 2 * t + (r & 1) + (r >> 1) * 8;
          if constexpr (D == 64) {
            const uint2 x = lds8(vals + u * kPageBytes + value_at<D>(row, g >> 1) + (g & 1) * 8);
            vr[r][0] = x.x; vr[r][1] = x.y;
          } else {
#pragma unroll
            for (int c = 0; c < D / 128; ++c) {
              const uint4 x = lds16(vals + u * kPageBytes + value_at<D>(row, g * (D / 128) + c));
              vr[r][c * 4] = x.x; vr[r][c * 4 + 1] = x.y; vr[r][c * 4 + 2] = x.z; vr[r][c * 4 + 3] = x.w;
            }
          }
          if (E4M3 && masked && (key0 + u * kPage + row >= len || base + u >= p1)) {      // codes behind the last key may stand for NaN
#pragma unroll
            for (int w = 0; w < D / 32; ++w) vr[r][w] = 0;
          }
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w)
#pragma unroll
          for (int high = 0; high < 2; ++high) {
            uint32_t f[4];
            value_pairs<E4M3>(vr[0][w], vr[1][w], high, f[0], f[1]);
            value_pairs<E4M3>(vr[2][w], vr[3][w], high, f[2], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16_16816(o[n][w * 2 + high], f, pf[u][n][0], pf[u][n][1]);
          }
      }
      __syncwarp();
      copy_values(at_slot);
      at_slot = at_slot + 1 == kSlots ? 0 : at_slot + 1;
    }

    if (spoiled != INT_MAX) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (spoiled < limit[n][e & 1]) o[n][k][e] = CUDART_NAN_F;
    }
    Piece next;
    if (at < end) {                             // the next piece's rows come while this one's go out
      next = locate(at);
      load_q(next);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 4);
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 8);
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 16);
      }
    if (a.even) {                            // a warp's own piece: a lane has D / 8 columns of each of its rows
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = n * 8 + 2 * t + c;
          if (r >= rows) continue;
          if (whole) {
            const float inv = l[n][c] == 0.f ? 0.f : kUnit / l[n][c];
            uint16_t* to = static_cast<uint16_t*>(a.out) + (head * a.rows + r0 + r) * D + g * (D / 8);
#pragma unroll
            for (int k = 0; k < kSteps; k += 4) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = pack_out16x2(o[n][k + e][c] * inv, o[n][k + e][c + 2] * inv, a.bf16);
              *reinterpret_cast<uint4*>(to + 2 * k) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            float* to = a.part + (slot * kRows + r) * D + g * (D / 8);
#pragma unroll
            for (int k = 0; k < kSteps; k += 2)
              *reinterpret_cast<float4*>(to + 2 * k) = make_float4(o[n][k][c], o[n][k][c + 2], o[n][k + 1][c], o[n][k + 1][c + 2]);
          }
          if (g == 0) leave_sums(a, whole, slot, head, r0 + r, r, kRows, m[n][c], l[n][c]);
        }
      x = next;
      continue;
    }
    // ---- the warps' parts together, where their rings were
    cp_async_wait<0>();
    __syncwarp();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = n * 8 + 2 * t + c;
        if (g == 0) {
          sm_ml(warp)[r * 2] = m[n][c];
          sm_ml(warp)[r * 2 + 1] = l[n][c];
        }
        float* to = sm_o(warp) + r * (D + 4) + g * (D / 8);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) *reinterpret_cast<float2*>(to + 2 * k) = make_float2(o[n][k][c], o[n][k][c + 2]);
      }
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_ml(w)[r * 2]);
      const float ref = top == -CUDART_INF_F ? 0.f : top;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float half = half_step(sm_ml(w)[r * 2], ref), f = half * half;
        sum += sm_ml(w)[r * 2 + 1] * half * half;
        const float4 x = *reinterpret_cast<const float4*>(sm_o(w) + r * (D + 4) + d);
        acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : kUnit / sum;
        uint2 packed = make_uint2(pack_out16x2(acc.x * inv, acc.y * inv, a.bf16), pack_out16x2(acc.z * inv, acc.w * inv, a.bf16));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (head * a.rows + r0 + r) * D + d) = packed;
      } else {
        *reinterpret_cast<float4*>(a.part + (slot * kRows + r) * D + d) = acc;
      }
      if (d == 0) leave_sums(a, whole, slot, head, r0 + r, r, kRows, top, sum);
    }
    __syncthreads();
  }
}

// The parts of segment (head, row block rb) of sequence b: how many, and part i's slot.
struct Parts {
  int n;
  int64_t slot0, step;
  bool even;
  __device__ __forceinline__ int64_t slot(int i) const { return even && i > 0 ? (slot0 & ~(int64_t)1) + i * step : slot0 + i * step; }
};
__device__ __forceinline__ Parts parts_of(const DecodeArgs& a, int b, int h, int rb) {
  Parts x;
  const int pages = pages_of(a, b), lanes = a.c.heads * a.blocks, first = a.plan[kPlanHead + b];
  x.even = a.even;
  if (a.even) {
    const int per = a.plan[0], x0 = first * lanes + (h * a.blocks + rb) * (pages + kOpening), u0 = (x0 + kOpening) / per;
    x.n = pages == 0 ? 0 : (x0 + kOpening + pages - 1) / per - u0 + 1;
    // the first part is its warp's second piece unless the warp's range begins in the segment
    x.slot0 = 2 * (int64_t)u0 + (u0 * per < x0 ? 1 : 0);
    x.step = 2;
  } else {
    x.n = a.plan[kPlanHead + b + 1] - first;
    x.slot0 = (int64_t)first * lanes + (int64_t)h * x.n * a.blocks + rb;
    x.step = a.blocks;
  }
  return x;
}

// The parts of a row together: a warp for each query row of a KV head after an even cut (a few parts each), a CTA where few segments were cut for all
// CTAs.  Rows of segments that were not cut have nothing to do.
template <int D, int W>
__global__ void __launch_bounds__(kThreads) merge_kernel(const DecodeArgs a, int row_block) {
  const int tid = threadIdx.x, lane = tid & 31, warp = W == 1 ? 0 : tid >> 5;
  const int64_t all = (int64_t)blockIdx.x * (kWarps / W) + (W == 1 ? tid >> 5 : 0);
  const int64_t head = all / a.rows;
  if (head >= (int64_t)a.batch * a.c.heads) return;
  const int row = (int)(all % a.rows), rb = row / row_block, r = row % row_block;
  const int b = (int)(head / a.c.heads), h = (int)(head % a.c.heads);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Parts x = parts_of(a, b, h, rb);
  if (x.n <= 1) return;
  __shared__ float sm[W][2];
  __shared__ float4 sm_o[W][D / 4];
  float top = -CUDART_INF_F;
  for (int i = W == 1 ? lane : tid; i < x.n; i += 32 * W) top = fmaxf(top, a.part_ml[(x.slot(i) * row_block + r) * 2]);
#pragma unroll
  for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (W > 1) {
    if (lane == 0) sm[warp][0] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, sm[w][0]);
  }
  const float ref = top == -CUDART_INF_F ? 0.f : top;
  constexpr int kEach = (D / 4 + 31) / 32;
  float4 acc[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int i = warp; i < x.n; i += W) {
    const int64_t slot = x.slot(i) * row_block + r;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + slot * 2);
    const float half = half_step(ml.x, ref), f = half * half;
    sum += ml.y * half * half;
    const float4* p = reinterpret_cast<const float4*>(a.part + slot * D);
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (lane + e * 32 < D / 4) {
        const float4 v = p[lane + e * 32];
        acc[e].x += v.x * f; acc[e].y += v.y * f; acc[e].z += v.z * f; acc[e].w += v.w * f;
      }
  }
  if (W > 1) {
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (lane + e * 32 < D / 4) sm_o[warp][lane + e * 32] = acc[e];
    if (lane == 0) sm[warp][1] = sum;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (lane + e * 32 < D / 4) {
          const float4 v = sm_o[w][lane + e * 32];
          acc[e].x += v.x; acc[e].y += v.y; acc[e].z += v.z; acc[e].w += v.w;
        }
      sum += sm[w][1];
    }
  }
  const float inv = sum == 0.f ? 0.f : kUnit / sum;
  uint16_t* out = static_cast<uint16_t*>(a.out) + (head * a.rows + row) * D;
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (lane + e * 32 < D / 4)
      *reinterpret_cast<uint2*>(out + (lane + e * 32) * 4) =
          make_uint2(pack_out16x2(acc[e].x * inv, acc[e].y * inv, a.bf16), pack_out16x2(acc[e].z * inv, acc[e].w * inv, a.bf16));
  if (a.lse != nullptr && lane == 0) a.lse[head * a.rows + row] = sum == 0.f ? CUDART_INF_F : ref + log2f(sum);
}

// mass_j += sum over rows of 2^(score - log of the row's sum): a CTA for each KV head and 1024 keys, four keys a thread, a row's four scores in one load.
constexpr int kEachKey = 4, kMassThreads = 256, kMassKeys = kEachKey * kMassThreads;
__global__ void __launch_bounds__(kMassThreads) mass_kernel(const DecodeArgs a, int row_block, int chunks) {
  const int64_t head = blockIdx.x / chunks;
  const int b = (int)(head / a.c.heads), h = (int)(head % a.c.heads), j0 = blockIdx.x % chunks * kMassKeys + threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int len = min(len_of(a, b), a.mass_cap);
  if (j0 - (int)threadIdx.x >= len) return;
  const int at = a.mass_index != nullptr ? a.mass_index[b] : b;
  if (at < 0 || at >= a.mass_rows) {
    if (threadIdx.x == 0) atomicOr(a.c.status, kStatusBadPageId);
    return;
  }
  float* mass = a.mass + ((int64_t)at * a.c.heads + h) * a.mass_cap;
  float had[kEachKey], got[kEachKey];
#pragma unroll
  for (int k = 0; k < kEachKey; ++k) {
    had[k] = j0 + k * kMassThreads < len ? mass[j0 + k * kMassThreads] : 0.f;
    got[k] = 0.f;
  }
  for (int rb = 0; rb < a.blocks; ++rb) {
    const float* s = a.scores + ((head * a.blocks + rb) * a.c.max_pages * kPage + j0) * a.score_cols;
    const float* lse = a.lse + head * a.rows + rb * row_block;
    const int rows = min(row_block, a.rows - rb * row_block);
    if (a.score_cols % 4 == 0) {
      for (int r = 0; r < rows; r += 4) {
        float4 v[kEachKey];
#pragma unroll
        for (int k = 0; k < kEachKey; ++k)
          if (j0 + k * kMassThreads < len) v[k] = __ldcs(reinterpret_cast<const float4*>(s + (int64_t)k * kMassThreads * a.score_cols + r));
        float n[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) n[e] = r + e < rows ? lse[r + e] : CUDART_INF_F;
#pragma unroll
        for (int k = 0; k < kEachKey; ++k)
          if (j0 + k * kMassThreads < len) {
            const float w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (r + e < rows) got[k] += fast_exp2(w[e] - n[e]);
          }
      }
    } else {
      for (int r = 0; r < rows; ++r)
#pragma unroll
        for (int k = 0; k < kEachKey; ++k)
          if (j0 + k * kMassThreads < len) got[k] += fast_exp2(s[(int64_t)k * kMassThreads * a.score_cols + r] - lse[r]);
    }
  }
#pragma unroll
  for (int k = 0; k < kEachKey; ++k)
    if (j0 + k * kMassThreads < len) mass[j0 + k * kMassThreads] = had[k] + got[k];
}

// Behind the kernel before it in the stream: its blocks come as soon as there is room, and wait for that kernel's end before they read.
template <class... Params, class... Args>
cudaError_t launch_behind(void (*kernel)(Params...), int64_t grid, int threads, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int D, int NT, bool E4M3>
cudaError_t launch_decode_as(const DecodeArgs& a, cudaStream_t s) {
  constexpr int kRows = NT * 8;
  const size_t smem = (size_t)kWarps * Shape<D, NT>::kWarpBytes + ((size_t)2 * a.batch + 1) * 4;
  static SharedMemoryLimit limit;
  cudaError_t e = limit.raise(reinterpret_cast<const void*>(decode_kernel<D, NT, E4M3>), (int)smem);
  if (e != cudaSuccess) return e;
  if ((e = launch_behind(decode_kernel<D, NT, E4M3>, a.n_cta, kThreads, smem, s, a)) != cudaSuccess) return e;
  const int64_t rows = (int64_t)a.batch * a.c.heads * a.rows;
  if (a.even) e = launch_behind(merge_kernel<D, 1>, (rows + kWarps - 1) / kWarps, kThreads, 0, s, a, kRows);
  else if (a.c.max_pages > kLeastPart) e = launch_behind(merge_kernel<D, kWarps>, rows, kThreads, 0, s, a, kRows);      // (else no segment is cut)
  if (e != cudaSuccess || a.mass == nullptr) return e;
  const int chunks = (int)(((int64_t)a.c.max_pages * kPage + kMassKeys - 1) / kMassKeys);
  return launch_behind(mass_kernel, (int64_t)chunks * a.batch * a.c.heads, kMassThreads, 0, s, a, kRows, chunks);
}

template <int D, int NT>
cudaError_t launch_decode_codes(const DecodeArgs& a, bool e4m3, cudaStream_t s) {
  return e4m3 ? launch_decode_as<D, NT, true>(a, s) : launch_decode_as<D, NT, false>(a, s);
}

template <int D, int NT>
constexpr int ctas_of() { return Shape<D, NT>::kCtas; }

}  // namespace

// Query rows of a block: 8, or 16 for more of up to 128 columns.  What is in a block reads every code once, another block reads it again (mostly from L2).
// Blocks of 32 for width 64 were slower, 39 to 48 us against 33 for 20 rows each of 16 sequences of up to 4096 tokens: their registers leave too little
// under way at once.
static int tiles_of(int dim, int rows) { return dim == 256 || rows <= 8 ? 1 : 2; }

DecodeShape decode_shape(int dim, int rows, int sms) {
  DecodeShape d;
  const int tiles = tiles_of(dim, rows);
  d.row_block = tiles * 8;
  d.blocks = (rows + d.row_block - 1) / d.row_block;
  const int ctas = dim == 256 ? ctas_of<256, 1>() : dim == 128 ? (tiles == 2 ? ctas_of<128, 2>() : ctas_of<128, 1>())
                 : tiles == 2 ? ctas_of<64, 2>() : ctas_of<64, 1>();
  d.n_cta = sms * ctas;
  d.slots = 2 * d.n_cta * kWarps;
  d.score_cols = rows >= d.row_block ? d.row_block : (rows + 1) & ~1;
  return d;
}

cudaError_t launch_decode(DecodeArgs a, bool e4m3, cudaStream_t s) {
  a.even = 2 * (int64_t)a.batch * a.c.heads * a.blocks > a.n_cta;
  const int tiles = tiles_of(a.c.dim, a.rows);
  switch (a.c.dim) {
    case 64: return tiles == 2 ? launch_decode_codes<64, 2>(a, e4m3, s) : launch_decode_codes<64, 1>(a, e4m3, s);
    case 128: return tiles == 2 ? launch_decode_codes<128, 2>(a, e4m3, s) : launch_decode_codes<128, 1>(a, e4m3, s);
    default: return launch_decode_codes<256, 1>(a, e4m3, s);
  }
}

}  // namespace kv8
}  // namespace fa
