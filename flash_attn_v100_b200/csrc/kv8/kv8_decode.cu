// Attention of each sequence's newest tokens on the paged 8-bit cache.
//
//   s_rj = f(q_r . k_j ks_j),  p_rj = 2^(s_rj - m_r),  o_r = sum_j p_rj vs_j v_j / sum_j p_rj
//
// with one scale ks, vs for the 16 tokens of a page and head.  Bound by HBM (2 D bytes a token and KV head against 4 D flop a row), so the
// rows of a KV head (its query heads times the new tokens) share every code that is read, in blocks of 8 or 16.  Keys, and then output dimensions,
// are the 16 rows of mma.sync.m16n8k16 and the query rows its 8 columns: S^T = K Q^T, O^T = V^T P^T.
// Codes go from global memory straight to registers in the operands' layout: a lane's 16 bytes of a key row are four steps of the (permuted)
// contraction, and its 16 bytes of four tokens' values the rows of eight tiles of O^T.  They become fp16 there, exactly.
// K's scale multiplies the finished scores.  V's scale goes into the exponent: with m the running maximum of s + log2 vs the weight that meets the
// codes is 2^(s + log2 vs - m) <= 1, so fp16 keeps 11 bits of the products that matter whatever the pages' scales are; the sum of weights
// takes 2^(s - m) in fp32.
// The pages of all sequences and heads are cut evenly over the CTAs; where there are fewer segments than half the CTAs each is cut into equal
// parts, at least kLeastPart pages.  Parts of a cut segment go through global memory to a second launch.
#include <math_constants.h>

#include "kv8.cuh"

namespace fa {
namespace kv8 {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kLeastPart = 8;

__device__ __forceinline__ float log2_of(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// int8 codes are taken as fp16 1152 + code (0x6400 | (byte ^ 0x80)); for keys the 1152 stays in the product and its multiple of the query row's sum is
// taken off the score.
constexpr uint32_t kMagic = 0x64646464u, kBias2 = 0x64806480u;

// Four codes of a key row as the two halves of a step's contraction.
template <bool E4M3>
__device__ __forceinline__ void key_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    w ^= 0x80808080u;
    lo = __byte_perm(w, kMagic, 0x4140);
    hi = __byte_perm(w, kMagic, 0x4342);
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

// How the pages are cut.  even: CTA c takes the pages [c * per, (c + 1) * per) of all segments in order.  else: every segment of sequence b has
// ceil(pages / per) parts, and CTA c takes one.  first[b]: pages (parts) of a KV head and row block before sequence b.
struct Plan {
  bool even;
  int per;
  const int* first;
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
  __syncthreads();
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

__device__ __forceinline__ Plan make_plan(const DecodeArgs& a, int* first, int* warp_sums) {
  Plan p;
  const int lanes = a.c.heads * a.blocks, segments = a.batch * lanes;
  const int64_t units = (int64_t)running_sum(a.batch, first, warp_sums, [&](int b) { return pages_of(a, b); }) * lanes;
  p.even = 2 * segments > a.n_cta;
  p.first = first;
  if (p.even) {
    p.per = max(1, (int)((units + a.n_cta - 1) / a.n_cta));
  } else {
    // no more parts than CTAs: sum of ceil(pages / per) <= units / per + segments
    p.per = max(kLeastPart, (int)((units + a.n_cta - segments - 1) / (a.n_cta - segments)));
    running_sum(a.batch, first, warp_sums, [&](int b) { return (pages_of(a, b) + p.per - 1) / p.per; });
  }
  return p;
}

// The last b with first[b] * lanes <= x that is not empty (there is one).
__device__ __forceinline__ int find(const int* first, int batch, int64_t x, int lanes) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if ((int64_t)first[mid] * lanes <= x) lo = mid; else hi = mid;
  }
  return lo;
}

template <int D, int NT, bool E4M3>
struct Shape {
  static constexpr int kTile = D == 256 || (D == 128 && NT == 2) ? 1 : 2;      // pages of a warp's step
  static constexpr int kChunks = D / 64;       // 16-byte pieces of a key row that a lane takes
  static constexpr int kSteps = D / 16;        // of the contraction, and tiles of O^T
  static constexpr int kRows = NT * 8;
  static constexpr int kCtas = D == 256 ? 2 : NT == 2 ? (D == 64 ? 3 : 2) : (D == 64 ? 4 : 3);
};

template <int D, int NT, bool E4M3>
__global__ void __launch_bounds__(kThreads, Shape<D, NT, E4M3>::kCtas) decode_kernel(const DecodeArgs a) {
  using S = Shape<D, NT, E4M3>;
  constexpr int kTile = S::kTile, kChunks = S::kChunks, kSteps = S::kSteps, kRows = S::kRows;
  extern __shared__ int smem[];
  int* first = smem;                                              // [batch + 1]
  float* sm_o = reinterpret_cast<float*>(smem + ((a.batch + 1 + 3) & ~3));      // [kWarps][kRows][D + 4]
  float* sm_ml = sm_o + kWarps * kRows * (D + 4);                 // [kWarps][kRows][2]
  __shared__ int warp_sums[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int lanes = a.c.heads * a.blocks;
  const Plan plan = make_plan(a, first, warp_sums);
  if (blockIdx.x == 0) {
    for (int i = tid; i <= a.batch; i += kThreads) a.plan[kPlanHead + i] = first[i];
    if (tid == 0) {
      a.plan[0] = plan.even;
      a.plan[1] = plan.per;
    }
  }
  // Sequences without keys.
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (pages_of(a, b) != 0) continue;
    const int64_t n = (int64_t)a.c.heads * a.rows * D;
    uint16_t* o = static_cast<uint16_t*>(a.out) + b * n;
    for (int64_t i = tid; i < n; i += kThreads) o[i] = 0;
  }
  int64_t at = plan.even ? (int64_t)blockIdx.x * plan.per : blockIdx.x;
  int64_t end = (int64_t)first[a.batch] * lanes;
  end = plan.even ? min(end, at + plan.per) : min(end, at + 1);
  const int64_t range0 = at;
  while (at < end) {
    // ---- the piece: pages [p0, p1) of sequence b, KV head h, rows from r0 on
    const int b = find(first, a.batch, at, lanes);
    const int pages = pages_of(a, b), parts = first[b + 1] - first[b];
    const int64_t in = at - (int64_t)first[b] * lanes;
    int h, rb, p0, p1;
    int64_t slot;
    if (plan.even) {
      const int seg = (int)(in / pages);
      h = seg / a.blocks;
      rb = seg % a.blocks;
      p0 = (int)(in % pages);
      p1 = (int)min((int64_t)pages, p0 + (end - at));
      slot = 2 * (int64_t)blockIdx.x + (at == range0 ? 0 : 1);
      at += p1 - p0;
    } else {
      rb = (int)(in % a.blocks);
      h = (int)(in / a.blocks / parts);
      const int part = (int)(in / a.blocks % parts);
      p0 = (int)((int64_t)pages * part / parts);
      p1 = (int)((int64_t)pages * (part + 1) / parts);
      slot = blockIdx.x;
      at = end;
    }
    const bool whole = p0 == 0 && p1 == pages;
    const int len = len_of(a, b), r0 = rb * kRows, rows = min(kRows, a.rows - r0);
    const int64_t head = (int64_t)b * a.c.heads + h;
    // ---- query rows as the second operand, fp16; bf16 rows are brought into its range by a power of two
    uint32_t qf[NT][kSteps][2];
    float factor[NT][2], offset[NT][2];         // of the lane's columns 2t and 2t + 1
    int limit[NT][2];                           // keys that they see
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = n * 8 + g;
      const uint16_t* q = static_cast<const uint16_t*>(a.q) + (head * a.rows + r0 + min(r, rows - 1)) * D;
      float sum = 0.f, up = 1.f;
      uint32_t raw[kSteps][2];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const uint4 x0 = *reinterpret_cast<const uint4*>(q + (c * 4 + t) * 16), x1 = *reinterpret_cast<const uint4*>(q + (c * 4 + t) * 16 + 8);
        const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[c * 4 + i / 2][i & 1] = w[i];
      }
      if (a.bf16) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) most = __vmaxu2(most, __vmaxu2(raw[i][0] & 0x7fff7fffu, raw[i][1] & 0x7fff7fffu));
        most = max(most & 0xffffu, most >> 16);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = min(max((int)(most >> 7) - 127, -126), 126);      // the largest magnitude's exponent
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            raw[i][j] = pack_half2(__uint_as_float(raw[i][j] << 16) * down, __uint_as_float(raw[i][j] & 0xffff0000u) * down);
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          qf[n][i][j] = raw[i][j];
          if constexpr (!E4M3) {
            const float2 f = __half22float2(*reinterpret_cast<__half2*>(&raw[i][j]));
            sum += f.x + f.y;
          }
        }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = n * 8 + 2 * t + c;
        offset[n][c] = E4M3 ? 0.f : -1152.f * __shfl_sync(0xffffffffu, sum, (2 * t + c) * 4);
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

    // ---- the warp's steps: pages p0 + (warp + kWarps * i) * kTile + {0 .. kTile - 1}
    const int steps = (p1 - p0 + kTile - 1) / kTile;
    const int mine = (steps - warp + kWarps - 1) / kWarps;      // <= 0: none
    constexpr int kAhead = 32 / kTile;                          // steps whose pages a warp looks up at once, a lane each
    int id_next = 0, id = 0;
    float2 sc_next = make_float2(0.f, 0.f), sc = sc_next;
    const auto look_up = [&](int i0) {                          // pages of the steps i0 .. i0 + kAhead - 1
      const int p = p0 + (warp + kWarps * (i0 + lane / kTile)) * kTile + lane % kTile;
      id_next = 0;
      sc_next = make_float2(0.f, 0.f);
      if (p < p1) {
        id_next = a.c.table[(int64_t)b * a.c.width + p];
        const bool fine = page_ok(a.c, id_next);
        if (!fine) {
          atomicOr(a.c.status, kStatusBadPageId);
          id_next = 0;
        }
        sc_next = *reinterpret_cast<const float2*>(a.c.scale + ((int64_t)id_next * a.c.heads + h) * 2);
        // a scale that is not finite spoils what sees the page, whatever the codes
        if (!fine || !(fabsf(sc_next.x) <= 3.4028235e38f)) sc_next.x = CUDART_NAN_F;
        sc_next.y = log2_of(sc_next.y);
      }
    };
    const int64_t page_bytes = (int64_t)a.c.heads * kPage * D;
    const uint8_t* kbase = a.c.k + (int64_t)h * kPage * D + g * D + t * 16;
    const uint8_t* vbase = a.c.v + (int64_t)h * kPage * D + 2 * t * D + g * (D / 8);
    uint32_t kr[kTile][2][kChunks][4];          // key rows g and g + 8
    uint32_t vr[kTile][4][D / 32];              // value rows 2t, 2t + 1, 2t + 8, 2t + 9
    const auto load_keys = [&](const int (&pg)[kTile]) {
#pragma unroll
      for (int u = 0; u < kTile; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const uint4 x = load_stream16(kbase + pg[u] * page_bytes + half * 8 * D + c * 64);
            kr[u][half][c][0] = x.x; kr[u][half][c][1] = x.y; kr[u][half][c][2] = x.z; kr[u][half][c][3] = x.w;
          }
    };
    const auto load_values = [&](const int (&pg)[kTile]) {
#pragma unroll
      for (int u = 0; u < kTile; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint8_t* p = vbase + pg[u] * page_bytes + ((r & 1) + (r >> 1) * 8) * D;
          if constexpr (D == 64) {
            const uint2 x = load_stream8(p);
            vr[u][r][0] = x.x; vr[u][r][1] = x.y;
          } else {
#pragma unroll
            for (int c = 0; c < D / 128; ++c) {
              const uint4 x = load_stream16(p + c * 16);
              vr[u][r][c * 4] = x.x; vr[u][r][c * 4 + 1] = x.y; vr[u][r][c * 4 + 2] = x.z; vr[u][r][c * 4 + 3] = x.w;
            }
          }
        }
    };
    int pg[kTile];                              // pages of the step whose loads come next
    if (mine > 0) {
      look_up(0);
      id = id_next;
      sc = sc_next;
      if (mine > kAhead) look_up(kAhead);
#pragma unroll
      for (int u = 0; u < kTile; ++u) pg[u] = __shfl_sync(0xffffffffu, id, u);
      load_keys(pg);
      load_values(pg);
    }
    for (int i = 0; i < mine; ++i) {
      const int base = p0 + (warp + kWarps * i) * kTile, j = i % kAhead;
      float ks[kTile], lv[kTile];
#pragma unroll
      for (int u = 0; u < kTile; ++u) {
        ks[u] = __shfl_sync(0xffffffffu, sc.x, j * kTile + u);
        lv[u] = __shfl_sync(0xffffffffu, sc.y, j * kTile + u);
      }
      // ---- S^T = K Q^T
      float s[kTile][NT][4];
#pragma unroll
      for (int u = 0; u < kTile; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int u = 0; u < kTile; ++u) {
            uint32_t f[4];
            key_pairs<E4M3>(kr[u][0][c][w], f[0], f[2]);
            key_pairs<E4M3>(kr[u][1][c][w], f[1], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16_16816(s[u][n], f, qf[n][c * 4 + w][0], qf[n][c * 4 + w][1]);
          }
      if (j == kAhead - 1) {
        id = id_next;
        sc = sc_next;
        if (i + 1 + kAhead < mine) look_up(i + 1 + kAhead);
      }
      const bool more = i + 1 < mine;
      if (more) {
#pragma unroll
        for (int u = 0; u < kTile; ++u) pg[u] = __shfl_sync(0xffffffffu, id, (j + 1) % kAhead * kTile + u);
        load_keys(pg);
      }
      // ---- scores in base 2
      const int key0 = base * kPage;
#pragma unroll
      for (int u = 0; u < kTile; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[u][n][e] = (s[u][n][e] + offset[n][e & 1]) * (factor[n][e & 1] * ks[u]);
      if (a.capped) {
#pragma unroll
        for (int u = 0; u < kTile; ++u)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[u][n][e] = a.cap * tanhf(s[u][n][e] * a.inv_cap);
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
      // ---- running maximum of s + log2 vs
      uint32_t pf[kTile][NT][2];
      bool moved = false;
      float shrink[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = -CUDART_INF_F;
#pragma unroll
          for (int u = 0; u < kTile; ++u) x = fmaxf(x, fmaxf(s[u][n][c], s[u][n][c + 2]) + fminf(fmaxf(lv[u], -60.f), 60.f));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float top = fmaxf(m[n][c], x);
          shrink[n][c] = top == -CUDART_INF_F ? 1.f : fast_exp2(m[n][c] - top);
          moved |= top != m[n][c];
          m[n][c] = top;
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          l[n][0] *= shrink[n][0];
          l[n][1] *= shrink[n][1];
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][k][e] *= shrink[n][e & 1];
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float ref[2] = {m[n][0] == -CUDART_INF_F ? 0.f : m[n][0], m[n][1] == -CUDART_INF_F ? 0.f : m[n][1]};
#pragma unroll
        for (int u = 0; u < kTile; ++u) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float d = s[u][n][e] - ref[e & 1];
            l[n][e & 1] += fast_exp2(d);
            p[e] = fast_exp2(d + lv[u]);
          }
          pf[u][n][0] = transpose8x8(pack_half2(p[0], p[1]));
          pf[u][n][1] = transpose8x8(pack_half2(p[2], p[3]));
        }
      }
      // ---- O^T += V^T P^T
      if (E4M3 && masked) {                     // codes behind the last key may stand for NaN
#pragma unroll
        for (int u = 0; u < kTile; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = key0 + u * kPage + 2 * t + (r & 1) + (r >> 1) * 8;
            if (key >= len || base + u >= p1)
#pragma unroll
              for (int w = 0; w < D / 32; ++w) vr[u][r][w] = 0;
          }
      }
#pragma unroll
      for (int w = 0; w < D / 32; ++w)
#pragma unroll
        for (int high = 0; high < 2; ++high)
#pragma unroll
          for (int u = 0; u < kTile; ++u) {
            uint32_t f[4];
            value_pairs<E4M3>(vr[u][0][w], vr[u][1][w], high, f[0], f[1]);
            value_pairs<E4M3>(vr[u][2][w], vr[u][3][w], high, f[2], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16_16816(o[n][w * 2 + high], f, pf[u][n][0], pf[u][n][1]);
          }
      if (more) load_values(pg);
    }

    // ---- the warps' parts together
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = n * 8 + 2 * t + c;
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 4);
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 8);
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 16);
        if (g == 0) {
          sm_ml[(warp * kRows + r) * 2] = m[n][c];
          sm_ml[(warp * kRows + r) * 2 + 1] = l[n][c];
        }
        float* to = sm_o + (warp * kRows + r) * (D + 4) + g * (D / 8);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) *reinterpret_cast<float2*>(to + 2 * k) = make_float2(o[n][k][c], o[n][k][c + 2]);
      }
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_ml[(w * kRows + r) * 2]);
      const float ref = top == -CUDART_INF_F ? 0.f : top;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = fast_exp2(sm_ml[(w * kRows + r) * 2] - ref);
        sum += sm_ml[(w * kRows + r) * 2 + 1] * f;
        const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * kRows + r) * (D + 4) + d);
        acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint2 packed = make_uint2(pack_out16x2(acc.x * inv, acc.y * inv, a.bf16), pack_out16x2(acc.z * inv, acc.w * inv, a.bf16));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (head * a.rows + r0 + r) * D + d) = packed;
        if (a.lse != nullptr && d == 0) a.lse[head * a.rows + r0 + r] = sum == 0.f ? CUDART_INF_F : ref + log2f(sum);
      } else {
        *reinterpret_cast<float4*>(a.part + (slot * kRows + r) * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * kRows + r) * 2) = make_float2(top, sum);
      }
    }
    __syncthreads();
  }
}

// The parts of a row together: a CTA for each query row of a KV head; rows of segments that were not cut have nothing to do.
template <int D>
__global__ void __launch_bounds__(kThreads) merge_kernel(const DecodeArgs a, int row_block) {
  const int64_t head = blockIdx.x / a.rows;
  const int row = blockIdx.x % a.rows, rb = row / row_block, r = row % row_block;
  const int b = (int)(head / a.c.heads), h = (int)(head % a.c.heads);
  const int pages = pages_of(a, b), lanes = a.c.heads * a.blocks, per = a.plan[1];
  const int64_t first = a.plan[kPlanHead + b];
  const bool even = a.plan[0] != 0;
  int n;
  int64_t slot0, step, u0 = 0;
  if (even) {
    u0 = first * lanes + (int64_t)(h * a.blocks + rb) * pages;
    n = pages == 0 ? 0 : (int)((u0 + pages - 1) / per - u0 / per + 1);
    slot0 = u0 / per * 2;
    step = 2;
  } else {
    n = (int)(a.plan[kPlanHead + b + 1] - first);
    slot0 = first * lanes + (int64_t)h * n * a.blocks + rb;
    step = a.blocks;
  }
  if (n <= 1) return;
  // in an even cut the first part is its CTA's second piece unless it begins where the CTA does
  const auto slot = [&](int i) { return slot0 + i * step + (even && i == 0 && u0 % per != 0 ? 1 : 0); };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ float sm[kWarps][2];
  __shared__ float4 sm_o[kWarps][D / 4];
  float top = -CUDART_INF_F;
  for (int i = tid; i < n; i += kThreads) top = fmaxf(top, a.part_ml[(slot(i) * row_block + r) * 2]);
#pragma unroll
  for (int d = 16; d; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) sm[warp][0] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w][0]);
  const float ref = top == -CUDART_INF_F ? 0.f : top;
  constexpr int kEach = (D / 4 + 31) / 32;
  float4 acc[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int i = warp; i < n; i += kWarps) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (slot(i) * row_block + r) * 2);
    const float f = fast_exp2(ml.x - ref);
    sum += ml.y * f;
    const float4* p = reinterpret_cast<const float4*>(a.part + (slot(i) * row_block + r) * D);
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (lane + e * 32 < D / 4) {
        const float4 x = p[lane + e * 32];
        acc[e].x += x.x * f; acc[e].y += x.y * f; acc[e].z += x.z * f; acc[e].w += x.w * f;
      }
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (lane + e * 32 < D / 4) sm_o[warp][lane + e * 32] = acc[e];
  if (lane == 0) sm[warp][1] = sum;
  __syncthreads();
  if (tid < D / 4) {
    float4 x = sm_o[0][tid];
    sum = sm[0][1];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      const float4 y = sm_o[w][tid];
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      sum += sm[w][1];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint2 packed = make_uint2(pack_out16x2(x.x * inv, x.y * inv, a.bf16), pack_out16x2(x.z * inv, x.w * inv, a.bf16));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (head * a.rows + row) * D + tid * 4) = packed;
    if (a.lse != nullptr && tid == 0) a.lse[head * a.rows + row] = sum == 0.f ? CUDART_INF_F : ref + log2f(sum);
  }
}

// mass_j += sum over rows of 2^(score - log-sum): a thread for each key.
__global__ void __launch_bounds__(256) mass_kernel(const DecodeArgs a, int row_block) {
  const int64_t head = blockIdx.y;
  const int b = (int)(head / a.c.heads), h = (int)(head % a.c.heads);
  const int len = min(len_of(a, b), a.mass_cap);
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= len) return;
  const int at = a.mass_index != nullptr ? a.mass_index[b] : b;
  if (at < 0 || at >= a.mass_rows) {
    if (j == 0) atomicOr(a.c.status, kStatusBadPageId);
    return;
  }
  float sum = 0.f;
  for (int rb = 0; rb < a.blocks; ++rb) {
    const float* s = a.scores + (((head * a.blocks + rb) * a.c.max_pages) * kPage + j) * a.score_cols;
    const float* lse = a.lse + head * a.rows + rb * row_block;
    const int rows = min(row_block, a.rows - rb * row_block);
    for (int r = 0; r < rows; ++r) sum += fast_exp2(s[r] - lse[r]);
  }
  a.mass[((int64_t)at * a.c.heads + h) * a.mass_cap + j] += sum;
}

template <int D, int NT, bool E4M3>
cudaError_t launch_decode_as(const DecodeArgs& a, cudaStream_t s) {
  constexpr int kRows = NT * 8;
  const size_t smem = (((size_t)a.batch + 1 + 3) & ~(size_t)3) * 4 + (size_t)kWarps * kRows * (D + 6) * 4;
  static SharedMemoryLimit limit;
  cudaError_t e = limit.raise(reinterpret_cast<const void*>(decode_kernel<D, NT, E4M3>), (int)smem);
  if (e != cudaSuccess) return e;
  decode_kernel<D, NT, E4M3><<<a.n_cta, kThreads, smem, s>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  merge_kernel<D><<<(unsigned)((int64_t)a.batch * a.c.heads * a.rows), kThreads, 0, s>>>(a, kRows);
  if ((e = cudaGetLastError()) != cudaSuccess || a.mass == nullptr) return e;
  const dim3 grid((unsigned)(((int64_t)a.c.max_pages * kPage + 255) / 256), (unsigned)(a.batch * a.c.heads));
  mass_kernel<<<grid, 256, 0, s>>>(a, kRows);
  return cudaGetLastError();
}

template <int D, int NT>
cudaError_t launch_decode_codes(const DecodeArgs& a, bool e4m3, cudaStream_t s) {
  return e4m3 ? launch_decode_as<D, NT, true>(a, s) : launch_decode_as<D, NT, false>(a, s);
}

template <int D, int NT>
constexpr int ctas_of() { return Shape<D, NT, false>::kCtas; }

}  // namespace

DecodeShape decode_shape(int dim, int rows, int sms) {
  DecodeShape d;
  const bool wide = rows > 8 && dim <= 128;
  d.row_block = wide ? 16 : 8;
  d.blocks = (rows + d.row_block - 1) / d.row_block;
  const int ctas = dim == 64 ? (wide ? ctas_of<64, 2>() : ctas_of<64, 1>()) : dim == 128 ? (wide ? ctas_of<128, 2>() : ctas_of<128, 1>()) : ctas_of<256, 1>();
  d.n_cta = sms * ctas;
  d.slots = 2 * d.n_cta;
  d.score_cols = rows >= d.row_block ? d.row_block : (rows + 1) & ~1;
  return d;
}

cudaError_t launch_decode(DecodeArgs a, bool e4m3, cudaStream_t s) {
  const bool wide = a.rows > 8 && a.c.dim <= 128;
  switch (a.c.dim) {
    case 64: return wide ? launch_decode_codes<64, 2>(a, e4m3, s) : launch_decode_codes<64, 1>(a, e4m3, s);
    case 128: return wide ? launch_decode_codes<128, 2>(a, e4m3, s) : launch_decode_codes<128, 1>(a, e4m3, s);
    default: return launch_decode_codes<256, 1>(a, e4m3, s);
  }
}

}  // namespace kv8
}  // namespace fa
