// What the operators on the paged 8-bit cache share: arguments, codes, loads.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common.cuh"
#include "../smem_limit.cuh"

namespace fa {
namespace kv8 {

constexpr int kPage = 16;
constexpr float kLeastScale = 7.888609052210118e-31f;      // 2^-100: a reciprocal stays finite
__host__ __device__ constexpr float top_of(bool e4m3) { return e4m3 ? 448.f : 127.f; }

struct Cache {
  uint8_t *k, *v;
  float* scale;           // [pages, heads, 2]
  int64_t pages;
  int heads, dim;
  const int* table;
  int width, max_pages;
  int* status;
};

struct AppendArgs {
  Cache c;
  const void *k, *v;
  int64_t k_stride, v_stride, total;
  const int *positions, *cu;
  int batch;
};

struct DecodeArgs {
  Cache c;
  const void* q;
  void* out;
  const int* lens;
  int batch, rows, tokens;      // rows: query rows of a KV head, (heads of its group) x tokens
  bool bf16, capped;
  float scale;                  // of scores in base 2
  float cap, inv_cap, cap_exp, near;      // cap of scores in base 2, 1 / cap, 2 log2 e / cap, cap / 4
  float* mass;
  const int* mass_index;
  int mass_rows, mass_cap;
  int n_cta, blocks;            // blocks: row blocks of a KV head
  bool even;                    // cut evenly over all warps
  int *plan;                    // [kPlanHead + batch + 1]
  float *part, *part_ml;        // [slots][row block][dim], [slots][row block][2]
  float *scores, *lse;          // [batch, heads, blocks, max tokens, score columns], [batch, heads, rows]
  int score_cols;
};

struct EvictArgs {
  Cache c;
  const float* mass;
  const int* mass_index;
  int mass_rows, mass_cap;
  const int* lens;
  int batch;
  const int* new_table;
  int new_width, budget, sink, recent;
  int *kept, *new_lens;
  float* new_mass;
};

cudaError_t launch_append(const AppendArgs& a, bool e4m3, bool bf16, cudaStream_t s);
cudaError_t launch_evict(const EvictArgs& a, bool e4m3, int sms, cudaStream_t s);

// Sizes of a decode that its caller and its workspace go by.
struct DecodeShape {
  int row_block, blocks, n_cta, slots, score_cols;
};
DecodeShape decode_shape(int dim, int rows, int sms);
cudaError_t launch_decode(DecodeArgs a, bool e4m3, cudaStream_t s);

constexpr int kPlanHead = 4;      // places of a large and of a small unit, small units taken
constexpr int kMaxBatch = 4096;      // sequences of one launch: their page counts' running sum is kept in shared memory

__device__ __forceinline__ bool page_ok(const Cache& c, int id) { return id >= 0 && id < c.pages; }

__device__ __forceinline__ uint4 load_stream16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}

// Four codes as fp32 values, and four values (in units of the scale) as codes, rounded to nearest even.
template <bool E4M3>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
  if constexpr (E4M3) {
    uint32_t lo, hi;
    asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(lo), "=r"(hi) : "r"(w));
    const float2 f0 = __half22float2(*reinterpret_cast<__half2*>(&lo)), f1 = __half22float2(*reinterpret_cast<__half2*>(&hi));
    x[0] = f0.x; x[1] = f0.y; x[2] = f1.x; x[3] = f1.y;
  } else {
    w ^= 0x80808080u;      // 2^23 + code + 128, exactly
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __fadd_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 + i)), -8388736.f);
  }
}
template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4]) {
  if constexpr (E4M3) {
    uint32_t r;
    asm("{.reg .b16 a, b; cvt.rn.satfinite.e4m3x2.f32 a, %2, %1; cvt.rn.satfinite.e4m3x2.f32 b, %4, %3; mov.b32 %0, {a, b};}"
        : "=r"(r) : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]));
    return r;
  } else {
    // 1.5 * 2^23 + x leaves the rounded value's low byte at the bottom; |x| is at most 127 but for a rounding
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fadd_rn(x[i], 12582912.f));
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
}
// Codes of one scale as codes of another, `ratio` = scale before / scale <= 1.
template <bool E4M3>
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
  float x[4];
  decode4<E4M3>(w, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __fmul_rn(x[i], ratio);
  return encode4<E4M3>(x);
}

}  // namespace kv8
}  // namespace fa
