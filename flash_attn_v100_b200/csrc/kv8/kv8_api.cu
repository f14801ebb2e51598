// C-ABI entry points of the operators on the paged 8-bit cache (see include/fa_b200_kv8.h): argument checks and launches.
#include "../../../include/fa_b200_kv8.h"

#include <math.h>

#include <atomic>

#include "../api_common.cuh"
#include "kv8.cuh"

namespace {

namespace k8 = fa::kv8;

__device__ int g_status;      // of a device: every launch on it shares the word, which needs no allocation and no clearing before a capture

std::atomic<uint64_t> g_devices;

cudaError_t status_word(int** word) {
  static std::atomic<int*> cached[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && (*word = cached[dev].load(std::memory_order_acquire)) != nullptr) return cudaSuccess;
  void* p = nullptr;
  if ((e = cudaGetSymbolAddress(&p, g_status)) != cudaSuccess) return e;
  *word = static_cast<int*>(p);
  if (dev >= 0 && dev < 64) {
    cached[dev].store(*word, std::memory_order_release);
    g_devices.fetch_or(1ull << dev);
  }
  return cudaSuccess;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

int check_cache(const FakCache* p) {
  FA_REQUIRE(p != nullptr && p->k && p->v && p->scale && p->table, "null pointer");
  FA_REQUIRE(p->codes == FAK_INT8 || p->codes == FAK_E4M3, "unknown codes %d", p->codes);
  FA_REQUIRE(p->pages > 0 && p->pages < (1ll << 31) && p->heads > 0 && p->heads < 32768, "bad cache sizes: pages=%lld heads=%d", (long long)p->pages, p->heads);
  FA_REQUIRE(p->max_pages > 0 && p->width >= p->max_pages && p->max_pages <= (1 << 26), "bad table sizes: width=%d max_pages=%d", p->width, p->max_pages);
  FA_REQUIRE(aligned16(p->k) && aligned16(p->v) && (reinterpret_cast<uintptr_t>(p->scale) & 7) == 0, "k, v and scale must be 16- and 8-byte aligned");
  if (p->dim != 64 && p->dim != 128 && p->dim != 256) return fail(FAK_ERR_UNSUPPORTED, "head dimension %d is not built (64, 128, 256)", p->dim);
  return FAK_OK;
}

int make_cache(const FakCache* p, k8::Cache& c) {
  int* word = nullptr;
  const cudaError_t e = status_word(&word);
  if (e != cudaSuccess) return done(e, "the status word");
  c = {static_cast<uint8_t*>(p->k), static_cast<uint8_t*>(p->v), p->scale, p->pages, p->heads, p->dim, p->table, p->width, p->max_pages, word};
  return FAK_OK;
}

// Sequences of one launch of a decode: their running sum of pages has to fit in shared memory, and the pages of all heads and row blocks, with what a segment
// costs beside them, in 31 bits.
int64_t slab_of(const FakCache* p, int blocks) {
  int64_t n = k8::kMaxBatch;
  const int64_t by_pages = ((1ll << 31) - 1) / (((int64_t)p->max_pages + 16) * p->heads * blocks);
  if (n > by_pages) n = by_pages;
  return n < 1 ? 1 : n;
}

struct Layout {
  size_t plan, part, part_ml, lse, scores, bytes;
};
Layout layout_of(const FakCache* p, int64_t batch, int rows, bool with_mass, const k8::DecodeShape& d) {
  Layout w;
  const size_t heads = (size_t)batch * p->heads;
  w.plan = 0;
  w.part = round256((k8::kPlanHead + (size_t)batch + 1) * 4);
  w.part_ml = w.part + round256((size_t)d.slots * d.row_block * p->dim * 4);
  w.lse = w.part_ml + round256((size_t)d.slots * d.row_block * 2 * 4);
  w.scores = w.lse + (with_mass ? round256(heads * rows * 4) : 0);
  w.bytes = w.scores + (with_mass ? round256(heads * d.blocks * p->max_pages * k8::kPage * d.score_cols * 4) : 0);
  return w;
}

int check_decode(const FakCache* p, int batch, int q_heads, int tokens) {
  const int rc = check_cache(p);
  if (rc != FAK_OK) return rc;
  FA_REQUIRE(batch >= 0 && batch <= (1 << 24) && tokens > 0 && tokens <= 65536, "bad sizes: batch=%d tokens=%d", batch, tokens);
  FA_REQUIRE(q_heads > 0 && q_heads <= (1 << 20) && q_heads % p->heads == 0, "q_heads=%d is not a multiple of heads=%d", q_heads, p->heads);
  FA_REQUIRE((int64_t)(q_heads / p->heads) * tokens <= 65536, "a KV head has %lld query rows, 65536 are the most", (long long)(q_heads / p->heads) * tokens);
  return FAK_OK;
}

}  // namespace

extern "C" {

const char* fak_last_error(void) { return g_err; }

int fak_status(void* stream, int* status, int clear) {
  FA_REQUIRE(status != nullptr, "null pointer");
  int* word = nullptr;
  cudaError_t e = status_word(&word);
  if (e == cudaSuccess) e = cudaMemcpyAsync(status, word, sizeof(int), cudaMemcpyDeviceToHost, st(stream));
  if (e == cudaSuccess && clear) e = cudaMemsetAsync(word, 0, sizeof(int), st(stream));
  if (e == cudaSuccess) e = cudaStreamSynchronize(st(stream));
  if (e != cudaSuccess) return done(e, "fak_status");
  if (*status != 0) return fail(FAK_ERR_DEVICE_STATUS, "a kernel on the 8-bit cache met a page or a row of sums outside the cache (status %d)", *status);
  return FAK_OK;
}

uint64_t fak_devices(void) { return g_devices.load(); }

int fak_append_paged(const FakCache* cache, const void* k, const void* v, int64_t k_stride, int64_t v_stride, int dtype, const int32_t* positions,
                     const int32_t* cu_seqlens, int batch, int64_t total, void* stream) {
  int rc = check_cache(cache);
  if (rc != FAK_OK) return rc;
  FA_REQUIRE(dtype_ok(dtype), "unknown dtype %d", dtype);
  FA_REQUIRE(batch >= 0 && total >= 0 && total < kMaxRows && (cu_seqlens != nullptr || total == batch), "bad sizes: batch=%d total=%lld", batch,
             (long long)total);
  if (total == 0 || batch == 0) return FAK_OK;
  FA_REQUIRE(k && v, "null pointer");
  FA_REQUIRE(aligned16(k) && aligned16(v) && k_stride % 8 == 0 && v_stride % 8 == 0, "k and v must have 16-byte aligned rows");
  FA_REQUIRE(k_stride >= (int64_t)cache->heads * cache->dim && v_stride >= (int64_t)cache->heads * cache->dim, "a token's row is longer than the stride");
  FA_REQUIRE(total * cache->heads / 2 < kMaxRows, "too many rows: %lld tokens of %d heads", (long long)total, cache->heads);
  k8::AppendArgs a{};
  if ((rc = make_cache(cache, a.c)) != FAK_OK) return rc;
  a.k = k; a.v = v; a.k_stride = k_stride; a.v_stride = v_stride; a.total = total; a.positions = positions; a.cu = cu_seqlens; a.batch = batch;
  return done(k8::launch_append(a, cache->codes == FAK_E4M3, dtype == FAK_BF16, st(stream)), "append_paged");
}

size_t fak_decode_workspace(const FakCache* cache, int batch, int q_heads, int tokens, int with_mass) {
  if (check_decode(cache, batch, q_heads, tokens) != FAK_OK || batch == 0) return 0;
  const int rows = q_heads / cache->heads * tokens;
  const k8::DecodeShape d = k8::decode_shape(cache->dim, rows, sm_count());
  const int64_t slab = slab_of(cache, d.blocks);
  return layout_of(cache, batch < slab ? batch : slab, rows, with_mass != 0, d).bytes;
}

int fak_decode_paged(const FakCache* cache, const void* q, void* out, const int32_t* lens, int batch, int q_heads, int tokens, int dtype, float softcap,
                     float* mass, const int32_t* mass_index, int mass_rows, int mass_cap, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_decode(cache, batch, q_heads, tokens);
  if (rc != FAK_OK) return rc;
  FA_REQUIRE(dtype_ok(dtype), "unknown dtype %d", dtype);
  FA_REQUIRE(softcap == 0.f || (softcap >= 1e-30f && softcap <= 1e30f), "softcap must be 0 or from 1e-30 to 1e30");
  if (batch == 0) return FAK_OK;
  FA_REQUIRE(q && out && lens && workspace, "null pointer");
  FA_REQUIRE(aligned16(q) && aligned16(out) && aligned16(workspace), "q, out and the workspace must be 16-byte aligned");
  FA_REQUIRE(mass == nullptr || (mass_rows > 0 && mass_cap > 0 && (mass_index != nullptr || mass_rows >= batch)), "bad sizes: mass_rows=%d mass_cap=%d", mass_rows,
             mass_cap);
  const int rows = q_heads / cache->heads * tokens;
  const k8::DecodeShape d = k8::decode_shape(cache->dim, rows, sm_count());
  const int64_t slab = batch < slab_of(cache, d.blocks) ? batch : slab_of(cache, d.blocks);
  const Layout w = layout_of(cache, slab, rows, mass != nullptr, d);
  FA_REQUIRE(workspace_bytes >= w.bytes, "the workspace has %zu bytes, %zu are needed", workspace_bytes, w.bytes);
  FA_REQUIRE(((int64_t)cache->max_pages + 16) * cache->heads * d.blocks < (1ll << 31), "too many pages: %d of a sequence, %d heads, %d row blocks", cache->max_pages,
             cache->heads, d.blocks);
  k8::DecodeArgs a{};
  if ((rc = make_cache(cache, a.c)) != FAK_OK) return rc;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  const double log2e = 1.4426950408889634, root = 1.0 / sqrt((double)cache->dim);
  a.rows = rows; a.tokens = tokens; a.bf16 = dtype == FAK_BF16; a.capped = softcap > 0.f;
  a.scale = (float)(root * log2e);
  a.cap = (float)(softcap * log2e);
  a.inv_cap = a.capped ? (float)(1.0 / (softcap * log2e)) : 0.f;
  a.cap_exp = a.capped ? (float)(2.0 / softcap) : 0.f;
  a.near = 0.25f * a.cap;
  a.n_cta = d.n_cta; a.blocks = d.blocks; a.score_cols = d.score_cols;
  a.plan = reinterpret_cast<int*>(base + w.plan);
  a.part = reinterpret_cast<float*>(base + w.part);
  a.part_ml = reinterpret_cast<float*>(base + w.part_ml);
  a.lse = mass != nullptr ? reinterpret_cast<float*>(base + w.lse) : nullptr;
  a.scores = mass != nullptr ? reinterpret_cast<float*>(base + w.scores) : nullptr;
  a.mass_cap = mass_cap;
  const int64_t row_bytes = (int64_t)q_heads * tokens * cache->dim * 2;
  for (int64_t b0 = 0; b0 < batch; b0 += slab) {
    a.batch = (int)(batch - b0 < slab ? batch - b0 : slab);
    a.c.table = cache->table + b0 * cache->width;
    a.lens = lens + b0;
    a.q = static_cast<const uint8_t*>(q) + b0 * row_bytes;
    a.out = static_cast<uint8_t*>(out) + b0 * row_bytes;
    a.mass = mass != nullptr && mass_index == nullptr ? mass + b0 * cache->heads * mass_cap : mass;
    a.mass_index = mass_index != nullptr ? mass_index + b0 : nullptr;
    a.mass_rows = mass_index != nullptr ? mass_rows : (int)(mass_rows - b0);
    if ((rc = done(k8::launch_decode(a, cache->codes == FAK_E4M3, st(stream)), "decode_paged")) != FAK_OK) return rc;
  }
  return FAK_OK;
}

int fak_evict_paged(const FakCache* cache, const float* mass, const int32_t* mass_index, int mass_rows, int mass_cap, const int32_t* lens, int batch,
                    const int32_t* new_table, int new_width, int budget, int sink, int recent, int32_t* kept, int32_t* new_lens, float* new_mass,
                    void* stream) {
  int rc = check_cache(cache);
  if (rc != FAK_OK) return rc;
  FA_REQUIRE(batch >= 0 && budget > 0 && sink >= 0 && recent >= 0 && (int64_t)sink + recent <= budget, "bad sizes: budget=%d sink=%d recent=%d", budget, sink,
             recent);
  FA_REQUIRE((int64_t)new_width * k8::kPage >= budget, "a row of the new table has %d pages, fewer than %d tokens need", new_width, budget);
  FA_REQUIRE(mass_rows > 0 && mass_cap > 0 && (mass_index != nullptr || mass_rows >= batch), "bad sizes: mass_rows=%d mass_cap=%d", mass_rows, mass_cap);
  FA_REQUIRE((int64_t)batch * cache->heads < (1ll << 27) && (int64_t)batch * cache->heads * ((budget + 15) / 16) < kMaxRows, "too many rows: batch=%d heads=%d budget=%d",
             batch, cache->heads, budget);
  if (batch == 0) return FAK_OK;
  FA_REQUIRE(mass && lens && new_table && kept && new_lens && new_mass, "null pointer");
  k8::EvictArgs a{};
  if ((rc = make_cache(cache, a.c)) != FAK_OK) return rc;
  a.mass = mass; a.mass_index = mass_index; a.mass_rows = mass_rows; a.mass_cap = mass_cap; a.lens = lens; a.batch = batch;
  a.new_table = new_table; a.new_width = new_width; a.budget = budget; a.sink = sink; a.recent = recent;
  a.kept = kept; a.new_lens = new_lens; a.new_mass = new_mass;
  return done(k8::launch_evict(a, cache->codes == FAK_E4M3, sm_count(), st(stream)), "evict_paged");
}

}  // extern "C"
