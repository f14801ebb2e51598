/* C ABI of the operators on a paged cache in 8 bits (libfa_b200_kv8.so, sm_100a): what writes it, what reads it, what makes it shorter.
 *
 * The cache keeps 16 tokens a page: codes [pages, heads, 16, dim] for keys and for values and a scale for each page, head and kind,
 * [pages, heads, 2] fp32 (0: keys, 1: values), from 0 up.  A code stands for code * scale; codes are int8 in -127..127 or e4m3, none of them
 * NaN (what spoils a page is an infinite scale).  dim is 64, 128 or 256.  table [batch, *] int32 with row stride `width` holds a sequence's pages
 * in order; of a row the first `max_pages` entries are looked at, and a sequence has at most 16 * max_pages tokens.
 *
 * Conventions: device pointers on the current device, 16-byte aligned where tensors of 8 or 16 bits are meant; every call is asynchronous
 * on `stream` (a cudaStream_t); nothing is allocated.  Return value: 0, or a negative code with a text in fak_last_error().  A page
 * outside the cache is never touched: the kernel records it in a status word of the device (fak_status) and goes on. */
#ifndef FA_B200_KV8_H
#define FA_B200_KV8_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { FAK_F16 = 0, FAK_BF16 = 1 };           /* rows: queries, new keys and values, results */
enum { FAK_INT8 = 0, FAK_E4M3 = 1 };          /* codes */
enum { FAK_OK = 0, FAK_ERR_INVALID_ARGUMENT = -1, FAK_ERR_UNSUPPORTED = -2, FAK_ERR_CUDA = -4, FAK_ERR_DEVICE_STATUS = -5 };

typedef struct {
  void *k, *v;
  float* scale;
  int64_t pages;
  int32_t heads, dim, codes;
  const int32_t* table;
  int32_t width, max_pages;
} FakCache;

const char* fak_last_error(void);

/* Waits for `stream` and reads the status word of the current device: FAK_ERR_DEVICE_STATUS if a page outside the cache was met (bit 1 of
 * *status) since it was last cleared. */
int fak_status(void* stream, int* status, int clear);
/* Devices (bit i: device i) that an operator has been called on. */
uint64_t fak_devices(void);

/* New rows into pages.  k, v: `total` tokens of [heads, dim], k_stride and v_stride elements from token to token (multiples of 8).  Sequence b has the
 * tokens cu_seqlens[b] to cu_seqlens[b + 1] (null: token b alone, total == batch) and puts them at positions[b] and on (null: 0; negative: a
 * sequence that is left out).
 * For each page, head and kind with new rows: a = their largest magnitude, NaN as infinity; the scale becomes max(a * (1 / top),
 * 2^-100), top = 127 or 448, and at least the scale before where rows of the sequence come in front of the new ones in the page; their codes are then
 * rounded again from code * (scale before / scale).  A new code is x * (1 / scale), rounded to nearest even, or 0 under an infinite scale. */
int fak_append_paged(const FakCache* cache, const void* k, const void* v, int64_t k_stride, int64_t v_stride, int dtype, const int32_t* positions,
                     const int32_t* cu_seqlens, int batch, int64_t total, void* stream);

/* Attention of the `tokens` newest tokens of each sequence, q and out [batch, q_heads, tokens, dim]; lens [batch] counts them in.  Token t of
 * a sequence sees the keys before lens - tokens + t + 1, and no page behind those reaches it; a row that sees none gives zeros.  Scores (q . k) / sqrt(dim), with softcap (0, or
 * from 1e-30 to 1e30) softcap * tanh(score / softcap).  mass [mass_rows, heads, mass_cap] fp32, where given: every key's weights, summed over the rows of its head, are added to row
 * mass_index[b] (null: b), which must be another one for each b.  The workspace (16-byte aligned) has fak_decode_workspace bytes. */
size_t fak_decode_workspace(const FakCache* cache, int batch, int q_heads, int tokens, int with_mass);
int fak_decode_paged(const FakCache* cache, const void* q, void* out, const int32_t* lens, int batch, int q_heads, int tokens, int dtype, float softcap,
                     float* mass, const int32_t* mass_index, int mass_rows, int mass_cap, void* workspace, size_t workspace_bytes, void* stream);

/* Keeps `budget` tokens of each longer sequence, head by head, and all of a shorter one: the first `sink`, the last `recent`, and of the rest
 * those with the largest mass (NaN above all, ties to the lowest index).  They go in order to the pages of new_table (row stride new_width), which
 * must be none of those that are read; a new page's scale is the largest of its tokens' and codes are rounded again from code * (scale
 * before / scale).  kept [batch, heads, budget] receives their indices (-1 behind the last), new_mass [batch, heads, budget] their mass (0), new_lens [batch]. */
int fak_evict_paged(const FakCache* cache, const float* mass, const int32_t* mass_index, int mass_rows, int mass_cap, const int32_t* lens, int batch,
                    const int32_t* new_table, int new_width, int budget, int sink, int recent, int32_t* kept, int32_t* new_lens, float* new_mass,
                    void* stream);

#ifdef __cplusplus
}
#endif
#endif
