// paged.hpp -- launchers of the paged-cache kernels (paged_cache.hip,
// paged_attention.hip) and of sampling (sample.hip).
//
// The cache holds int8 codes in pages of `page` tokens (16, 32, 64 or 128) with
// one fp32 scale per page, key/value head and side; a value is code * scale.
//   k codes: [pages][kv_heads][page / 16][head_dim / 16][16 tokens][16 dimensions]
//   v codes: [pages][kv_heads][page / 16][head_dim][16 tokens]
// (blocks of 16 tokens in the order in which the matrix operands of attention
// take them: the 16 bytes of neighbouring lanes lie side by side.  With keys
// token by token each lane's 16 bytes are in a line of their own, 50 cache
// accesses a load instead of 16: four prompts of 2048 tokens took 310 us, and
// 284 us with the blocks)
//   scales:  [pages][kv_heads]
// A slot is page * page_size + offset; -1 (and anything outside the cache) is
// no slot.
#pragma once

#include "lamd.hpp"
#include "loom_accel_amd.h"

namespace lamd {

struct KvPages {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    int pages, page, kv_heads, hd;
};

// Offsets within a page's head (page * hd codes).
__host__ __device__ inline int k_offset(int token, int d, int hd) {
    return (token >> 4) * 16 * hd + (d >> 4) * 256 + (token & 15) * 16 + (d & 15);
}
__host__ __device__ inline int v_offset(int token, int d, int hd) {
    return (token >> 4) * 16 * hd + d * 16 + (token & 15);
}

enum RowType : int { ROW_F32 = 0, ROW_BF16 = 1, ROW_F64 = 2 };

// Tables of `requests` requests: table[r][i] is the page of positions
// [i*page, (i+1)*page) of request r (-1 past held[r]); free_pages holds the
// pages that nobody has, the next one to give at free_pages[*free_count - 1].
struct PageTables {
    int32_t* table;
    int32_t* held;
    int32_t* free_pages;
    int32_t* free_count;
    int requests, max_pages, pages, page;
};

struct PlanOut {
    int32_t* row_start;  // requests + 1
    int32_t* lens;       // requests
    int32_t* request;    // rows
    int32_t* positions;  // rows
    int32_t* slots;      // rows
    int32_t* scratch;    // 4 * requests
};

hipError_t launch_page_reset(const PageTables& t, hipStream_t s);
hipError_t launch_page_plan(const PageTables& t, const int32_t* lens, const int32_t* new_tokens, int rows,
                            const PlanOut& o, hipStream_t s);
hipError_t launch_page_release(const PageTables& t, const uint8_t* done, hipStream_t s);

// head_dim of the paged kernels
inline bool paged_hd_ok(int hd) { return hd == 32 || hd == 64 || hd == 128 || hd == 256; }

hipError_t launch_kv_append(const KvPages& c, const void* k, const void* v, int type, int rows, long k_stride,
                            long v_stride, const int32_t* slots, hipStream_t s);
hipError_t launch_kv_read(const KvPages& c, const int32_t* slots, int rows, float* k, float* v, hipStream_t s);

struct PagedAttn {
    KvPages c;
    const int32_t* table;  // requests x max_pages
    int max_pages, requests;
    const int32_t* row_start;  // requests + 1
    const int32_t* positions;  // rows
    const void* q;
    void* out;
    int type, rows, heads;
    long q_stride, out_stride;  // elements between rows
    float scale;
    int max_context;  // no position is at or past it
    void* workspace;
};
size_t paged_attn_workspace(int rows, int heads, int kv_heads, int hd, int requests, int max_context);
hipError_t launch_paged_attn(const PagedAttn& a, hipStream_t s);

// Checks of the entry points (paged_api.hip): 0, or -1 with the message set.
int check_kv_pages(const loom_amd_kv_pages* c, KvPages* out);
int check_paged_rows(const KvPages& c, int requests, int max_pages, int rows, int heads, int max_context);

struct SampleArgs {
    const float* logits;
    long stride;
    int vocab, rows;
    const float* temperature;  // each of the four: rows values, or null
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniform;  // rows
    int32_t* ids;          // rows
    void* workspace;
};
size_t sample_workspace(int vocab, int rows);
hipError_t launch_sample(const SampleArgs& a, hipStream_t s);

}  // namespace lamd
