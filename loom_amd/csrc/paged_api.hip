// paged_api.hip -- loom_amd_page_*, loom_amd_kv_*, loom_amd_paged_attention
// and loom_amd_sample entry points (include/loom_accel_amd.h).
#include <math.h>

#include "api_util.hpp"
#include "loom_accel_amd.h"
#include "paged.hpp"

namespace lamd {

static bool page_ok(int p) { return p == 16 || p == 32 || p == 64 || p == 128; }

static int check_table(const loom_amd_page_table* t, PageTables* out) {
    if (!t) return fail("page table is null");
    if (!t->pages || !t->held || !t->free_pages || !t->free_count) return fail("page table: null buffer");
    if (t->requests <= 0 || t->max_pages <= 0 || t->num_pages <= 0) {
        return fail("page table: requests, max_pages and num_pages must be positive");
    }
    if (!page_ok(t->page_size)) return fail("page_size must be 16, 32, 64 or 128");
    if ((long)t->num_pages * t->page_size > 0x7fffffffl || (long)t->max_pages * t->page_size > 0x7fffffffl) {
        return fail("page table: more than 2^31 - 1 tokens");
    }
    *out = PageTables{t->pages, t->held, t->free_pages, t->free_count,
                      t->requests, t->max_pages, t->num_pages, t->page_size};
    return 0;
}

int check_kv_pages(const loom_amd_kv_pages* c, KvPages* out) {
    if (!c) return fail("kv pages are null");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail("kv pages: null buffer");
    if (c->num_pages <= 0 || c->kv_heads <= 0) return fail("kv pages: num_pages and kv_heads must be positive");
    if (!page_ok(c->page_size)) return fail("page_size must be 16, 32, 64 or 128");
    if (!paged_hd_ok(c->head_dim)) return fail("head_dim of a paged cache must be 32, 64, 128 or 256");
    if (c->kv_heads > 65535) return fail("kv pages: more than 65535 heads");
    if ((long)c->num_pages * c->page_size > 0x7fffffffl) return fail("kv pages: more than 2^31 - 1 tokens");
    if (((uintptr_t)c->k & 15) || ((uintptr_t)c->v & 15)) return fail("kv pages: codes must be 16-byte aligned");
    *out = KvPages{c->k, c->v, c->k_scale, c->v_scale, c->num_pages, c->page_size, c->kv_heads, c->head_dim};
    return 0;
}

static int check_attention(int rows, int heads, int kv_heads, int requests) {
    if (rows < 0 || heads <= 0 || kv_heads <= 0 || requests <= 0) return fail("bad shape");
    if (heads % kv_heads != 0) return fail("kv_heads must divide heads");
    if ((int64_t)rows * heads > 0x7fffffff) return fail("rows * heads exceeds 2^31 - 1");
    return 0;
}

int check_paged_rows(const KvPages& c, int requests, int max_pages, int rows, int heads, int max_context) {
    if (check_attention(rows, heads, c.kv_heads, requests)) return -1;
    if (max_pages <= 0 || (int64_t)max_pages * c.page > 0x7fffffff) return fail("bad max_pages");
    if (max_context < 0 || max_context > max_pages * c.page) {
        return fail("max_context must be within max_pages * page_size");
    }
    return 0;
}

}  // namespace lamd

using namespace lamd;

extern "C" {

int loom_amd_page_table_reset(const loom_amd_page_table* table, void* stream) {
    PageTables t;
    if (check_table(table, &t)) return -1;
    hipError_t e = launch_page_reset(t, (hipStream_t)stream);
    return e == hipSuccess ? 0 : fail_hip("page_table_reset", e);
}

int loom_amd_page_table_plan(const loom_amd_page_table* table, const int32_t* lens, const int32_t* new_tokens,
                             int rows, const loom_amd_page_plan* plan, void* stream) {
    PageTables t;
    if (check_table(table, &t)) return -1;
    if (!lens || !new_tokens || !plan || !plan->row_start || !plan->lens || !plan->scratch) return fail("null buffer");
    if (rows < 0) return fail("bad shape");
    if (rows > 0 && (!plan->request || !plan->positions || !plan->slots)) return fail("null buffer");
    if ((uintptr_t)plan->scratch & 15) return fail("plan scratch must be 16-byte aligned");
    const PlanOut o{plan->row_start, plan->lens, plan->request, plan->positions, plan->slots, plan->scratch};
    hipError_t e = launch_page_plan(t, lens, new_tokens, rows, o, (hipStream_t)stream);
    return e == hipSuccess ? 0 : fail_hip("page_table_plan", e);
}

int loom_amd_page_table_release(const loom_amd_page_table* table, const uint8_t* done, void* stream) {
    PageTables t;
    if (check_table(table, &t)) return -1;
    if (!done) return fail("null buffer");
    hipError_t e = launch_page_release(t, done, (hipStream_t)stream);
    return e == hipSuccess ? 0 : fail_hip("page_table_release", e);
}

int loom_amd_kv_append(const loom_amd_kv_pages* cache, const void* k, const void* v, int type, int rows,
                       int64_t k_stride, int64_t v_stride, const int32_t* slots, void* stream) {
    KvPages c;
    if (check_kv_pages(cache, &c)) return -1;
    if (type != LOOM_AMD_ROW_F32 && type != LOOM_AMD_ROW_BF16) return fail("rows of keys and values are fp32 or bf16");
    if (rows < 0) return fail("bad shape");
    if (rows == 0) return 0;
    if (!k || !v || !slots) return fail("null buffer");
    const int64_t width = (int64_t)c.kv_heads * c.hd;
    if (rows > 1 && (k_stride < width || v_stride < width)) return fail("row strides must cover kv_heads * head_dim");
    hipError_t e = launch_kv_append(c, k, v, type, rows, k_stride, v_stride, slots, (hipStream_t)stream);
    return e == hipSuccess ? 0 : fail_hip("kv_append", e);
}

int loom_amd_kv_read(const loom_amd_kv_pages* cache, const int32_t* slots, int rows, float* k, float* v,
                     void* stream) {
    KvPages c;
    if (check_kv_pages(cache, &c)) return -1;
    if (rows < 0) return fail("bad shape");
    if (rows == 0) return 0;
    if (!slots || !k || !v) return fail("null buffer");
    if (((uintptr_t)k & 15) || ((uintptr_t)v & 15)) return fail("outputs of kv_read must be 16-byte aligned");
    hipError_t e = launch_kv_read(c, slots, rows, k, v, (hipStream_t)stream);
    return e == hipSuccess ? 0 : fail_hip("kv_read", e);
}

int loom_amd_paged_attention_workspace(int rows, int heads, int kv_heads, int head_dim, int requests,
                                       int max_context, size_t* bytes) {
    if (!bytes) return fail("bytes is null");
    *bytes = 0;
    if (check_attention(rows, heads, kv_heads, requests)) return -1;
    if (!paged_hd_ok(head_dim)) return fail("head_dim of a paged cache must be 32, 64, 128 or 256");
    if (max_context < 0) return fail("bad shape");
    if (rows > 0) *bytes = paged_attn_workspace(rows, heads, kv_heads, head_dim, requests, max_context);
    return 0;
}

int loom_amd_paged_attention(const loom_amd_kv_pages* cache, const int32_t* pages, int requests, int max_pages,
                             const int32_t* row_start, const int32_t* positions, const void* q, int type, int rows,
                             int heads, int64_t q_stride, float scale, int max_context, void* out,
                             int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream) {
    KvPages c;
    if (check_kv_pages(cache, &c)) return -1;
    if (check_paged_rows(c, requests, max_pages, rows, heads, max_context)) return -1;
    if (type != LOOM_AMD_ROW_F32 && type != LOOM_AMD_ROW_BF16 && type != LOOM_AMD_ROW_F64) {
        return fail("rows of queries are fp32, bf16 or fp64");
    }
    if (!isfinite(scale)) return fail("scale must be finite");
    if (rows == 0) return 0;
    if (!pages || !row_start || !positions || !q || !out) return fail("null buffer");
    const int64_t width = (int64_t)heads * c.hd;
    if (rows > 1 && (q_stride < width || out_stride < width)) return fail("row strides must cover heads * head_dim");
    const size_t need = paged_attn_workspace(rows, heads, c.kv_heads, c.hd, requests, max_context);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        return fail("workspace of " + std::to_string(workspace_bytes) + " bytes, need " + std::to_string(need));
    }
    if ((uintptr_t)workspace & 15) return fail("workspace must be 16-byte aligned");
    PagedAttn a{c, pages, max_pages, requests, row_start, positions, q, out, type, rows, heads,
                (long)q_stride, (long)out_stride, scale, max_context, workspace};
    hipError_t e = launch_paged_attn(a, (hipStream_t)stream);
    return e == hipSuccess ? 0 : fail_hip("paged_attention", e);
}

static int check_sample(int vocab, int rows) {
    if (vocab <= 0 || rows < 0) return fail("bad shape");
    if (vocab > LOOM_AMD_SAMPLE_MAX_VOCAB) return fail("vocab is limited to 8388608");
    return 0;
}

int loom_amd_sample_workspace(int vocab, int rows, size_t* bytes) {
    if (!bytes) return fail("bytes is null");
    *bytes = 0;
    if (check_sample(vocab, rows)) return -1;
    *bytes = sample_workspace(vocab, rows);
    return 0;
}

int loom_amd_sample(const float* logits, int64_t stride, int vocab, int rows, const float* temperature,
                    const int32_t* top_k, const float* top_p, const float* min_p, const float* uniform,
                    int32_t* ids, void* workspace, size_t workspace_bytes, void* stream) {
    if (check_sample(vocab, rows)) return -1;
    if (rows == 0) return 0;
    if (!logits || !uniform || !ids) return fail("null buffer");
    if (rows > 1 && stride < vocab) return fail("row stride must cover vocab");
    const size_t need = sample_workspace(vocab, rows);
    if (!workspace || workspace_bytes < need) {
        return fail("workspace of " + std::to_string(workspace_bytes) + " bytes, need " + std::to_string(need));
    }
    if ((uintptr_t)workspace & 15) return fail("workspace must be 16-byte aligned");
    SampleArgs a{logits, (long)stride, vocab, rows, temperature, top_k, top_p, min_p, uniform, ids, workspace};
    hipError_t e = launch_sample(a, (hipStream_t)stream);
    return e == hipSuccess ? 0 : fail_hip("sample", e);
}

}  // extern "C"
