// Host side of the batched serving operators: argument checks, launch plans
// and workspaces of vkv_page_map, vkv_pages_append, vkv_paged_attn,
// vkv_prompt_attn and vkv_logprobs.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "vkv.h"
#include "vkv_internal.h"
#include "vkv_serve.h"

using namespace vkv;

namespace {

vkv_status bad(const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return host_fail(VKV_STATUS_INVALID_ARGUMENT, buf);
}

vkv_status small_ws(const char *what, size_t have, size_t need) {
    char buf[256];
    std::snprintf(buf, sizeof(buf), "%s: workspace of %zu bytes, %zu needed", what, have, need);
    return host_fail(VKV_STATUS_BUFFER_TOO_SMALL, buf);
}

hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }

// Launches go to the stream's device, whichever is current.
struct StreamDevice {
    int prev = -1;
    bool changed = false;
    explicit StreamDevice(hipStream_t st) {
        hipDevice_t dev = 0;
        if (st && hipStreamGetDevice(st, &dev) == hipSuccess && hipGetDevice(&prev) == hipSuccess && prev != dev)
            changed = hipSetDevice(dev) == hipSuccess;
    }
    ~StreamDevice() {
        if (changed) (void)hipSetDevice(prev);
    }
};

int elem_bytes(int32_t dtype) {
    return dtype == VKV_DTYPE_F32 ? 4 : dtype == VKV_DTYPE_F16 || dtype == VKV_DTYPE_BF16 ? 2 : 0;
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// An array of rows read and written 16 bytes at a time; *stride: 0 = packed.
vkv_status check_rows(const char *what, const char *name, const void *p, int64_t width, int32_t dtype, int64_t *stride) {
    if (*stride == 0) *stride = width;
    const int eb = elem_bytes(dtype);
    if (!p) return bad("%s: %s is null", what, name);
    if (*stride < width || *stride > (int64_t)1 << 40) return bad("%s: %s: row stride %lld below the row's %lld values", what, name, (long long)*stride, (long long)width);
    if (!aligned(p, 16) || *stride * eb % 16 != 0) return bad("%s: %s: rows must be 16-byte aligned", what, name);
    return VKV_STATUS_OK;
}

vkv_status check_ints(const char *what, const void *p) {
    if (!p) return bad("%s: null argument", what);
    if (!aligned(p, 4)) return bad("%s: int32 and f32 arrays must be 4-byte aligned", what);
    return VKV_STATUS_OK;
}

bool page_size_ok(int32_t n) { return n == 16 || n == 32 || n == 64 || n == 128 || n == 256; }

vkv_status check_pool(const char *what, const vkv_pages *p) {
    if (!p) return bad("%s: null pages", what);
    if (p->dtype != VKV_DTYPE_E4M3 && p->dtype != VKV_DTYPE_I8) return bad("%s: pages of dtype %d", what, p->dtype);
    if (!page_size_ok(p->page_size)) return bad("%s: page size %d (16, 32, 64, 128 or 256)", what, p->page_size);
    if (p->head_dim != 64 && p->head_dim != 128) return bad("%s: head dim %d (64 or 128)", what, p->head_dim);
    if (p->n_layers < 1 || p->n_pages < 1 || p->n_kv_heads < 1 || p->n_kv_heads > 4096 ||
        (int64_t)p->n_pages * p->page_size > INT32_MAX)
        return bad("%s: %d layers of %d pages of %d kv heads", what, p->n_layers, p->n_pages, p->n_kv_heads);
    // 16-token blocks of a layer are counted in 32 bits
    if ((int64_t)p->n_pages * p->n_kv_heads * (p->page_size / 16) > INT32_MAX)
        return bad("%s: %d pages of %d kv heads", what, p->n_pages, p->n_kv_heads);
    return VKV_STATUS_OK;
}

vkv_status check_pages(const char *what, const vkv_pages *p, int32_t layer) {
    if (vkv_status s = check_pool(what, p)) return s;
    if (!p->k || !p->v || !p->k_scale || !p->v_scale) return bad("%s: null pages", what);
    if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->k_scale, 4) || !aligned(p->v_scale, 4))
        return bad("%s: codes must be 16-byte aligned, scales 4-byte", what);
    if (layer < 0 || layer >= p->n_layers) return bad("%s: layer %d outside [0, %d)", what, layer, p->n_layers);
    return VKV_STATUS_OK;
}

vkv_status check_heads(const char *what, int32_t n_q_heads, int32_t n_kv_heads) {
    if (n_kv_heads < 1 || n_kv_heads > 4096 || n_q_heads < n_kv_heads || n_q_heads % n_kv_heads != 0 || n_q_heads > 65536)
        return bad("%s: %d query heads over %d kv heads", what, n_q_heads, n_kv_heads);
    return VKV_STATUS_OK;
}

template <typename P> P *layer_at(P *base, const vkv_pages *p, int32_t layer, int64_t per_head) {
    return base + (int64_t)layer * p->n_pages * p->n_kv_heads * per_head;
}

// Up to so many work groups of kPromptRows rows, which leave CUs idle, prompts
// of more than a tile of keys go by kPromptRowsFew rows and their keys over the
// waves (f32, 32 heads over 8 of 128: 200 tokens 56 work groups, 21.0 -> 15.8 us;
// 700 tokens 176, 45.3 -> 41.9; 1000 tokens 256, 61.3 against 63.2; bf16 200
// tokens 13.4 -> 11.0, 700 tokens 25.8 against 27.9, 1500 tokens 376, 45.6
// against 62.1; a single token 8.9 against 10.5).
constexpr int64_t kPromptGroupsFew = 192;

// Work groups of the paged attention beyond which longer chunks only save
// partials: four per CU (16 rows of 8192 tokens 40.8 us, 46.3 with twice as
// many; 131 rows of up to 500 21.4 us, 30.5).  A chunk's start and end, and its
// place in the merge, want 256 keys at least (1 x 8192 tokens 11.9 us, 15.2
// with 128; with 512, 4 x 8192 tokens 24.6 instead of 19.5).
constexpr int64_t kAttnGroups = 1024;
constexpr int64_t kAttnChunkMin = 256;

int64_t attn_units(int32_t n_rows, int32_t n_q_heads, int32_t n_kv_heads) {
    return (int64_t)n_rows * n_kv_heads * ((n_q_heads / n_kv_heads + 7) / 8);
}

// Keys per work group and chunks per row.  A row begins at the multiple of 32
// at or below its first key.
void attn_plan(int64_t units, int32_t max_len, int32_t window, int32_t *chunk, int32_t *n_chunks) {
    const int64_t span = std::max<int64_t>(1, window > 0 && window < max_len ? std::min<int64_t>(max_len, (int64_t)window + 31) : max_len);
    int64_t c = (span * units + kAttnGroups - 1) / kAttnGroups;
    c = (c + kPagedChunkStep - 1) / kPagedChunkStep * kPagedChunkStep;
    c = std::min<int64_t>(std::max(c, kAttnChunkMin), kPagedChunkMax);
    *chunk = (int32_t)c;
    *n_chunks = (int32_t)((span + c - 1) / c);
}

// No fewer (row, chunk) pairs than any plan of so many rows and tokens, or of
// fewer, has, with any window: a chunk is at its least, its most, or at
// least what leaves kAttnGroups units, `per_row` to a row.
int64_t attn_parts_most(int64_t n_rows, int64_t per_row, int32_t max_len) {
    const int64_t span = (int64_t)max_len + 31;
    const int64_t few = (span + kPagedChunkMax - 1) / kPagedChunkMax, many = (span + kAttnChunkMin - 1) / kAttnChunkMin;
    return std::max(n_rows * few, std::min(n_rows * many, kAttnGroups / per_row + n_rows));
}

int64_t attn_bytes(int64_t parts, int32_t n_q_heads, int32_t head_dim) { return parts * n_q_heads * (head_dim + 2) * 4; }

int prompt_planes(int32_t dtype) { return dtype == VKV_DTYPE_F32 ? 2 : 1; }
int64_t prompt_tiles(int32_t n_seq, int32_t n_tokens, int keys) { return (int64_t)n_tokens / keys + n_seq; }

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

int64_t prompt_info_bytes(int64_t tiles, int32_t n_kv_heads) { return round256(tiles * n_kv_heads * 4); }

// a chunk's (maximum, sum, weighted sum, count) of each of 4 waves
int64_t logprobs_stats_bytes(int64_t chunks) { return chunks * 4 * 16; }

}  // namespace

extern "C" {

vkv_status vkv_page_map(const int32_t *len_old, const int32_t *len_new, int32_t n_req, int32_t page_size,
                        int32_t n_pages, int32_t *table, int32_t table_stride, int32_t *free_pages,
                        const int32_t *n_free, int32_t *n_free_out, int32_t max_tokens, int32_t *len_out,
                        int32_t *cu_new, int32_t *slots, int32_t *positions, int32_t *status, void *hip_stream) {
    const char *what = "page map";
    if (n_req < 1 || n_req > 1 << 24) return bad("%s: %d requests", what, n_req);
    if (!page_size_ok(page_size)) return bad("%s: page size %d (16, 32, 64, 128 or 256)", what, page_size);
    if (n_pages < 1 || (int64_t)n_pages * page_size > INT32_MAX) return bad("%s: %d pages", what, n_pages);
    if (table_stride < 1 || (int64_t)table_stride * page_size > INT32_MAX) return bad("%s: table stride %d", what, table_stride);
    if (max_tokens < 0 || max_tokens >= 1 << 30) return bad("%s: max_tokens %d", what, max_tokens);
    for (const void *p : {(const void *)len_old, (const void *)len_new, (const void *)table, (const void *)free_pages,
                          (const void *)n_free, (const void *)n_free_out, (const void *)len_out, (const void *)cu_new,
                          (const void *)status})
        if (vkv_status s = check_ints(what, p)) return s;
    if (max_tokens > 0)
        for (const void *p : {(const void *)slots, (const void *)positions})
            if (vkv_status s = check_ints(what, p)) return s;
    MapArgs a{len_old, len_new, n_req, page_size, n_pages, table, table_stride, free_pages, n_free, n_free_out,
              max_tokens, len_out, cu_new, slots, positions, status};
    StreamDevice on(as_stream(hip_stream));
    const hipError_t e = launch_page_map(a, as_stream(hip_stream));
    if (e != hipSuccess) return host_hip_fail(e, "page map launch");
    return host_ok();
}

vkv_status vkv_pages_append(const vkv_pages *pages, int32_t layer, const int32_t *slots, int32_t n_tokens,
                            int32_t dtype, const void *k, const void *v, int64_t row_stride, void *hip_stream) {
    const char *what = "pages append";
    if (vkv_status s = check_pages(what, pages, layer)) return s;
    if (!elem_bytes(dtype)) return bad("%s: rows of dtype %d", what, dtype);
    if (n_tokens < 0 || n_tokens >= 1 << 24) return bad("%s: %d tokens", what, n_tokens);
    if (n_tokens == 0) return host_ok();
    if (vkv_status s = check_ints(what, slots)) return s;
    const int64_t width = (int64_t)pages->n_kv_heads * pages->head_dim;
    if (vkv_status s = check_rows(what, "k", k, width, dtype, &row_stride)) return s;
    if (vkv_status s = check_rows(what, "v", v, width, dtype, &row_stride)) return s;
    const int64_t per_head = (int64_t)pages->page_size * pages->head_dim;
    AppendPagesArgs a{};
    a.k_codes = layer_at((uint8_t *)pages->k, pages, layer, per_head);
    a.v_codes = layer_at((uint8_t *)pages->v, pages, layer, per_head);
    a.k_scale = layer_at(pages->k_scale, pages, layer, 1);
    a.v_scale = layer_at(pages->v_scale, pages, layer, 1);
    a.slots = slots;
    a.k = k;
    a.v = v;
    a.row_stride = row_stride;
    a.n_tokens = n_tokens;
    a.n_slots = pages->n_pages * pages->page_size;
    a.page_size = pages->page_size;
    a.n_kv_heads = pages->n_kv_heads;
    StreamDevice on(as_stream(hip_stream));
    const hipError_t e = launch_pages_append(dtype, pages->dtype, pages->head_dim, a, as_stream(hip_stream));
    if (e != hipSuccess) return host_hip_fail(e, "pages append launch");
    return host_ok();
}

size_t vkv_paged_attn_workspace(const vkv_pages *pages, int32_t n_rows, int32_t n_q_heads, int32_t max_len) {
    if (check_pool("paged attention workspace", pages) || n_rows < 0 || max_len < 0 ||
        check_heads("paged attention workspace", n_q_heads, pages->n_kv_heads))
        return 0;
    const int64_t most = attn_parts_most(n_rows, attn_units(1, n_q_heads, pages->n_kv_heads), max_len);
    return (size_t)attn_bytes(most, n_q_heads, pages->head_dim);
}

vkv_status vkv_paged_attn(const vkv_pages *pages, int32_t layer, const int32_t *table, int32_t table_stride,
                          const int32_t *lens, int32_t n_rows, int32_t max_len, int32_t window, int32_t dtype,
                          const void *q, int64_t q_stride, void *out, int64_t out_stride, int32_t n_q_heads,
                          float scale, void *workspace, size_t workspace_bytes, void *hip_stream) {
    const char *what = "paged attention";
    if (vkv_status s = check_pages(what, pages, layer)) return s;
    if (vkv_status s = check_heads(what, n_q_heads, pages->n_kv_heads)) return s;
    if (!elem_bytes(dtype)) return bad("%s: rows of dtype %d", what, dtype);
    if (n_rows < 0 || max_len < 0 || window < 0 || table_stride < 0)
        return bad("%s: %d rows of up to %d tokens, window %d, table stride %d", what, n_rows, max_len, window, table_stride);
    if (table_stride > 0 && max_len > (int64_t)table_stride * pages->page_size)
        return bad("%s: max_len %d beyond %d pages of %d", what, max_len, table_stride, pages->page_size);
    if (max_len > 65535 * kPagedChunkMax - 32) return bad("%s: max_len %d", what, max_len);
    if (!std::isfinite(scale)) return bad("%s: scale", what);
    const int64_t units = attn_units(n_rows, n_q_heads, pages->n_kv_heads);
    if (std::max<int64_t>(units, (int64_t)n_rows * n_q_heads) >= 1 << 24) return bad("%s: %d rows of %d heads", what, n_rows, n_q_heads);
    if (n_rows == 0) return host_ok();
    if (vkv_status s = check_ints(what, table)) return s;
    if (vkv_status s = check_ints(what, lens)) return s;
    const int64_t width = (int64_t)n_q_heads * pages->head_dim;
    if (vkv_status s = check_rows(what, "q", q, width, dtype, &q_stride)) return s;
    if (vkv_status s = check_rows(what, "out", out, width, dtype, &out_stride)) return s;
    PagedAttnArgs a{};
    attn_plan(units, max_len, window, &a.chunk, &a.n_chunks);
    // (a grid has fewer than 2^32 threads)
    if ((units + 8 * (units / n_rows)) * a.n_chunks >= 1 << 24) return bad("%s: %d rows of up to %d tokens", what, n_rows, max_len);
    const int64_t parts = (int64_t)n_rows * n_q_heads * a.n_chunks;
    if (a.n_chunks > 1) {
        const int64_t need = attn_bytes((int64_t)n_rows * a.n_chunks, n_q_heads, pages->head_dim);
        if ((int64_t)workspace_bytes < need) return small_ws(what, workspace_bytes, (size_t)need);
        if (!workspace || !aligned(workspace, 16)) return bad("%s: workspace null or not 16-byte aligned", what);
    }
    const int64_t per_head = (int64_t)pages->page_size * pages->head_dim;
    a.k_codes = layer_at((const uint8_t *)pages->k, pages, layer, per_head);
    a.v_codes = layer_at((const uint8_t *)pages->v, pages, layer, per_head);
    a.k_scale = layer_at((const float *)pages->k_scale, pages, layer, 1);
    a.v_scale = layer_at((const float *)pages->v_scale, pages, layer, 1);
    a.table = table;
    a.lens = lens;
    a.q = q;
    a.out = out;
    a.part_o = (float *)workspace;
    a.part_ml = (float *)workspace + parts * pages->head_dim;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.table_stride = table_stride;
    a.n_rows = n_rows;
    a.max_len = max_len;
    a.window = window;
    a.n_pages = pages->n_pages;
    a.page_size = pages->page_size;
    a.n_kv_heads = pages->n_kv_heads;
    a.n_q_heads = n_q_heads;
    a.scale = scale;
    StreamDevice on(as_stream(hip_stream));
    const hipError_t e = launch_paged_attn(dtype, pages->dtype, pages->head_dim, a, as_stream(hip_stream));
    if (e != hipSuccess) return host_hip_fail(e, "paged attention launch");
    return host_ok();
}

size_t vkv_prompt_attn_workspace(int32_t dtype, int32_t n_seq, int32_t n_tokens, int32_t n_kv_heads, int32_t head_dim) {
    if (!elem_bytes(dtype) || n_seq < 0 || n_tokens < 0 || n_kv_heads < 1 || n_kv_heads > 4096 ||
        (head_dim != 64 && head_dim != 128))
        return 0;
    const int planes = prompt_planes(dtype), keys = prompt_keys(planes, head_dim);
    const int64_t tiles = prompt_tiles(n_seq, n_tokens, keys);
    return (size_t)(prompt_info_bytes(tiles, n_kv_heads) + tiles * n_kv_heads * planes * 2 * keys * head_dim * 2);
}

vkv_status vkv_prompt_attn(int32_t dtype, const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                           const void *v, int64_t v_stride, const int32_t *cu_seqlens, int32_t n_seq, int32_t n_tokens,
                           int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim, float scale, int32_t window,
                           void *out, int64_t out_stride, void *workspace, size_t workspace_bytes, void *hip_stream) {
    const char *what = "prompt attention";
    if (!elem_bytes(dtype)) return bad("%s: rows of dtype %d", what, dtype);
    if (vkv_status s = check_heads(what, n_q_heads, n_kv_heads)) return s;
    if (head_dim != 64 && head_dim != 128) return bad("%s: head dim %d (64 or 128)", what, head_dim);
    if (n_seq < 0 || n_tokens < 0 || window < 0) return bad("%s: %d prompts of %d tokens, window %d", what, n_seq, n_tokens, window);
    if (!std::isfinite(scale)) return bad("%s: scale", what);
    PromptArgs a{};
    const int keys = prompt_keys(prompt_planes(dtype), head_dim);
    a.n_tiles = prompt_tiles(n_seq, n_tokens, keys);
    const int64_t rows = (int64_t)n_tokens * (n_q_heads / n_kv_heads);
    const bool few = (rows / kPromptRows + n_seq) * n_kv_heads <= kPromptGroupsFew && n_tokens > keys;
    a.rows = few ? kPromptRowsFew : kPromptRows;
    a.n_slots = rows / a.rows + n_seq;
    if (a.n_tiles >= 1 << 24 || a.n_slots * n_kv_heads >= 1 << 23) return bad("%s: %d prompts of %d tokens", what, n_seq, n_tokens);
    if (n_seq == 0 || n_tokens == 0) return host_ok();
    if (vkv_status s = check_ints(what, cu_seqlens)) return s;
    const int64_t kv = (int64_t)n_kv_heads * head_dim, width = (int64_t)n_q_heads * head_dim;
    if (vkv_status s = check_rows(what, "q", q, width, dtype, &q_stride)) return s;
    if (vkv_status s = check_rows(what, "k", k, kv, dtype, &k_stride)) return s;
    if (vkv_status s = check_rows(what, "v", v, kv, dtype, &v_stride)) return s;
    if (vkv_status s = check_rows(what, "out", out, width, dtype, &out_stride)) return s;
    const size_t need = vkv_prompt_attn_workspace(dtype, n_seq, n_tokens, n_kv_heads, head_dim);
    if (workspace_bytes < need) return small_ws(what, workspace_bytes, need);
    if (!workspace || !aligned(workspace, 256)) return bad("%s: workspace null or not 256-byte aligned", what);
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.out_stride = out_stride;
    a.cu = cu_seqlens;
    a.n_seq = n_seq;
    a.n_tokens = n_tokens;
    a.n_q_heads = n_q_heads;
    a.n_kv_heads = n_kv_heads;
    a.window = window;
    a.scale = scale;
    a.info = (int32_t *)workspace;
    a.data = (uint8_t *)workspace + prompt_info_bytes(a.n_tiles, n_kv_heads);
    StreamDevice on(as_stream(hip_stream));
    const hipError_t e = launch_prompt_attn(dtype, head_dim, a, as_stream(hip_stream));
    if (e != hipSuccess) return host_hip_fail(e, "prompt attention launch");
    return host_ok();
}

size_t vkv_logprobs_workspace(int32_t n_rows, int64_t n_vocab, int32_t n_top) {
    if (n_rows < 0 || n_vocab < 1 || n_vocab > 1 << 30 || n_top < 0 || n_top > kLogprobsMaxTop) return 0;
    const int64_t most = logprobs_chunks_most(n_rows, n_vocab);
    return (size_t)(logprobs_stats_bytes(most) + most * n_top * 8);
}

vkv_status vkv_logprobs(int32_t dtype, const void *logits, int64_t row_stride, int32_t n_rows, int64_t n_vocab,
                        const int32_t *tokens, float *logprob, float *entropy, int32_t n_top, int32_t *top_ids,
                        float *top_logprobs, void *workspace, size_t workspace_bytes, void *hip_stream) {
    const char *what = "log probabilities";
    const int eb = elem_bytes(dtype);
    if (!eb) return bad("%s: logits of dtype %d", what, dtype);
    if (n_rows < 0 || n_rows > 65535 || n_vocab < 1 || n_vocab > 1 << 30)
        return bad("%s: %d rows of %lld logits", what, n_rows, (long long)n_vocab);
    if (n_top < 0 || n_top > kLogprobsMaxTop || n_top > n_vocab) return bad("%s: n_top %d", what, n_top);
    if (row_stride == 0) row_stride = n_vocab;
    if (row_stride < n_vocab || row_stride > (int64_t)1 << 40) return bad("%s: row stride %lld", what, (long long)row_stride);
    if (!tokens != !logprob) return bad("%s: tokens and logprob go together", what);
    if (n_rows == 0) return host_ok();
    if (!logits || !aligned(logits, 16)) return bad("%s: logits null or not 16-byte aligned", what);
    if (n_top > 0)
        for (const void *p : {(const void *)top_ids, (const void *)top_logprobs})
            if (vkv_status s = check_ints(what, p)) return s;
    if (!aligned(tokens, 4) || !aligned(logprob, 4) || !aligned(entropy, 4))
        return bad("%s: int32 and f32 arrays must be 4-byte aligned", what);
    const LogprobsPlan plan = logprobs_plan(n_rows, n_vocab, eb, n_top, n_rows == 1 || row_stride * eb % 16 == 0);
    const int64_t chunks = (int64_t)n_rows * plan.chunks;
    const int64_t stats = logprobs_stats_bytes(chunks), need = stats + chunks * n_top * 8;
    if ((int64_t)workspace_bytes < need) return small_ws(what, workspace_bytes, (size_t)need);
    if (!workspace || !aligned(workspace, 16)) return bad("%s: workspace null or not 16-byte aligned", what);
    LogprobsArgs a{logits, row_stride, n_rows, (int32_t)n_vocab, n_top, plan.chunks, plan.turns, tokens, logprob, entropy,
                   top_ids, top_logprobs, (float *)workspace, (unsigned long long *)((uint8_t *)workspace + stats)};
    StreamDevice on(as_stream(hip_stream));
    const hipError_t e = launch_logprobs(dtype, a, plan.blocks, as_stream(hip_stream));
    if (e != hipSuccess) return host_hip_fail(e, "log probabilities launch");
    return host_ok();
}

}  // extern "C"
