// Arguments and launches of the batched serving operators (vkv_pages.hip,
// vkv_prompt.hip, vkv_logprobs.hip), called by vkv_serve.cpp.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "vkv.h"

namespace vkv {

struct MapArgs {
    const int32_t *len_old, *len_new;
    int32_t n_req, page_size, n_pages;
    int32_t *table;
    int32_t table_stride;
    int32_t *free_pages;
    const int32_t *n_free;
    int32_t *n_free_out;
    int32_t max_tokens;
    int32_t *len_out, *cu_new, *slots, *positions, *status;
};

hipError_t launch_page_map(const MapArgs &a, hipStream_t st);

struct AppendPagesArgs {
    uint8_t *k_codes, *v_codes;    // of the layer
    float *k_scale, *v_scale;
    const int32_t *slots;
    const void *k, *v;
    int64_t row_stride;
    int32_t n_tokens, n_slots, page_size, n_kv_heads;
    int32_t looks;         // tokens that a work group looks at for first ones of their page (<= 64)
};
hipError_t launch_pages_append(int dtype, int code, int head_dim, const AppendPagesArgs &a, hipStream_t st);

// Keys per work group of the paged attention: a multiple of the 128 keys its
// waves take at once, and at most 64 blocks of 16 (one per lane).
constexpr int kPagedChunkStep = 128, kPagedChunkMax = 1024;

struct PagedAttnArgs {
    const uint8_t *k_codes, *v_codes;   // of the layer
    const float *k_scale, *v_scale;
    const int32_t *table;
    const int32_t *lens;
    const void *q;
    void *out;
    float *part_o;         // [row][query head][chunk][head_dim], not normalised
    float *part_ml;        // [row][query head][chunk] (maximum in log2 units, sum)
    int64_t q_stride, out_stride;
    int32_t table_stride, n_rows, max_len, window, n_pages, page_size, n_kv_heads, n_q_heads;
    int32_t chunk, n_chunks;
    float scale;
};

hipError_t launch_paged_attn(int dtype, int code, int head_dim, const PagedAttnArgs &a, hipStream_t st);

// Causal attention of packed prompts (vkv_prompt.hip).
// (token, query head of a kv head) rows per work group, and where they are few
constexpr int kPromptRows = 128, kPromptRowsFew = 32;
// Keys per tile: of K and V, `planes` 16-bit planes each, two tiles take 64 KiB
constexpr int prompt_keys(int planes, int head_dim) { return planes * head_dim <= 128 ? 64 : 32; }

struct PromptArgs {
    const void *q, *k, *v;
    void *out;
    int64_t q_stride, k_stride, v_stride, out_stride;
    const int32_t *cu;
    int32_t n_seq, n_tokens, n_q_heads, n_kv_heads, window;
    int64_t n_tiles;       // key tiles of a kv head
    int32_t rows;          // of a query tile
    int64_t n_slots;       // query tiles of a kv head
    float scale;
    int32_t *info;         // [kv head][tile]: exponents of K and V, whether V holds what is not finite
    uint8_t *data;         // [kv head][tile]: the tile's matrix operands
};

hipError_t launch_prompt_attn(int dtype, int head_dim, const PromptArgs &a, hipStream_t st);

// Log probabilities (vkv_logprobs.hip).
constexpr int kLogprobsMaxTop = 32;

struct LogprobsArgs {
    const void *logits;
    int64_t row_stride;
    int32_t n_rows, n_vocab, n_top, n_chunks, turns;
    const int32_t *tokens;
    float *logprob, *entropy;
    int32_t *top_ids;
    float *top_logprobs;
    float *stats;                       // [row][chunk][4 waves][4]: maximum, sum, weighted sum
    unsigned long long *keys;           // [row][chunk][n_top]
};

// 16-byte blocks per thread and piece, pieces per chunk, chunks per row;
// rows_aligned: every row begins at a 16-byte boundary
struct LogprobsPlan {
    int32_t blocks, turns, chunks;
};
LogprobsPlan logprobs_plan(int n_rows, int64_t n_vocab, int elem_bytes, int n_top, bool rows_aligned);
// no fewer chunks than any plan of so many rows, or of fewer, has
int64_t logprobs_chunks_most(int64_t n_rows, int64_t n_vocab);
hipError_t launch_logprobs(int dtype, const LogprobsArgs &a, int blocks, hipStream_t st);

}  // namespace vkv
