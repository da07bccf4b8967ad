// tvq_decode.h -- internal launcher declarations of the decoding operators
// (paged cache, beam search); the exported surface is include/tvq.h.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tvq {

// One layer's paged cache and the sequences in it.  Strides are in elements;
// a token's head_dim values are contiguous.
struct PagedView {
    int type = 0;  // TVQ_TYPE_F16 or TVQ_TYPE_BF16
    void* k = nullptr;
    void* v = nullptr;
    int64_t n_pages = 0;
    int page = 0, page_log2 = 0;  // tokens per page (a power of two)
    int kv_heads = 0, dim = 0;
    int64_t k_page = 0, k_tok = 0, k_head = 0, v_page = 0, v_tok = 0, v_head = 0;
    const int32_t* table = nullptr;  // [n_seq, n_cols] page numbers, rows table_stride apart
    int64_t table_stride = 0;
    int n_cols = 0;
    const int32_t* ctx = nullptr;  // [n_seq] tokens in the cache, the new ones included
    const int32_t* cu = nullptr;   // [n_seq + 1] first packed row of each sequence, or null: one row each
    int n_seq = 0;
    int n_rows = 0;
};

struct AppendArgs {
    PagedView c;
    int src_type = 0;  // TVQ_TYPE_*
    const void *k = nullptr, *v = nullptr, *q = nullptr;
    int64_t k_tok = 0, k_head = 0, v_tok = 0, v_head = 0, q_tok = 0, q_head = 0;
    int q_heads = 0;
    void* q_out = nullptr;  // [n_rows, q_heads, dim] in the cache's type
};
int launch_paged_append(const AppendArgs& a, cudaStream_t st);

struct PagedAttnArgs {
    PagedView c;
    const void* q = nullptr;
    int64_t q_tok = 0, q_head = 0;
    int q_heads = 0;
    int max_q = 0;   // no sequence has more new rows
    int window = 0;  // 0: every earlier key; w > 0: the last w keys, the row's own among them
    float scale = 0.0f;
    void* out = nullptr;   // [n_rows, q_heads, dim]
    float* lse = nullptr;  // [n_rows, q_heads] or null
    void* ws = nullptr;
    int64_t ws_bytes = 0;
};
int paged_attention_workspace(const PagedAttnArgs& a, int64_t* bytes);
int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st);

struct BeamSelectArgs {
    int type = 0;  // logits: TVQ_TYPE_*
    const void* logits = nullptr;
    int64_t stride = 0;
    const float* scores = nullptr;
    const uint8_t* finished = nullptr;  // [batch * beams] or null
    int batch = 0, beams = 0, keep = 0, vocab = 0, eos = 0;
    float* out_scores = nullptr;
    int64_t* out_tokens = nullptr;
    int32_t* out_parents = nullptr;
    void* ws = nullptr;
    int64_t ws_bytes = 0;
};
int beam_select_workspace(const BeamSelectArgs& a, int64_t* bytes);
int launch_beam_select(const BeamSelectArgs& a, cudaStream_t st);

struct BeamReorderArgs {
    const int32_t* table = nullptr;
    int64_t table_stride = 0;
    const int32_t* lens = nullptr;
    int rows = 0, cols = 0;
    const int32_t* parents = nullptr;
    int new_rows = 0;
    const int32_t* refs = nullptr;
    int64_t n_pages = 0;
    int32_t* new_table = nullptr;  // [new_rows, cols]
    int32_t* new_lens = nullptr;
    int32_t* new_refs = nullptr;
    int32_t* status = nullptr;  // [2]: pages taken, rows without room
    // the cache of every layer: [layers, n_pages, page, kv_heads, dim], strides in elements of 2 bytes
    void *k = nullptr, *v = nullptr;
    int layers = 0, page = 0, kv_heads = 0, dim = 0;
    int64_t k_layer = 0, k_page = 0, k_tok = 0, k_head = 0, v_layer = 0, v_page = 0, v_tok = 0, v_head = 0;
    void* ws = nullptr;
    int64_t ws_bytes = 0;
};
int beam_reorder_workspace(const BeamReorderArgs& a, int64_t* bytes);
int launch_beam_reorder(const BeamReorderArgs& a, cudaStream_t st);

}  // namespace tvq
