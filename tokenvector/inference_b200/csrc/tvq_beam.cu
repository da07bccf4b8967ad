// tvq_beam.cu -- beam search on the device: the choice of the best (beam,
// token) pairs out of a step's logits, and the reordering of the beams' paged
// caches that follows it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "tvq_common.cuh"
#include "tvq_decode.h"

namespace tvq {

namespace {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// ---------------------------------------------------------------- selection
// A logit's place in its row's order as one 64-bit key: the value's bits,
// made monotone, above; the complement of the token below, so that equal
// values go to the lowest token and no two keys of a row are equal.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t token) {
    uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (static_cast<uint64_t>(b) << 32) | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t b = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);
}
__device__ __forceinline__ uint32_t key_token(uint64_t key) { return 0xFFFFFFFFu - static_cast<uint32_t>(key); }

// The logit as the selection sees it: NaN is a masked token; a finished beam
// has only its end token.
template <typename T>
__device__ __forceinline__ float seen_logit(const T* row, int v, bool done, int eos) {
    if (done) return v == eos ? 0.0f : -INFINITY;
    const float x = to_f32(row[v]);
    return x != x ? -INFINITY : x;
}

template <typename U>
__device__ U block_max(U x, U* sm) {
    for (int w = 16; w > 0; w >>= 1) {
        const U y = __shfl_xor_sync(0xffffffffu, x, w);
        x = x > y ? x : y;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = x;
    __syncthreads();
    x = sm[0];
    for (int i = 1; i < static_cast<int>(blockDim.x >> 5); i++) x = sm[i] > x ? sm[i] : x;
    return x;
}

// The plain kernel of one row: its maximum, ln sum exp(x - max), then its
// `keep` best one after another, each the largest key below the one before.
template <typename T>
__global__ void __launch_bounds__(256) select_row_kernel(const BeamSelectArgs a, uint64_t* keys, float2* stats) {
    __shared__ uint64_t sm_k[8];
    __shared__ float sm_f[8];
    griddep_wait();
    const int r = blockIdx.x;
    const T* row = static_cast<const T*>(a.logits) + r * a.stride;
    const bool done = a.finished && a.finished[r];
    float m = -INFINITY;
    for (int v = threadIdx.x; v < a.vocab; v += 256) m = fmaxf(m, seen_logit(row, v, done, a.eos));
    m = block_max(m, sm_f);
    float sum = 0.0f;
    for (int v = threadIdx.x; v < a.vocab; v += 256) sum += expf(seen_logit(row, v, done, a.eos) - m);
    for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm_f[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        float t = 0.0f;
        for (int i = 0; i < 8; i++) t += sm_f[i];
        stats[r] = make_float2(m, logf(t));
    }
    uint64_t below = ~0ull;
    for (int k = 0; k < a.keep; k++) {
        uint64_t best = 0;
        for (int v = threadIdx.x; v < a.vocab; v += 256) {
            const uint64_t key = order_key(seen_logit(row, v, done, a.eos), v);
            if (key < below && key > best) best = key;
        }
        below = block_max(best, sm_k);
        if (threadIdx.x == 0) keys[static_cast<int64_t>(r) * a.keep + k] = below;
    }
}

// One request: the totals of its beams' lists, and the `keep` best of them.
__global__ void __launch_bounds__(256) select_merge_kernel(const BeamSelectArgs a, const uint64_t* keys,
                                                           const float2* stats) {
    __shared__ uint64_t sm_k[8];
    griddep_wait();
    const int b = blockIdx.x, n = a.beams * a.keep;
    uint64_t below = ~0ull;
    for (int k = 0; k < a.keep; k++) {
        uint64_t best = 0;
        for (int c = threadIdx.x; c < n; c += 256) {
            const int r = b * a.beams + c / a.keep;
            const float2 st = stats[r];
            const float x = key_value(keys[static_cast<int64_t>(b) * n + c]);
            float total = a.scores[r] + ((x - st.x) - st.y);
            if (total != total) total = -INFINITY;
            const uint64_t key = order_key(total, c);
            if (key < below && key > best) best = key;
        }
        below = block_max(best, sm_k);
        if (threadIdx.x == 0) {
            const int c = static_cast<int>(key_token(below)), o = b * a.keep + k;
            a.out_scores[o] = key_value(below);
            a.out_tokens[o] = key_token(keys[static_cast<int64_t>(b) * n + c]);
            a.out_parents[o] = c / a.keep;
        }
    }
}

// ---------------------------------------------------------------- reordering
// A copy that a row needs: page `src` -> page `dst` (or -1: none).
struct PageCopy {
    int src, dst, fill;
};

__device__ int block_scan(int x, int* sm, int* total) {  // exclusive, 1024 threads
    int inc = x;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) sm[w] = inc;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < 32; i++) {
        if (i < w) before += sm[i];
        all += sm[i];
    }
    *total = all;
    return before + inc - x;
}

// Tables, lengths, counts and the list of copies, by one CTA.
__global__ void __launch_bounds__(1024) reorder_tables_kernel(const BeamReorderArgs a, int* held, int* tails,
                                                              int* freelist, PageCopy* copies, int* err) {
    __shared__ int sm[32];
    griddep_wait();
    const int t = threadIdx.x;
    for (int64_t i = t; i < a.n_pages; i += 1024) {
        held[i] = 0;
        a.new_refs[i] = a.refs[i];
    }
    __syncthreads();
    auto used = [&](int len) { return min(a.cols, (len + a.page - 1) / a.page); };
    for (int64_t e = t; e < static_cast<int64_t>(a.rows) * a.cols; e += 1024) {
        const int r = static_cast<int>(e / a.cols), c = static_cast<int>(e - static_cast<int64_t>(r) * a.cols);
        const int pg = a.table[r * a.table_stride + c];
        if (c < used(a.lens[r]) && pg >= 0 && pg < a.n_pages) {
            atomicAdd(held + pg, 1);
            atomicSub(a.new_refs + pg, 1);
        }
    }
    // a row's tail page: >= 0 part-filled, -1 none (the row ends with a page), -2 no parent
    for (int r = t; r < a.new_rows; r += 1024) {
        const int q = a.parents[r];
        if (q >= a.rows) record_error(err, DEVERR_BAD_INDEX);
        const bool live = q >= 0 && q < a.rows;
        const int len = live ? a.lens[q] : 0, fill = len % a.page, at = len / a.page;
        int tail = live ? -1 : -2;
        if (live && fill > 0 && at < a.cols) {
            tail = a.table[q * a.table_stride + at];
            if (tail < 0 || tail >= a.n_pages) {
                record_error(err, DEVERR_BAD_PAGE);
                tail = -1;
            }
        }
        tails[r] = tail;
        a.new_lens[r] = len;
    }
    __syncthreads();
    int need = 0;
    for (int r0 = 0; r0 < a.new_rows; r0 += 1024) {
        const int r = r0 + t;
        bool fresh = false;
        if (r < a.new_rows && tails[r] > -2) {
            bool keeps = tails[r] >= 0 && a.refs[tails[r]] == held[tails[r]];
            for (int o = 0; keeps && o < r; o++) keeps = tails[o] != tails[r];
            fresh = !keeps && a.new_lens[r] / a.page < a.cols;
        }
        int all;
        const int rank = need + block_scan(fresh ? 1 : 0, sm, &all);
        if (r < a.new_rows) copies[r].dst = fresh ? rank : -1;  // its turn in the free list, for now
        need += all;
    }
    __syncthreads();
    int found = 0;
    for (int64_t i0 = 0; i0 < a.n_pages && found < need; i0 += 1024) {
        const int64_t i = i0 + t;
        const bool is_free = i < a.n_pages && a.refs[i] == 0;
        int all;
        const int rank = found + block_scan(is_free ? 1 : 0, sm, &all);
        if (is_free && rank < need) freelist[rank] = static_cast<int>(i);
        found += all;
    }
    __syncthreads();
    int short_of = 0;
    for (int r0 = 0; r0 < a.new_rows; r0 += 1024) {
        const int r = r0 + t;
        bool none = false;
        if (r < a.new_rows) {
            const int turn = copies[r].dst, len = a.new_lens[r], fill = len % a.page;
            const bool keeps = fill > 0 && turn < 0 && tails[r] >= 0;
            const int pg = turn >= 0 && turn < found ? freelist[turn] : -1;
            none = tails[r] > -2 && !keeps && pg < 0;
            copies[r] = PageCopy{tails[r], tails[r] >= 0 ? pg : -1, fill};
            const int q = a.parents[r], n = tails[r] > -2 ? used(len) : 0;
            for (int c = 0; c < a.cols; c++) {
                int e = c < n ? a.table[q * a.table_stride + c] : -1;
                if (c == len / a.page && tails[r] > -2 && !keeps) e = pg;
                a.new_table[static_cast<int64_t>(r) * a.cols + c] = e;
                if (e >= 0 && e < a.n_pages) atomicAdd(a.new_refs + e, 1);
            }
        }
        int all;
        block_scan(none ? 1 : 0, sm, &all);
        short_of += all;
    }
    if (t == 0) {
        a.status[0] = min(need, found);
        a.status[1] = short_of;
    }
}

// The filled part of the pages that rows copy, every layer, keys and values.
__global__ void __launch_bounds__(256) reorder_copy_kernel(const BeamReorderArgs a, const PageCopy* copies) {
    griddep_wait();
    const PageCopy c = copies[blockIdx.x];
    if (c.dst < 0) return;
    const int layer = blockIdx.y >> 1, d8 = a.dim / 8, per = a.kv_heads * d8;
    const bool v = blockIdx.y & 1;
    uint16_t* base = static_cast<uint16_t*>(v ? a.v : a.k) + layer * (v ? a.v_layer : a.k_layer);
    const int64_t page = v ? a.v_page : a.k_page, tok = v ? a.v_tok : a.k_tok, head = v ? a.v_head : a.k_head;
    for (int i = threadIdx.x; i < c.fill * per; i += 256) {
        const int t = i / per, h = (i - t * per) / d8, e = i - t * per - h * d8;
        const int64_t o = t * tok + h * head + e * 8;
        *reinterpret_cast<uint4*>(base + c.dst * page + o) = *reinterpret_cast<const uint4*>(base + c.src * page + o);
    }
}

int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

}  // namespace

int beam_select_workspace(const BeamSelectArgs& a, int64_t* bytes) {
    const int64_t rows = static_cast<int64_t>(a.batch) * a.beams;
    *bytes = up256(rows * a.keep * 8) + up256(rows * 8);
    return TVQ_OK;
}

int launch_beam_select(const BeamSelectArgs& a, cudaStream_t st) {
    const int64_t rows = static_cast<int64_t>(a.batch) * a.beams;
    uint64_t* keys = static_cast<uint64_t*>(a.ws);
    float2* stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(a.ws) + up256(rows * a.keep * 8));
    int rc;
    const dim3 grid(static_cast<unsigned>(rows));
    if (a.type == TVQ_TYPE_F32) rc = launch_pdl(select_row_kernel<float>, grid, dim3(256), 0, st, a, keys, stats);
    else if (a.type == TVQ_TYPE_F16) rc = launch_pdl(select_row_kernel<__half>, grid, dim3(256), 0, st, a, keys, stats);
    else rc = launch_pdl(select_row_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, a, keys, stats);
    if (rc) return rc;
    return launch_pdl(select_merge_kernel, dim3(static_cast<unsigned>(a.batch)), dim3(256), 0, st, a, keys, stats);
}

int beam_reorder_workspace(const BeamReorderArgs& a, int64_t* bytes) {
    *bytes = up256(a.n_pages * 4) + 2 * up256(a.new_rows * 4ll) + up256(a.new_rows * 12ll);
    return TVQ_OK;
}

int launch_beam_reorder(const BeamReorderArgs& a, cudaStream_t st) {
    int rc = 0;
    DeviceState* ds = device_state(&rc);
    if (!ds) return rc;
    uint8_t* w = static_cast<uint8_t*>(a.ws);
    int* held = reinterpret_cast<int*>(w);
    int* tails = reinterpret_cast<int*>(w + up256(a.n_pages * 4));
    int* freelist = reinterpret_cast<int*>(w + up256(a.n_pages * 4) + up256(a.new_rows * 4ll));
    PageCopy* copies = reinterpret_cast<PageCopy*>(w + up256(a.n_pages * 4) + 2 * up256(a.new_rows * 4ll));
    rc = launch_pdl(reorder_tables_kernel, dim3(1), dim3(1024), 0, st, a, held, tails, freelist, copies, ds->d_error);
    if (rc || a.new_rows == 0 || a.layers == 0) return rc;
    return launch_pdl(reorder_copy_kernel, dim3(a.new_rows, 2 * a.layers), dim3(256), 0, st, a, copies);
}

}  // namespace tvq
