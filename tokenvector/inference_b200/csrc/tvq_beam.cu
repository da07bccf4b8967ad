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

__device__ __forceinline__ float ex2(float x) {  // 2^x, relative error ~2^-22, 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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

// A float's bits in its order (-0 counts as 0).
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One slice of one row: its maximum m, sum exp(x - m), and its `keep` best
// keys, best first.  Bound: memory, each logit is read once (about ten instructions
// a logit; 128 threads of 64 logits, since finding the bar is quadratic in the
// threads: 256 of 32 took twice the time).  The keep-th largest of the threads'
// best values is a bar that at least `keep` logits reach, and above which only
// keep - 1 threads have any, so one pass collects all that can count and at
// most keep EPT, unless many equal the bar; then those are taken by their
// tokens, chunk by chunk.  The collected are ranked by counting.
// Slices of 8192 logits, or of 2048 while a step has too few rows to fill the
// GPU with the larger ones.
constexpr int SLT = 128;
template <typename T, int EPT>
__global__ void __launch_bounds__(SLT) select_slice_kernel(const BeamSelectArgs a, uint64_t* keys, float2* stats, int slices) {
    constexpr int VEC = 16 / sizeof(T), NV = EPT / VEC;
    extern __shared__ __align__(16) uint64_t found[];  // [keep * EPT]
    __shared__ __align__(16) uint32_t best[SLT];
    __shared__ uint32_t s_bar;
    __shared__ float s_sum[SLT / 32];
    __shared__ int s_n, s_scan[SLT / 32];
    griddep_wait();
    const int r = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const T* row = static_cast<const T*>(a.logits) + r * a.stride;
    // slices start at 16-byte boundaries; tokens outside the row carry numbers that
    // rank (as unsigned) behind every token of it
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int begin = slice * (SLT * EPT) - mis, v0 = begin + tid * VEC;
    const int64_t at = static_cast<int64_t>(r) * slices + slice;
    uint64_t* out = keys + at * a.keep;
    if (a.finished && a.finished[r]) {  // its row counts as 0 at eos, -inf elsewhere
        const int first = max(begin, 0);
        const bool has = a.eos >= first && a.eos < begin + SLT * EPT;
        if (tid < a.keep) {
            int v = first + tid - (has ? 1 : 0);
            if (has && v >= a.eos) v++;
            out[tid] = has && tid == 0 ? order_key(0.0f, a.eos) : order_key(-INFINITY, v);
        }
        if (tid == 0) stats[at] = has ? make_float2(0.0f, 1.0f) : make_float2(-INFINITY, 0.0f);
        return;
    }
    if (tid == 0) {
        s_n = 0;
        s_bar = 0xFFFFFFFFu;
    }
    float x[EPT], top = -INFINITY;
#pragma unroll
    for (int c = 0; c < NV; c++) {
        const int v = v0 + c * SLT * VEC;
        if (v >= 0 && v + VEC <= a.vocab) {
            union { T t[VEC]; uint4 u; } w;
            w.u = __ldcs(reinterpret_cast<const uint4*>(row + v));
#pragma unroll
            for (int e = 0; e < VEC; e++) x[c * VEC + e] = to_f32(w.t[e]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++)
                x[c * VEC + e] = v + e >= 0 && v + e < a.vocab ? to_f32(row[v + e]) : -INFINITY;
        }
    }
#pragma unroll
    for (int i = 0; i < EPT; i++) {
        x[i] = fmaxf(x[i], -INFINITY);  // NaN counts as -inf
        top = fmaxf(top, x[i]);
    }
    const uint32_t mine = order_bits(top);
    best[tid] = mine;
    __syncthreads();
    int above = 0;
    uint32_t most = 0;
#pragma unroll 8
    for (int i = 0; i < SLT; i += 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(best + i);
        above += (w.x > mine) + (w.y > mine) + (w.z > mine) + (w.w > mine);
        most = max(max(most, max(w.x, w.y)), max(w.z, w.w));
    }
    const uint32_t low = __reduce_min_sync(0xffffffffu, above < a.keep ? mine : 0xFFFFFFFFu);
    if ((tid & 31) == 0) atomicMin(&s_bar, low);
    __syncthreads();
    const float m = key_value(static_cast<uint64_t>(most) << 32), bar = key_value(static_cast<uint64_t>(s_bar) << 32);
    const float base = m == -INFINITY ? 0.0f : m;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int cap = a.keep * EPT;
#pragma unroll
    for (int i = 0; i < EPT; i++) {
        sum[i & 3] += ex2((x[i] - base) * 1.4426950408889634f);  // (the difference first: the maximum's term is 1)
        if (x[i] >= bar) {
            const int n = atomicAdd(&s_n, 1);
            if (n < cap) found[n] = order_key(x[i], v0 + i / VEC * SLT * VEC + i % VEC);
        }
    }
    float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) all += __shfl_xor_sync(0xffffffffu, all, w);
    if ((tid & 31) == 0) s_sum[tid >> 5] = all;
    __syncthreads();
    if (tid == 0) {
        all = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
        stats[at] = make_float2(m, all);
    }
    int n = s_n;
    if (n > cap) {  // many equal the bar: those above it, then as many of them as are missing, lowest tokens first
        __syncthreads();
        if (tid == 0) s_n = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EPT; i++)
            if (x[i] > bar) found[atomicAdd(&s_n, 1)] = order_key(x[i], v0 + i / VEC * SLT * VEC + i % VEC);
        __syncthreads();
        n = s_n;
        const int want = n + max(0, a.keep - n);
#pragma unroll
        for (int ch = 0; ch < NV; ch++) {
            int cnt = 0;
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const int v = v0 + ch * SLT * VEC + e;
                cnt += x[ch * VEC + e] == bar && v >= 0 && v < a.vocab;
            }
            int inc = cnt;
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, inc, o);
                if ((tid & 31) >= o) inc += y;
            }
            __syncthreads();
            if ((tid & 31) == 31) s_scan[tid >> 5] = inc;
            __syncthreads();
            int before = n + inc - cnt, total = 0;
            for (int w = 0; w < SLT / 32; w++) {
                if (w < (tid >> 5)) before += s_scan[w];
                total += s_scan[w];
            }
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const int v = v0 + ch * SLT * VEC + e;
                if (x[ch * VEC + e] == bar && v >= 0 && v < a.vocab) {
                    if (before < want) found[before] = order_key(bar, v);
                    before++;
                }
            }
            n = min(want, n + total);
            if (n == want) break;
        }
        __syncthreads();
    }
    for (int i = tid; i < n; i += SLT) {
        const uint64_t key = found[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += found[j] > key;
        if (rank < a.keep) out[rank] = key;
    }
    // (a slice with fewer logits than `keep`: places behind every token's)
    if (tid >= n && tid < a.keep) out[tid] = order_key(-INFINITY, 0x80000000u + tid);
}

// A candidate's place in its request's order: total, then the lower beam, then
// its place in the beam's list.
struct Place {
    uint64_t hi, lo;
    __device__ bool above(const Place& o) const { return hi > o.hi || (hi == o.hi && lo > o.lo); }
};

// One request: the `keep` best of its beams' slices' lists.  (A candidate that
// is not among its beam's `keep` best has that many above it in any case.)
// The same bar: the keep-th largest of the lists' heads, found among the
// threads' best heads first, leaves candidates of at most `keep` lists.
// Bound: latency; a few rounds through L2.
constexpr int ST = 256;
__global__ void __launch_bounds__(ST) select_merge_kernel(const BeamSelectArgs a, const uint64_t* keys,
                                                          const float2* stats, int slices, int heads_cap) {
    extern __shared__ __align__(16) uint8_t sm[];
    Place* best = reinterpret_cast<Place*>(sm);  // [ST]
    Place* heads = best + ST;                    // [heads_cap]
    Place* found = heads + heads_cap;            // [min(lists, keep) keep]
    __shared__ float s_score[64], s_max[64], s_z[64];
    __shared__ Place s_bar;
    __shared__ int s_n[2];
    const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();
    for (int w = warp; w < a.beams; w += ST / 32) {
        const float2* st = stats + (static_cast<int64_t>(b) * a.beams + w) * slices;
        float m = -INFINITY, sum = 0.0f;
        for (int i = lane; i < slices; i += 32) m = fmaxf(m, st[i].x);
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        for (int i = lane; i < slices; i += 32) sum += st[i].y * expf(st[i].x - m);
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            s_score[w] = a.scores[b * a.beams + w];
            s_max[w] = m;
            s_z[w] = logf(sum);
        }
    }
    if (tid < 2) s_n[tid] = 0;
    __syncthreads();
    const int lists = a.beams * slices;
    const uint64_t* mine = keys + static_cast<int64_t>(b) * lists * a.keep;
    auto place = [&](int list, int i) {
        const int w = list / slices;
        Place p;
        p.lo = mine[static_cast<int64_t>(list) * a.keep + i];
        float total = s_score[w] + ((key_value(p.lo) - s_max[w]) - s_z[w]);
        if (total != total) total = -INFINITY;
        p.hi = order_key(total, w);
        return p;
    };
    auto rank_of = [](const Place* all, int n, const Place& p) {
        int rank = 0;
        for (int i = 0; i < n; i++) rank += all[i].above(p);
        return rank;
    };
    Place top{0, 0};
    for (int l = tid; l < lists; l += ST) {
        const Place p = place(l, 0);
        if (p.above(top)) top = p;
    }
    best[tid] = top;
    if (tid == 0) s_bar = Place{0, 0};
    __syncthreads();
    const int threads = min(lists, ST);
    if (tid < threads && rank_of(best, threads, top) == a.keep - 1) s_bar = top;
    __syncthreads();
    if (lists > ST) {  // the bar among all heads that reach the one among the threads'
        Place bar = s_bar;
        for (int l = tid; l < lists; l += ST) {
            const Place p = place(l, 0);
            if (!bar.above(p)) heads[atomicAdd(&s_n[1], 1)] = p;
        }
        __syncthreads();
        const int n = s_n[1];
        for (int i = tid; i < n; i += ST)
            if (rank_of(heads, n, heads[i]) == a.keep - 1) s_bar = heads[i];
        __syncthreads();
    }
    const Place bar = s_bar;
    for (int64_t c = tid; c < static_cast<int64_t>(lists) * a.keep; c += ST) {
        const int l = static_cast<int>(c / a.keep);
        const Place p = place(l, static_cast<int>(c - static_cast<int64_t>(l) * a.keep));
        if (!bar.above(p)) found[atomicAdd(&s_n[0], 1)] = p;
    }
    __syncthreads();
    const int n = s_n[0];
    for (int i = tid; i < n; i += ST) {
        const Place p = found[i];
        const int rank = rank_of(found, n, p);
        if (rank >= a.keep) continue;
        const int o = b * a.keep + rank;
        a.out_scores[o] = key_value(p.hi);
        a.out_tokens[o] = key_token(p.lo);
        a.out_parents[o] = key_token(p.hi);
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

namespace {

// Slices of a step's rows: 8192 logits each, 2048 while that leaves some of
// the 148 SMs without one.
constexpr int kSms = 148;
struct Slices {
    int ept, n, heads_cap, found_cap;
    int64_t keys, bytes;  // of the workspace: the lists', all
};
Slices slices_of(const BeamSelectArgs& a) {
    Slices s;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.beams;
    // (a row may start up to 15 bytes behind a 16-byte boundary: 7 logits of 2 bytes)
    auto count = [&](int ept) { return (a.vocab + 7 + SLT * ept - 1) / (SLT * ept); };
    s.ept = rows * count(64) < kSms ? 16 : 64;
    s.n = count(s.ept);
    const int lists = a.beams * s.n;
    s.heads_cap = lists > ST ? std::min(lists, a.keep * ((lists + ST - 1) / ST)) : 0;
    s.found_cap = std::min(lists, a.keep) * a.keep;
    s.keys = up256(rows * s.n * a.keep * 8);
    s.bytes = s.keys + up256(rows * s.n * 8);
    return s;
}

template <typename T, int EPT>
int launch_slices(const BeamSelectArgs& a, const Slices& s, uint64_t* keys, float2* stats, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>(s.n), static_cast<unsigned>(a.batch * a.beams));
    return launch_pdl(select_slice_kernel<T, EPT>, grid, dim3(SLT), static_cast<size_t>(a.keep) * EPT * 8, st, a, keys,
                      stats, s.n);
}

template <typename T>
int launch_select(const BeamSelectArgs& a, const Slices& s, cudaStream_t st) {
    uint64_t* keys = static_cast<uint64_t*>(a.ws);
    float2* stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(a.ws) + s.keys);
    const int rc = s.ept == 16 ? launch_slices<T, 16>(a, s, keys, stats, st) : launch_slices<T, 64>(a, s, keys, stats, st);
    if (rc) return rc;
    const size_t smem = (ST + s.heads_cap + s.found_cap) * sizeof(Place);
    static const cudaError_t attr =
        cudaFuncSetAttribute(select_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    TVQ_CUDA(attr);
    return launch_pdl(select_merge_kernel, dim3(static_cast<unsigned>(a.batch)), dim3(ST), smem, st, a, keys, stats, s.n,
                      s.heads_cap);
}

}  // namespace

int beam_select_workspace(const BeamSelectArgs& a, int64_t* bytes) {
    *bytes = slices_of(a).bytes;
    return TVQ_OK;
}

int launch_beam_select(const BeamSelectArgs& a, cudaStream_t st) {
    const Slices s = slices_of(a);
    if (a.type == TVQ_TYPE_F32) return launch_select<float>(a, s, st);
    if (a.type == TVQ_TYPE_F16) return launch_select<__half>(a, s, st);
    return launch_select<__nv_bfloat16>(a, s, st);
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
