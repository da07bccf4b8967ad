// tvq_beam.cu -- beam search on the device: the choice of the best (beam,
// token) pairs out of a step's logits, and the reordering of the beams' paged
// caches that follows it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "tvq_common.cuh"
#include "tvq_decode.h"

namespace tvq {

namespace {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

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

// Slices of the rows: each one's maximum m, sum exp(x - m), and its `keep`
// best keys, best first.  Each logit is read once; a slice's steps are short
// and follow one another (5026 f32 logits ~4 us with six CTAs on an SM, issue
// slots 56 % busy), so a pass takes what one logit needs and the rest is paid
// once a slice.  Measured with the merge: 256 rows of 50257 f32 22 us (f16 21:
// it is not the bytes), 1024 rows 52 us (4.0 TB/s), 4 rows 8.6 us.  Six CTAs an SM go over the slices,
// with a 32 KB buffer each that one bulk copy fills as soon as the slice before
// has been looked through; between them there is always some at work.
//   pass 1  the best value of every group of 4 threads (2 for keep > 32)
//   bar     the keep-th largest of those 32 (64): at least `keep` logits reach it
//   pass 2  the sum, and which logits reach the bar: hardly more than `keep`
//           (22 of 5000 at keep 16); they are collected and ranked by counting
// If more reach it than the list holds (many equal logits, or the best ones
// side by side), the bar is raised to the keep-th largest value by bisection,
// and those that equal it are taken by their tokens.
constexpr int SLT = 128;                 // threads
constexpr int SBUF = 32768;              // bytes of a slice
constexpr int SMAX = SBUF / 4 - 8;       // logits of a slice, so that a thread has whole words of at most 64 in all
constexpr int SCAP = 512;                // logits that reach the bar
template <typename T>
__global__ void __launch_bounds__(SLT) select_slice_kernel(const BeamSelectArgs a, uint64_t* keys, float2* stats,
                                                           int slices, int width, int* err) {
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ __align__(128) uint8_t sm[];  // the slice, then found[SCAP]
    uint64_t* found = reinterpret_cast<uint64_t*>(sm + SBUF);
    __shared__ __align__(16) uint32_t best[64];
    __shared__ __align__(8) uint64_t full;
    __shared__ float s_sum[SLT / 32];
    __shared__ int s_n, s_scan[SLT / 32];
    const int tid = threadIdx.x, rows = a.batch * a.beams, items = rows * slices;
    const int per = a.keep <= 32 ? 4 : 2;  // threads of a group
    if (tid == 0) {
        mbar_init(&full, 1);
        fence_barrier_init();
    }
    __syncthreads();
    griddep_wait();
    griddep_launch();  // the merge's CTAs get in place as the last slices run

    // A slice: tokens [first, end) of row r, copied as the 16-byte words that hold them, as far as these lie
    // within the logits (the rest of the first and last word of all is read one by one).
    const uintptr_t lo = reinterpret_cast<uintptr_t>(a.logits);
    const uintptr_t hi = lo + ((rows - 1) * a.stride + a.vocab) * sizeof(T);
    struct Slice {
        int r, first, end;
        uintptr_t from, word;  // address of token `first`; of the first word's start
        bool done;
    };
    auto slice_of = [&](int item) {
        Slice s;
        s.r = item / slices;
        s.first = (item - s.r * slices) * width;
        s.end = min(a.vocab, s.first + width);
        s.from = lo + (s.r * a.stride + s.first) * sizeof(T);
        s.word = s.from & ~uintptr_t(15);
        s.done = s.first >= s.end || (a.finished && a.finished[s.r]);
        return s;
    };
    auto fetch = [&](const Slice& s) {  // by thread 0
        if (s.done) return;
        const uintptr_t a0 = s.word < lo ? s.word + 16 : s.word;
        const uintptr_t past = (s.from + (s.end - s.first) * sizeof(T) + 15) & ~uintptr_t(15);
        const uintptr_t a1 = past > hi ? past - 16 : past;
        if (a1 > a0) {
            mbar_arrive_expect_tx(&full, static_cast<uint32_t>(a1 - a0));
            bulk_load(sm + (a0 - s.word), reinterpret_cast<const void*>(a0), static_cast<uint32_t>(a1 - a0), &full);
        } else {
            mbar_arrive(&full);
        }
    };
    uint32_t phase = 0;
    Slice next{};
    if (static_cast<int>(blockIdx.x) < items) {
        next = slice_of(blockIdx.x);
        if (tid == 0) fetch(next);
    }
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const Slice s = next;
        const bool more = item + static_cast<int>(gridDim.x) < items;
        if (more) next = slice_of(item + gridDim.x);
        uint64_t* out = keys + static_cast<int64_t>(item) * a.keep;
        if (s.done) {  // a finished row counts as 0 at eos, -inf elsewhere
            const bool has = a.eos >= s.first && a.eos < s.end;
            if (tid < a.keep) {
                int v = s.first + tid - (has ? 1 : 0);
                if (has && v >= a.eos) v++;
                // (a slice with fewer tokens than `keep`: places behind every token's)
                const bool real = v < s.end;
                out[tid] = has && tid == 0 ? order_key(0.0f, a.eos) : order_key(-INFINITY, real ? v : 0x80000000u + tid);
            }
            if (tid == 0) stats[item] = has ? make_float2(0.0f, 1.0f) : make_float2(-INFINITY, 0.0f);
            if (more && tid == 0) fetch(next);
            continue;
        }
        const int skip = static_cast<int>((s.from - s.word) / sizeof(T));  // entry e of the buffer is token first - skip + e
        const int count = s.end - s.first, words = (skip + count + VEC - 1) / VEC;
        T* data = reinterpret_cast<T*>(sm);
        if (!mbar_wait_for(&full, phase, nullptr, 0, TVQ_WAIT_LIMIT_NS)) record_error(err, DEVERR_TIMEOUT_ROWS);
        phase ^= 1;
        // the words that reach out of the slice: -inf there, and what the copy left out
        if (tid < 2 * VEC) {
            const int e = tid < VEC ? tid : (words - 1) * VEC + tid - VEC;
            const bool in = e >= skip && e < skip + count;
            const uintptr_t at = s.word + e / VEC * 16;
            if (!in) data[e] = from_f32<T>(-INFINITY);
            else if (at < lo || at + 16 > hi) data[e] = reinterpret_cast<const T*>(s.word)[e];
            fence_proxy_async_smem();  // (before the next copy into the buffer)
        }
        if (tid == 0) s_n = 0;
        __syncthreads();
        float top = -INFINITY;
#pragma unroll 4
        for (int w = tid; w < words; w += SLT) {
            union { T t[VEC]; uint4 u; } x;
            x.u = reinterpret_cast<const uint4*>(data)[w];
#pragma unroll
            for (int e = 0; e < VEC; e++) top = fmaxf(top, to_f32(x.t[e]));  // (NaN counts as -inf)
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        if (per == 4) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (tid % per == 0) best[tid / per] = order_bits(top);
        __syncthreads();
        // every warp: a lane's place among the groups' tops, and the lowest of those that have fewer than
        // `keep` above them
        const int lane = tid & 31;
        uint32_t low = 0xFFFFFFFFu, most = 0;
        for (int g = lane; g < SLT / per; g += 32) {
            const uint32_t mine = best[g];
            int above = 0;
#pragma unroll 8
            for (int i = 0; i < SLT / per; i += 4) {
                const uint4 w = *reinterpret_cast<const uint4*>(best + i);
                above += (w.x > mine) + (w.y > mine) + (w.z > mine) + (w.w > mine);
            }
            if (above < a.keep) low = min(low, mine);
            most = max(most, mine);
        }
        low = __reduce_min_sync(0xffffffffu, low);
        most = __reduce_max_sync(0xffffffffu, most);
        const float m = key_value(static_cast<uint64_t>(most) << 32);
        float bar = key_value(static_cast<uint64_t>(low) << 32);
        const float base = m == -INFINITY ? 0.0f : m;
        const int v0 = s.first - skip;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        uint64_t hits = 0;  // which of the thread's logits reach the bar (collected one by one in the loop, each took ~400 cycles)
#pragma unroll 2
        for (int w = tid, k = 0; w < words; w += SLT, k += VEC) {
            union { T t[VEC]; uint4 u; } x;
            x.u = reinterpret_cast<const uint4*>(data)[w];
            uint32_t some = 0;
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float y = fmaxf(to_f32(x.t[e]), -INFINITY);
                sum[e & 3] += ex2((y - base) * 1.4426950408889634f);  // (the difference first: the maximum's term is 1)
                some |= y >= bar ? 1u << e : 0u;
            }
            hits |= static_cast<uint64_t>(some) << k;
        }
        if (bar == -INFINITY)  // (entries outside the slice are -inf there: none of its logits)
            for (int w = tid, k = 0; w < words; w += SLT, k += VEC)
                for (int e = 0; e < VEC; e++)
                    if (static_cast<unsigned>(w * VEC + e - skip) >= static_cast<unsigned>(count)) hits &= ~(1ull << (k + e));
        if (hits) {
            for (int n = atomicAdd(&s_n, __popcll(hits)); hits && n < SCAP; hits &= hits - 1, n++) {
                const int k = __ffsll(hits) - 1, e = (tid + k / VEC * SLT) * VEC + k % VEC;
                found[n] = order_key(fmaxf(to_f32(data[e]), -INFINITY), v0 + e);
            }
        }
        float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) all += __shfl_xor_sync(0xffffffffu, all, w);
        if (lane == 0) s_sum[tid >> 5] = all;
        __syncthreads();
        if (tid == 0) stats[item] = make_float2(m, (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]));
        int n = s_n;
        if (n > SCAP) {
            // the keep-th largest value: the highest that `keep` logits reach
            auto value = [&](int e) { return fmaxf(to_f32(data[e]), -INFINITY); };
            uint32_t below = low, least = most;  // `keep` reach `below`; the highest such is in [below, least]
            while (below < least) {
                const uint32_t mid = below + (least - below + 1) / 2;
                int reach = 0;
                for (int e = skip + tid; e < skip + count; e += SLT) reach += order_bits(value(e)) >= mid;
                reach = __reduce_add_sync(0xffffffffu, reach);
                __syncthreads();
                if (lane == 0) s_scan[tid >> 5] = reach;
                __syncthreads();
                reach = 0;
                for (int w = 0; w < SLT / 32; w++) reach += s_scan[w];
                if (reach >= a.keep) below = mid;
                else least = mid - 1;
            }
            bar = key_value(static_cast<uint64_t>(below) << 32);
            // those above it, then as many that equal it as are missing, lowest tokens first
            __syncthreads();
            if (tid == 0) s_n = 0;
            __syncthreads();
            for (int e = skip + tid; e < skip + count; e += SLT) {
                const float y = value(e);
                if (y > bar) found[atomicAdd(&s_n, 1)] = order_key(y, v0 + e);
            }
            __syncthreads();
            n = s_n;
            const int want = max(n, a.keep);
            for (int e0 = skip; e0 < skip + count && n < want; e0 += SLT) {
                const int e = e0 + tid;
                const bool same = e < skip + count && value(e) == bar;
                const uint32_t votes = __ballot_sync(0xffffffffu, same);
                __syncthreads();
                if (lane == 0) s_scan[tid >> 5] = __popc(votes);
                __syncthreads();
                int place = n + __popc(votes & ((1u << lane) - 1)), total = 0;
                for (int w = 0; w < SLT / 32; w++) {
                    if (w < (tid >> 5)) place += s_scan[w];
                    total += s_scan[w];
                }
                if (same && place < want) found[place] = order_key(bar, v0 + e);
                n = min(want, n + total);
            }
            __syncthreads();
        }
        if (more && tid == 0) fetch(next);  // (nobody reads the buffer any more)
        for (int i = tid; i < n; i += SLT) {
            const uint64_t key = found[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < n; j++) rank += found[j] > key;
            if (rank < a.keep) out[rank] = key;
        }
        if (tid >= n && tid < a.keep) out[tid] = order_key(-INFINITY, 0x80000000u + tid);
        __syncthreads();  // `found` and the counters are free
    }
}

// A candidate's place in its request's order: total, then the lower beam, then
// its place in the beam's list.
struct Place {
    uint64_t hi, lo;
    __device__ int above(const Place& o) const {  // (without branches: with them a comparison took ~190 cycles)
        return static_cast<int>(hi > o.hi) | (static_cast<int>(hi == o.hi) & static_cast<int>(lo > o.lo));
    }
};

// One request: the `keep` best of its beams' slices' lists.  (A candidate that
// is not among its beam's `keep` best has that many above it in any case.)
// The same bar: the keep-th largest of the lists' heads, found among the
// threads' best heads first, leaves candidates of at most `keep` lists.
// Bound: latency, so what is read is asked for at once: all statistics, a
// list's head and AHEAD candidates for each thread; and its code runs once, so
// it is short: loops that were unrolled by four took 1.4 us more to fetch than
// they saved.  Measured: ~4 us for 4 beams of 24 slices, ~5 for 8 of 10.
constexpr int ST = 256, AHEAD = 4;
__global__ void __launch_bounds__(ST) select_merge_kernel(const BeamSelectArgs a, const uint64_t* keys,
                                                          const float2* stats, int slices, int heads_cap) {
    extern __shared__ __align__(128) uint8_t sm[];
    Place* best = reinterpret_cast<Place*>(sm);  // [ST]
    Place* heads = best + ST;                    // [heads_cap]
    Place* found = heads + heads_cap;            // [min(lists, keep) keep]
    __shared__ float s_score[64], s_max[64], s_z[64];
    __shared__ Place s_bar;
    __shared__ int s_n[2];
    const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int lists = a.beams * slices, all = lists * a.keep;
    griddep_wait();
    const uint64_t* mine = keys + static_cast<int64_t>(b) * all;
    const uint64_t head = tid < lists ? mine[static_cast<int64_t>(tid) * a.keep] : 0;
    uint64_t ahead[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) ahead[i] = tid + i * ST < all ? mine[tid + i * ST] : 0;
    if (tid < 2) s_n[tid] = 0;
    if (tid == 0) s_bar = Place{0, 0};
    for (int w = warp; w < a.beams; w += ST / 32) {
        const float2* st = stats + (static_cast<int64_t>(b) * a.beams + w) * slices;
        float2 one = lane < slices ? st[lane] : make_float2(-INFINITY, 0.0f);
        const float score = a.scores[b * a.beams + w];
        float m = one.x;
        for (int i = lane + 32; i < slices; i += 32) m = fmaxf(m, st[i].x);
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float sum = lane < slices ? one.y * expf(one.x - m) : 0.0f;
        for (int i = lane + 32; i < slices; i += 32) sum += st[i].y * expf(st[i].x - m);
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            s_score[w] = score;
            s_max[w] = m;
            s_z[w] = logf(sum);
        }
    }
    __syncthreads();
    // (quotients of numbers below 2^22 by way of the reciprocal: right, and a tenth of the division's code)
    const float by_slices = 1.0f / slices, by_keep = 1.0f / a.keep;
    auto place = [&](uint64_t key, int list) {
        const int w = static_cast<int>((list + 0.5f) * by_slices);
        float total = s_score[w] + ((key_value(key) - s_max[w]) - s_z[w]);
        if (total != total) total = -INFINITY;
        return Place{order_key(total, w), key};
    };
    // a warp's lanes compare p with all
    auto rank_of = [&](const Place* set, int n, const Place& p) {
        int rank = 0;
#pragma unroll 1
        for (int i = lane; i < n; i += 32) rank += set[i].above(p);
        return __reduce_add_sync(0xffffffffu, rank);
    };
    Place top{0, 0};
    if (tid < lists) top = place(head, tid);
    for (int l = tid + ST; l < lists; l += ST) {
        const Place p = place(mine[static_cast<int64_t>(l) * a.keep], l);
        if (p.above(top)) top = p;
    }
    best[tid] = top;
    __syncthreads();
    const int threads = min(lists, ST);
#pragma unroll 1
    for (int i = warp; i < threads; i += ST / 32) {
        const Place p = best[i];
        if (rank_of(best, threads, p) == a.keep - 1 && lane == 0) s_bar = p;
    }
    __syncthreads();
    if (lists > ST) {  // the bar among all heads that reach the one among the threads'
        const Place first = s_bar;
        for (int l = tid; l < lists; l += ST) {
            const Place p = place(mine[static_cast<int64_t>(l) * a.keep], l);
            if (!first.above(p)) heads[atomicAdd(&s_n[1], 1)] = p;
        }
        __syncthreads();
        const int n = s_n[1];
#pragma unroll 1
        for (int i = warp; i < n; i += ST / 32) {
            const Place p = heads[i];
            if (rank_of(heads, n, p) == a.keep - 1 && lane == 0) s_bar = p;
        }
        __syncthreads();
    }
    const Place bar = s_bar;
    auto collect = [&](uint64_t key, int c) {
        const Place p = place(key, static_cast<int>((c + 0.5f) * by_keep));
        if (!bar.above(p)) found[atomicAdd(&s_n[0], 1)] = p;
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
        if (tid + i * ST < all) collect(ahead[i], tid + i * ST);
    for (int c = tid + AHEAD * ST; c < all; c += ST) collect(mine[c], c);
    __syncthreads();
    const int n = s_n[0];
#pragma unroll 1
    for (int i = warp; i < n; i += ST / 32) {
        const Place p = found[i];
        const int rank = rank_of(found, n, p);
        if (lane != 0 || rank >= a.keep) continue;
        const int o = b * a.keep + rank;
        a.out_scores[o] = key_value(p.hi);
        a.out_tokens[o] = key_token(p.lo);
        a.out_parents[o] = key_token(p.hi);
    }
}

// ---------------------------------------------------------------- reordering
// A copy that a row needs: `fill` tokens of page src to page dst.
struct PageCopy {
    int src, dst, fill;
};
// What becomes of a new row: its parent's first `n` pages, and page `page` in
// column `at` (at -1: none of its own; page -1: none to be had).
struct RowPlan {
    int parent, n, at, page;
};

constexpr int RT = 1024;  // threads of a CTA
// Exclusive sum over the CTA; counts in both halves of the word do not meet.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* sm, uint32_t* total) {
    uint32_t inc = x;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) sm[w] = inc;
    __syncthreads();
    uint32_t part = sm[lane];  // (32 warps)
    const uint32_t own = part;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, part, o);
        if (lane >= o) part += y;
    }
    *total = __shfl_sync(0xffffffffu, part, 31);
    return __shfl_sync(0xffffffffu, part - own, w) + inc - x;
}

// Every thread's writes to memory before are seen by every thread of the cluster after (through L2: read them with __ldcg).
template <int RC>
__device__ __forceinline__ void cluster_sync() {
    if constexpr (RC == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Tables, lengths, counts and the list of copies.  A step's tables are a few
// KB; what takes the time is the chain of reads that depend on one another, and
// the atomics of one SM (one address a cycle), so a cluster of eight CTAs does
// large ones, and one CTA small ones, where a barrier across the cluster costs
// more (the rule and its figures are at the launch); both in three phases.
// (The new tables themselves are written by the next kernel.)  full[page],
// part[page]: how often the old tables hold it as a full page and as a
// part-filled one; owner[page]: the lowest new row whose tail it is.  A page
// that some row holds as a full one is nobody's to go on in, also where another
// row ends in it (rows of different lengths that share a prefix).
template <int RC>
__global__ void __cluster_dims__(RC, 1, 1) __launch_bounds__(RT)
    reorder_tables_kernel(const BeamReorderArgs a, int* full, int* part, int* owner, int* freelist, RowPlan* rows,
                          PageCopy* copies, int* n_copies, int* err) {
    __shared__ uint32_t sm[32];
    griddep_wait();
    griddep_launch();
    constexpr int ALL = RC * RT;
    const int t = threadIdx.x, g = blockIdx.x * RT + t;  // the cluster is the grid
    const int log2 = __ffs(a.page) - 1;
    auto used = [&](int len) { return min(a.cols, (len >> log2) + ((len & (a.page - 1)) != 0)); };  // (any int)
    // (row, column) of the entries g, g + ALL, ... of a table: one division, not one each
    const int r_first = g / max(a.cols, 1), c_first = g - r_first * a.cols;
    const int r_step = ALL / max(a.cols, 1), c_step = ALL - r_step * a.cols;
    auto step = [&](int& r, int& c) {
        r += r_step;
        c += c_step;
        if (c >= a.cols) {
            c -= a.cols;
            r++;
        }
    };

    // ---- 1: counters; the first free pages, at most one for each new row
    for (int64_t i = g; i < a.n_pages; i += ALL) {
        full[i] = part[i] = 0;
        owner[i] = INT_MAX;
    }
    int found = 0;
    if (blockIdx.x == 0) {
        for (int64_t i0 = 0; i0 < a.n_pages && found < a.new_rows; i0 += RT * 8) {
            const int64_t i = i0 + t * 8;
            uint32_t free = 0;
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (i + e < a.n_pages && __ldg(a.refs + i + e) == 0) free |= 1u << e;
            uint32_t all;
            int rank = found + static_cast<int>(block_scan(__popc(free), sm, &all));
            for (; free && rank < a.new_rows; free &= free - 1, rank++) freelist[rank] = static_cast<int>(i) + __ffs(free) - 1;
            found += static_cast<int>(all);
        }
    }
    cluster_sync<RC>();

    // ---- 2: what the old tables hold; the new rows' parents, and their tails' owners
    constexpr int B = 4;  // entries whose reads are on their way together
    for (int r = r_first, c = c_first; r < a.rows && a.cols > 0;) {
        int pg[B], len[B], cc[B];
#pragma unroll
        for (int k = 0; k < B; k++, step(r, c)) {
            const bool in = r < a.rows;
            pg[k] = in ? __ldg(a.table + r * a.table_stride + c) : -1;
            len[k] = in ? __ldg(a.lens + r) : 0;
            cc[k] = c;
        }
#pragma unroll
        for (int k = 0; k < B; k++)
            if (cc[k] < used(len[k]) && pg[k] >= 0 && pg[k] < a.n_pages)
                atomicAdd((cc[k] < len[k] >> log2 ? full : part) + pg[k], 1);
    }
    for (int r = g; r < a.new_rows; r += ALL) {
        const int q = a.parents[r];
        if (q >= a.rows) record_error(err, DEVERR_BAD_INDEX);
        const bool live = q >= 0 && q < a.rows;
        const int len = live ? max(0, a.lens[q]) : 0, at = len >> log2;  // (at indexes the table: never below 0)
        int tail = -1;  // the page that is part-filled, if one is
        if (live && (len & (a.page - 1)) && at < a.cols) {
            tail = a.table[q * a.table_stride + at];
            if (tail < 0 || tail >= a.n_pages) {
                record_error(err, DEVERR_BAD_PAGE);
                tail = -1;
            } else {
                atomicMin(owner + tail, r);
            }
        }
        a.new_lens[r] = len;
        rows[r] = RowPlan{live ? q : -1, live ? used(len) : 0, at, tail};
    }
    cluster_sync<RC>();

    // ---- 3: who keeps its tail, who takes which free page (one CTA); the counts without the old tables (the others, if any)
    if (blockIdx.x == 0) {
        int taken = 0, short_of = 0, copied = 0;
        for (int r0 = 0; r0 < a.new_rows; r0 += RT) {
            const int r = r0 + t;
            RowPlan p{-1, 0, -1, -1};
            bool filled = false, keeps = false;  // it ends in a part-filled page, and stays there
            int fill = 0;
            if (r < a.new_rows) {
                const int4 w = __ldcg(reinterpret_cast<const int4*>(rows + r));
                p = RowPlan{w.x, w.y, w.z, w.w};
                filled = p.page >= 0;
                fill = __ldcg(a.new_lens + r) & (a.page - 1);
                keeps = filled && __ldcg(owner + p.page) == r && __ldcg(full + p.page) == 0 &&
                        a.refs[p.page] == __ldcg(part + p.page);
            }
            const bool fresh = p.parent >= 0 && !keeps && p.at < a.cols;
            uint32_t all;
            const int turn = taken + static_cast<int>(block_scan(fresh, sm, &all));
            const bool got = fresh && turn < found;
            taken += static_cast<int>(all);
            const uint32_t mine = (got && filled) | (p.parent >= 0 && !keeps && !got ? 0x10000u : 0u);
            const uint32_t before = block_scan(mine, sm, &all);
            const int page = got ? __ldcg(freelist + turn) : -1;
            if (got && filled) copies[copied + (before & 0xFFFFu)] = PageCopy{p.page, page, fill};
            copied += static_cast<int>(all & 0xFFFFu);
            short_of += static_cast<int>(all >> 16);
            if (r < a.new_rows) rows[r] = RowPlan{p.parent, p.n, fresh ? p.at : -1, page};
        }
        if (t == 0) {
            a.status[0] = min(taken, found);
            a.status[1] = short_of;
            *n_copies = copied;
        }
    }
    if (RC == 1 || blockIdx.x > 0)
        for (int64_t i = RC == 1 ? t : g - RT; i < a.n_pages; i += RC == 1 ? RT : ALL - RT)
            a.new_refs[i] = a.refs[i] - __ldcg(full + i) - __ldcg(part + i);
}

// The new tables and what they hold, and the filled part of the pages that
// rows copy, every layer, keys and values.  Bound: memory.  A thread writes one
// entry of the tables or none, then CTAs go over (copy, layer, k or v); a
// thread has eight 16-byte pieces on their way.  Measured with the kernel
// before: 256 rows of 12 layers, 142 MB: 35 us, the copy 2 us a layer of it
// (5.9 TB/s).
constexpr int CT = 128, CU = 8;
__global__ void __launch_bounds__(CT) reorder_copy_kernel(const BeamReorderArgs a, const RowPlan* rows,
                                                          const PageCopy* copies, const int* n_copies) {
    griddep_wait();
    const int64_t entries = static_cast<int64_t>(a.new_rows) * a.cols;
    for (int64_t i = blockIdx.x * CT + threadIdx.x; i < entries; i += gridDim.x * CT) {
        const int r = static_cast<int>(i / a.cols), c = static_cast<int>(i - static_cast<int64_t>(r) * a.cols);
        const int4 p = __ldg(reinterpret_cast<const int4*>(rows + r));  // RowPlan: parent, n, at, page
        const int page = c == p.z ? p.w : c < p.y ? __ldg(a.table + p.x * a.table_stride + c) : -1;
        a.new_table[i] = page;
        if (page >= 0 && page < a.n_pages) atomicAdd(a.new_refs + page, 1);
    }
    const int items = *n_copies * 2 * a.layers, d8 = a.dim / 8, per = a.kv_heads * d8;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int which = item % (2 * a.layers), layer = which >> 1;
        const PageCopy c = copies[item / (2 * a.layers)];
        const bool v = which & 1;
        uint16_t* base = static_cast<uint16_t*>(v ? a.v : a.k) + layer * (v ? a.v_layer : a.k_layer);
        const int64_t page = v ? a.v_page : a.k_page, tok = v ? a.v_tok : a.k_tok, head = v ? a.v_head : a.k_head;
        const uint16_t* src = base + c.src * page;
        uint16_t* dst = base + c.dst * page;
        const int total = c.fill * per;
        // pieces in the order of the storage: token, head or head, token
        const bool by_head = head > tok;
        const int inner = by_head ? c.fill : a.kv_heads;
        const int64_t in_step = by_head ? tok : head, out_step = by_head ? head : tok;
        for (int i0 = threadIdx.x; i0 < total; i0 += CT * CU) {
            uint4 x[CU];
            int64_t at[CU];
#pragma unroll
            for (int u = 0; u < CU; u++) {
                const int i = i0 + u * CT;
                const int j = i / d8, o = j / inner;
                at[u] = o * out_step + (j - o * inner) * in_step + (i - j * d8) * 8;
                if (i < total) x[u] = __ldcs(reinterpret_cast<const uint4*>(src + at[u]));
            }
#pragma unroll
            for (int u = 0; u < CU; u++)
                if (i0 + u * CT < total) *reinterpret_cast<uint4*>(dst + at[u]) = x[u];
        }
    }
}

int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

}  // namespace

namespace {

// Slices of a step's rows, for the six CTAs that go over them on each of the
// 148 SMs: as few rounds of as narrow slices as will do, where a slice costs
// what 3000 logits do besides its own (the two passes over its tops), and has
// at least 2048.
constexpr int kSms = 148, kSliceCtas = 6 * kSms, kSliceCost = 3000;
struct Slices {
    int n, width, heads_cap, found_cap;
    int64_t keys, bytes;  // of the workspace: the lists', all
};
Slices slices_of(const BeamSelectArgs& a) {
    Slices s;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.beams;
    const int least = (a.vocab + SMAX - 1) / SMAX;
    int64_t cost = INT64_MAX;
    s.n = least;
    for (int n = least; n <= std::max(least, std::min(a.vocab / 2048, 3 * least + 24)); n++) {
        const int64_t c = (rows * n + kSliceCtas - 1) / kSliceCtas * ((a.vocab + n - 1) / n + kSliceCost);
        if (c < cost) {
            cost = c;
            s.n = n;
        }
    }
    s.width = (a.vocab + s.n - 1) / s.n;
    const int lists = a.beams * s.n;
    s.heads_cap = lists > ST ? std::min(lists, a.keep * ((lists + ST - 1) / ST)) : 0;
    s.found_cap = std::min(lists, a.keep) * a.keep;
    s.keys = up256(rows * s.n * a.keep * 8);
    s.bytes = s.keys + up256(rows * s.n * 8);
    return s;
}

template <typename T>
int launch_select(const BeamSelectArgs& a, const Slices& s, cudaStream_t st) {
    int rc = 0;
    DeviceState* ds = device_state(&rc);
    if (!ds) return rc;
    uint64_t* keys = static_cast<uint64_t*>(a.ws);
    float2* stats = reinterpret_cast<float2*>(static_cast<uint8_t*>(a.ws) + s.keys);
    rc = allow_smem<select_merge_kernel>(200 * 1024);
    if (rc) return rc;
    const int64_t items = static_cast<int64_t>(a.batch) * a.beams * s.n;
    rc = launch_pdl(select_slice_kernel<T>, dim3(static_cast<unsigned>(std::min<int64_t>(items, kSliceCtas))), dim3(SLT),
                    static_cast<size_t>(SBUF + SCAP * 8), st, a, keys, stats, s.n, s.width, ds->d_error);
    if (rc) return rc;
    const size_t smem = (ST + s.heads_cap + s.found_cap) * sizeof(Place);
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
    *bytes = 256 + 3 * up256(a.n_pages * 4) + up256(a.new_rows * 4ll) + up256(a.new_rows * 16ll) + up256(a.new_rows * 12ll);
    return TVQ_OK;
}

int launch_beam_reorder(const BeamReorderArgs& a, cudaStream_t st) {
    int rc = 0;
    DeviceState* ds = device_state(&rc);
    if (!ds) return rc;
    uint8_t* w = static_cast<uint8_t*>(a.ws);
    auto take = [&](int64_t bytes) {
        uint8_t* p = w;
        w += up256(bytes);
        return p;
    };
    int* n_copies = reinterpret_cast<int*>(take(4));
    int* full = reinterpret_cast<int*>(take(a.n_pages * 4));
    int* part = reinterpret_cast<int*>(take(a.n_pages * 4));
    int* owner = reinterpret_cast<int*>(take(a.n_pages * 4));
    int* freelist = reinterpret_cast<int*>(take(a.new_rows * 4ll));
    RowPlan* rows = reinterpret_cast<RowPlan*>(take(a.new_rows * 16ll));
    PageCopy* copies = reinterpret_cast<PageCopy*>(take(a.new_rows * 12ll));
    // One CTA and the cluster, both kernels of a reorder with hardly anything to copy: by entries of the table 92: 8.0
    // and 8.3 us, 736: 9.4 and 9.7, 1472: 9.7 and 9.9, 2944: 10.6 and 10.4, 5888: 13.5 and 11.2, 20288: 24.5 and 12.6;
    // by pages (16 rows) 1000: 9.3 and 9.3, 2000: 9.9 and 9.5, 8000: 12.4 and 10.4, 64000: 33 and 11.6.
    const bool small = static_cast<int64_t>(std::max(a.rows, a.new_rows)) * a.cols <= 2 * RT && a.n_pages <= RT;
    rc = launch_pdl(small ? reorder_tables_kernel<1> : reorder_tables_kernel<8>, dim3(small ? 1 : 8), dim3(RT), 0, st, a,
                    full, part, owner, freelist, rows, copies, n_copies, ds->d_error);
    if (rc || a.new_rows == 0) return rc;
    const int64_t items = std::max<int64_t>(2ll * a.new_rows * a.layers, (static_cast<int64_t>(a.new_rows) * a.cols + CT - 1) / CT);
    if (items == 0) return rc;
    return launch_pdl(reorder_copy_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(items, ds->sm_count * 12ll))), dim3(CT),
                      0, st, a, rows, copies, n_copies);
}

}  // namespace tvq
