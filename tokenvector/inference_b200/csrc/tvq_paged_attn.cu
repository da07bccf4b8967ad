// tvq_paged_attn.cu -- attention of new tokens over a paged cache.
//
// Row i of a sequence with n new rows and L cached tokens (the new ones
// included) sits at p = L - n + i and sees the keys j <= p (j > p - window).
// With x_j = log2(e) scale q.k_j, over any split of the keys into parts,
//   m = max x_j, l = sum 2^(x_j - m), o = sum 2^(x_j - m) v_j per part,
//   M = max m, L = sum 2^(m - M) l, out = sum 2^(m - M) o / L,
//   lse = ln 2 (M + log2 L),
// so the keys are read once and parts are joined at the end.  The query heads
// that share a kv head are rows of one product: row r = i * group + g.
//
// attn_rows_kernel: sequences of at most 16 such rows (single tokens, a few
// drafted ones).  Every key and value is used for at most 16 rows, so the
// bytes of the cache bound it, and what counts is that enough of them are in
// flight and that every SM has the same share:
//  - all tiles (8 KB of keys and values) of all (sequence, kv head) pairs
//    stand in one line, which is cut into equal pieces, one for each of the
//    eight warps of each SM, whatever the lengths.  Every CTA finds its pieces
//    from the lengths on the device; neighbouring pieces go to different SMs.
//  - a warp is a pipeline of its own: its tiles come through its own ring of
//    three stages by TMA (a tile's pages are boxes of a {value, token, half,
//    head, page} tensor map, so any strides will do), across the ends of
//    pairs, and it keeps its own m, l, o.  192 KB are in flight on each SM,
//    and nothing in the CTA waits for another warp.  (Eight warps that share
//    each pair and join it in shared memory took ~4000 cycles a pair more,
//    which doubled the time of many short sequences.)
//  - two producer warps fill the eight rings, eight lanes for each, whichever
//    has a free stage: a TMA load costs its thread ~200 cycles, which
//    doubled a tile's time when the consumers issued their own.
//  - mma.sync m16n8k16 with the rows padded to 16: a warp's tile takes ~1000
//    cycles from ring to ring, and the eight together 125 a tile where its
//    bytes take ~330, so the wider tcgen05 tile (128 rows) would buy nothing.
//  - a pair that lies in one piece is written at once; the parts of the others
//    go to the workspace in f32, and attn_join_kernel joins them in order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "tvq_common.cuh"
#include "tvq_decode.h"
#include "tvq_kernels.h"

namespace tvq {

namespace {

constexpr int NW = 8;              // consumer warps of the rows kernel's CTA
constexpr int NTHR = (NW + 2) * 32;  // and two producer warps, a ring for every eight lanes
constexpr int MAX_ROWS = 16;       // rows of a pair (new tokens x heads of the group)

// device error codes: the wait that gave up first
enum : int { DEVERR_PATTN_EMPTY = 71, DEVERR_PATTN_FULL = 72 };

__device__ __forceinline__ float ex2(float x) {  // 2^x, relative error ~2^-22, 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A bounded wait that a page number out of range (recorded in the same word,
// and no reason to stop) does not cut short.
__device__ __forceinline__ bool wait_full(uint64_t* bar, uint32_t parity, int* err) {
    const bool ok = mbar_wait_for(bar, parity, nullptr, DEVERR_PATTN_FULL, TVQ_WAIT_LIMIT_NS);
    if (!ok) record_error(err, DEVERR_PATTN_FULL);
    return ok;
}

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// 5-D TMA tile load {value, token, half, head, page}; what lies outside is zero.
__device__ __forceinline__ void tma_load_5d(const CUtensorMap* map, uint64_t* bar, uint32_t dst, int c0, int c1, int c2,
                                            int c3, int c4) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// d += A (16 x 16) B (16 x 8), f32 sums
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One sequence as both kernels see it.
struct Seq {
    int row0;  // first packed row
    int n;     // new rows
    int len;   // tokens in the cache
};
__device__ __forceinline__ Seq load_seq(const PagedView& c, int s) {
    Seq q;
    q.len = __ldg(c.ctx + s);
    if (c.cu) {
        q.row0 = max(0, __ldg(c.cu + s));
        q.n = max(0, min(__ldg(c.cu + s + 1), c.n_rows) - q.row0);
    } else {
        q.row0 = s;
        q.n = 1;
    }
    return q;
}

// The tiles of KT keys [first, end) that the rows of a sequence see together:
// one at least, so that rows without keys are written too.
template <int KT>
__device__ __forceinline__ int2 seq_tiles(const Seq& q, int window) {
    const int p0 = q.len - q.n;
    const int first = window > 0 ? max(0, p0 - window + 1) / KT : 0;
    return make_int2(first, max(first + 1, (max(q.len, 0) + KT - 1) / KT));
}

// ---------------------------------------------------------------- few rows
template <int DP>
struct RowsCfg {
    static constexpr int KT = DP == 128 ? 16 : 32;       // keys per tile
    static constexpr int HALF = KT * 128;                // 64 values of a tile's keys, 128-byte swizzle
    static constexpr int HALVES = DP / 64;
    static constexpr int STAGE = 2 * HALVES * HALF;      // one tile, 8 KB: keys, then values
    static constexpr int STAGES = 3;                     // of each warp
    static constexpr int OFF_BAR = NW * STAGES * STAGE;  // full[NW][STAGES], empty[NW][STAGES]
    static constexpr int OFF_MISC = OFF_BAR + 2 * NW * STAGES * 8;  // int64 at[NW], int seq[NW], int scan[NW + 2]
    static constexpr int SMEM = OFF_MISC + NW * 16 + 8;
};

struct RowsPlan {
    uint8_t* parts;  // [pieces][2]: f32 [rows_cap][DP], then float2 (m, l) [rows_cap]
    int2* spans;     // [n_seq * kv_heads]: a pair's first and last piece
    int rows_cap;    // no pair has more rows
    int64_t slot;    // bytes of one part
    // One TMA load: `box` tokens (a power of two: a page, or a tile of a larger
    // one) of 64 values, or of both halves (box_halves 2: 128 values and box =
    // KT).  by_value: the head dim is no multiple of 64, the halves start at
    // values 0 and 64 of one dimension that ends with the head dim.
    int box, box_halves, by_value;
};

// Where a walk over a piece stands: a pair and its tiles in the piece.
struct Cursor {
    int s, hk;
    int64_t left;    // tiles of the piece from this pair's first one on
    Seq q;
    int2 all;        // the pair's tiles
    int first, end;  // those in the piece
};

template <typename T, int DP>
__global__ void __launch_bounds__(NTHR, 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const PagedAttnArgs a, const RowsPlan plan, int* err) {
    using C = RowsCfg<DP>;
    constexpr int KT = C::KT;
    extern __shared__ __align__(1024) uint8_t sm[];
    int64_t* s_at = reinterpret_cast<int64_t*>(sm + C::OFF_MISC);
    int* s_seq = reinterpret_cast<int*>(s_at + NW);
    int* s_scan = s_seq + NW;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // whose ring this thread serves: its warp's, or eight lanes' of a producer warp
    const int mine = warp < NW ? warp : (warp - NW) * 4 + (lane >> 3);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR) + mine * C::STAGES;
    uint64_t* empty = full + NW * C::STAGES;
    uint8_t* ring = sm + mine * (C::STAGES * C::STAGE);
    const int group = a.q_heads / a.c.kv_heads;
    const int fit = MAX_ROWS / group;  // new rows of a sequence that this kernel takes
    if (tid == 0) {
        for (int i = 0; i < 2 * NW * C::STAGES; i++) mbar_init(reinterpret_cast<uint64_t*>(sm + C::OFF_BAR) + i, 1);
        fence_barrier_init();
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    griddep_wait();
    griddep_launch();  // the join kernel's CTAs fit beside this one's and wait there

    // ---- the pieces of the line of tiles
    auto weight = [&](int s) -> int {
        if (s >= a.c.n_seq) return 0;
        const Seq q = load_seq(a.c, s);
        if (q.n == 0 || q.n > fit) return 0;
        const int2 t = seq_tiles<KT>(q, a.window);
        return t.y - t.x;
    };
    auto scan = [&](int x, int* all) {  // inclusive, over the CTA
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) s_scan[warp] = x;
        __syncthreads();
        int sum = 0;
        for (int w = 0; w < NW + 2; w++) {
            if (w < warp) x += s_scan[w];
            sum += s_scan[w];
        }
        *all = sum;
        return x;
    };
    int64_t total = 0;
    int w0 = 0, inc0 = 0;
    for (int s0 = 0; s0 < a.c.n_seq; s0 += NTHR) {
        int all;
        w0 = weight(s0 + tid);
        inc0 = scan(w0, &all);
        total += all;
    }
    total *= a.c.kv_heads;
    const int64_t pieces = static_cast<int64_t>(gridDim.x) * NW;
    const int64_t per = max(static_cast<int64_t>(1), (total + pieces - 1) / pieces);
    int64_t before = 0;
    for (int s0 = 0; s0 < a.c.n_seq; s0 += NTHR) {
        int all = 0;
        int w = w0, inc = inc0;
        if (a.c.n_seq > NTHR) {
            w = weight(s0 + tid);
            inc = scan(w, &all);
        }
        const int64_t hi = (before + inc) * a.c.kv_heads, lo = hi - static_cast<int64_t>(w) * a.c.kv_heads;
        if (w > 0)
            for (int i = 0; i < NW; i++) {
                const int64_t at = per * (static_cast<int64_t>(i) * gridDim.x + blockIdx.x);
                if (at >= lo && at < hi) {
                    s_seq[i] = s0 + tid;
                    s_at[i] = lo;
                }
            }
        before += all;
    }
    __syncthreads();
    const int piece = mine * gridDim.x + blockIdx.x;
    const int64_t begin = per * piece, stop = min(total, begin + per);
    if (warp < NW && begin >= stop) return;

    Cursor cur;
    auto enter = [&](Cursor& c, int skip) {  // s, hk, left and q set: the pair's tiles from `skip` on
        c.all = seq_tiles<KT>(c.q, a.window);
        c.first = c.all.x + skip;
        c.end = static_cast<int>(min(static_cast<int64_t>(c.all.y), c.first + c.left));
    };
    auto next_pair = [&](Cursor& c) {  // false: the piece is done
        c.left -= c.end - c.first;
        if (c.left <= 0) return false;
        if (++c.hk == a.c.kv_heads) {
            c.hk = 0;
            do {
                c.q = load_seq(a.c, ++c.s);
            } while (c.q.n == 0 || c.q.n > fit);
        }
        enter(c, 0);
        return true;
    };
    cur.left = stop - begin;
    if (cur.left > 0) {
        cur.s = s_seq[mine];
        cur.q = load_seq(a.c, cur.s);
        const int64_t in_seq = begin - s_at[mine];
        const int2 t = seq_tiles<KT>(cur.q, a.window);
        cur.hk = static_cast<int>(in_seq / (t.y - t.x));
        enter(cur, static_cast<int>(in_seq - static_cast<int64_t>(cur.hk) * (t.y - t.x)));
    }

    if (warp >= NW) {
        // ------------------------------------------------ producers
        // Eight lanes for a ring.  Its tiles come in windows of eight page
        // lookups (lane i: the i-th box), the next window's under way while this
        // one's tiles are issued; each of the lanes issues one load of a tile.
        const int boxes = KT / plan.box, loads_h = C::HALVES / plan.box_halves, ops = 2 * boxes * loads_h;
        const int sub = lane & 7, lead = lane & 24;
        const bool is_v = sub & 1, issues = sub < ops;
        const int b = (sub >> 1) / loads_h, h = (sub >> 1) - b * loads_h;
        const uint32_t dst = smem_u32(ring) + (is_v ? C::HALVES * C::HALF : 0) + h * C::HALF + b * plan.box * 128;
        const CUtensorMap* map = is_v ? &tmV : &tmK;
        const int x = plan.by_value ? h * 64 : 0, y = plan.by_value ? 0 : h;
        struct Window {
            int t, end, hk, page;
        };
        int next_t = cur.left > 0 ? cur.first : 0;
        bool more = cur.left > 0;
        auto look = [&]() {
            Window w;
            w.t = w.end = next_t;
            w.hk = cur.hk;
            w.page = 0;
            if (!more) return w;
            w.end = min(cur.end, next_t + 8 / boxes);
            const int j = w.t * KT + sub * plan.box;
            if (j < w.end * KT && j < cur.q.len) {
                const int col = j >> a.c.page_log2;
                w.page = col < a.c.n_cols ? __ldg(a.c.table + cur.s * a.c.table_stride + col) : -1;
            }
            next_t = w.end;
            if (next_t == cur.end) {
                more = next_pair(cur);
                next_t = cur.first;
            }
            return w;
        };
        auto checked = [&](Window w) {
            if (static_cast<unsigned>(w.page) >= static_cast<unsigned>(a.c.n_pages)) {
                record_error(err, DEVERR_BAD_PAGE);
                w.page = -1;  // outside the tensor map: zeros
            }
            return w;
        };
        int n = 0, stage = 0, phase = 1, pos = 0;  // tiles issued, the ring's place, tiles of the window issued
        Window win = look(), then = look();
        if (win.t < win.end) win = checked(win);
        bool ok = true;
        uint32_t idle = 0;
        uint64_t since = 0;
        while (true) {
            const bool has = win.t + pos < win.end;
            if (!__any_sync(0xffffffffu, has)) break;
            bool ready = has && mbar_test(empty + stage, phase);
            ready = __shfl_sync(0xffffffffu, ready, lead);
            const int pg = __shfl_sync(0xffffffffu, win.page, lead + ((pos * boxes + b) & 7));
            if (ready) {
                if (sub == 0) mbar_arrive_expect_tx(full + stage, C::STAGE);
                if (issues)
                    tma_load_5d(map, full + stage, dst + stage * C::STAGE, x,
                                ((win.t + pos) * KT + b * plan.box) & (a.c.page - 1), y, win.hk, pg);
                n++;
                if (++stage == C::STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
                if (win.t + ++pos == win.end) {
                    win = then;
                    pos = 0;
                    if (win.t < win.end) {
                        win = checked(win);
                        then = look();
                    }
                }
            }
            if (__any_sync(0xffffffffu, ready)) {
                idle = 0;
            } else if ((++idle & 63u) == 0u) {  // nothing free for a while: the bound of every wait here
                if (idle == 64u) since = globaltimer_ns();
                else ok = globaltimer_ns() - since < TVQ_WAIT_LIMIT_NS;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) {
                    record_error(err, DEVERR_PATTN_EMPTY);
                    break;
                }
            } else {
                __nanosleep(32);
            }
        }
        // every load lands before the CTA may end
        if (sub == 0)
            for (int i = max(0, n - C::STAGES); i < n; i++)
                wait_full(full + i % C::STAGES, (i / C::STAGES) & 1, nullptr);
        return;
    }

    // ---------------------------------------------------- consumers
    const float scale2 = a.scale * 1.4426950408889634f;
    const int g = lane >> 2, quad = lane & 3;
    int stage = 0, phase = 0;
    bool ok = true;
    for (bool go = true; go; go = next_pair(cur)) {
        // ---- the pair's rows as A fragments
        const int rows = cur.q.n * group;
        uint32_t qf[DP / 16][4];
        int pos[2];     // of this thread's two rows (below 0: sees nothing)
        int64_t at[2];  // their place in out (below 0: none)
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const int r = g + hf * 8;
            const int i = r / group, gi = r - i * group;
            const bool in = r < rows;
            pos[hf] = in ? cur.q.len - cur.q.n + i : -1;
            at[hf] = in ? static_cast<int64_t>(cur.q.row0 + i) * a.q_heads + cur.hk * group + gi : -1;
            const T* q = static_cast<const T*>(a.q) + (in ? (cur.q.row0 + i) * a.q_tok + (cur.hk * group + gi) * a.q_head : 0);
#pragma unroll
            for (int kk = 0; kk < DP / 16; kk++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int d = kk * 16 + e * 8 + quad * 2;
                    qf[kk][e * 2 + hf] = in && d < a.c.dim ? __ldg(reinterpret_cast<const uint32_t*>(q + d)) : 0u;
                }
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[DP / 8][4];
#pragma unroll
        for (int n = 0; n < DP / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;

        for (int t = cur.first; t < cur.end; t++) {
            if (ok) ok = __all_sync(0xffffffffu, wait_full(full + stage, phase, err));
            const uint32_t ks = smem_u32(ring) + stage * C::STAGE, vs = ks + C::HALVES * C::HALF;
            if ((t + 1) * KT > cur.q.len) {
                // the values behind the sequence's end may be anything, and 0 x NaN is NaN: zeros
                const int from = max(0, cur.q.len - t * KT);
                for (int i = from * 8 + lane; i < KT * 8; i += 32)
#pragma unroll
                    for (int h = 0; h < C::HALVES; h++)
                        *reinterpret_cast<uint4*>(ring + stage * C::STAGE + (C::HALVES + h) * C::HALF + i * 16) =
                            make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async_smem();
                __syncwarp();
            }
            float sc[KT / 8][4];
#pragma unroll
            for (int n = 0; n < KT / 8; n++) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
            {
                const int r = ((lane >> 4) << 3) + (lane & 7), cc = (lane >> 3) & 1;
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk++) {
                    const uint32_t half = ks + (kk / 4) * C::HALF;
#pragma unroll
                    for (int n = 0; n < KT / 16; n++) {
                        uint32_t b[4];
                        ldsm4(half + (n * 16 + r) * 128 + ((((kk & 3) * 2 + cc) ^ (r & 7)) << 4), b);
                        mma16816<T>(sc[2 * n], qf[kk], b[0], b[1]);
                        mma16816<T>(sc[2 * n + 1], qf[kk], b[2], b[3]);
                    }
                }
            }
            uint32_t pf[KT / 16][4];
            const int j0 = t * KT + quad * 2;
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int hi = pos[hf], lo = a.window > 0 ? hi - a.window : -1;  // keys in (lo, hi]
                float x[KT / 4], top = -INFINITY;
#pragma unroll
                for (int e = 0; e < KT / 4; e++) {
                    const int j = j0 + (e >> 1) * 8 + (e & 1);
                    const float y = sc[e >> 1][hf * 2 + (e & 1)] * scale2;
                    x[e] = j <= hi && j > lo ? y : -INFINITY;
                    top = fmaxf(top, x[e]);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float m2 = fmaxf(m[hf], top);
                const float base = m2 == -INFINITY ? 0.0f : m2;
                const float f = ex2(m[hf] - base);
                m[hf] = m2;
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < KT / 4; e++) {
                    x[e] = ex2(x[e] - base);
                    sum += x[e];
                }
                l[hf] = l[hf] * f + sum;
                // the weights meet V in its own type: 2^-11 (f16) or 2^-8 (bf16) of each, as the
                // rounding of the result; l sums them unrounded
#pragma unroll
                for (int n = 0; n < KT / 16; n++) {
                    pf[n][hf] = pack2<T>(x[4 * n], x[4 * n + 1]);
                    pf[n][2 + hf] = pack2<T>(x[4 * n + 2], x[4 * n + 3]);
                }
#pragma unroll
                for (int n = 0; n < DP / 8; n++) {
                    o[n][hf * 2] *= f;
                    o[n][hf * 2 + 1] *= f;
                }
            }
            {
                const int r = (((lane >> 3) & 1) << 3) + (lane & 7), cc = lane >> 4;
#pragma unroll
                for (int n = 0; n < DP / 16; n++) {
                    const uint32_t half = vs + (n / 4) * C::HALF;
#pragma unroll
                    for (int k = 0; k < KT / 16; k++) {
                        uint32_t b[4];
                        ldsm4_t(half + (k * 16 + r) * 128 + ((((n & 3) * 2 + cc) ^ (r & 7)) << 4), b);
                        mma16816<T>(o[2 * n], pf[k], b[0], b[1]);
                        mma16816<T>(o[2 * n + 1], pf[k], b[2], b[3]);
                    }
                }
            }
            __syncwarp();  // every lane is done with the stage
            if (lane == 0) mbar_arrive(empty + stage);
            if (++stage == C::STAGES) {
                stage = 0;
                phase ^= 1;
            }
        }

        // ---- the pair's end: written, or left for the join
        const bool begins = cur.first == cur.all.x, whole = begins && cur.end == cur.all.y;
        if (begins && lane == 0) {
            const int64_t at0 = stop - cur.left;  // the pair's first tile in the line
            plan.spans[static_cast<int64_t>(cur.s) * a.c.kv_heads + cur.hk] =
                make_int2(piece, static_cast<int>((at0 + cur.all.y - cur.all.x - 1) / per));
        }
        uint8_t* part = plan.parts + (static_cast<int64_t>(piece) * 2 + (begins ? 1 : 0)) * plan.slot;
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            float sum = l[hf];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (at[hf] < 0) continue;
            const int r = g + hf * 8;
            if (whole) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                T* out = static_cast<T*>(a.out) + at[hf] * a.c.dim + quad * 2;
#pragma unroll
                for (int n = 0; n < DP / 8; n++)
                    if (n * 8 < a.c.dim)
                        *reinterpret_cast<uint32_t*>(out + n * 8) = pack2<T>(o[n][hf * 2] * inv, o[n][hf * 2 + 1] * inv);
                if (quad == 0 && a.lse)
                    a.lse[at[hf]] = sum == 0.0f ? -INFINITY : (m[hf] + log2f(sum)) * 0.6931471805599453f;
            } else {
                float* out = reinterpret_cast<float*>(part) + r * DP + quad * 2;
#pragma unroll
                for (int n = 0; n < DP / 8; n++)
                    if (n * 8 < a.c.dim)
                        *reinterpret_cast<float2*>(out + n * 8) = make_float2(o[n][hf * 2], o[n][hf * 2 + 1]);
                if (quad == 0)
                    *reinterpret_cast<float2*>(part + (static_cast<int64_t>(plan.rows_cap) * DP * 4 + r * 8)) =
                        make_float2(m[hf], sum);
            }
        }
    }
}

// The rows of pairs that lie in several pieces: out = sum 2^(m - M) o / L over
// the parts, in their order.  SHARE of a CTA's eight warps take a row together
// (each its own parts), a lane has DP / 32 values.  Bound: latency (the parts
// are in L2), so a row's parts are spread over as many warps as there are.
constexpr int JW = 8;
template <typename T, int DP, int SHARE>
__global__ void __launch_bounds__(JW * 32) attn_join_kernel(const PagedAttnArgs a, const RowsPlan plan) {
    constexpr int E = DP / 32, ROWS = JW / SHARE;
    __shared__ float s_o[JW][DP];
    __shared__ float2 s_ml[JW];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.q_heads / a.c.kv_heads;
    const int64_t all = static_cast<int64_t>(a.c.n_seq) * a.c.kv_heads * plan.rows_cap;
    bool waited = false;
    for (int64_t u0 = static_cast<int64_t>(blockIdx.x) * ROWS; u0 < all; u0 += static_cast<int64_t>(gridDim.x) * ROWS) {
        const int64_t u = u0 + warp / SHARE, pair = u / plan.rows_cap;
        const int r = static_cast<int>(u - pair * plan.rows_cap);
        const int s = static_cast<int>(pair / a.c.kv_heads), hk = static_cast<int>(pair - static_cast<int64_t>(s) * a.c.kv_heads);
        Seq q{0, 0, 0};
        if (u < all) q = load_seq(a.c, s);  // (the rows kernel started this one after its own wait: they are there)
        if (!waited) griddep_wait();
        waited = true;
        int2 span = make_int2(0, 0);
        if (q.n > 0 && q.n <= MAX_ROWS / group && r < q.n * group) span = plan.spans[pair];
        const bool act = span.x != span.y;
        float t = -INFINITY, sum = 0.0f, o[E];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = 0.0f;
        if (act)
#pragma unroll 4
            for (int c = span.x + warp % SHARE; c <= span.y; c += SHARE) {
                const uint8_t* part = plan.parts + (static_cast<int64_t>(c) * 2 + (c == span.x ? 1 : 0)) * plan.slot;
                const float2 ml = *reinterpret_cast<const float2*>(part + (static_cast<int64_t>(plan.rows_cap) * DP * 4 + r * 8));
                float x[E];
#pragma unroll
                for (int e = 0; e < E; e++) x[e] = reinterpret_cast<const float*>(part)[r * DP + e * 32 + lane];
                const float t2 = fmaxf(t, ml.x), base = t2 == -INFINITY ? 0.0f : t2;
                const float f = ex2(t - base), w = ex2(ml.x - base);
                t = t2;
                sum = sum * f + ml.y * w;
#pragma unroll
                for (int e = 0; e < E; e++) o[e] = o[e] * f + x[e] * w;
            }
        if constexpr (SHARE > 1) {
            if (lane == 0) s_ml[warp] = make_float2(t, sum);
#pragma unroll
            for (int e = 0; e < E; e++) s_o[warp][e * 32 + lane] = o[e];
            __syncthreads();
            const int w0 = warp - warp % SHARE;
            t = s_ml[w0].x;
#pragma unroll
            for (int w = 1; w < SHARE; w++) t = fmaxf(t, s_ml[w0 + w].x);
            const float base = t == -INFINITY ? 0.0f : t;
            sum = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < SHARE; w++) {
                const float f = ex2(s_ml[w0 + w].x - base);
                sum += s_ml[w0 + w].y * f;
#pragma unroll
                for (int e = 0; e < E; e++) o[e] += s_o[w0 + w][e * 32 + lane] * f;
            }
            __syncthreads();
        }
        if (act && warp % SHARE == 0) {
            const int i = r / group, gi = r - i * group;
            const int64_t at = static_cast<int64_t>(q.row0 + i) * a.q_heads + hk * group + gi;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            T* out = static_cast<T*>(a.out) + at * a.c.dim;
#pragma unroll
            for (int e = 0; e < E; e++)
                if (e * 32 + lane < a.c.dim) out[e * 32 + lane] = from_f32<T>(o[e] * inv);
            if (lane == 0 && a.lse) a.lse[at] = sum == 0.0f ? -INFINITY : (t + log2f(sum)) * 0.6931471805599453f;
        }
    }
    if (!waited) griddep_wait();
}

// ---------------------------------------------------------------- many rows
// The sequence that packed row `row` belongs to (the last s with cu[s] <= row).
__device__ __forceinline__ int seq_of_row(const int32_t* cu, int n_seq, int row) {
    int lo = 0, hi = n_seq;  // cu[lo] <= row < cu[hi] (cu[n_seq] taken as the end)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(cu + mid) <= row) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The plain kernel: one warp per (row, head), keys one after another, the
// softmax's running maximum and sum in f32 (m' = max(m, s), l' = l 2^(m - m')
// + 2^(s - m'), o' likewise), four values of the head dim per lane.
template <typename T>
__global__ void __launch_bounds__(128) paged_attention_row_kernel(const PagedAttnArgs a, int skip, int* err) {
    griddep_wait();
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (unit >= static_cast<int64_t>(a.c.n_rows) * a.q_heads) return;
    const int row = static_cast<int>(unit / a.q_heads), h = static_cast<int>(unit - static_cast<int64_t>(row) * a.q_heads);
    const int hk = h / (a.q_heads / a.c.kv_heads);
    const int s = a.c.cu ? seq_of_row(a.c.cu, a.c.n_seq, row) : row;
    const int n = a.c.cu ? __ldg(a.c.cu + s + 1) - __ldg(a.c.cu + s) : 1;
    const int i = a.c.cu ? row - __ldg(a.c.cu + s) : 0;
    if (i < 0 || i >= n || i >= a.max_q) return;  // a row of no sequence
    if (n <= skip) return;
    const int p = __ldg(a.c.ctx + s) - n + i;
    const float scale2 = a.scale * 1.4426950408889634f;
    float q[4], o[4] = {0, 0, 0, 0};
    const int d0 = lane * 4;
    const bool in = d0 < a.c.dim;
    const T* qp = static_cast<const T*>(a.q) + row * a.q_tok + h * a.q_head + d0;
    for (int c = 0; c < 4; c++) q[c] = in ? to_f32(qp[c]) * scale2 : 0.0f;
    float m = -INFINITY, l = 0.0f;
    const int first = a.window > 0 ? max(0, p - a.window + 1) : 0;
    for (int j = first; j <= p; j++) {
        const int col = j >> a.c.page_log2, slot = j & (a.c.page - 1);
        const int pg = col < a.c.n_cols ? __ldg(a.c.table + s * a.c.table_stride + col) : -1;
        float k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
        if (static_cast<unsigned>(pg) >= static_cast<unsigned>(a.c.n_pages)) {
            record_error(err, DEVERR_BAD_PAGE);
        } else if (in) {
            const T* kp = static_cast<const T*>(a.c.k) + pg * a.c.k_page + slot * a.c.k_tok + hk * a.c.k_head + d0;
            const T* vp = static_cast<const T*>(a.c.v) + pg * a.c.v_page + slot * a.c.v_tok + hk * a.c.v_head + d0;
            for (int c = 0; c < 4; c++) { k[c] = to_f32(kp[c]); v[c] = to_f32(vp[c]); }
        }
        float x = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
        for (int w = 16; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
        const float m2 = fmaxf(m, x);
        const float f = m2 == -INFINITY ? 0.0f : exp2f(m - m2), e = m2 == -INFINITY ? 0.0f : exp2f(x - m2);
        m = m2;
        l = l * f + e;
        for (int c = 0; c < 4; c++) o[c] = o[c] * f + e * v[c];
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    T* op = static_cast<T*>(a.out) + unit * a.c.dim + d0;
    if (in)
        for (int c = 0; c < 4; c++) op[c] = from_f32<T>(o[c] * inv);
    if (lane == 0 && a.lse) a.lse[unit] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace

namespace {

int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

// Workspace of the rows kernel: spans of all pairs, then two parts per piece.
struct RowsSpace {
    int64_t spans = 0, slot = 0, bytes = 0;
    int rows_cap = 0;
};
RowsSpace rows_space(const PagedAttnArgs& a, int sms) {
    RowsSpace w;
    const int group = a.q_heads / a.c.kv_heads;
    if (group > MAX_ROWS || a.max_q == 0) return w;
    const int dp = a.c.dim > 64 ? 128 : 64;
    w.rows_cap = std::min(MAX_ROWS / group, a.max_q) * group;
    w.slot = up256(w.rows_cap * (dp * 4ll + 8));
    w.spans = up256(8ll * a.c.n_seq * a.c.kv_heads);
    w.bytes = w.spans + 2ll * sms * NW * w.slot;
    return w;
}

}  // namespace

int paged_attention_workspace(const PagedAttnArgs& a, int64_t* bytes) {
    int rc = 0;
    DeviceState* ds = device_state(&rc);
    if (!ds) return rc;
    *bytes = rows_space(a, ds->sm_count).bytes;
    return TVQ_OK;
}

namespace {

// The cache as a {value, token, half, head, page} tensor map, boxes of 64
// values x `box` tokens x `halves` (128-byte swizzle).  A head dim that is no
// multiple of 64 stays one dimension, so that nothing behind it is read.
int cache_map(CUtensorMap* map, const PagedView& c, const void* ptr, int64_t tok, int64_t head, int64_t page, int box,
              int halves) {
    const bool whole = c.dim % 64 == 0;
    const uint64_t dims[5] = {static_cast<uint64_t>(whole ? 64 : c.dim), static_cast<uint64_t>(c.page),
                              static_cast<uint64_t>(whole ? c.dim / 64 : 1), static_cast<uint64_t>(c.kv_heads),
                              static_cast<uint64_t>(c.n_pages)};
    const uint64_t strides[4] = {static_cast<uint64_t>(tok) * 2, 128, static_cast<uint64_t>(head) * 2,
                                 static_cast<uint64_t>(page) * 2};
    const uint32_t boxes[5] = {64, static_cast<uint32_t>(box), static_cast<uint32_t>(halves), 1, 1};
    return make_tma_16bit(map, ptr, 5, dims, strides, boxes);
}

template <typename T, int DP>
int launch_rows(const PagedAttnArgs& a, DeviceState* ds, cudaStream_t st) {
    using C = RowsCfg<DP>;
    static const cudaError_t attr =
        cudaFuncSetAttribute(attn_rows_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    TVQ_CUDA(attr);
    const RowsSpace w = rows_space(a, ds->sm_count);
    RowsPlan plan;
    plan.spans = static_cast<int2*>(a.ws);
    plan.parts = static_cast<uint8_t*>(a.ws) + w.spans;
    plan.rows_cap = w.rows_cap;
    plan.slot = w.slot;
    plan.box = std::min(a.c.page, C::KT);
    plan.by_value = a.c.dim % 64 != 0;
    plan.box_halves = a.c.dim == 128 && plan.box == C::KT ? 2 : 1;
    CUtensorMap tmK, tmV;
    int rc = cache_map(&tmK, a.c, a.c.k, a.c.k_tok, a.c.k_head, a.c.k_page, plan.box, plan.box_halves);
    if (rc) return rc;
    rc = cache_map(&tmV, a.c, a.c.v, a.c.v_tok, a.c.v_head, a.c.v_page, plan.box, plan.box_halves);
    if (rc) return rc;
    rc = launch_pdl(attn_rows_kernel<T, DP>, dim3(ds->sm_count), dim3(NTHR), C::SMEM, st, tmK, tmV, a, plan,
                    ds->d_error);
    if (rc) return rc;
    // One CTA of the join fits beside the rows kernel's on an SM.  Rows for all of them: eight warps a row;
    // more rows: a warp each.
    const int64_t rows = static_cast<int64_t>(a.c.n_seq) * a.c.kv_heads * w.rows_cap;
    if (rows <= ds->sm_count)
        return launch_pdl(attn_join_kernel<T, DP, JW>, dim3(static_cast<unsigned>(rows)), dim3(JW * 32), 0, st, a, plan);
    const int64_t ctas = std::min<int64_t>((rows + JW - 1) / JW, ds->sm_count * 8ll);
    return launch_pdl(attn_join_kernel<T, DP, 1>, dim3(static_cast<unsigned>(ctas)), dim3(JW * 32), 0, st, a, plan);
}

template <typename T>
int launch_attention(const PagedAttnArgs& a, DeviceState* ds, cudaStream_t st) {
    const int group = a.q_heads / a.c.kv_heads;
    int rc = TVQ_OK;
    if (group <= MAX_ROWS) rc = a.c.dim > 64 ? launch_rows<T, 128>(a, ds, st) : launch_rows<T, 64>(a, ds, st);
    if (rc || static_cast<int64_t>(a.max_q) * group <= MAX_ROWS) return rc;
    const int64_t units = static_cast<int64_t>(a.c.n_rows) * a.q_heads;
    return launch_pdl(paged_attention_row_kernel<T>, dim3(static_cast<unsigned>((units + 3) / 4)), dim3(128), 0, st, a,
                      MAX_ROWS / group, ds->d_error);
}

}  // namespace

int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
    int rc = 0;
    DeviceState* ds = device_state(&rc);
    if (!ds) return rc;
    TVQ_CHECK(ds->cc_major == 10, TVQ_ERR_UNSUPPORTED, "the paged attention needs an sm_100 device");
    if (a.c.n_rows == 0 || a.max_q == 0) return TVQ_OK;
    return a.c.type == TVQ_TYPE_F16 ? launch_attention<__half>(a, ds, st) : launch_attention<__nv_bfloat16>(a, ds, st);
}

}  // namespace tvq
