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
// attn_rows_kernel: calls without a sequence of more than 16 such rows (single
// tokens, a few drafted ones).  Every key and value is used for at most 16 rows, so the
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
// Measured: 24 sequences of up to 24000 tokens, 32 heads on 8 of 128: 223 us,
// 6.2 TB/s, 95 % of a copy's rate.  48 sequences of up to 1024, 25 heads of 64,
// whose tokens have their heads side by side: 45 us, of which ~10 are the start
// and the join, and 128-byte pieces get 4.9 TB/s (2 KB ones 5.8).  One token
// of one sequence of 700: 8.4 us, all latency.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "tvq_common.cuh"
#include "tvq_decode.h"
#include "tvq_exact.cuh"
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

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// The softmax's weights meet V in its type, as multiples of 2^-24 at the
// smallest in float16.  A factor 2^UP, which the sum l carries as well, keeps
// the largest (1, or the tile kernel's 2^8) just within the type's 65504, so
// that a weight is whole down to 2^(-14 - UP) of the largest and counts down to
// 2^(-25 - UP): many keys beside one that has nearly all the weight are not
// lost.  It costs nothing, the exponent's offset being subtracted in any case.
// (bfloat16 has float's range.)
template <typename T, int LARGEST>  // log2 of the largest weight
constexpr int UP = std::is_same<T, __half>::value ? 15 - LARGEST : 0;

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

// a / b for a >= 0, b > 0; short for what fits 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// One sequence as the kernels see it.
struct Seq {
    int row0;  // first packed row
    int n;     // new rows
    int m;     // those that the call takes: the first max_q, as the workspace is sized for
    int len;   // tokens in the cache
};
__device__ __forceinline__ Seq load_seq(const PagedAttnArgs& a, int s) {
    const PagedView& c = a.c;
    Seq q;
    q.len = __ldg(c.ctx + s);
    if (c.cu) {
        q.row0 = __ldg(c.cu + s);
        q.n = __ldg(c.cu + s + 1) - q.row0;
        q.m = q.row0 < 0 ? 0 : max(0, min(min(q.n, a.max_q), c.n_rows - q.row0));
    } else {
        q.row0 = s;
        q.n = q.m = 1;
    }
    return q;
}

// The tiles of KT keys [first, end) that the rows of a sequence see together:
// one at least, so that rows without keys are written too.
template <int KT>
__device__ __forceinline__ int2 seq_tiles(const Seq& q, int window) {
    const int p0 = q.len - q.n;
    const int first = window > 0 ? max(0, p0 - window + 1) / KT : 0;
    return make_int2(first, max(first + 1, (max(p0 + q.m, 0) + KT - 1) / KT));
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
    const int group = a.q_heads / a.c.kv_heads;  // (max_q * group <= MAX_ROWS: few_rows)
    static_assert(2 * NW * C::STAGES <= NTHR - 32);
    if (tid < 2 * NW * C::STAGES) {
        mbar_init(reinterpret_cast<uint64_t*>(sm + C::OFF_BAR) + tid, 1);
        fence_barrier_init();
    } else if (tid == NTHR - 1) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    griddep_wait();
    griddep_launch();  // the join kernel's CTAs fit beside this one's and wait there

    // ---- the pieces of the line of tiles
    auto weight = [&](int s) -> int {
        if (s >= a.c.n_seq) return 0;
        const Seq q = load_seq(a, s);
        if (q.m == 0) return 0;
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
    const int64_t per = max(static_cast<int64_t>(1), quotient(total + pieces - 1, pieces));
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
                c.q = load_seq(a, ++c.s);
            } while (c.q.m == 0);
        }
        enter(c, 0);
        return true;
    };
    cur.left = stop - begin;
    if (cur.left > 0) {
        cur.s = s_seq[mine];
        cur.q = load_seq(a, cur.s);
        const int64_t in_seq = begin - s_at[mine];
        const int2 t = seq_tiles<KT>(cur.q, a.window);
        cur.hk = static_cast<int>(quotient(in_seq, t.y - t.x));
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
            bool read;  // (a box behind the sequence's end or before all windows is zeros)
        };
        int next_t = cur.left > 0 ? cur.first : 0;
        bool more = cur.left > 0;
        auto look = [&]() {
            Window w;
            w.t = w.end = next_t;
            w.hk = cur.hk;
            w.page = -1;  // outside the tensor map: zeros
            w.read = false;
            if (!more) return w;
            w.end = min(cur.end, next_t + 8 / boxes);
            const int j = w.t * KT + sub * plan.box;
            const int low = a.window > 0 ? cur.q.len - cur.q.n - a.window + 1 : 0;  // the first key that a row sees
            if (j < w.end * KT && j < cur.q.len && j + plan.box > low) {
                w.read = true;
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
            if (w.read && static_cast<unsigned>(w.page) >= static_cast<unsigned>(a.c.n_pages)) {
                record_error(err, DEVERR_BAD_PAGE);
                w.page = -1;
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
    constexpr float up = UP<T, 0>, down = 1.0f / (1 << UP<T, 0>);
    const int g = lane >> 2, quad = lane & 3;
    int stage = 0, phase = 0;
    bool ok = true;
    for (bool go = true; go; go = next_pair(cur)) {
        // ---- the pair's rows as A fragments
        const int rows = cur.q.m * group;
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
                // (rounded up: not even the rounding of huge scores makes a weight larger than 2^up)
                const float to = m2 == -INFINITY ? 0.0f : m2, base = __fadd_ru(to, -up);
                const float f = ex2(m[hf] - to);
                m[hf] = m2;
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < KT / 4; e++) {
                    x[e] = ex2(x[e] - base);
                    sum += x[e];
                }
                l[hf] = l[hf] * f + sum;
                // the weights meet V in its own type (see UP): 2^-11 (f16) or 2^-8 (bf16) of each, as the
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
                make_int2(piece, static_cast<int>(quotient(at0 + cur.all.y - cur.all.x - 1, per)));
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
                    a.lse[at[hf]] = sum == 0.0f ? -INFINITY : (m[hf] + log2f(sum * down)) * 0.6931471805599453f;
            } else {
                float* out = reinterpret_cast<float*>(part) + r * DP + quad * 2;
#pragma unroll
                for (int n = 0; n < DP / 8; n++)
                    if (n * 8 < a.c.dim)
                        *reinterpret_cast<float2*>(out + n * 8) = make_float2(o[n][hf * 2] * down, o[n][hf * 2 + 1] * down);
                if (quad == 0)
                    *reinterpret_cast<float2*>(part + (static_cast<int64_t>(plan.rows_cap) * DP * 4 + r * 8)) =
                        make_float2(m[hf], sum * down);
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
__global__ void __launch_bounds__(JW * 32, 6) attn_join_kernel(const PagedAttnArgs a, const RowsPlan plan) {
    constexpr int E = DP / 32, ROWS = JW / SHARE, AHEAD = DP == 128 ? 2 : 4;
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
        Seq q{};
        if (u < all) q = load_seq(a, s);  // (the rows kernel started this one after its own wait: they are there)
        if (!waited) griddep_wait();
        waited = true;
        int2 span = make_int2(0, 0);
        if (r < q.m * group) span = plan.spans[pair];
        const bool act = span.x != span.y;
        float t = -INFINITY, sum = 0.0f, o[E];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = 0.0f;
        if (act)
            for (int c0 = span.x + warp % SHARE; c0 <= span.y; c0 += SHARE * AHEAD) {
                float2 ml[AHEAD];
                float x[AHEAD][E];
#pragma unroll
                for (int i = 0; i < AHEAD; i++) {  // (asked for together: one after the other, each took ~800 cycles)
                    const int c = c0 + i * SHARE;
                    ml[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
                    for (int e = 0; e < E; e++) x[i][e] = 0.0f;
                    if (c > span.y) continue;
                    const uint8_t* part = plan.parts + (static_cast<int64_t>(c) * 2 + (c == span.x ? 1 : 0)) * plan.slot;
                    ml[i] = *reinterpret_cast<const float2*>(part + (static_cast<int64_t>(plan.rows_cap) * DP * 4 + r * 8));
#pragma unroll
                    for (int e = 0; e < E; e++) x[i][e] = reinterpret_cast<const float*>(part)[r * DP + e * 32 + lane];
                }
                float t2 = t;
#pragma unroll
                for (int i = 0; i < AHEAD; i++) t2 = fmaxf(t2, ml[i].x);
                const float base = t2 == -INFINITY ? 0.0f : t2, f = ex2(t - base);
                t = t2;
                sum *= f;
#pragma unroll
                for (int e = 0; e < E; e++) o[e] *= f;
#pragma unroll
                for (int i = 0; i < AHEAD; i++) {
                    const float w = ex2(ml[i].x - base);
                    sum += ml[i].y * w;
#pragma unroll
                    for (int e = 0; e < E; e++) o[e] += x[i][e] * w;
                }
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
// attn_tile_kernel: calls with more than 16 rows in some sequence, on the
// tcgen05 tensor cores.  A unit is two tiles of up to 128 rows (whole tokens:
// 128 / group of them, with all heads of the group) of one (sequence, kv head),
// which share the stream of 128-key tiles of K and V; where a sequence's rows
// end with the first of the two, both take those rows, one the even key tiles
// and one the odd.  All (unit, key tile) stand in one line that is cut into
// equal pieces, one for each SM, as above, so ragged prompts, causal triangles
// and few rows over many keys all fill the GPU; units cut by a piece's end are
// joined by attn_tile_join_kernel.
//
// Per tile t and key tile j, in tensor memory: S_t = Q_t K_j^T (128 x 128
// f32), its softmax's weights P_t (16-bit, over S_t's columns: those of keys
// 0-63 from column 0, of keys 64-127 from column 64), O_t += P_t V_j.
//   warp 0       TMA: Q of a unit, then K_j, V_j through one ring
//   warp 1       MMA issuer: for each j, PV_A(j-1), S_A(j), PV_B(j-1), S_B(j),
//                so one tile's softmax runs under the other's products
//   warp 2       tensor memory; zeros over the values behind a sequence's end
//                (they may be anything, and 0 x NaN is NaN)
//   warp 3       walks the piece and leaves the units for the others in shared
//                memory, up to four ahead
//   warps 4-19   softmax, eight for each tile: two threads have a row, 64 keys
//                each (one thread with 128 keys has too little to do at once:
//                its instructions waited 1.4 cycles each for one another)
// O stays relative to the row's first maximum until the running one exceeds it
// by 2^8 (then O and l are scaled by the softmax warps): weights stay below
// 2^8, within either 16-bit type (see UP), and nearly no tile is scaled twice.
// The weights of the first 32 keys of each thread are handed over by themselves,
// so that half of PV runs while the other weights are made (414 -> 403 us below).
// A commit of S_t(j) covers PV_t(j-1), issued before it, so scaling O needs no
// barrier of its own; and in-order execution of the products lets S_t(j)
// overwrite P_t(j-1) right behind the product that reads it.
// Bound: the two products of a tile and j (2 x 512 cycles at D = 128) wait for
// its softmax and the softmax for them.  Its 128 x 128 exponentials take the
// special-function units 1024 cycles, with reading, maximum, exchange and
// writing ~1900, so the tensor cores rest in between.
// (Polynomials on the FMA pipe for a part of the exponentials did not help:
// the chain through a softmax is as long, with more to issue.  Nor did an
// issuer that takes whichever tile is ready, or one that starts a unit's first
// S before the last PV of the unit before: their code comes between the
// products, which cost the long chunk 25 % and 4 %.)
// Measured: a chunk of 4096 tokens behind 16384, 16 heads on 4 of 128: 404 us,
// 1191 TFLOP/s, 72 % of a large product's rate at full clock; called again and
// again, under the power limit, 470 us, 1023 TFLOP/s, 73 % of what the product
// sustains.  Nine prompts of up to 1023, 12 heads of 64: 51 us, where a unit's end and the next one's first tile take
// ~4 us beside its few tiles, and the start ~6.
constexpr int TM = 128, TKEYS = 128;
constexpr int TTHR = 640;
enum : int {
    DEVERR_PTILE_EMPTY = 73, DEVERR_PTILE_Q = 74, DEVERR_PTILE_KV = 75, DEVERR_PTILE_P = 76, DEVERR_PTILE_S = 77,
    DEVERR_PTILE_O = 78, DEVERR_PTILE_FIX = 79, DEVERR_PTILE_DRAIN = 80, DEVERR_PTILE_WORK = 81
};

template <int DP>
struct TileCfg {
    static constexpr int HALVES = DP / 64;
    static constexpr int HALF = 128 * 128;               // 128 rows of 64 values, 128-byte swizzle
    static constexpr int QT = HALVES * HALF;             // one tile of Q
    static constexpr int STAGE = HALVES * HALF;          // 128 keys or values
    static constexpr int STAGES = 163840 / STAGE;        // 5 or 10
    static constexpr int OFF_RING = 2 * QT;
    static constexpr int OFF_BAR = OFF_RING + STAGES * STAGE;
    static constexpr int BARS = 3 * STAGES + 23;
    static constexpr int OFF_WORK = OFF_BAR + (BARS + 1) * 8;  // Work[4]
    static constexpr int OFF_X = OFF_WORK + 4 * 96;      // float [2][2][128]: what the halves of a row tell each other
    static constexpr int OFF_MISC = OFF_X + 2 * 2 * 128 * 4;  // int64 at, int seq, tmem
    static constexpr int SMEM = OFF_MISC + 16;
    static constexpr int64_t SLOT = 2 * TM * (DP * 4 + 8);
    static constexpr uint32_t COL_S = 0, COL_O = 256, COLS = 512;
};

struct Begun {
    int rows, row0, m, hk;  // rows of the unit (0: none); the sequence's; the kv head
    int unit, last, pad[2];  // which unit of the sequence; the last piece that has a part of it
};
struct TilePlan {
    uint8_t* parts;  // [grid][2] slots: float4 [DP / 4][256 rows] (a warp's rows side by side), then float2 (m, l) [256]
    struct Begun* begun;  // [grid]: the unit that a piece begins and does not end
    int tokens;      // of a tile: 128 / group
    int box, box_halves, by_value;  // as RowsPlan's, KT = 128
    float scale2;    // log2(e) |scale|, not 0
    int negative;
};

// A unit's tiles of rows: tokens [i0, i0 + cnt) each, key tiles [first, end).
struct Unit {
    int i0[2], cnt[2], first[2], end[2];
    int f, e;  // of both
};
__device__ __forceinline__ Unit make_unit(const Seq& q, int u, int tokens, int window) {
    Unit w;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        w.i0[t] = (2 * u + t) * tokens;
        w.cnt[t] = max(0, min(tokens, q.m - w.i0[t]));
        const int pa = q.len - q.n + w.i0[t], pb = pa + w.cnt[t] - 1;
        w.first[t] = window > 0 ? max(0, pa - window + 1) / TKEYS : 0;
        w.end[t] = max(w.first[t] + 1, (max(pb + 1, 0) + TKEYS - 1) / TKEYS);
        if (w.cnt[t] == 0) w.first[t] = w.end[t] = 0;
    }
    w.f = w.first[0];
    w.e = max(w.end[0], w.end[1]);
    return w;
}
__device__ __forceinline__ int seq_units(const Seq& q, int tokens) { return (q.m + 2 * tokens - 1) / (2 * tokens); }

// A unit's share of a CTA's piece: key tiles [a, b), of them [lo, hi) for each
// row tile (lo >= hi: none).
struct Work {
    int hk, row0, n, len, a, b, more;
    int whole, begins;  // the piece holds all of the unit's key tiles; the first of them
    int i0[2], cnt[2], lo[2], hi[2];
    int s;
    int dup;  // both row tiles are the first one: key tiles lo, lo + 2, ... each
};
static_assert(sizeof(Work) <= 96);

// Q_t K_j^T with B transposed as given by idesc; A in tensor memory for P V.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// A B operand whose N runs along the rows of 128 bytes (V: [key][value]): groups
// of 64 values HALF bytes apart, groups of 8 keys 1024 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t saddr, uint32_t group) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(group >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}
__device__ __forceinline__ void tma_load_4d(const CUtensorMap* map, uint64_t* bar, uint32_t dst, int c0, int c1, int c2,
                                            int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
        " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// wait_full with a code
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, int* err, int code) {
    const bool ok = mbar_wait_for(bar, parity, nullptr, code, TVQ_WAIT_LIMIT_NS);
    if (!ok) record_error(err, code);
    return ok;
}

template <typename T, int DP>
__global__ void __launch_bounds__(TTHR, 1)
    attn_tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const PagedAttnArgs a, const TilePlan plan, int* err) {
    using C = TileCfg<DP>;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint64_t* kv_full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    uint64_t* kv_empty = kv_full + C::STAGES;
    uint64_t* q_full = kv_empty + C::STAGES;  // [2] each
    uint64_t* q_empty = q_full + 2;
    uint64_t* s_full = q_empty + 2;
    uint64_t* p_full = s_full + 2;
    uint64_t* o_full = p_full + 2;
    uint64_t* drain = o_full + 2;
    uint64_t* w_full = drain + 1;  // [4] each
    uint64_t* w_empty = w_full + 4;
    uint64_t* p_half = w_empty + 4;  // [2] the weights of keys 0-31 and 64-95
    uint64_t* b_ready = p_half + 2;  // tile B's part of tile A's rows is there
    uint64_t* b_free = b_ready + 1;  // and has been read
    uint64_t* v_fixed = b_free + 1;  // [STAGES] the values there end with the sequence
    Work* works = reinterpret_cast<Work*>(sm + C::OFF_WORK);
    int64_t* s_at = reinterpret_cast<int64_t*>(sm + C::OFF_MISC);
    int* s_seq = reinterpret_cast<int*>(s_at + 1);
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(s_seq + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.q_heads / a.c.kv_heads;
    if (tid < C::BARS) {
        uint64_t* bar = kv_full + tid;
        int users = 1;
        if (bar >= kv_empty && bar < q_full) users = 2;                                          // the issuer and the fixing warp
        if ((bar >= p_full && bar < o_full) || (bar >= p_half && bar < v_fixed)) users = 8;     // a tile's warps
        if (bar >= w_empty && bar < p_half) users = 19;  // TMA, MMA, fixing and sixteen softmax warps
        mbar_init(bar, users);
        fence_barrier_init();
    } else if (tid == TTHR - 1) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (warp == 2) {
        tmem_alloc(tmem_holder, C::COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    griddep_wait();
    griddep_launch();  // the join's CTAs take the place of this kernel's as these end

    // ---- the piece of the line of key tiles
    auto weight = [&](int s) -> int64_t {  // of one kv head
        if (s >= a.c.n_seq) return 0;
        const Seq q = load_seq(a, s);
        if (q.m == 0) return 0;
        int64_t sum = 0;
        for (int u = 0; u < seq_units(q, plan.tokens); u++) {
            const Unit w = make_unit(q, u, plan.tokens, a.window);
            sum += w.e - w.f;
        }
        return sum;
    };
    auto scan = [&](int64_t x, int64_t* all) {  // inclusive, over the CTA (the ring's memory is free yet)
        int64_t* buf = reinterpret_cast<int64_t*>(sm + C::OFF_RING);
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) buf[warp] = x;
        __syncthreads();
        int64_t sum = 0;
        for (int w = 0; w < TTHR / 32; w++) {
            if (w < warp) x += buf[w];
            sum += buf[w];
        }
        *all = sum;
        return x;
    };
    int64_t total = 0, w0 = 0, inc0 = 0;
    for (int s0 = 0; s0 < a.c.n_seq; s0 += TTHR) {
        int64_t all;
        w0 = weight(s0 + tid);
        inc0 = scan(w0, &all);
        total += all;
    }
    total *= a.c.kv_heads;
    const int64_t per = max(static_cast<int64_t>(1), quotient(total + gridDim.x - 1, gridDim.x));
    const int64_t begin = per * blockIdx.x, stop = min(total, begin + per);
    int64_t before = 0;
    for (int s0 = 0; s0 < a.c.n_seq; s0 += TTHR) {
        int64_t all = 0, w = w0, inc = inc0;
        if (a.c.n_seq > TTHR) {
            w = weight(s0 + tid);
            inc = scan(w, &all);
        }
        const int64_t hi = (before + inc) * a.c.kv_heads, lo = hi - w * a.c.kv_heads;
        if (w > 0 && begin >= lo && begin < hi) {
            *s_seq = s0 + tid;
            *s_at = lo;
        }
        before += all;
    }
    fence_proxy_async_smem();  // (the scan's words in the ring, before TMA writes there)
    __syncthreads();
    bool ok = true;
    // the k-th unit of the piece; false: there is none (or a wait gave up)
    auto take = [&](int k) -> bool {
        ok = ok && wait_bar(w_full + (k & 3), (k >> 2) & 1, err, DEVERR_PTILE_WORK);
        return ok && works[k & 3].more;
    };
    auto done = [&](int k) {  // by one thread of a warp, once the warp needs nothing more of it
        mbar_arrive(w_empty + (k & 3));
    };
    if (warp < 4) {
        if (warp == 3) {
            // ------------------------------------------------ the walk
            if (lane == 0) {
                Begun begun{};
                int s = 0, hk = 0, u = 0, skip = 0, units = 0;
                int64_t left = stop - begin;
                Seq q{};
                if (left > 0) {
                    s = *s_seq;
                    q = load_seq(a, s);
                    int64_t in = begin - *s_at, one = 0;  // one: tiles of one kv head
                    units = seq_units(q, plan.tokens);
                    for (int i = 0; i < units; i++) {
                        const Unit w = make_unit(q, i, plan.tokens, a.window);
                        one += w.e - w.f;
                    }
                    hk = static_cast<int>(quotient(in, one));
                    in -= hk * one;
                    for (u = 0; u < units; u++) {
                        const Unit w = make_unit(q, u, plan.tokens, a.window);
                        if (in < w.e - w.f) break;
                        in -= w.e - w.f;
                    }
                    skip = static_cast<int>(in);
                }
                for (int k = 0;; k++) {
                    ok = ok && wait_bar(w_empty + (k & 3), ((k >> 2) & 1) ^ 1, err, DEVERR_PTILE_WORK);
                    if (!ok) break;
                    Work& o = works[k & 3];
                    o.more = left > 0;
                    if (left > 0) {
                        const Unit w = make_unit(q, u, plan.tokens, a.window);
                        o.s = s;
                        o.hk = hk;
                        o.row0 = q.row0;
                        o.n = q.n;
                        o.len = q.len;
                        o.a = w.f + skip;
                        o.b = static_cast<int>(min(static_cast<int64_t>(w.e), o.a + left));
                        o.begins = skip == 0;
                        o.whole = skip == 0 && o.b == w.e;
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            o.i0[t] = w.i0[t];
                            o.cnt[t] = w.cnt[t];
                            o.lo[t] = max(w.first[t], o.a);
                            o.hi[t] = min(w.end[t], o.b);
                        }
                        o.dup = w.cnt[1] == 0;
                        if (o.dup) {
                            o.i0[1] = w.i0[0];
                            o.cnt[1] = w.cnt[0];
                            o.lo[1] = o.a + 1;
                            o.hi[1] = o.b;
                        }
                        if (o.begins && !o.whole)
                            begun = Begun{w.cnt[0] + w.cnt[1], q.row0, q.m, hk, u,
                                          static_cast<int>(quotient(stop - left + w.e - w.f - 1, per))};
                        left -= o.b - o.a;
                        skip = 0;
                        if (left > 0 && ++u == units) {
                            u = 0;
                            if (++hk == a.c.kv_heads) {
                                hk = 0;
                                do {
                                    q = load_seq(a, ++s);
                                } while (q.m == 0);
                                units = seq_units(q, plan.tokens);
                            }
                        }
                    }
                    mbar_arrive(w_full + (k & 3));
                    if (!o.more) break;
                }
                plan.begun[blockIdx.x] = begun;
            }
            __syncwarp();
        } else if (warp == 0) {
            // ------------------------------------------------ TMA
            const int boxes = TKEYS / plan.box, loads_h = C::HALVES / plan.box_halves, ops = boxes * loads_h;
            const int b = lane / loads_h, h = lane - b * loads_h;
            const bool issues = lane < ops;
            const int x = plan.by_value ? h * 64 : 0, y = plan.by_value ? 0 : h;
            const uint32_t ring = smem_u32(sm) + C::OFF_RING + h * C::HALF + b * plan.box * 128;
            int n = 0, stage = 0, phase = 1, nq0 = 0, nq1 = 0;
            for (int k = 0; __all_sync(0xffffffffu, take(k)); k++) {
                const Work& w = works[k & 3];
                const int hk = w.hk, len = w.len, end = w.b;
                const int low = a.window > 0 ? len - w.n + w.i0[0] - a.window + 1 : 0;  // the first key that a row sees
                const int32_t* row = a.c.table + w.s * a.c.table_stride;
                auto look = [&](int j) {
                    const int key = j * TKEYS + b * plan.box;
                    if (!issues || j >= end || key >= len || key + plan.box <= low) return 0;
                    const int col = key >> a.c.page_log2;
                    return col < a.c.n_cols ? __ldg(row + col) : -1;
                };
                int page = look(w.a);
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    int& nq = t ? nq1 : nq0;
                    if (w.lo[t] >= w.hi[t] || (t == 1 && w.dup)) continue;
                    ok = ok && wait_bar(q_empty + t, (nq & 1) ^ 1, err, DEVERR_PTILE_EMPTY);
                    if (ok && lane == 0) {
                        mbar_arrive_expect_tx(q_full + t, C::HALVES * plan.tokens * group * 128);
                        for (int i = 0; i < C::HALVES; i++)
                            tma_load_4d(&tmQ, q_full + t, smem_u32(sm) + t * C::QT + i * C::HALF, plan.by_value ? i * 64 : 0,
                                        plan.by_value ? 0 : i, hk * group, w.row0 + w.i0[t]);
                    }
                    if (ok) nq++;
                }
                ok = __all_sync(0xffffffffu, ok);
                for (int j = w.a; ok && j < end; j++) {
                    int now = page;
                    page = look(j + 1);
                    const int key = j * TKEYS + b * plan.box;
                    if (key >= len || key + plan.box <= low) {
                        now = -1;  // behind the sequence's end or before all windows: outside the tensor map, zeros
                    } else if (issues && static_cast<unsigned>(now) >= static_cast<unsigned>(a.c.n_pages)) {
                        record_error(err, DEVERR_BAD_PAGE);
                        now = -1;
                    }
                    const int slot = key & (a.c.page - 1);
                    for (int v = 0; v < 2; v++) {
                        ok = __all_sync(0xffffffffu, wait_bar(kv_empty + stage, phase, err, DEVERR_PTILE_EMPTY));
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(kv_full + stage, C::STAGE);
                        __syncwarp();
                        if (issues)
                            tma_load_5d(v ? &tmV : &tmK, kv_full + stage, ring + stage * C::STAGE, x, slot, y, hk, now);
                        n++;
                        if (++stage == C::STAGES) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) done(k);
            }
            // every load lands before the CTA may end
            if (lane == 0) {
                for (int i = max(0, n - C::STAGES); i < n; i++)
                    wait_bar(kv_full + i % C::STAGES, (i / C::STAGES) & 1, nullptr, DEVERR_PTILE_DRAIN);
                if (nq0) wait_bar(q_full, (nq0 - 1) & 1, nullptr, DEVERR_PTILE_DRAIN);
                if (nq1) wait_bar(q_full + 1, (nq1 - 1) & 1, nullptr, DEVERR_PTILE_DRAIN);
            }
            __syncwarp();
        } else if (warp == 1) {
            // ------------------------------------------------ MMA issuer
            constexpr uint32_t ty = std::is_same<T, __half>::value ? 0u : 1u;
            // (bit 13 negates Q: with a negative scale the largest score is still the largest product)
            const uint32_t idesc_s = (1u << 4) | (ty << 7) | (ty << 10) | (static_cast<uint32_t>(TKEYS >> 3) << 17) |
                                     (static_cast<uint32_t>(TM >> 4) << 24) | (plan.negative ? 1u << 13 : 0u);
            constexpr uint32_t idesc_o = (1u << 4) | (ty << 7) | (ty << 10) | (1u << 16) |
                                         (static_cast<uint32_t>(DP >> 3) << 17) | (static_cast<uint32_t>(TM >> 4) << 24);
            if (lane == 0) {
                // the ring holds K_a, V_a, K_a+1, ...: step j uses V_{j-1} (stage sv) and K_j (stage sk)
                int sk = 0, pk = 0, nq = 0, np = 0;  // nq, np: a bit for each row tile's parity
                uint32_t fixes = 0;                  // and one for each stage
                auto scores = [&](int t, int q, uint32_t ka) {  // S_t = Q_q K^T
                    const uint64_t qd = smem_desc_k_sw128(smem_u32(sm) + q * C::QT), kd = smem_desc_k_sw128(ka);
#pragma unroll
                    for (int i = 0; i < DP / 16; i++) {  // (values behind the head dim are zeros in both)
                        const uint64_t off = ((i >> 2) * C::HALF + (i & 3) * 32) >> 4;
                        umma_f16(tmem + C::COL_S + t * TKEYS, qd + off, kd + off, idesc_s, i > 0);
                    }
                    umma_commit(s_full + t);
                };
                auto values = [&](int t, uint32_t va, bool first) {  // O_t (+)= P_t V
                    const uint64_t vd = smem_desc_mn_sw128(va, C::HALF);
                    for (int c = 0; ok && c < 2; c++) {  // keys 0-31 and 64-95, while the others' weights are made
                        ok = wait_bar((c ? p_full : p_half) + t, (np >> t) & 1, err, DEVERR_PTILE_P);
                        if (!ok) return;
                        tc_fence_after();
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int at = (i >> 1) * 4 + c * 2 + (i & 1);  // of the eight times 16 keys
                            umma_ts(tmem + C::COL_O + t * DP, tmem + C::COL_S + t * TKEYS + (at >> 2) * 64 + (at & 3) * 8,
                                    vd + at * (2048 >> 4), idesc_o, (!first || c > 0 || i > 0) ? 1u : 0u);
                        }
                    }
                    np ^= 1 << t;
                };
                auto fixed = [&](int sv) {  // the values of stage sv end with the sequence
                    ok = ok && wait_bar(v_fixed + sv, fixes >> sv & 1, err, DEVERR_PTILE_FIX);
                    fixes ^= 1u << sv;
                };
                auto next = [&](int& sv, int& pv) {  // behind V_{sv}: the stages of V and K
                    umma_commit(kv_empty + sk);
                    sv = sk + 1;
                    pv = pk;
                    if (sv == C::STAGES) {
                        sv = 0;
                        pv ^= 1;
                    }
                    sk = sv + 1;
                    pk = pv;
                    if (sk == C::STAGES) {
                        sk = 0;
                        pk ^= 1;
                    }
                };
                for (int k = 0; take(k); k++) {
                    const Work& w = works[k & 3];
                    const int first = w.a, end = w.b, len = w.len;
                    const int lo[2] = {w.lo[0], w.lo[1]}, hi[2] = {w.hi[0], w.hi[1]};
                    int sv = 0, pv = 0;
                    if (!w.dup) {
                        // the key tiles in the midst of both row tiles' (their last S and first PV excepted) have a loop
                        // without questions, if they are many: the code between the products is time (441 -> 422 us for
                        // the long chunk), but code that runs a few times costs more to fetch than it saves
                        const int mid = max(lo[0], lo[1]) + 2, mid_end = min(hi[0], hi[1]) - 1;
                        for (int j = first; ok && j <= end; j++) {
                            if (j == mid && mid_end - mid >= 8) {
                                for (; ok && j < mid_end; j++) {
                                    const uint32_t ka = smem_u32(sm) + C::OFF_RING + sk * C::STAGE;
                                    const uint32_t va = smem_u32(sm) + C::OFF_RING + sv * C::STAGE;
                                    ok = wait_bar(kv_full + sk, pk, err, DEVERR_PTILE_KV) &&
                                         wait_bar(kv_full + sv, pv, err, DEVERR_PTILE_KV);
#pragma unroll
                                    for (int t = 0; t < 2; t++) {
                                        if (ok) values(t, va, false);
                                        if (ok) scores(t, t, ka);
                                    }
                                    if (!ok) break;
                                    umma_commit(kv_empty + sv);
                                    next(sv, pv);
                                }
                                if (!ok) break;
                            }
                            const uint32_t ka = smem_u32(sm) + C::OFF_RING + sk * C::STAGE;
                            const uint32_t va = smem_u32(sm) + C::OFF_RING + sv * C::STAGE;
                            if (j < end) ok = wait_bar(kv_full + sk, pk, err, DEVERR_PTILE_KV);
                            if (ok && j > first) ok = wait_bar(kv_full + sv, pv, err, DEVERR_PTILE_KV);
                            // (V of the last key tile, the only one that may end with the sequence)
                            if (j == end && end * TKEYS > len) fixed(sv);
#pragma unroll
                            for (int t = 0; t < 2; t++) {
                                if (ok && j - 1 >= lo[t] && j - 1 < hi[t]) {
                                    values(t, va, j - 1 == lo[t]);
                                    if (ok && j == hi[t]) umma_commit(o_full + t);
                                }
                                if (ok && j >= lo[t] && j < hi[t]) {
                                    if (j == lo[t]) {
                                        ok = wait_bar(q_full + t, (nq >> t) & 1, err, DEVERR_PTILE_Q);
                                        nq ^= 1 << t;
                                        if (!ok) break;
                                    }
                                    scores(t, t, ka);
                                    if (j == hi[t] - 1) umma_commit(q_empty + t);
                                }
                            }
                            if (!ok) break;
                            if (j > first) umma_commit(kv_empty + sv);
                            if (j < end) next(sv, pv);
                        }
                    } else {
                        // key tiles a, a + 2, ... are tile A's, the others B's; S(j) depends on nothing of j - 1, the other's
                        for (int j = first; ok && j <= end; j++) {
                            const uint32_t va = smem_u32(sm) + C::OFF_RING + sv * C::STAGE;
                            if (j < end) {
                                ok = wait_bar(kv_full + sk, pk, err, DEVERR_PTILE_KV);
                                if (ok) {
                                    if (j == first) {
                                        ok = wait_bar(q_full, nq & 1, err, DEVERR_PTILE_Q);
                                        nq ^= 1;
                                    }
                                    if (ok) {
                                        scores((j - first) & 1, 0, smem_u32(sm) + C::OFF_RING + sk * C::STAGE);
                                        if (j == end - 1) umma_commit(q_empty);
                                    }
                                }
                            }
                            if (ok && j > first) {
                                const int t = (j - first + 1) & 1;  // the tile that has j - 1
                                ok = wait_bar(kv_full + sv, pv, err, DEVERR_PTILE_KV);
                                if (j * TKEYS > len) fixed(sv);
                                if (ok) values(t, va, j - 1 < first + 2);
                                if (ok && j + 1 >= end) umma_commit(o_full + t);
                                if (ok) umma_commit(kv_empty + sv);
                            }
                            if (ok && j < end) next(sv, pv);
                        }
                    }
                    done(k);
                }
                // all products are done before tensor memory is freed
                umma_commit(drain);
                wait_bar(drain, 0, err, DEVERR_PTILE_DRAIN);
            }
            __syncwarp();
        } else if (warp == 2) {
            // ------------------------------------------------ values behind a sequence's end
            // This warp uses every ring entry (and frees it with the issuer), so that it neither falls behind the
            // ring nor meets a barrier whose parity is a phase before last's; the issuer waits for the fix of a
            // stage before it frees it, so a stage's fixes do not overtake it either.
            int stage = 0, phase = 0;
            for (int k = 0; __all_sync(0xffffffffu, take(k)); k++) {
                const int first = works[k & 3].a, end = works[k & 3].b, len = works[k & 3].len;
                for (int i = 2 * first; ok && i < 2 * end; i++) {  // K_a, V_a, K_a+1, ...
                    ok = __all_sync(0xffffffffu, wait_bar(kv_full + stage, phase, err, DEVERR_PTILE_FIX));
                    if (!ok) break;
                    if ((i & 1) && (i + 1) / 2 * TKEYS > len) {
                        const int from = max(0, len - i / 2 * TKEYS);
                        uint8_t* v = sm + C::OFF_RING + stage * C::STAGE;
                        for (int e = from * 8 + lane; e < TKEYS * 8; e += 32)
#pragma unroll
                            for (int h = 0; h < C::HALVES; h++)
                                *reinterpret_cast<uint4*>(v + h * C::HALF + e * 16) = make_uint4(0u, 0u, 0u, 0u);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(v_fixed + stage);
                    }
                    if (lane == 0) mbar_arrive(kv_empty + stage);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                __syncwarp();
                if (lane == 0) done(k);
            }
        }
    } else {
        // ------------------------------------------------ softmax
        const int t = (warp - 4) >> 3, half = (warp >> 2) & 1 ? 0 : 1, wl = warp & 3;  // warps 4-7, 12-15: keys 0-63
        const int row = wl * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(wl * 32) << 16);
        // this thread's 64 scores; its weights go over the first 32 columns of them
        const uint32_t s_addr = lanes + C::COL_S + t * TKEYS + half * 64;
        const uint32_t o_addr = lanes + C::COL_O + t * DP;
        float* x_mine = reinterpret_cast<float*>(sm + C::OFF_X) + (t * 2 + half) * 128 + row;
        const float* x_other = reinterpret_cast<float*>(sm + C::OFF_X) + (t * 2 + (half ^ 1)) * 128 + row;
        const float* x_b = reinterpret_cast<float*>(sm + C::OFF_X) + 2 * 128 + row;  // tile B's, at a unit's end
        const uint32_t pair_bar = 1 + t * 4 + wl;  // of the two warps that share 32 rows
        const float scale2 = plan.scale2;
        constexpr float up = UP<T, 8>, down = 1.0f / (1 << UP<T, 8>);
        const int ri = row / group, gi = row - ri * group;  // this row's token of the tile, its head of the group
        int ns = 0, no = 0, nd = 0;
        // (both warps of a pair go on, or neither: they meet at barriers)
        for (int k = 0; named_bar_and(pair_bar, 64, take(k)); k++) {
            const Work& w = works[k & 3];
            const int lo = w.lo[t], hi = w.hi[t];
            const bool valid = ri < w.cnt[t];
            // of the tile's rows: keys up to pmin are seen by all, keys up to pmax - window by none
            const int pmin = w.len - w.n + w.i0[t], pmax = pmin + w.cnt[t] - 1;
            const int pos = valid ? pmin + ri : -1;
            float m = -INFINITY, l = 0.0f;  // m of the raw products
            for (int j = lo; j < hi; j += w.dup ? 2 : 1) {
                if (ok) ok = wait_bar(s_full + t, ns & 1, err, DEVERR_PTILE_S);
                __syncwarp();
                ns++;
                tc_fence_after();
                // 64 scores do not fit a thread's registers next to what is made of them: the second 32 are read twice.
                const int k0 = j * TKEYS + half * 64;
                const bool edge = k0 + 63 > pmin || (a.window > 0 && k0 <= pmax - a.window);
                auto hide = [&](int c, uint32_t (&s)[32]) {
                    const int top = pos - k0 - c * 32, bot = a.window > 0 ? top - a.window : -1;  // columns in (bot, top]
                    uint32_t seen = top >= 31 ? 0xFFFFFFFFu : top < 0 ? 0u : (2u << top) - 1;
                    if (bot >= 0) seen &= bot >= 31 ? 0u : ~((2u << bot) - 1);
                    if (__all_sync(0xffffffffu, seen == 0xFFFFFFFFu)) return;
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (!(seen >> e & 1)) s[e] = 0xFF800000u;  // -inf
                };
                auto most = [](const uint32_t (&s)[32]) {  // (NaN goes through: the row is then NaN)
                    float mx[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        mx[q] = max3(__uint_as_float(s[q * 8]), __uint_as_float(s[q * 8 + 1]), __uint_as_float(s[q * 8 + 2]));
                        mx[q] = max3(mx[q], __uint_as_float(s[q * 8 + 3]), __uint_as_float(s[q * 8 + 4]));
                        mx[q] = max3(mx[q], __uint_as_float(s[q * 8 + 5]), __uint_as_float(s[q * 8 + 6]));
                    }
                    mx[0] = max3(mx[0], mx[1], __uint_as_float(s[7]));
                    mx[2] = max3(mx[2], mx[3], __uint_as_float(s[15]));
                    return max3(max3(mx[0], mx[2], __uint_as_float(s[23])), __uint_as_float(s[31]), __uint_as_float(s[31]));
                };
                uint32_t s0[32], s1[32];
                tmem_ld32(s_addr, s0);
                tmem_ld32(s_addr + 32, s1);
                tmem_ld_wait();
                if (edge) {
                    hide(0, s0);
                    hide(1, s1);
                }
                const float mine = most(s0);
                float tile = max3(mine, most(s1), mine);
                *x_mine = tile;
                named_bar_sync(pair_bar, 64);
                tile = max3(tile, *x_other, tile);
                if (tile != tile) l = tile;
                // l == 0 and O == 0 as long as m is -inf: nothing to scale then
                const bool grow = m != -INFINITY && (tile - m) * scale2 > 8.0f;
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? ex2((m - tile) * scale2) : 1.0f;
                    if (j > lo && half == 0) {
#pragma unroll 1
                        for (int c = 0; c < DP / 16; c++) {
                            uint32_t o[16];
                            tmem_ld16(o_addr + c * 16, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(o_addr + c * 16, o);
                        }
                    }
                    l *= f;
                    if (grow) m = tile;
                }
                if (m == -INFINITY) m = tile;
                // One FMA makes the exponent scale2 s - scale2 m + up.  Where the bits of scale2 m end above 2^-4 its
                // rounding is off by whole powers of two: there m is subtracted from the scores first, where they are.
                float base = m == -INFINITY ? up : up - m * scale2;
                if (__any_sync(0xffffffffu, fabsf(base) > 1048576.0f)) {
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t s[16];
                        tmem_ld16(s_addr + c * 16, s);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; e++) s[e] = __float_as_uint(__uint_as_float(s[e]) - (m == -INFINITY ? 0.0f : m));
                        tmem_st16(s_addr + c * 16, s);
                    }
                    tmem_st_wait();
                    tmem_ld32(s_addr, s0);
                    tmem_ld_wait();
                    if (edge) hide(0, s0);
                    base = up;
                }
                const uint64_t scale22 = f2_pack(scale2, scale2), base2 = f2_pack(base, base);
                uint64_t sum2[2] = {0ull, 0ull};
                // the weights meet V in its own type (see UP): 2^-11 (f16) or 2^-8 (bf16) of each, as the
                // rounding of the result; l sums them unrounded
                auto weigh = [&](int c, const uint32_t (&s)[32]) {  // (their columns lie within the scores read so far)
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        float y, z;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), scale22, base2), y, z);
                        y = ex2(y);
                        z = ex2(z);
                        sum2[e & 1] = f2_add(sum2[e & 1], f2_pack(y, z));
                        p[e] = pack2<T>(y, z);
                    }
                    tmem_st16(s_addr + c * 16, p);
                };
                tmem_ld32(s_addr + 32, s1);
                weigh(0, s0);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_half + t);
                tmem_ld_wait();
                if (edge) hide(1, s1);
                weigh(1, s1);
                float sa, sb, sc, sd;
                f2_unpack(sum2[0], sa, sb);
                f2_unpack(sum2[1], sc, sd);
                l += (sa + sb) + (sc + sd);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + t);
            }
            // ---- the tile's end
            const bool whole = w.whole, dup = w.dup;
            uint8_t* part = plan.parts + (static_cast<int64_t>(blockIdx.x) * 2 + w.begins) * C::SLOT;
            const int64_t at = static_cast<int64_t>(w.row0 + w.i0[t] + ri) * a.q_heads + w.hk * group + gi;
            named_bar_sync(pair_bar, 64);  // (the last maxima have been read)
            *x_mine = l;
            named_bar_sync(pair_bar, 64);
            l += *x_other;
            if (lo < hi) {
                if (ok) ok = __all_sync(0xffffffffu, wait_bar(o_full + t, no & 1, err, DEVERR_PTILE_O));
                no++;
                tc_fence_after();
            }
            float mt = l == 0.0f ? -INFINITY : m * scale2, fa = 1.0f, fb = 0.0f;
            if (dup) {  // tile A takes up what tile B has of the same rows
                if (t == 1) {
                    named_bar_sync(pair_bar, 64);  // (the sums have been read)
                    *x_mine = half ? l : mt;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(b_ready);
                } else {
                    if (ok) ok = __all_sync(0xffffffffu, wait_bar(b_ready, nd & 1, err, DEVERR_PTILE_O));
                    tc_fence_after();
                    const float2 b = make_float2(x_b[0], x_b[128]);
                    const float top = fmaxf(mt, b.x), base = top == -INFINITY ? 0.0f : top;
                    fa = ex2(mt - base);
                    fb = ex2(b.x - base);
                    l = l * fa + b.y * fb;
                    mt = top;
                }
            }
            const bool both = dup && w.lo[1] < w.hi[1];
            if (lo < hi && !(dup && t == 1)) {
                const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : down;
                const float ga = fa * inv, gb = fb * inv;
                const int odd = lane & 1;
                const int64_t own = valid ? at : -1, other = __shfl_xor_sync(0xffffffffu, own, 1);
                const int64_t at_even = odd ? other : own, at_odd = odd ? own : other;
#pragma unroll 1
                for (int c = half * (DP / 32); c < (half + 1) * (DP / 32); c++) {
                    uint32_t o[16], ob[16];
                    __syncwarp();
                    tmem_ld16(o_addr + c * 16, o);
                    if (both) tmem_ld16(o_addr + DP + c * 16, ob);
                    tmem_ld_wait();
                    float y[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        y[e] = __uint_as_float(o[e]) * ga;
                        if (both) y[e] = fmaf(__uint_as_float(ob[e]), gb, y[e]);
                    }
                    if (whole) {
                        // two lanes write the 32 bytes of a row, then those of the other's (16 bytes a row and store
                        // cost the same as 32)
                        uint32_t u[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) u[e] = pack2<T>(y[2 * e], y[2 * e + 1]);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? u[e] : u[4 + e], 1);
                            if (odd) u[e] = got;  // row of the even lane, then the own one
                            else u[4 + e] = got;  // the own row, then the odd lane's
                        }
                        if (c * 16 + odd * 8 >= a.c.dim) continue;
                        T* out = static_cast<T*>(a.out) + c * 16 + odd * 8;
                        if (at_even >= 0) *reinterpret_cast<uint4*>(out + at_even * a.c.dim) = make_uint4(u[0], u[1], u[2], u[3]);
                        if (at_odd >= 0) *reinterpret_cast<uint4*>(out + at_odd * a.c.dim) = make_uint4(u[4], u[5], u[6], u[7]);
                    } else if (valid) {
                        float4* out = reinterpret_cast<float4*>(part) + c * 4 * (2 * TM) + t * TM + row;
#pragma unroll
                        for (int e = 0; e < 4; e++) out[e * 2 * TM] = make_float4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
                    }
                }
                tc_fence_before();
            }
            if (half == 0 && !(dup && t == 1)) {
                if (valid && whole && a.lse) a.lse[at] = l == 0.0f ? -INFINITY : (mt + log2f(l * down)) * 0.6931471805599453f;
                if (valid && !whole)  // (a row tile without keys in the piece: m -inf)
                    *reinterpret_cast<float2*>(part + 2 * TM * DP * 4 + (t * TM + row) * 8) = make_float2(mt, l * down);
            }
            if (dup && t == 0) {
                __syncwarp();
                if (lane == 0) mbar_arrive(b_free);
            } else if (dup) {  // its output and statistics may be written again
                if (ok) ok = __all_sync(0xffffffffu, wait_bar(b_free, nd & 1, err, DEVERR_PTILE_O));
                tc_fence_after();
            }
            nd += dup;
            __syncwarp();
            if (lane == 0) done(k);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 2) tmem_dealloc(tmem, C::COLS);
}

// The rows of units that lie in several pieces: as attn_join_kernel.  DP / 4
// lanes have a row, 16 bytes each, and two rows go at once, so that hardly more
// CTAs come than are under way together (a warp a row: 7.5 us for 148 units
// cut in two, D = 64, of which this leaves ~3).
template <typename T, int DP>
__global__ void __launch_bounds__(256) attn_tile_join_kernel(const PagedAttnArgs a, const TilePlan plan) {
    using C = TileCfg<DP>;
    constexpr int LANES = DP / 4, SIDE = 256 / LANES, R = 2;
    griddep_wait();
    const int4 b0 = *reinterpret_cast<const int4*>(plan.begun + blockIdx.x);
    const int2 b1 = *reinterpret_cast<const int2*>(&plan.begun[blockIdx.x].unit);
    const int group = a.q_heads / a.c.kv_heads, hk = b0.w, unit = b1.x, last = b1.y;
    // a warp: eight rows, four float4 of each
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int x = warp % (LANES / 4) * 4 + (lane >> 3), row0 = blockIdx.y * SIDE * R + warp / (LANES / 4) * 8 + (lane & 7);
    if (b0.x == 0) return;
    int64_t at[R];  // the rows' places in out (below 0: none)
    float m[R], sum[R], o[R][4];
    bool any = false;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int row = row0 + i * SIDE, r = row & (TM - 1), ri = r / group;
        const int tok = (2 * unit + (row >> 7)) * plan.tokens + ri;
        at[i] = ri < plan.tokens && tok < b0.z ? static_cast<int64_t>(b0.y + tok) * a.q_heads + hk * group + (r - ri * group) : -1;
        any |= at[i] >= 0;
        m[i] = -INFINITY;
        sum[i] = 0.0f;
        for (int e = 0; e < 4; e++) o[i][e] = 0.0f;
    }
    if (!any) return;
#pragma unroll 2
    for (int c = blockIdx.x; c <= last; c++) {
        const uint8_t* part = plan.parts + (static_cast<int64_t>(c) * 2 + (c == static_cast<int>(blockIdx.x) ? 1 : 0)) * C::SLOT;
        float2 ml[R];
        float4 y[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            ml[i] = make_float2(-INFINITY, 0.0f);
            if (at[i] < 0) continue;
            const int row = row0 + i * SIDE;
            ml[i] = *reinterpret_cast<const float2*>(part + 2 * TM * DP * 4 + row * 8);
            y[i] = reinterpret_cast<const float4*>(part)[x * 2 * TM + row];
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            if (ml[i].x == -INFINITY) continue;  // (y is not written then)
            const float m2 = fmaxf(m[i], ml[i].x);
            const float f = ex2(m[i] - m2), w = ex2(ml[i].x - m2);
            m[i] = m2;
            sum[i] = sum[i] * f + ml[i].y * w;
            o[i][0] = o[i][0] * f + y[i].x * w;
            o[i][1] = o[i][1] * f + y[i].y * w;
            o[i][2] = o[i][2] * f + y[i].z * w;
            o[i][3] = o[i][3] * f + y[i].w * w;
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
        if (at[i] < 0) continue;
        const float inv = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];
        if (x * 4 < a.c.dim)
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at[i] * a.c.dim + x * 4) =
                make_uint2(pack2<T>(o[i][0] * inv, o[i][1] * inv), pack2<T>(o[i][2] * inv, o[i][3] * inv));
        if (x == 0 && a.lse) a.lse[at[i]] = sum[i] == 0.0f ? -INFINITY : (m[i] + log2f(sum[i])) * 0.6931471805599453f;
    }
}

}  // namespace

namespace {

int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

bool few_rows(const PagedAttnArgs& a) {
    return static_cast<int64_t>(a.max_q) * (a.q_heads / a.c.kv_heads) <= MAX_ROWS;
}

// Workspace of the rows kernel: spans of all pairs, then two parts per piece.
struct RowsSpace {
    int64_t spans = 0, slot = 0, bytes = 0;
    int rows_cap = 0;
};
RowsSpace rows_space(const PagedAttnArgs& a, int sms) {
    RowsSpace w;
    const int group = a.q_heads / a.c.kv_heads;
    if (!few_rows(a) || a.max_q == 0) return w;
    const int dp = a.c.dim > 64 ? 128 : 64;
    w.rows_cap = std::min(MAX_ROWS / group, a.max_q) * group;
    w.slot = up256(w.rows_cap * (dp * 4ll + 8));
    w.spans = up256(8ll * a.c.n_seq * a.c.kv_heads);
    w.bytes = w.spans + 2ll * sms * NW * w.slot;
    return w;
}

// Workspace of the tile kernel: the pieces' units, two parts per piece.
struct TileSpace {
    int64_t begun = 0, bytes = 0;
};
TileSpace tile_space(const PagedAttnArgs& a, int sms) {
    TileSpace w;
    if (few_rows(a)) return w;
    w.begun = up256(sizeof(Begun) * sms);
    w.bytes = w.begun + 2ll * sms * (a.c.dim > 64 ? TileCfg<128>::SLOT : TileCfg<64>::SLOT);
    return w;
}

}  // namespace

int paged_attention_workspace(const PagedAttnArgs& a, int64_t* bytes) {
    int rc = 0;
    DeviceState* ds = device_state(&rc);
    if (!ds) return rc;
    *bytes = rows_space(a, ds->sm_count).bytes + tile_space(a, ds->sm_count).bytes;
    return TVQ_OK;
}

namespace {

// The cache as a {value, token, half, head, page} tensor map, boxes of 64
// values x `box` tokens x `halves` (128-byte swizzle).  A head dim that is no
// multiple of 64 stays one dimension, so that nothing behind it is read.  A
// cache without pages has one in its map, at any address: the kernels check
// page numbers against n_pages and ask for page -1, zeros, instead.
int cache_map(CUtensorMap* map, const PagedAttnArgs& a, const void* ptr, int64_t tok, int64_t head, int64_t page, int box,
              int halves) {
    const PagedView& c = a.c;
    if (c.n_pages == 0) ptr = a.out;
    const bool whole = c.dim % 64 == 0;
    const uint64_t dims[5] = {static_cast<uint64_t>(whole ? 64 : c.dim), static_cast<uint64_t>(c.page),
                              static_cast<uint64_t>(whole ? c.dim / 64 : 1), static_cast<uint64_t>(c.kv_heads),
                              static_cast<uint64_t>(std::max<int64_t>(c.n_pages, 1))};
    const uint64_t strides[4] = {static_cast<uint64_t>(tok) * 2, 128, static_cast<uint64_t>(head) * 2,
                                 static_cast<uint64_t>(page) * 2};
    const uint32_t boxes[5] = {64, static_cast<uint32_t>(box), static_cast<uint32_t>(halves), 1, 1};
    return make_tma_16bit(map, ptr, 5, dims, strides, boxes);
}

template <typename T, int DP>
int launch_rows(const PagedAttnArgs& a, DeviceState* ds, cudaStream_t st) {
    using C = RowsCfg<DP>;
    int rc = allow_smem<attn_rows_kernel<T, DP>>(C::SMEM);
    if (rc) return rc;
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
    rc = cache_map(&tmK, a, a.c.k, a.c.k_tok, a.c.k_head, a.c.k_page, plan.box, plan.box_halves);
    if (rc) return rc;
    rc = cache_map(&tmV, a, a.c.v, a.c.v_tok, a.c.v_head, a.c.v_page, plan.box, plan.box_halves);
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

template <typename T, int DP>
int launch_tiles(const PagedAttnArgs& a, DeviceState* ds, cudaStream_t st) {
    using C = TileCfg<DP>;
    int rc = allow_smem<attn_tile_kernel<T, DP>>(C::SMEM);
    if (rc) return rc;
    const int group = a.q_heads / a.c.kv_heads;
    uint8_t* ws = static_cast<uint8_t*>(a.ws);
    TilePlan plan;
    plan.begun = reinterpret_cast<Begun*>(ws);
    plan.parts = ws + tile_space(a, ds->sm_count).begun;
    plan.tokens = TM / group;
    plan.box = std::min(a.c.page, TKEYS);
    plan.by_value = a.c.dim % 64 != 0;
    plan.box_halves = a.c.dim == 128 && plan.box == TKEYS ? 2 : 1;
    plan.negative = a.scale < 0.0f;
    plan.scale2 = std::max(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);  // (0 x -inf would be NaN)
    CUtensorMap tmQ, tmK, tmV;
    const bool whole = a.c.dim % 64 == 0;
    const uint64_t dims[4] = {static_cast<uint64_t>(whole ? 64 : a.c.dim), static_cast<uint64_t>(whole ? a.c.dim / 64 : 1),
                              static_cast<uint64_t>(a.q_heads), static_cast<uint64_t>(a.c.n_rows)};
    const uint64_t strides[3] = {128, static_cast<uint64_t>(a.q_head) * 2, static_cast<uint64_t>(a.q_tok) * 2};
    const uint32_t box[4] = {64, 1, static_cast<uint32_t>(group), static_cast<uint32_t>(plan.tokens)};
    rc = make_tma_16bit(&tmQ, a.q, 4, dims, strides, box);
    if (rc) return rc;
    rc = cache_map(&tmK, a, a.c.k, a.c.k_tok, a.c.k_head, a.c.k_page, plan.box, plan.box_halves);
    if (rc) return rc;
    rc = cache_map(&tmV, a, a.c.v, a.c.v_tok, a.c.v_head, a.c.v_page, plan.box, plan.box_halves);
    if (rc) return rc;
    rc = launch_pdl(attn_tile_kernel<T, DP>, dim3(ds->sm_count), dim3(TTHR), C::SMEM, st, tmQ, tmK, tmV, a, plan,
                    ds->d_error);
    if (rc) return rc;
    return launch_pdl(attn_tile_join_kernel<T, DP>, dim3(ds->sm_count, DP / 8), dim3(256), 0, st, a, plan);
}

// Steps (no sequence has more than 16 rows): the rows kernel, which waits for
// nothing but the cache.  Else the tile kernel for all sequences, those of few
// rows among them too.  Both kernels with few rows, L2 cold: 48 sequences of 700
// keys, 25 heads of 64, one token each: rows 64 us, tiles 100, sixteen tokens 72
// and 102; 24 of 14000 keys, 32 heads on 8 of 128, four tokens: 248 and 252; 16 of
// 6000, 32 on 4, two tokens: 65 and 63.  So the rows kernel is ahead or level up to
// the 16 rows that its matrix instruction has.
template <typename T>
int launch_attention(const PagedAttnArgs& a, DeviceState* ds, cudaStream_t st) {
    if (few_rows(a)) return a.c.dim > 64 ? launch_rows<T, 128>(a, ds, st) : launch_rows<T, 64>(a, ds, st);
    return a.c.dim > 64 ? launch_tiles<T, 128>(a, ds, st) : launch_tiles<T, 64>(a, ds, st);
}

}  // namespace

int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
    int rc = 0;
    DeviceState* ds = device_state(&rc);
    if (!ds) return rc;
    TVQ_CHECK(a.q_heads / a.c.kv_heads <= TM, TVQ_ERR_UNSUPPORTED, "more than 128 query heads to a kv head");
    TVQ_CHECK(ds->cc_major == 10, TVQ_ERR_UNSUPPORTED, "the paged attention needs an sm_100 device");
    if (a.c.n_rows == 0 || a.max_q == 0) return TVQ_OK;
    return a.c.type == TVQ_TYPE_F16 ? launch_attention<__half>(a, ds, st) : launch_attention<__nv_bfloat16>(a, ds, st);
}

}  // namespace tvq
