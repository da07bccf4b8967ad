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
//  - one CTA per SM; all 32-key tiles of all (sequence, kv head) pairs stand
//    in one line, and CTA c takes the c-th equal piece of it, whatever the
//    lengths.  Every CTA finds its piece from the lengths on the device.
//  - two producer warps (keys, values) bring the piece's tiles through a 192 KB
//    ring by TMA (a tile's pages are boxes of a {value, token, half, head,
//    page} tensor map, so any strides will do), across the ends of pairs; six
//    consumer warps take the tiles in turn, each with its own m, l, o, and join them at the end
//    of a pair, while the next pair's tiles are on their way.
//  - mma.sync m16n8k16 with the rows padded to 16: at D = 128 the products
//    of a 16 KB tile take 128 of the ~650 cycles that its bytes take, so the
//    wider tcgen05 tile (128 rows) would buy nothing here.
//  - a pair that several CTAs share is joined by the one that finishes last
//    (a counter per CTA in the workspace, zero between calls), in the order
//    of the parts, so results do not depend on who that is.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "tvq_common.cuh"
#include "tvq_decode.h"
#include "tvq_kernels.h"

namespace tvq {

namespace {

constexpr int NW = 6;              // consumer warps of the rows kernel
constexpr int NC = NW * 32;        // consumer threads
constexpr int NTHR = NC + 64;      // and two producer warps
constexpr int MAX_ROWS = 16;       // rows of a pair (new tokens x heads of the group)

// device error codes: the wait that gave up first
enum : int { DEVERR_PATTN_EMPTY = 71, DEVERR_PATTN_FULL = 72, DEVERR_PATTN_DRAIN = 73 };

__device__ __forceinline__ float ex2(float x) {  // 2^x, relative error ~2^-22, 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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
    static constexpr int KT = 32;                        // keys per tile
    static constexpr int HALF = KT * 128;                // 64 values of a tile's keys, 128-byte swizzle
    static constexpr int HALVES = DP / 64;
    static constexpr int STAGE = 2 * HALVES * HALF;      // one tile: keys, then values
    static constexpr int STAGES = 196608 / STAGE;        // 24 or 12
    // A stage is always the same warp's, which waits for its phases one after
    // another.  Were it to pass from warp to warp, one that is ahead could take
    // the parity of the phase before last for that of the one it waits for.
    static_assert(STAGES % NW == 0);
    static constexpr int OFF_PART = STAGES * STAGE;      // [NW / 2][16][DP] f32
    static constexpr int OFF_ML = OFF_PART + NW / 2 * 16 * DP * 4;     // float2 [2][NW][16]
    static constexpr int OFF_BAR = OFF_ML + 2 * NW * 16 * 8;      // full[STAGES], empty[STAGES]
    static constexpr int OFF_MISC = OFF_BAR + 2 * STAGES * 8;     // scan[NW + 2], last, at[2]
    static constexpr int SMEM = OFF_MISC + 64;
    static constexpr int64_t SLOT = 16 * (DP * 4 + 8);   // workspace bytes of one partial
};

struct RowsPlan {
    int* counters;   // [grid]
    uint8_t* parts;  // [grid][2] slots
    int min_tiles;   // no CTA gets a smaller piece
    // One TMA load: `box` tokens (a power of two: a page, or a tile of a larger
    // one) of 64 values, or of both halves (box_halves 2: 128 values and box =
    // KT).  by_value: the head dim is no multiple of 64, the halves start at
    // values 0 and 64 of one dimension that ends with the head dim.
    int box, box_halves, by_value;
};

// Where a walk over a CTA's piece stands: a pair and its tiles in the piece.
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
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR);
    uint64_t* empty = full + C::STAGES;
    int* s_scan = reinterpret_cast<int*>(sm + C::OFF_MISC);
    int* s_last = s_scan + NW + 2;
    int64_t* s_at = reinterpret_cast<int64_t*>(s_scan + NW + 4);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.q_heads / a.c.kv_heads;
    const int fit = MAX_ROWS / group;  // new rows of a sequence that this kernel takes
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; i++) {
            mbar_init(full + i, 2);
            mbar_init(empty + i, 1);
        }
        fence_barrier_init();
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    griddep_wait();

    // ---- this CTA's piece of the line of tiles
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
    const int64_t per = max(static_cast<int64_t>(plan.min_tiles), (total + gridDim.x - 1) / gridDim.x);
    const int64_t begin = per * blockIdx.x, stop = min(total, begin + per);
    if (begin >= stop) return;
    int64_t before = 0;
    for (int s0 = 0; s0 < a.c.n_seq; s0 += NTHR) {
        int all = 0;
        int w = w0, inc = inc0;
        if (a.c.n_seq > NTHR) {
            w = weight(s0 + tid);
            inc = scan(w, &all);
        }
        const int64_t hi = (before + inc) * a.c.kv_heads, lo = hi - static_cast<int64_t>(w) * a.c.kv_heads;
        if (begin >= lo && begin < hi) {
            s_at[0] = s0 + tid;
            s_at[1] = lo;
        }
        before += all;
    }
    __syncthreads();

    Cursor cur;
    auto enter = [&](int skip) {  // cur.s, hk, left and q set: the pair's tiles from `skip` on
        cur.all = seq_tiles<KT>(cur.q, a.window);
        cur.first = cur.all.x + skip;
        cur.end = static_cast<int>(min(static_cast<int64_t>(cur.all.y), cur.first + cur.left));
    };
    auto next_pair = [&]() {  // false: the piece is done
        cur.left -= cur.end - cur.first;
        if (cur.left <= 0) return false;
        if (++cur.hk == a.c.kv_heads) {
            cur.hk = 0;
            do {
                cur.q = load_seq(a.c, ++cur.s);
            } while (cur.q.n == 0 || cur.q.n > fit);
        }
        enter(0);
        return true;
    };
    cur.s = static_cast<int>(s_at[0]);
    cur.q = load_seq(a.c, cur.s);
    cur.left = stop - begin;
    {
        const int64_t in_seq = begin - s_at[1];
        const int2 t = seq_tiles<KT>(cur.q, a.window);
        cur.hk = static_cast<int>(in_seq / (t.y - t.x));
        enter(static_cast<int>(in_seq - static_cast<int64_t>(cur.hk) * (t.y - t.x)));
    }

    if (warp >= NW) {
        // ------------------------------------------------ producers: keys, values
        // lane i looks up the page of the i-th load of a window of 32 loads
        const bool is_v = warp > NW;
        const CUtensorMap* map = is_v ? &tmV : &tmK;
        const uint32_t base = smem_u32(sm) + (is_v ? C::HALVES * C::HALF : 0);
        const int per_tile = KT / plan.box, loads_h = C::HALVES / plan.box_halves;
        int n = 0, stage = 0, phase = 1;  // tiles issued; the ring's place and the empty barriers' parity
        bool ok = true;
        do {
            const int loads = (cur.end - cur.first) * per_tile;
            for (int l0 = 0; ok && l0 < loads; l0 += 32) {
                const int j = cur.first * KT + (l0 + lane) * plan.box;
                int page = -1;
                if (l0 + lane < loads && j < cur.q.len) {
                    const int col = j >> a.c.page_log2;
                    if (col < a.c.n_cols) page = __ldg(a.c.table + cur.s * a.c.table_stride + col);
                    // (a page past the cache's end is outside the tensor map: zeros)
                    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.c.n_pages)) {
                        record_error(err, DEVERR_BAD_PAGE);
                        page = -1;
                    }
                }
                const int here = min(32, loads - l0);
                for (int i = 0; i < here; i += per_tile) {
                    ok = __all_sync(0xffffffffu, mbar_wait(empty + stage, phase, err, DEVERR_PATTN_EMPTY));
                    if (!ok) break;
                    uint64_t* bar = full + stage;
                    if (lane == 0) mbar_arrive_expect_tx(bar, C::STAGE / 2);
                    for (int b = 0; b < per_tile; b++) {
                        const int pg = __shfl_sync(0xffffffffu, page, i + b);
                        const int slot = (cur.first * KT + (l0 + i + b) * plan.box) & (a.c.page - 1);
                        if (lane == 0) {
                            const uint32_t dst = base + stage * C::STAGE + b * plan.box * 128;
                            for (int h = 0; h < loads_h; h++)
                                tma_load_5d(map, bar, dst + h * C::HALF, plan.by_value ? h * 64 : 0, slot,
                                            plan.by_value ? 0 : h, cur.hk, pg);
                        }
                    }
                    n++;
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        } while (ok && next_pair());
        // every load lands before the CTA may end
        if (lane == 0)
            for (int i = max(0, n - C::STAGES); i < n; i++)
                mbar_wait(full + i % C::STAGES, (i / C::STAGES) & 1, nullptr, DEVERR_PATTN_DRAIN);
        return;
    }

    // ---------------------------------------------------- consumers
    const float scale2 = a.scale * 1.4426950408889634f;
    const int g = lane >> 2, quad = lane & 3;
    int parity = 0, n0 = 0;  // n0: the pair's first tile in the order of the ring
    int turn = warp, stage = warp % C::STAGES, phase = 0;  // this warp's next tile there
    bool ok = true;
    for (bool go = true; go; n0 += cur.end - cur.first, go = next_pair(), parity ^= 1) {
        // ---- the pair's rows as A fragments
        const int rows = cur.q.n * group;
        uint32_t qf[DP / 16][4];
        int pos[2];  // of this thread's two rows (below 0: sees nothing)
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const int r = g + hf * 8;
            const int i = r / group, gi = r - i * group;
            const bool in = r < rows;
            pos[hf] = in ? cur.q.len - cur.q.n + i : -1;
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

        for (const int n1 = n0 + cur.end - cur.first; turn < n1; turn += NW) {
            const int t = cur.first + turn - n0;
            if (ok) ok = mbar_wait(full + stage, phase, err, DEVERR_PATTN_FULL);
            const uint32_t ks = smem_u32(sm) + stage * C::STAGE, vs = ks + C::HALVES * C::HALF;
            if ((t + 1) * KT > cur.q.len) {
                // the values behind the sequence's end may be anything, and 0 x NaN is NaN: zeros
                const int from = max(0, cur.q.len - t * KT);
                for (int i = from * 8 + lane; i < KT * 8; i += 32)
#pragma unroll
                    for (int h = 0; h < C::HALVES; h++)
                        *reinterpret_cast<uint4*>(sm + stage * C::STAGE + (C::HALVES + h) * C::HALF + i * 16) =
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
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + stage);
            stage += NW;
            if (stage >= C::STAGES) {
                stage -= C::STAGES;
                phase ^= 1;
            }
        }

        // ---- join the warps' parts
        float2* ml = reinterpret_cast<float2*>(sm + C::OFF_ML) + parity * NW * 16;
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            float x = l[hf];
            x += __shfl_xor_sync(0xffffffffu, x, 1);
            x += __shfl_xor_sync(0xffffffffu, x, 2);
            if (quad == 0) ml[warp * 16 + g + hf * 8] = make_float2(m[hf], x);
        }
        named_bar_sync(1, NC);
        const bool whole = cur.first == cur.all.x && cur.end == cur.all.y;
        const int slot = cur.first == cur.all.x ? 1 : 0;  // a pair that goes on after this piece, or came into it
        uint8_t* part = plan.parts + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * C::SLOT;
        float* buf = reinterpret_cast<float*>(sm + C::OFF_PART);
        auto top_of = [&](int r) {
            float t = ml[r].x;
#pragma unroll
            for (int w = 1; w < NW; w++) t = fmaxf(t, ml[w * 16 + r].x);
            return t;
        };
        {
            float f[2];
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const float t = top_of(g + hf * 8);
                f[hf] = t == -INFINITY ? 0.0f : ex2(m[hf] - t);
            }
            float* mine = buf + warp % (NW / 2) * (16 * DP);
            if (warp >= NW / 2) {
#pragma unroll
                for (int n = 0; n < DP / 8; n++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
                        *reinterpret_cast<float2*>(mine + (g + hf * 8) * DP + n * 8 + quad * 2) =
                            make_float2(o[n][hf * 2] * f[hf], o[n][hf * 2 + 1] * f[hf]);
            }
            named_bar_sync(1, NC);
            if (warp < NW / 2) {
#pragma unroll
                for (int n = 0; n < DP / 8; n++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        float2* w = reinterpret_cast<float2*>(mine + (g + hf * 8) * DP + n * 8 + quad * 2);
                        const float2 y = *w;
                        *w = make_float2(fmaf(o[n][hf * 2], f[hf], y.x), fmaf(o[n][hf * 2 + 1], f[hf], y.y));
                    }
            }
            named_bar_sync(1, NC);
        }
        for (int e = tid; e < rows * (DP / 4); e += NC) {
            const int r = e / (DP / 4), d = (e - r * (DP / 4)) * 4;
            if (d >= a.c.dim) continue;
            float4 y = *reinterpret_cast<const float4*>(buf + r * DP + d);
#pragma unroll
            for (int w = 1; w < NW / 2; w++) {
                const float4 z = *reinterpret_cast<const float4*>(buf + w * 16 * DP + r * DP + d);
                y.x += z.x;
                y.y += z.y;
                y.z += z.z;
                y.w += z.w;
            }
            const float t = top_of(r);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float2 z = ml[w * 16 + r];
                sum += t == -INFINITY ? 0.0f : z.y * ex2(z.x - t);
            }
            if (whole) {
                const int i = r / group, gi = r - i * group;
                const int64_t at = static_cast<int64_t>(cur.q.row0 + i) * a.q_heads + cur.hk * group + gi;
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.c.dim + d) =
                    make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
                if (d == 0 && a.lse) a.lse[at] = sum == 0.0f ? -INFINITY : (t + log2f(sum)) * 0.6931471805599453f;
            } else {
                *reinterpret_cast<float4*>(part + (r * DP + d) * 4) = y;
                if (d == 0) *reinterpret_cast<float2*>(part + 16 * DP * 4 + r * 8) = make_float2(t, sum);
            }
        }
        if (whole) continue;

        // ---- join the CTAs' parts: CTA c0 began the pair, c1 ends it
        const int64_t at0 = stop - cur.left - (cur.first - cur.all.x);  // the pair's first tile in the line
        const int c0 = static_cast<int>(at0 / per), c1 = static_cast<int>((at0 + cur.all.y - cur.all.x - 1) / per);
        __threadfence();
        named_bar_sync(1, NC);
        if (tid == 0) *s_last = atomicAdd(plan.counters + c0, 1) == c1 - c0;
        named_bar_sync(1, NC);
        if (!*s_last) continue;
        __threadfence();
        for (int e = tid; e < rows * (DP / 4); e += NC) {
            const int r = e / (DP / 4), d = (e - r * (DP / 4)) * 4;
            if (d >= a.c.dim) continue;
            auto slot_of = [&](int c) { return plan.parts + (static_cast<int64_t>(c) * 2 + (c == c0 ? 1 : 0)) * C::SLOT; };
            float t = -INFINITY;
            for (int c = c0; c <= c1; c++)
                t = fmaxf(t, __ldcg(reinterpret_cast<const float2*>(slot_of(c) + 16 * DP * 4 + r * 8)).x);
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float sum = 0.0f;
            for (int c = c0; c <= c1; c++) {
                const float2 z = __ldcg(reinterpret_cast<const float2*>(slot_of(c) + 16 * DP * 4 + r * 8));
                const float f = t == -INFINITY ? 0.0f : ex2(z.x - t);
                const float4 x = __ldcg(reinterpret_cast<const float4*>(slot_of(c) + (r * DP + d) * 4));
                sum = fmaf(z.y, f, sum);
                y.x = fmaf(x.x, f, y.x);
                y.y = fmaf(x.y, f, y.y);
                y.z = fmaf(x.z, f, y.z);
                y.w = fmaf(x.w, f, y.w);
            }
            const int i = r / group, gi = r - i * group;
            const int64_t at = static_cast<int64_t>(cur.q.row0 + i) * a.q_heads + cur.hk * group + gi;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.c.dim + d) =
                make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
            if (d == 0 && a.lse) a.lse[at] = sum == 0.0f ? -INFINITY : (t + log2f(sum)) * 0.6931471805599453f;
        }
        if (tid == 0) plan.counters[c0] = 0;
    }
}

// ---------------------------------------------------------------- many rows
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

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

constexpr int64_t kCounterBytes = 4096;  // at the workspace's start: a counter per CTA of any kernel here

}  // namespace

int paged_attention_workspace(const PagedAttnArgs& a, int64_t* bytes) {
    int rc = 0;
    DeviceState* ds = device_state(&rc);
    if (!ds) return rc;
    *bytes = kCounterBytes + 2ll * ds->sm_count * (a.c.dim > 64 ? RowsCfg<128>::SLOT : RowsCfg<64>::SLOT);
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
    RowsPlan plan;
    plan.counters = static_cast<int*>(a.ws);
    plan.parts = static_cast<uint8_t*>(a.ws) + kCounterBytes;
    plan.min_tiles = 4;
    plan.box = std::min(a.c.page, C::KT);
    plan.by_value = a.c.dim % 64 != 0;
    plan.box_halves = a.c.dim == 128 && plan.box == C::KT ? 2 : 1;
    CUtensorMap tmK, tmV;
    int rc = cache_map(&tmK, a.c, a.c.k, a.c.k_tok, a.c.k_head, a.c.k_page, plan.box, plan.box_halves);
    if (rc) return rc;
    rc = cache_map(&tmV, a.c, a.c.v, a.c.v_tok, a.c.v_head, a.c.v_page, plan.box, plan.box_halves);
    if (rc) return rc;
    return launch_pdl(attn_rows_kernel<T, DP>, dim3(ds->sm_count), dim3(NTHR), C::SMEM, st, tmK, tmV, a, plan,
                      ds->d_error);
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
    TVQ_CHECK(ds->sm_count * 4 <= kCounterBytes, TVQ_ERR_UNSUPPORTED, "more SMs than counters");
    if (a.c.n_rows == 0 || a.max_q == 0) return TVQ_OK;
    return a.c.type == TVQ_TYPE_F16 ? launch_attention<__half>(a, ds, st) : launch_attention<__nv_bfloat16>(a, ds, st);
}

}  // namespace tvq
