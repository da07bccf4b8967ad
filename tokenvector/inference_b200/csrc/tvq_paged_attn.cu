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
// attn_rows_kernel: sequences of at most 32 such rows (single tokens, a few
// drafted ones).  Every key and value is used for at most 32 rows, so the
// bytes of the cache bound it, and what counts is that enough of them are in
// flight and that every SM has the same share:
//  - one CTA per SM; all 16-key tiles of all (sequence, kv head) pairs stand
//    in one line, and CTA c takes the c-th equal piece of it, whatever the
//    lengths.  Every CTA finds its piece from the lengths on the device.
//  - the eight warps of a CTA are pipelines of their own: warp w takes the
//    tiles w, w + 8, ... of a pair, brings them through its own ring in
//    shared memory (cp.async, no barrier), and keeps its own m, l, o.  The
//    ring runs on across the ends of pairs, so the next pair's tiles are on
//    their way while the warps join their parts of this one.
//  - mma.sync m16n8k16 with the rows padded to 16 or 32: at D = 128 the two
//    products take 64 of an SM's ~350 cycles per 16 KB of cache, so that the
//    wider tcgen05 tile (128 rows) would buy nothing here.
//  - a pair that several CTAs share is joined by the one that finishes last
//    (a counter per CTA in the workspace, zero between calls), in the order
//    of the parts, so results do not depend on who that is.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "tvq_common.cuh"
#include "tvq_decode.h"

namespace tvq {

namespace {

constexpr int KT = 16;      // keys per tile
constexpr int NW = 8;       // warps per CTA of the rows kernel
constexpr int NTHR = NW * 32;

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

// 16 bytes global -> shared; zeros when !in (the address is then not read)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
    const int n = in ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

// The 16-key tiles [first, end) that the rows of a sequence see together: one
// at least, so that rows without keys are written too.
__device__ __forceinline__ int2 seq_tiles(const Seq& q, int window) {
    const int p0 = q.len - q.n;
    const int first = window > 0 ? max(0, p0 - window + 1) / KT : 0;
    return make_int2(first, max(first + 1, (max(q.len, 0) + KT - 1) / KT));
}

// ---------------------------------------------------------------- few rows
template <int DP, int MT>
struct RowsCfg {
    static constexpr int ROWB = DP * 2;                  // bytes of a key
    static constexpr int STAGE = 2 * KT * ROWB;          // one tile: keys, then values
    static constexpr int STAGES = DP == 128 ? 3 : 6;     // 192 KB of ring either way
    static constexpr int RING = NW * STAGES * STAGE;
    static constexpr int PART = 16 * DP * 4;             // one warp's o of 16 rows
    static constexpr int OFF_PART = RING;                // [4][16][DP] f32
    static constexpr int OFF_ML = OFF_PART + 4 * PART;   // float2 [MLB][NW][16 * MT]
    static constexpr int MLB = DP == 128 && MT == 2 ? 1 : 2;  // two, as far as they fit: one barrier less
    static constexpr int SMEM = OFF_ML + MLB * NW * 16 * MT * 8;
    static constexpr int64_t SLOT = 16 * MT * (DP * 4 + 8);  // workspace bytes of one partial
};

struct RowsPlan {
    int* counters;   // [grid]
    uint8_t* parts;  // [grid][2] slots
    int min_tiles;   // no CTA gets a smaller piece
};

// Where a warp stands in its CTA's piece: a pair and a tile of it.
struct Cursor {
    int s, hk;
    int64_t left;  // tiles of the piece from this pair's first tile in it on
    Seq q;
    int t, end;    // this warp's next tile, the end of the pair's tiles in the piece
    int first;     // the pair's first tile in the piece
    int2 all;      // the pair's tiles
};

template <typename T, int DP, int MT>
__global__ void __launch_bounds__(NTHR, 1) attn_rows_kernel(const PagedAttnArgs a, const RowsPlan plan, int* err) {
    using C = RowsCfg<DP, MT>;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ int s_scan[NW];
    __shared__ int64_t s_at[2];
    __shared__ int s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.q_heads / a.c.kv_heads;
    griddep_wait();

    // ---- this CTA's piece of the line of tiles
    auto weight = [&](int s) -> int {
        if (s >= a.c.n_seq) return 0;
        const Seq q = load_seq(a.c, s);
        if (q.n == 0 || q.n > 16 * MT / group) return 0;
        const int2 t = seq_tiles(q, a.window);
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
        for (int w = 0; w < NW; w++) {
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
        int all;
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
        if (a.c.n_seq > NTHR) before += all;
    }
    __syncthreads();

    Cursor cur;
    cur.s = static_cast<int>(s_at[0]);
    const int64_t in_seq = begin - s_at[1];
    auto enter = [&](Cursor& c, int skip) {  // c.s, c.hk, c.left set; the pair's tiles from `skip` on
        c.all = seq_tiles(c.q, a.window);
        c.first = c.all.x + skip;
        c.end = static_cast<int>(min(static_cast<int64_t>(c.all.y), c.first + c.left));
        c.t = c.first + warp;
    };
    auto next_pair = [&](Cursor& c) {  // false: the piece is done
        c.left -= c.end - c.first;
        if (c.left <= 0) return false;
        if (++c.hk == a.c.kv_heads) {
            c.hk = 0;
            do {
                c.q = load_seq(a.c, ++c.s);
            } while (c.q.n == 0 || c.q.n > 16 * MT / group);
        }
        enter(c, 0);
        return true;
    };
    cur.q = load_seq(a.c, cur.s);
    cur.left = stop - begin;
    {
        const int2 t = seq_tiles(cur.q, a.window);
        cur.hk = static_cast<int>(in_seq / (t.y - t.x));
        enter(cur, static_cast<int>(in_seq - static_cast<int64_t>(cur.hk) * (t.y - t.x)));
    }

    // ---- the warp's ring: tiles are issued STAGES - 1 ahead, one group each
    Cursor ahead = cur;
    bool more = true;
    uint8_t* ring = sm + warp * (C::STAGES * C::STAGE);
    const uint32_t ring_u = smem_u32(ring);
    int page = -1;  // of the tile's first (even lanes) or second (odd lanes) eight keys
    auto look = [&]() {  // the next tile with work, and its page
        while (more && ahead.t >= ahead.end) more = next_pair(ahead);
        if (!more) return;
        const int col = (ahead.t * KT + (lane & 1) * 8) >> a.c.page_log2;
        page = col < a.c.n_cols ? __ldg(a.c.table + ahead.s * a.c.table_stride + col) : -1;
    };
    auto issue = [&](int stage) {
        if (more) {
            const uint32_t dst = ring_u + stage * C::STAGE;
            constexpr int CH = C::ROWB / 16;  // 16-byte pieces of a key
            const int c = lane % CH;
            const int64_t kh = ahead.hk * a.c.k_head + c * 8, vh = ahead.hk * a.c.v_head + c * 8;
#pragma unroll
            for (int i = 0; i < KT * CH / 32; i++) {
                const int r = lane / CH + i * (32 / CH);
                const int j = ahead.t * KT + r;
                const int pg = __shfl_sync(0xffffffffu, page, r >> 3);
                const bool ok = static_cast<unsigned>(pg) < static_cast<unsigned>(a.c.n_pages);
                if (!ok && j < ahead.q.len) record_error(err, DEVERR_BAD_PAGE);
                const bool in = ok && j < ahead.q.len && c * 8 < a.c.dim;
                const int slot = j & (a.c.page - 1);
                const T* k = static_cast<const T*>(a.c.k) + (in ? pg * a.c.k_page + slot * a.c.k_tok + kh : 0);
                const T* v = static_cast<const T*>(a.c.v) + (in ? pg * a.c.v_page + slot * a.c.v_tok + vh : 0);
                const uint32_t o = dst + r * C::ROWB + ((c ^ (r & 7)) << 4);
                cp16(o, k, in);
                cp16(o + KT * C::ROWB, v, in);
            }
            ahead.t += NW;
        }
        cp_commit();
        look();
    };
    look();
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; i++) issue(i);
    int stage = 0, fill = C::STAGES - 1;

    const float scale2 = a.scale * 1.4426950408889634f;
    const int g = lane >> 2, quad = lane & 3;
    int parity = 0;
    for (bool go = true; go; go = next_pair(cur), parity ^= C::MLB - 1) {
        // ---- the pair's rows as A fragments
        const int rows = cur.q.n * group;
        uint32_t qf[MT][DP / 16][4];
        int pos[MT][2];  // of this thread's two rows in each block of 16 (below 0: sees nothing)
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int r = mt * 16 + g + hf * 8;
                const int i = r / group, gi = r - i * group;
                const bool in = r < rows;
                pos[mt][hf] = in ? cur.q.len - cur.q.n + i : -1;
                const T* q = static_cast<const T*>(a.q) + (in ? (cur.q.row0 + i) * a.q_tok + (cur.hk * group + gi) * a.q_head : 0);
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int d = kk * 16 + e * 8 + quad * 2;
                        qf[mt][kk][e * 2 + hf] = in && d < a.c.dim ? __ldg(reinterpret_cast<const uint32_t*>(q + d)) : 0u;
                    }
            }
        float m[MT][2], l[MT][2], o[MT][DP / 8][4];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.0f;
#pragma unroll
            for (int n = 0; n < DP / 8; n++) o[mt][n][0] = o[mt][n][1] = o[mt][n][2] = o[mt][n][3] = 0.0f;
        }

        for (; cur.t < cur.end; cur.t += NW) {
            cp_wait<C::STAGES - 2>();
            __syncwarp();  // the tile is there for every lane, and every lane is done with the one before
            issue(fill);
            const uint32_t ks = ring_u + stage * C::STAGE, vs = ks + KT * C::ROWB;
            float sc[MT][2][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int n = 0; n < 2; n++) sc[mt][n][0] = sc[mt][n][1] = sc[mt][n][2] = sc[mt][n][3] = 0.0f;
            {
                const int r = ((lane >> 4) << 3) + (lane & 7), cc = (lane >> 3) & 1;
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk++) {
                    uint32_t b[4];
                    ldsm4(ks + r * C::ROWB + (((kk * 2 + cc) ^ (r & 7)) << 4), b);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        mma16816<T>(sc[mt][0], qf[mt][kk], b[0], b[1]);
                        mma16816<T>(sc[mt][1], qf[mt][kk], b[2], b[3]);
                    }
                }
            }
            uint32_t pf[MT][4];
            const int j0 = cur.t * KT + quad * 2;
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int hi = pos[mt][hf], lo = a.window > 0 ? hi - a.window : -1;  // keys in (lo, hi]
                    float x[4], top = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = j0 + (e >> 1) * 8 + (e & 1);
                        const float y = sc[mt][e >> 1][hf * 2 + (e & 1)] * scale2;
                        x[e] = j <= hi && j > lo ? y : -INFINITY;
                        top = fmaxf(top, x[e]);
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float m2 = fmaxf(m[mt][hf], top);
                    const float base = m2 == -INFINITY ? 0.0f : m2;
                    const float f = ex2(m[mt][hf] - base);
                    m[mt][hf] = m2;
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[e] = ex2(x[e] - base);
                        sum += x[e];
                    }
                    l[mt][hf] = l[mt][hf] * f + sum;
                    // the weights meet V in its own type: 2^-11 (f16) or 2^-8 (bf16) of each, as the
                    // rounding of the result; l sums them unrounded
                    pf[mt][hf] = pack2<T>(x[0], x[1]);
                    pf[mt][2 + hf] = pack2<T>(x[2], x[3]);
#pragma unroll
                    for (int n = 0; n < DP / 8; n++) {
                        o[mt][n][hf * 2] *= f;
                        o[mt][n][hf * 2 + 1] *= f;
                    }
                }
            {
                const int r = (((lane >> 3) & 1) << 3) + (lane & 7), cc = lane >> 4;
#pragma unroll
                for (int n = 0; n < DP / 16; n++) {
                    uint32_t b[4];
                    ldsm4_t(vs + r * C::ROWB + (((n * 2 + cc) ^ (r & 7)) << 4), b);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        mma16816<T>(o[mt][2 * n], pf[mt], b[0], b[1]);
                        mma16816<T>(o[mt][2 * n + 1], pf[mt], b[2], b[3]);
                    }
                }
            }
            if (++stage == C::STAGES) stage = 0;
            if (++fill == C::STAGES) fill = 0;
        }

        // ---- join the eight warps' parts
        if constexpr (C::MLB == 1) __syncthreads();
        float2* ml = reinterpret_cast<float2*>(sm + C::OFF_ML) + parity * NW * 16 * MT;
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                float x = l[mt][hf];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                if (quad == 0) ml[warp * 16 * MT + mt * 16 + g + hf * 8] = make_float2(m[mt][hf], x);
            }
        __syncthreads();
        const bool whole = cur.first == cur.all.x && cur.end == cur.all.y;
        const int slot = cur.first == cur.all.x ? 1 : 0;  // a pair that goes on after this piece, or came into it
        uint8_t* part = plan.parts + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * C::SLOT;
        float* buf = reinterpret_cast<float*>(sm + C::OFF_PART);
        auto top_of = [&](int r) {
            float t = ml[r].x;
#pragma unroll
            for (int w = 1; w < NW; w++) t = fmaxf(t, ml[w * 16 * MT + r].x);
            return t;
        };
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float f[2];
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const float t = top_of(mt * 16 + g + hf * 8);
                f[hf] = t == -INFINITY ? 0.0f : ex2(m[mt][hf] - t);
            }
            float* mine = buf + (warp & 3) * (16 * DP);
            if (mt > 0) __syncthreads();  // the block before is read
            if (warp >= 4) {
#pragma unroll
                for (int n = 0; n < DP / 8; n++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
                        *reinterpret_cast<float2*>(mine + (g + hf * 8) * DP + n * 8 + quad * 2) =
                            make_float2(o[mt][n][hf * 2] * f[hf], o[mt][n][hf * 2 + 1] * f[hf]);
            }
            __syncthreads();
            if (warp < 4) {
#pragma unroll
                for (int n = 0; n < DP / 8; n++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        float2* w = reinterpret_cast<float2*>(mine + (g + hf * 8) * DP + n * 8 + quad * 2);
                        const float2 y = *w;
                        *w = make_float2(fmaf(o[mt][n][hf * 2], f[hf], y.x), fmaf(o[mt][n][hf * 2 + 1], f[hf], y.y));
                    }
            }
            __syncthreads();
            for (int e = tid; e < 16 * (DP / 4); e += NTHR) {
                const int r = e / (DP / 4), d = (e - r * (DP / 4)) * 4, row = mt * 16 + r;
                if (row >= rows || d >= a.c.dim) continue;
                float4 y = *reinterpret_cast<const float4*>(buf + r * DP + d);
#pragma unroll
                for (int w = 1; w < 4; w++) {
                    const float4 z = *reinterpret_cast<const float4*>(buf + w * 16 * DP + r * DP + d);
                    y.x += z.x;
                    y.y += z.y;
                    y.z += z.z;
                    y.w += z.w;
                }
                const float t = top_of(row);
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    const float2 z = ml[w * 16 * MT + row];
                    sum += t == -INFINITY ? 0.0f : z.y * ex2(z.x - t);
                }
                if (whole) {
                    const int i = row / group, gi = row - i * group;
                    const int64_t at = static_cast<int64_t>(cur.q.row0 + i) * a.q_heads + cur.hk * group + gi;
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.c.dim + d) =
                        make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
                    if (d == 0 && a.lse) a.lse[at] = sum == 0.0f ? -INFINITY : (t + log2f(sum)) * 0.6931471805599453f;
                } else {
                    *reinterpret_cast<float4*>(part + (static_cast<int64_t>(row) * DP + d) * 4) = y;
                    if (d == 0) *reinterpret_cast<float2*>(part + 16 * MT * DP * 4 + row * 8) = make_float2(t, sum);
                }
            }
        }
        if (whole) continue;

        // ---- join the CTAs' parts: CTA c0 began the pair, c1 ends it
        const int64_t at0 = begin + (stop - begin - cur.left) - (cur.first - cur.all.x);  // of the pair's first tile
        const int c0 = static_cast<int>(at0 / per), c1 = static_cast<int>((at0 + cur.all.y - cur.all.x - 1) / per);
        __threadfence();
        __syncthreads();
        if (tid == 0) s_last = atomicAdd(plan.counters + c0, 1) == c1 - c0;
        __syncthreads();
        if (!s_last) continue;
        __threadfence();
        for (int e = tid; e < rows * (DP / 4); e += NTHR) {
            const int row = e / (DP / 4), d = (e - row * (DP / 4)) * 4;
            if (d >= a.c.dim) continue;
            auto slot_of = [&](int c) { return plan.parts + (static_cast<int64_t>(c) * 2 + (c == c0 ? 1 : 0)) * C::SLOT; };
            float t = -INFINITY;
            for (int c = c0; c <= c1; c++)
                t = fmaxf(t, __ldcg(reinterpret_cast<const float2*>(slot_of(c) + 16 * MT * DP * 4 + row * 8)).x);
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float sum = 0.0f;
            for (int c = c0; c <= c1; c++) {
                const float2 z = __ldcg(reinterpret_cast<const float2*>(slot_of(c) + 16 * MT * DP * 4 + row * 8));
                const float f = t == -INFINITY ? 0.0f : ex2(z.x - t);
                const float4 x = __ldcg(reinterpret_cast<const float4*>(slot_of(c) + (static_cast<int64_t>(row) * DP + d) * 4));
                sum = fmaf(z.y, f, sum);
                y.x = fmaf(x.x, f, y.x);
                y.y = fmaf(x.y, f, y.y);
                y.z = fmaf(x.z, f, y.z);
                y.w = fmaf(x.w, f, y.w);
            }
            const int i = row / group, gi = row - i * group;
            const int64_t at = static_cast<int64_t>(cur.q.row0 + i) * a.q_heads + cur.hk * group + gi;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.c.dim + d) =
                make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
            if (d == 0 && a.lse) a.lse[at] = sum == 0.0f ? -INFINITY : (t + log2f(sum)) * 0.6931471805599453f;
        }
        if (tid == 0) plan.counters[c0] = 0;
    }
    cp_wait<0>();
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
    const bool two = static_cast<int64_t>(a.max_q) * (a.q_heads / a.c.kv_heads) > 16;
    const int64_t slot = a.c.dim > 64 ? (two ? RowsCfg<128, 2>::SLOT : RowsCfg<128, 1>::SLOT)
                                      : (two ? RowsCfg<64, 2>::SLOT : RowsCfg<64, 1>::SLOT);
    *bytes = kCounterBytes + 2ll * ds->sm_count * slot;
    return TVQ_OK;
}

namespace {

template <typename T, int DP, int MT>
int launch_rows(const PagedAttnArgs& a, DeviceState* ds, cudaStream_t st) {
    using C = RowsCfg<DP, MT>;
    static const cudaError_t attr = cudaFuncSetAttribute(attn_rows_kernel<T, DP, MT>,
                                                         cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    TVQ_CUDA(attr);
    RowsPlan plan;
    plan.counters = static_cast<int*>(a.ws);
    plan.parts = static_cast<uint8_t*>(a.ws) + kCounterBytes;
    plan.min_tiles = NW;
    return launch_pdl(attn_rows_kernel<T, DP, MT>, dim3(ds->sm_count), dim3(NTHR), C::SMEM, st, a, plan, ds->d_error);
}

template <typename T>
int launch_attention(const PagedAttnArgs& a, DeviceState* ds, cudaStream_t st) {
    const int group = a.q_heads / a.c.kv_heads;
    const bool two = static_cast<int64_t>(a.max_q) * group > 16;
    int rc;
    if (a.c.dim > 64) rc = two ? launch_rows<T, 128, 2>(a, ds, st) : launch_rows<T, 128, 1>(a, ds, st);
    else rc = two ? launch_rows<T, 64, 2>(a, ds, st) : launch_rows<T, 64, 1>(a, ds, st);
    if (rc || static_cast<int64_t>(a.max_q) * group <= 32) return rc;
    const int64_t units = static_cast<int64_t>(a.c.n_rows) * a.q_heads;
    return launch_pdl(paged_attention_row_kernel<T>, dim3(static_cast<unsigned>((units + 3) / 4)), dim3(128), 0, st, a,
                      32 / group, ds->d_error);
}

}  // namespace

int launch_paged_attention(const PagedAttnArgs& a, cudaStream_t st) {
    int rc = 0;
    DeviceState* ds = device_state(&rc);
    if (!ds) return rc;
    if (a.c.n_rows == 0 || a.max_q == 0) return TVQ_OK;
    return a.c.type == TVQ_TYPE_F16 ? launch_attention<__half>(a, ds, st) : launch_attention<__nv_bfloat16>(a, ds, st);
}

}  // namespace tvq
