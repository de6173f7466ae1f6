// Gated GQA attention over a paged bf16 KV cache: one new token per request
// (decode) and ragged chunks of several prompts (prefill).
//
// Per query row the semantics of the reference's attention() (c/qwen.c:598-663):
// zero-centred RMSNorm of q and k per head, partial NeoX RoPE on the first
// `rot` dims, K/V append, softmax attention over rows 0..pos, ctx *=
// sigmoid(gate). Only where a row lives differs: row pos of request r, KV
// head kh is row (table[r][pos / page] * KH + kh) * page + pos % page.
//
// Every page id and position is checked on the device before it is used; a
// bad one raises g_pages_error, is left out, and touches no memory.
#include "common.cuh"
#include "kernels.h"

namespace coli {

// Argument errors found on the device (first one wins, read and cleared by
// the host): the backend stays usable.
enum { PAGES_OK = 0, PAGES_BAD_ID = 1, PAGES_BAD_POS = 2, PAGES_BAD_ROWS = 3, PAGES_CONFLICT = 4, PAGES_BAD_REQ = 5 };
__device__ int g_pages_error;
__device__ __forceinline__ void pages_error(int code) { atomicCAS(&g_pages_error, 0, code); }

// Angle table of position pos, entries [0, rot / 2): the product and its
// reduction to a turn in double, the sine and cosine of what is left in float.
__device__ __forceinline__ void pages_rope_table(float *cs, float *sn, int pos, int rot, const RopeFreq &f, int tid0,
                                                 int nthr)
{
    constexpr double TURN = 6.283185307179586476925286766559;
    for (int j = tid0; j < (rot >> 1); j += nthr) {
        const double a = (double)pos * f.f[j];
        const float r = (float)(a - rint(a * (1.0 / TURN)) * TURN);
        sincosf(r, &sn[j], &cs[j]);
    }
}

// First row of K/V of request r, KV head kh, position pos; -1 for a page id
// outside the pool.
__device__ __forceinline__ long long pages_row(const PageView &v, int r, int kh, int pos)
{
    const int pi = pos / v.page, id = v.table[(size_t)r * v.max_pages + pi];
    if ((unsigned)id >= (unsigned)v.n_pages) { pages_error(PAGES_BAD_ID); return -1; }
    return ((long long)id * v.KH + kh) * v.page + (pos - pi * v.page);
}

// Request r's first row, number of rows and first position; 0 rows where it
// is idle or says something impossible.
__device__ __forceinline__ int pages_rows_of(const GqaPagesArgs &p, int r, int &row0, int &pos0)
{
    int n = 1;
    row0 = r;
    pos0 = p.base[r];
    if (p.cu) {
        row0 = p.cu[r];
        n = p.cu[r + 1] - row0;
        if (n == 0) return 0;
        if (row0 < 0 || n < 0 || n > p.S || row0 > p.S - n) { pages_error(PAGES_BAD_ROWS); return 0; }
        if (pos0 < 0) { pages_error(PAGES_BAD_POS); return 0; }
    } else if (pos0 < 0) {
        return 0;
    }
    if ((long long)pos0 + n > (long long)p.pv.max_pages * p.pv.page) { pages_error(PAGES_BAD_POS); return 0; }
    return n;
}

// Request of a row (the last r with cu[r] <= row < cu[r + 1]), -1 for a row
// behind the last sequence.
__device__ __forceinline__ int pages_req_of(const GqaPagesArgs &p, int row)
{
    if (!p.cu) return row;
    for (int r = 0; r < p.n_req; ++r)
        if (row >= p.cu[r] && row < p.cu[r + 1]) return r;
    return -1;
}

// ------------------------------------------------------------------ decode
// The work is one list of 16-token tiles, request by request and KV head by KV
// head, cut into equal consecutive ranges, one per CTA: a batch of any lengths
// keeps every SM streaming to the end, and a single long request is split over
// all of them. A range covers pieces of consecutive units (a unit: one request
// and KV head). A piece that is a whole unit writes ctx itself; the others
// leave (O, max, sum) in the workspace and pages_join_kernel merges a unit's
// pieces. A CTA has at most two such pieces, its first and its last, so the
// workspace does not depend on the batch.
//
// Inside a CTA warp w takes tiles w, w + 4, .. of the range through its own TMA
// ring (one 8 KiB box per tile of K and of V, mbarrier completion), which
// runs on across unit borders; the page ids of a warp's next 32 tiles are
// looked up by its 32 lanes at once, a batch ahead of their use. Per tile
// S^T[16 tok x 8 heads] = K Q^T and O^T += V^T P^T on bf16 mma.sync, the
// (up to) 8 query heads of the KV head being the N of the MMA. At 8 heads that
// is 8 FLOP per byte read: HBM bounds it, and tcgen05's 64-row minimum would
// leave 7/8 of its rows empty.
// The new token's K and V rows are normed, roped and appended by the warp that
// owns the unit's last tile: to the page, and over the tile's copy in shared
// memory, so no tile load waits for an append.
// fp32 activations: q and the probabilities are two bf16 parts each (hi + lo,
// 16 bits of mantissa), two MMAs instead of one per fragment.
constexpr int PD_WARPS = 4, PD_THREADS = 32 * PD_WARPS;
constexpr int PD_MIN_TILES = PD_WARPS;      // fewest tiles of a CTA: one per warp
template <typename TI> struct PdSmem {
    static constexpr bool SPLIT = sizeof(TI) == 4;
    static constexpr int STAGES = SPLIT ? 2 : 3;   // 128 / 192 KiB of tiles in flight per SM
    uint8_t ring[PD_WARPS][STAGES][2 * GQA_TILE_BYTES];
    float4 merge[PD_WARPS][8][32];          // a half of a warp's accumulators; also its cs / sn / vw scratch
    __nv_bfloat16 q[SPLIT ? 2 : 1][GQA_GRP * GQA_HD];
    TI gate[GQA_GRP * GQA_HD];
    float w[2][GQA_HD];                     // q / k norm weights
    float ml[PD_WARPS][GQA_GRP][2];
    int pre[1024 + 4];                      // tiles (of one KV head) before each request
    int part[PD_WARPS];
    uint64_t full[PD_WARPS][STAGES];
};

// The range of CTA c is tiles [c * per, (c + 1) * per) of `total`.
__device__ __forceinline__ int pd_per(int total, int ctas)
{
    const int per = (total + ctas - 1) / ctas;
    return max(PD_MIN_TILES, (per + PD_WARPS - 1) / PD_WARPS * PD_WARPS);
}

template <typename TI>
__global__ void __launch_bounds__(PD_THREADS, 1)
pages_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, GqaPagesArgs p,
                    PagesPart part, const __grid_constant__ RopeFreq f)
{
    using Smem = PdSmem<TI>;
    constexpr int STAGES = Smem::STAGES, QP = Smem::SPLIT ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
    const int KH = p.pv.KH, G = p.H / KH, page = p.pv.page;
    griddep_launch();                       // the join may be scheduled; it waits for this grid
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(&sm.full[warp][s], 1);
        fence_mbar_init();
    }
    if (tid == 0) { tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); }

    // tiles before each request
    {
        const int each = (p.n_req + PD_THREADS - 1) / PD_THREADS, r0 = tid * each;
        int n[8], mine = 0;
        for (int i = 0; i < each; ++i) {
            int row0, pos0;
            n[i & 7] = r0 + i < p.n_req && pages_rows_of(p, r0 + i, row0, pos0) ? pos0 / GQA_TILE + 1 : 0;
            mine += n[i & 7];
        }
        int inc = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += y;
        }
        if (lane == 31) sm.part[warp] = inc;
        for (int i = tid; i < 2 * GQA_HD; i += PD_THREADS) sm.w[i / GQA_HD][i % GQA_HD] = i < GQA_HD ? p.qnw[i] : p.knw[i - GQA_HD];
        for (int i = tid; i < QP * GQA_GRP * GQA_HD / 8; i += PD_THREADS)
            reinterpret_cast<uint4 *>(sm.q)[i] = make_uint4(0, 0, 0, 0);   // heads past the group's stay zero
        __syncthreads();
        int at = inc - mine;
        for (int w = 0; w < warp; ++w) at += sm.part[w];
        for (int i = 0; i < each; ++i) {
            if (r0 + i <= p.n_req) sm.pre[r0 + i] = at;
            at += n[i & 7];
        }
        if (tid == PD_THREADS - 1) sm.pre[p.n_req] = at;
        __syncthreads();
    }
    const int total = sm.pre[p.n_req] * KH;
    const int per = pd_per(total, gridDim.x);
    const int c0 = min(total, cta * per), c1 = min(total, c0 + per);
    // request of flat tile t: the last r with pre[r] * KH <= t
    auto find = [&](int t) {
        int lo = 0, hi = p.n_req - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (sm.pre[mid] * KH <= t) lo = mid; else hi = mid - 1;
        }
        return lo;
    };

    // ---- the warp's tiles: ordinal i is flat tile c0 + warp + 4 i
    const int mine = max(0, (c1 - c0 - warp + PD_WARPS - 1) / PD_WARPS);
    int ahead_id = 0, ahead_row = 0, at_group = 0;        // of ordinals (batch of 32) + lane
    auto look_up = [&](int batch) {
        const int i = batch * 32 + lane;
        if (i >= mine) return;
        const int t = c0 + warp + PD_WARPS * i, r = find(t), nt = sm.pre[r + 1] - sm.pre[r];
        const int rel = t - sm.pre[r] * KH, kh = rel / nt, tok = (rel - kh * nt) * GQA_TILE, pi = tok / page;
        ahead_id = p.pv.table[(size_t)r * p.pv.max_pages + pi];
        ahead_row = kh * page + tok - pi * page;
    };
    auto take = [&]() {                                   // the batch looked up becomes the one in use
        if ((unsigned)ahead_id >= (unsigned)p.pv.n_pages) { pages_error(PAGES_BAD_ID); ahead_id = 0; }
        at_group = (int)(((long long)ahead_id * KH * page + ahead_row) >> 3);
    };
    auto issue = [&](int i) {                             // whole warp; i < mine
        const int group = __shfl_sync(0xffffffffu, at_group, i & 31), s = i % STAGES;
        if (lane == 0) {
            uint8_t *kb = sm.ring[warp][s];
            mbar_expect_tx(&sm.full[warp][s], 2 * GQA_TILE_BYTES);
            tma_load_4d(kb, &tmK, 0, 0, 0, group, &sm.full[warp][s]);
            tma_load_4d(kb + GQA_TILE_BYTES, &tmV, 0, 0, 0, group, &sm.full[warp][s]);
        }
    };
    look_up(0);
    take();
    look_up(1);
    for (int i = 0; i < STAGES && i < mine; ++i) issue(i);

    float *cs = reinterpret_cast<float *>(sm.merge[warp]), *sn = cs + GQA_HD / 2, *vw = sn + GQA_HD / 2;
    const TI *qg = static_cast<const TI *>(p.qg);
    Raw8<TI> rq[2], rg[2], rk, rv;                        // the next unit's two heads of this warp
    auto load_heads = [&](int r, int kh) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int h = 2 * warp + u;
            if (h < G) {
                const TI *src = qg + ((size_t)r * p.H + kh * G + h) * 2 * GQA_HD + lane * 8;
                rq[u].load(src);
                rg[u].load(src + GQA_HD);
            }
        }
    };

    int t = c0, r = 0, kh = 0, i = 0, join_to = -1;
    if (t < c1) {
        r = find(t);
        kh = (t - sm.pre[r] * KH) / (sm.pre[r + 1] - sm.pre[r]);
        load_heads(r, kh);
    }
    const int r8 = lane & 7, mi = lane >> 3, h0 = (lane & 3) * 2, dr = lane >> 2;
    while (t < c1) {
        const int nt = sm.pre[r + 1] - sm.pre[r], u0 = sm.pre[r] * KH + kh * nt, u1 = u0 + nt, end = min(u1, c1);
        const int pos = p.base[r], T = pos + 1;
        // ---- q of the unit's heads, normed and roped, and the gate
        pages_rope_table(cs, sn, pos, p.rot, f, lane, 32);
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int h = 2 * warp + u;
            if (h < G) {
                float x[8], w[8], y[8];
                rq[u].unpack(x);
                load8<float>(sm.w[0] + lane * 8, w);
                gqa_norm_rope(y, x, w, p.eps, p.rot, cs, sn, vw, lane);
                // q to bf16 (a rounding of 2^-9 of each element; fp32 inputs: hi and lo parts)
                store8(sm.q[0] + h * GQA_HD + lane * 8, y);
                if constexpr (Smem::SPLIT) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] -= __bfloat162float(__float2bfloat16_rn(y[e]));
                    store8(sm.q[QP - 1] + h * GQA_HD + lane * 8, y);
                }
                rg[u].store(sm.gate + h * GQA_HD + lane * 8);
            }
        }
        // the last tile's owner fetches the row to append
        const bool append = u1 <= c1 && ((u1 - 1 - c0) & (PD_WARPS - 1)) == warp;
        if (append) {
            const size_t in = ((size_t)r * KH + kh) * GQA_HD + lane * 8;
            rk.load(static_cast<const TI *>(p.k) + in);
            rv.load(static_cast<const TI *>(p.v) + in);
        }
        __syncthreads();
        // Q^T as the B operand: b0 = (dim = 16kk + 2(lane&3) + {0,1}, head = lane>>2), b1 = dim + 8
        uint32_t qf[QP][16][2];
#pragma unroll
        for (int q = 0; q < QP; ++q)
#pragma unroll
            for (int kk = 0; kk < 16; ++kk) {
                const __nv_bfloat16 *src = sm.q[q] + (lane >> 2) * GQA_HD + kk * 16 + (lane & 3) * 2;
                qf[q][kk][0] = *reinterpret_cast<const uint32_t *>(src);
                qf[q][kk][1] = *reinterpret_cast<const uint32_t *>(src + 8);
            }
        // the next unit's heads, in flight during this unit's tiles
        int nr = r, nkh = kh + 1;
        if (nkh == KH) {
            nkh = 0;
            for (++nr; nr < p.n_req && sm.pre[nr + 1] == sm.pre[nr];) ++nr;
        }
        if (end < c1) load_heads(nr, nkh);

        float acc[16][4];
#pragma unroll
        for (int mt = 0; mt < 16; ++mt) acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        const float sl2 = p.scale_log2;
        for (; i < mine && c0 + warp + PD_WARPS * i < end; ++i) {
            const int s = i % STAGES, tile = c0 + warp + PD_WARPS * i - u0, tok0 = tile * GQA_TILE;
            mbar_wait(&sm.full[warp][s], (i / STAGES) & 1);   // a time-out raises the error word; the rest runs on what is there
            uint8_t *kt = sm.ring[warp][s], *vt = kt + GQA_TILE_BYTES;
            const uint32_t kb = smem_u32(kt), vb = kb + GQA_TILE_BYTES;
            const int valid = min(GQA_TILE, T - tok0);
            if (append && tile == nt - 1) {
                // position pos: into the page and over the loaded tile (whose row is the page's old contents)
                float x[8], w[8], y[8], v[8];
                rk.unpack(x);
                rv.unpack(v);
                load8<float>(sm.w[1] + lane * 8, w);
                gqa_norm_rope(y, x, w, p.eps, p.rot, cs, sn, vw, lane);
                const int row = pos - tok0, off = (row >> 3) * 4096 + (lane >> 3) * 1024 + (row & 7) * 128 + (((lane & 7) ^ (row & 7)) << 4);
                store8(reinterpret_cast<__nv_bfloat16 *>(kt + off), y);
                store8(reinterpret_cast<__nv_bfloat16 *>(vt + off), v);
                const long long at = pages_row(p.pv, r, kh, pos);
                if (at >= 0) {
                    store8(p.pv.k + at * GQA_HD + lane * 8, y);
                    store8(p.pv.v + at * GQA_HD + lane * 8, v);
                }
            }
            if (valid < GQA_TILE) {
                // rows past the end are never weighted; cleared so that stale
                // non-finite cache contents cannot come through as 0 * inf
                for (int j = lane; j < (GQA_TILE - valid) * 32; j += 32) {
                    const int row = valid + (j >> 5), c = (j & 31) >> 3, ch = j & 7;
                    *reinterpret_cast<uint4 *>(vt + (row >> 3) * 4096 + c * 1024 + (row & 7) * 128 + ch * 16) = make_uint4(0, 0, 0, 0);
                }
            }
            __syncwarp();
            // S^T[16 tok x 8 heads] = K[16 x 256] . Q^T[256 x 8]
            float sc[4] = {0.f, 0.f, 0.f, 0.f};
            {
                const uint32_t base = kb + (mi & 1) * 4096 + r8 * 128;
#pragma unroll
                for (int kk = 0; kk < 16; ++kk) {
                    const int chunk = (kk & 3) * 2 + (mi >> 1);
                    uint32_t a0, a1, a2, a3;
                    ldsm_x4(base + (kk >> 2) * 1024 + ((chunk ^ r8) << 4), a0, a1, a2, a3);
#pragma unroll
                    for (int q = 0; q < QP; ++q) mma_bf16_16816(sc, a0, a1, a2, a3, qf[q][kk][0], qf[q][kk][1]);
                }
            }
            // online softmax per head (heads h0, h0 + 1), log2 domain
            const int ta = lane >> 2, tb = ta + 8;
            const float x0 = ta < valid ? sc[0] * sl2 : -INFINITY, x1 = ta < valid ? sc[1] * sl2 : -INFINITY;
            const float x2 = tb < valid ? sc[2] * sl2 : -INFINITY, x3 = tb < valid ? sc[3] * sl2 : -INFINITY;
            float t0 = fmaxf(x0, x2), t1 = fmaxf(x1, x3);
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) {
                t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
                t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
            }
            const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
            const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
            const float p0 = exp2f(x0 - b0), p1 = exp2f(x1 - b1), p2 = exp2f(x2 - b0), p3 = exp2f(x3 - b1);
            if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
                const float al0 = exp2f(m0 - b0), al1 = exp2f(m1 - b1);
                l0 *= al0;
                l1 *= al1;
#pragma unroll
                for (int mt = 0; mt < 16; ++mt) { acc[mt][0] *= al0; acc[mt][1] *= al1; acc[mt][2] *= al0; acc[mt][3] *= al1; }
                m0 = n0;
                m1 = n1;
            }
            l0 += p0 + p2;
            l1 += p1 + p3;
            uint32_t pb[QP][2];
            pb[0][0] = pack_bf16(p0, p1);
            pb[0][1] = pack_bf16(p2, p3);
            if constexpr (Smem::SPLIT) {
                auto lo = [](float x) { return x - __bfloat162float(__float2bfloat16_rn(x)); };
                pb[QP - 1][0] = pack_bf16(lo(p0), lo(p1));
                pb[QP - 1][1] = pack_bf16(lo(p2), lo(p3));
            }
#pragma unroll
            for (int q = 0; q < QP; ++q) { pb[q][0] = movmatrix_t(pb[q][0]); pb[q][1] = movmatrix_t(pb[q][1]); }
            // O^T[256 dims x 8 heads] += V^T[256 x 16 tok] . P^T[16 tok x 8 heads]
            {
                const uint32_t base = vb + (mi >> 1) * 4096 + r8 * 128;
#pragma unroll
                for (int mt = 0; mt < 16; ++mt) {
                    const int chunk = (mt & 3) * 2 + (mi & 1);
                    uint32_t a0, a1, a2, a3;
                    ldsm_x4_t(base + (mt >> 2) * 1024 + ((chunk ^ r8) << 4), a0, a1, a2, a3);
#pragma unroll
                    for (int q = 0; q < QP; ++q) mma_bf16_16816(acc[mt], a0, a1, a2, a3, pb[q][0], pb[q][1]);
                }
            }
            __syncwarp();
            const int next = i + STAGES;
            if (next < mine) {
                if ((next & 31) == 0) { take(); look_up(next / 32 + 1); }
                if (lane == 0) fence_proxy_async();
                issue(next);
            }
        }
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, o);
            l1 += __shfl_xor_sync(0xffffffffu, l1, o);
        }
        // ---- merge the warps' parts, half of the accumulators at a time:
        // warp w adds the 16-dim blocks 2w and 2w + 1 of each half
        if (lane < 4) {
            sm.ml[warp][h0][0] = m0; sm.ml[warp][h0][1] = l0;
            sm.ml[warp][h0 + 1][0] = m1; sm.ml[warp][h0 + 1][1] = l1;
        }
        const bool first = t == u0, whole = first && end == u1;
        const int slot = 2 * cta + (first ? 1 : 0);
        float f0[PD_WARPS], f1[PD_WARPS], L0 = 0.f, L1 = 0.f, M0 = -INFINITY, M1 = -INFINITY;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
                const float (&a)[4] = acc[half * 8 + mt];
                sm.merge[warp][mt][lane] = make_float4(a[0], a[1], a[2], a[3]);
            }
            __syncthreads();
            if (half == 0) {
#pragma unroll
                for (int w = 0; w < PD_WARPS; ++w) { M0 = fmaxf(M0, sm.ml[w][h0][0]); M1 = fmaxf(M1, sm.ml[w][h0 + 1][0]); }
#pragma unroll
                for (int w = 0; w < PD_WARPS; ++w) {
                    const float a = sm.ml[w][h0][0], b = sm.ml[w][h0 + 1][0];
                    f0[w] = a == -INFINITY ? 0.f : exp2f(a - M0);
                    f1[w] = b == -INFINITY ? 0.f : exp2f(b - M1);
                    L0 += sm.ml[w][h0][1] * f0[w];
                    L1 += sm.ml[w][h0 + 1][1] * f1[w];
                }
                if (!whole && warp == 0 && lane < 4) {
                    float2 *ml = part.ml + (size_t)slot * GQA_GRP + h0;
                    ml[0] = make_float2(M0, L0);
                    ml[1] = make_float2(M1, L1);
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < PD_WARPS; ++w) {
                    const float4 a = sm.merge[w][2 * warp + u][lane];
                    o.x += a.x * f0[w]; o.y += a.y * f1[w]; o.z += a.z * f0[w]; o.w += a.w * f1[w];
                }
                const int d = (half * 8 + 2 * warp + u) * 16 + dr;
                if (whole) {
                    TI *out = static_cast<TI *>(p.ctx) + ((size_t)r * p.H + kh * G + h0) * GQA_HD + d;
                    const TI *g = sm.gate + h0 * GQA_HD + d;
                    if (h0 < G) {
                        out[0] = from_f32<TI>(o.x / L0 * sigmoidf_(to_f32(g[0])));
                        out[8] = from_f32<TI>(o.z / L0 * sigmoidf_(to_f32(g[8])));
                    }
                    if (h0 + 1 < G) {
                        out[GQA_HD] = from_f32<TI>(o.y / L1 * sigmoidf_(to_f32(g[GQA_HD])));
                        out[GQA_HD + 8] = from_f32<TI>(o.w / L1 * sigmoidf_(to_f32(g[GQA_HD + 8])));
                    }
                } else {
                    float *out = part.o + ((size_t)slot * GQA_GRP + h0) * GQA_HD + d;
                    out[0] = o.x; out[8] = o.z;
                    out[GQA_HD] = o.y; out[GQA_HD + 8] = o.w;
                }
            }
            __syncthreads();                // the area, q and the gate are written again
        }
        if (first && !whole) join_to = (u1 - 1) / per;
        t = end;
        if (t < c1) { r = nr; kh = nkh; }
    }
    // the unit that begins in this CTA and goes on: its pieces are this CTA's last and the firsts of cta + 1 .. join_to
    if (tid == 0) part.units[cta] = make_int4(join_to, r, kh, 0);
}

// One CTA per (first CTA of a split unit, query head): merges the unit's
// pieces. Warp w takes pieces w, w + 8, .. with a running maximum, lane = 8
// dims; then thread d merges the warps' results of dim d.
template <typename TI>
__global__ void __launch_bounds__(GQA_HD)
pages_join_kernel(GqaPagesArgs p, PagesPart part)
{
    constexpr int W = GQA_HD / 32;
    __shared__ float sm_ml[W][2];
    __shared__ __align__(16) float sm_o[W][GQA_HD];
    const int a = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();                         // a programmatic dependent of the decode kernel
    const int4 unit = part.units[a];
    if (unit.x < 0) return;
    const int n = unit.x - a + 1, G = p.H / p.pv.KH, head = unit.z * G + h;
    const size_t row = (size_t)unit.y * p.H + head;
    const float gate = to_f32(static_cast<const TI *>(p.qg)[row * 2 * GQA_HD + GQA_HD + tid]);
    float m = -INFINITY, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    constexpr int U = 4;                    // pieces whose loads a warp issues together
    for (int s0 = warp; s0 < n; s0 += U * W) {
        float2 ml[U];
        float4 x[U], y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * W;
            ml[u] = make_float2(-INFINITY, 0.f);
            if (s < n) {
                const size_t at = (size_t)(s ? 2 * (a + s) : 2 * a + 1) * GQA_GRP + h;
                ml[u] = part.ml[at];
                x[u] = *reinterpret_cast<const float4 *>(part.o + at * GQA_HD + 8 * lane);
                y[u] = *reinterpret_cast<const float4 *>(part.o + at * GQA_HD + 8 * lane + 4);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (ml[u].x == -INFINITY) continue;
            const float mn = fmaxf(m, ml[u].x);
            const float fo = m == -INFINITY ? 0.f : exp2f(m - mn), fs = exp2f(ml[u].x - mn);
            const float v[8] = {x[u].x, x[u].y, x[u].z, x[u].w, y[u].x, y[u].y, y[u].z, y[u].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = o[e] * fo + v[e] * fs;
            l = l * fo + ml[u].y * fs;
            m = mn;
        }
    }
    if (lane == 0) { sm_ml[warp][0] = m; sm_ml[warp][1] = l; }
    *reinterpret_cast<float4 *>(&sm_o[warp][8 * lane]) = make_float4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<float4 *>(&sm_o[warp][8 * lane + 4]) = make_float4(o[4], o[5], o[6], o[7]);
    __syncthreads();
    float M = -INFINITY, O = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm_ml[w][0]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float f = sm_ml[w][0] == -INFINITY ? 0.f : exp2f(sm_ml[w][0] - M);
        O += sm_o[w][tid] * f;
        L += sm_ml[w][1] * f;
    }
    static_cast<TI *>(p.ctx)[row * GQA_HD + tid] = from_f32<TI>(O / L * sigmoidf_(gate));
}

template <typename TI>
static cudaError_t pages_decode_run(const CUtensorMap &tk, const CUtensorMap &tv, const GqaPagesArgs &a, const PagesPart &part,
                                    const RopeFreq &f, int ctas, cudaStream_t st)
{
    const int smem = (int)sizeof(PdSmem<TI>) + 1024;
    static_assert(sizeof(PdSmem<TI>) + 1024 <= 232448, "decode shared memory exceeds the 227 KiB per-CTA limit");
    cudaError_t e = cudaFuncSetAttribute(pages_decode_kernel<TI>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    pages_decode_kernel<TI><<<ctas, PD_THREADS, smem, st>>>(tk, tv, a, part, f);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, a.H / a.pv.KH); cfg.blockDim = dim3(GQA_HD); cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, pages_join_kernel<TI>, a, part);
}

cudaError_t launch_pages_decode(const CUtensorMap &tk, const CUtensorMap &tv, const GqaPagesArgs &a, const PagesPart &part,
                                const RopeFreq &f, int in_bf16, int ctas, cudaStream_t st)
{
    return in_bf16 ? pages_decode_run<__nv_bfloat16>(tk, tv, a, part, f, ctas, st)
                   : pages_decode_run<float>(tk, tv, a, part, f, ctas, st);
}

// ------------------------------------------------------------------ append
// A warp per (row, KV head), lane = 8 dims: k normed and roped, v as it is,
// both rounded to bf16, the cache's type.
template <typename TI>
__global__ void __launch_bounds__(128)
pages_append_kernel(GqaPagesArgs p, const __grid_constant__ RopeFreq f)
{
    __shared__ __align__(16) float cs[4][GQA_HD / 2], sn[4][GQA_HD / 2];
    __shared__ float vec[4][GQA_HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int row0, pos0;
    if (blockIdx.x == 0)                     // what no row belongs to is looked over here
        for (int i = threadIdx.x; i < p.n_req; i += 128) pages_rows_of(p, i, row0, pos0);
    const int row = blockIdx.x, r = pages_req_of(p, row);
    if (r < 0) return;
    const int n = pages_rows_of(p, r, row0, pos0);
    if (n == 0) return;
    const int pos = pos0 + row - row0;
    pages_rope_table(cs[warp], sn[warp], pos, p.rot, f, lane, 32);
    __syncwarp();
    for (int kh = warp; kh < p.pv.KH; kh += 4) {
        const long long at = pages_row(p.pv, r, kh, pos);
        if (at < 0) continue;
        const size_t in = ((size_t)row * p.pv.KH + kh) * GQA_HD + lane * 8;
        float x[8], w[8], y[8], v[8];
        load8<TI>(static_cast<const TI *>(p.k) + in, x);
        load8<TI>(static_cast<const TI *>(p.v) + in, v);
        load8<float>(p.knw + lane * 8, w);
        gqa_norm_rope(y, x, w, p.eps, p.rot, cs[warp], sn[warp], vec[warp], lane);
        store8(p.pv.k + at * GQA_HD + lane * 8, y);
        store8(p.pv.v + at * GQA_HD + lane * 8, v);
    }
}

// ------------------------------------------------------------------ attention
// A warp per (row, query head), lane = 8 dims, one key at a time with a
// running maximum and sum; fp32 throughout.
template <typename TI>
__global__ void __launch_bounds__(128)
pages_attend_kernel(GqaPagesArgs p, const __grid_constant__ RopeFreq f)
{
    __shared__ __align__(16) float cs[4][GQA_HD / 2], sn[4][GQA_HD / 2];
    __shared__ float vec[4][GQA_HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x, h = blockIdx.y * 4 + warp, r = pages_req_of(p, row);
    if (r < 0 || h >= p.H) return;
    int row0, pos0;
    const int n = pages_rows_of(p, r, row0, pos0);
    if (n == 0) return;
    const int pos = pos0 + row - row0, kh = h / (p.H / p.pv.KH);
    pages_rope_table(cs[warp], sn[warp], pos, p.rot, f, lane, 32);
    __syncwarp();
    const TI *qg = static_cast<const TI *>(p.qg) + ((size_t)row * p.H + h) * 2 * GQA_HD + lane * 8;
    float x[8], w[8], q[8], g[8], o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    load8<TI>(qg, x);
    load8<TI>(qg + GQA_HD, g);
    load8<float>(p.qnw + lane * 8, w);
    gqa_norm_rope(q, x, w, p.eps, p.rot, cs[warp], sn[warp], vec[warp], lane);
    float m = -INFINITY, l = 0.f;
    for (int t = 0; t <= pos; ++t) {
        const long long at = pages_row(p.pv, r, kh, t);
        if (at < 0) continue;
        float kk[8], vv[8], s = 0.f;
        load8<__nv_bfloat16>(p.pv.k + at * GQA_HD + lane * 8, kk);
        load8<__nv_bfloat16>(p.pv.v + at * GQA_HD + lane * 8, vv);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(q[i], kk[i], s);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= p.scale_log2;
        const float mn = fmaxf(m, s), al = exp2f(m - mn), e = exp2f(s - mn);
        l = l * al + e;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = o[i] * al + e * vv[i];
        m = mn;
    }
    TI *out = static_cast<TI *>(p.ctx) + ((size_t)row * p.H + h) * GQA_HD + lane * 8;
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = from_f32<TI>(o[i] * inv * sigmoidf_(g[i]));
}

cudaError_t launch_pages_append(const GqaPagesArgs &a, const RopeFreq &f, int in_bf16, cudaStream_t st)
{
    if (in_bf16) pages_append_kernel<__nv_bfloat16><<<a.S, 128, 0, st>>>(a, f);
    else pages_append_kernel<float><<<a.S, 128, 0, st>>>(a, f);
    return cudaGetLastError();
}
cudaError_t launch_pages_attend(const GqaPagesArgs &a, const RopeFreq &f, int in_bf16, cudaStream_t st)
{
    const dim3 grid(a.S, (a.H + 3) / 4);
    if (in_bf16) pages_attend_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a, f);
    else pages_attend_kernel<float><<<grid, 128, 0, st>>>(a, f);
    return cudaGetLastError();
}

}  // namespace coli
