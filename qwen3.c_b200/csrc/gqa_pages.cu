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

// Angle table of position pos, entries [0, rot / 2): the angle in turns is the
// fraction of an exact 64-bit product, so far positions lose nothing.
__device__ __forceinline__ void pages_rope_table(float *cs, float *sn, int pos, int rot, const unsigned long long *turn,
                                                 int tid0, int nthr)
{
    for (int j = tid0; j < (rot >> 1); j += nthr) {
        const int top = (int)(((unsigned long long)pos * turn[j]) >> 32);      // 2^-32 turns, [-1/2, 1/2)
        sincospif((float)top * 4.656612873077393e-10f, &sn[j], &cs[j]);        // 2^-31: in half turns
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
// Units are (request, KV head) pairs, in that order. A unit is a run of ring
// entries: its q rows, its 16-token tiles, its gate rows; the list of all
// entries is cut into equal consecutive ranges, one per warp of the grid (4
// warps per CTA, one CTA per SM): batches of any lengths keep every SM
// streaming to the end, and one long request is spread over all of them.
//
// A warp works on its own. Everything it reads comes through its own 3-stage
// ring of 16 KiB (mbarrier completion), which runs on across units, so that no
// unit waits for its own loads: tiles as one TMA box of K and one of V, q and
// gate rows as bulk copies. 32 entries are looked up at once by the 32 lanes, a
// batch ahead of their use. The warp norms and ropes q, and writes the ctx of
// a unit that it holds whole. What warps of one CTA share of a unit is merged
// in shared memory when the ranges are done; what CTAs share goes through the
// workspace to pages_join_kernel: at most two pieces per CTA, whatever the
// batch.
//
// Per tile S^T[16 tok x 8 heads] = K Q^T and O^T += V^T P^T on bf16 mma.sync,
// the (up to) 8 query heads of the KV head being the N of the MMA: 8 FLOP per
// byte read, so HBM bounds it, and tcgen05's 64-row minimum would leave 7/8 of
// its rows empty. The tensor pipe has room to spare, so q and the softmax
// numerators are not rounded to one bf16 but enter as PARTS of them (hi + lo,
// 16 bits, for bf16 activations; three parts, 24 bits, for fp32 ones), one MMA
// for each.
//
// The new token's K and V rows are normed, roped and appended by the warp that
// owns the unit's last tile: to the page, and over the tile's copy in shared
// memory, so no tile load waits for an append.
//
// Short calls are bound by latency, instruction fetch a large part of it: what
// runs once per unit is kept in rolled loops over heads.
constexpr int PD_WARPS = 4, PD_THREADS = 32 * PD_WARPS, PD_STAGES = 3, PD_STAGE = 2 * GQA_TILE_BYTES;
constexpr int PD_OROW = 132;                 // floats between heads of O: 8 banks apart for the writers' heads
template <typename TI> struct PdEntry {      // layout of the q entry and of the gate entry in a stage
    static constexpr bool F32 = sizeof(TI) == 4;
    static constexpr int BYTES = GQA_HD * (int)sizeof(TI);    // a head's q (or gate), the new k, the new v
    static constexpr int ROW = BYTES + 8 * (int)sizeof(TI);   // apart: no bank conflicts between a quad's and the next head's reads
    static constexpr int KV = GQA_GRP * ROW;
    // the roped dims times 1 + w, fp32, in rows of YROW: behind the raw rows, or in their place
    static constexpr int Y = F32 ? 0 : (GQA_GRP + 2) * ROW, YROW = F32 ? ROW / 4 : 264;
    static constexpr int O = GQA_GRP * ROW;                   // gate entry: half of O, fp32, behind the gate rows
    static_assert((GQA_GRP + 2) * ROW <= PD_STAGE && Y + (GQA_GRP + 1) * YROW * 4 <= PD_STAGE && O + GQA_GRP * PD_OROW * 4 <= PD_STAGE && ROW % 16 == 0, "");
};
struct PdSmem {
    uint8_t ring[PD_WARPS][PD_STAGES][PD_STAGE];
    float w1[2][GQA_HD];                    // 1 + q / k norm weights
    float cs[PD_WARPS][GQA_HD / 2], sn[PD_WARPS][GQA_HD / 2];
    unsigned long long turn[GQA_HD / 2];
    float2 ml[PD_WARPS][2][GQA_GRP];        // (max, sum) of a warp's continued / opened piece
    int4 cont[PD_WARPS], open[PD_WARPS];    // (there: 1, and ends here: 2; request; KV head; parked / last CTA)
    int pre[1024 + 4];                      // entries (of one KV head) before each request
    int part[PD_WARPS];
    uint64_t full[PD_WARPS][PD_STAGES];
};
static_assert(sizeof(PdSmem) + 1024 <= 232448, "decode shared memory exceeds the 227 KiB per-CTA limit");

__device__ __forceinline__ void load4(const __nv_bfloat16 *p, float (&x)[4])
{
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u.x));
    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u.y));
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}
__device__ __forceinline__ void load4(const float *p, float (&x)[4])
{
    const float4 a = *reinterpret_cast<const float4 *>(p);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float (&x)[4])
{
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}
__device__ __forceinline__ void store4(float *p, const float (&x)[4])
{
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
// (x, y) as PARTS bf16 pairs whose sum is (x, y) to 8 PARTS bits
template <int PARTS>
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t (&out)[PARTS])
{
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        out[i] = pack_bf16(x, y);
        x -= __uint_as_float(out[i] << 16);
        y -= __uint_as_float(out[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ float2 pair_of(const __nv_bfloat16 *p)
{
    const uint32_t u = *reinterpret_cast<const uint32_t *>(p);
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 pair_of(const float *p) { return *reinterpret_cast<const float2 *>(p); }

template <typename TI>
__global__ void __launch_bounds__(PD_THREADS, 1)
pages_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, GqaPagesArgs p,
                    PagesPart part, const __grid_constant__ RopeFreq f)
{
    using E = PdEntry<TI>;
    constexpr int PARTS = E::F32 ? 3 : 2;
    extern __shared__ uint8_t smem_raw[];
    PdSmem &sm = *reinterpret_cast<PdSmem *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
    const int KH = p.pv.KH, G = p.H / KH, page = p.pv.page;
    griddep_launch();                       // the join may be scheduled; it waits for this grid
    if (lane == 0) {
        for (int s = 0; s < PD_STAGES; ++s) mbar_init(&sm.full[warp][s], 1);
        fence_mbar_init();
        sm.cont[warp] = sm.open[warp] = make_int4(0, 0, 0, 0);
    }
    if (tid == 0) { tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV); }

    // entries before each request: its tiles, a q and a gate entry
    {
        const int each = (p.n_req + PD_THREADS - 1) / PD_THREADS, r0 = min(p.n_req, tid * each), r1 = min(p.n_req, r0 + each);
        auto entries = [&](int r) {
            int row0, pos0;
            return pages_rows_of(p, r, row0, pos0) ? pos0 / GQA_TILE + 3 : 0;
        };
        int mine = 0;
#pragma unroll 1
        for (int r = r0; r < r1; ++r) mine += entries(r);
        if (tid < p.rot / 2) sm.turn[tid] = f.turn[tid];
        for (int j = tid; j < 2 * GQA_HD; j += PD_THREADS) sm.w1[0][j] = 1.f + p.qnw[j];   // knw follows qnw
        int inc = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += y;
        }
        if (lane == 31) sm.part[warp] = inc;
        __syncthreads();
        int at = inc - mine;
        for (int w = 0; w < warp; ++w) at += sm.part[w];
#pragma unroll 1
        for (int r = r0; r < r1; ++r) { sm.pre[r] = at; at += entries(r); }
        if (tid == PD_THREADS - 1) sm.pre[p.n_req] = at;
        __syncthreads();
    }
    const int total = sm.pre[p.n_req] * KH, workers = gridDim.x * PD_WARPS;
    const int per = max(1, (total + workers - 1) / workers);
    const int v0 = min(total, (cta * PD_WARPS + warp) * per), v1 = min(total, v0 + per);
    // request of entry v: the last r with pre[r] * KH <= v
    auto find = [&](int v) {
        int lo = 0, hi = p.n_req - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (sm.pre[mid] * KH <= v) lo = mid; else hi = mid - 1;
        }
        return lo;
    };

    // ---- the ring: what the warp reads for entries v0 .. v1 - 1. A piece that
    // starts inside a unit needs the q rows too (as entry v0 - 1), and a unit
    // whose tiles are all here the gate rows, though its last entry is the
    // next range's (as entry v1).
    int ahead = -1, ahead_id = 0, ahead_row = 0, what = 0, base_v = v0 - 1, issued = 0;   // ahead: -1 none, 0 tile, 1 q, 2 gate
    uint32_t todo = 0;
    auto look_up = [&](int base) {
        const int v = base + lane, at = min(max(v, v0), v1 - 1);
        ahead = -1;
        if (v > v1 || v0 >= v1) return;
        const int r = find(at), n = sm.pre[r + 1] - sm.pre[r], rel0 = at - sm.pre[r] * KH;
        int kh = (int)__fdividef((float)rel0, (float)n);        // at most KH <= 64: off by one at most
        kh -= kh * n > rel0;
        kh += (kh + 1) * n <= rel0;
        const int rel = rel0 - kh * n, nt = n - 2;
        const bool begins = at - rel + 1 >= v0;                 // the unit's first tile is in the range
        if (v < v0) ahead = rel >= 1 && rel <= nt ? 1 : -1;
        else if (v == v1) ahead = rel == nt && begins ? 2 : -1;
        else if (rel == 0) ahead = v + 1 < v1 ? 1 : -1;
        else if (rel <= nt) ahead = 0;
        else ahead = begins ? 2 : -1;
        ahead_row = r * KH + kh;
        if (ahead == 0) {
            const int pi = p.pv.tiles_div(rel - 1);
            ahead_id = p.pv.table[(size_t)r * p.pv.max_pages + pi];
            ahead_row = kh * page + (rel - 1) * GQA_TILE - pi * page;
        }
    };
    auto take = [&]() {                     // the batch looked up becomes the one in use
        if (ahead == 0 && (unsigned)ahead_id >= (unsigned)p.pv.n_pages) { pages_error(PAGES_BAD_ID); ahead_id = 0; }
        what = ahead == 0 ? (int)(((long long)ahead_id * KH * page + ahead_row) >> 3) : -1 - (2 * ahead_row + (ahead & 1));
        todo = __ballot_sync(0xffffffffu, ahead >= 0);
    };
    auto issue_next = [&]() {               // whole warp: the next entry into the next stage
        while (todo == 0) {
            if (base_v > v1 + 32) return;
            take();
            look_up(base_v);
            base_v += 32;
        }
        const int e = __shfl_sync(0xffffffffu, what, __ffs(todo) - 1), s = issued % PD_STAGES;
        todo &= todo - 1;
        ++issued;
        uint8_t *to = sm.ring[warp][s];
        uint64_t *bar = &sm.full[warp][s];
        if (e >= 0) {
            if (lane == 0) {
                mbar_expect_tx(bar, PD_STAGE);
                tma_load_4d(to, &tmK, 0, 0, 0, e, bar);
                tma_load_4d(to + GQA_TILE_BYTES, &tmV, 0, 0, 0, e, bar);
            }
        } else {                            // rows of unit `u`, a bulk copy per lane
            const int u = (-1 - e) >> 1, is_q = (-1 - e) & 1, r = p.pv.heads_div(u), n = is_q ? G + 2 : G;
            if (lane == 0) mbar_expect_tx(bar, n * E::BYTES);
            __syncwarp();
            const TI *from = static_cast<const TI *>(p.qg) + ((size_t)r * p.H + (u - r * KH) * G + lane) * 2 * GQA_HD + (is_q ? 0 : GQA_HD);
            if (lane == G) from = static_cast<const TI *>(p.k) + (size_t)u * GQA_HD;
            if (lane == G + 1) from = static_cast<const TI *>(p.v) + (size_t)u * GQA_HD;
            if (lane < n) bulk_load(to + (lane < G ? lane * E::ROW : E::KV + (lane - G) * E::ROW), from, E::BYTES, bar);
        }
    };
    // ---- entry by entry; each leaves its stage to the one PD_STAGES behind it
    float *cs = sm.cs[warp], *sn = sm.sn[warp];
    const int r8 = lane & 7, mi = lane >> 3, h0 = (lane & 3) * 2, dr = lane >> 2;
    const float sl2 = p.scale_log2;
    // the unit in work: request, KV head, position, tiles, the tiles of this piece
    int r = 0, kh = 0, pos = -1, nt = 0, u0 = 0, tile = 0, end_tile = 0, next_v = v0, next_r = 0, next_kh = 0;
    bool begins = false, ends = false;
    uint32_t qf[PARTS][16][2];              // q as the B operand: head lane / 4, dims 16kk + 2 (lane % 4) + {0, 1, 8, 9}
    uint4 new_k = make_uint4(0, 0, 0, 0);   // the row to append, bf16
    uint4 new_vb = make_uint4(0, 0, 0, 0);
    float acc[16][4], m0 = 0.f, m1 = 0.f, l0 = 0.f, l1 = 0.f;
    if (v0 < v1) {
        next_r = find(v0);
        next_kh = (v0 - sm.pre[next_r] * KH) / (sm.pre[next_r + 1] - sm.pre[next_r]);
    }
    enum { AT_Q, AT_TILE, AT_GATE } at = AT_Q;
#pragma unroll 1
    for (int i = -PD_STAGES;; ++i) {
        if (i >= 0) {
            if (at == AT_Q) {
                // ---- the next unit with tiles in the range
                for (;;) {
                    if (next_v >= v1) break;
                    r = next_r; kh = next_kh;
                    const int n = sm.pre[r + 1] - sm.pre[r];
                    nt = n - 2;
                    u0 = sm.pre[r] * KH + kh * n;
                    tile = max(next_v - u0 - 1, 0);
                    end_tile = min(v1 - u0 - 1, nt);
                    next_v = min(v1, u0 + n);
                    if (++next_kh == KH) {
                        next_kh = 0;
                        for (++next_r; next_r < p.n_req && sm.pre[next_r + 1] == sm.pre[next_r];) ++next_r;
                    }
                    if (tile < end_tile) break;
                    tile = end_tile = 0;
                }
                if (tile >= end_tile) break;
            }
            const int s = i % PD_STAGES;
            mbar_wait(&sm.full[warp][s], (i / PD_STAGES) & 1);   // a time-out raises the error word; the rest runs on what is there
            uint8_t *st = sm.ring[warp][s];
            if (at == AT_Q) {
                begins = tile == 0;
                ends = end_tile == nt;
                if (pos != p.base[r]) {
                    pos = p.base[r];
                    pages_rope_table(cs, sn, pos, p.rot, sm.turn, lane, 32);
                }
                __syncwarp();
                // rs: the norm's factor of a row, which the rotation commutes with; lanes 4h .. 4h + 3
                // hold the quarters of head h's fragments, and all 32 lanes 8 dims each of the new k
                const int h = lane >> 2, d0 = 2 * (lane & 3), half = p.rot >> 1;
                const TI *x = reinterpret_cast<const TI *>(st + min(h, G - 1) * E::ROW);
                const TI *xk = reinterpret_cast<const TI *>(st + E::KV);
                float s0 = 0.f, s1 = 0.f, sk = 0.f, k[8], val[8];
#pragma unroll
                for (int kk = 0; kk < 16; ++kk) {
                    const float2 a = pair_of(x + 16 * kk + d0), b = pair_of(x + 16 * kk + 8 + d0);
                    s0 += a.x * a.x + a.y * a.y;
                    s1 += b.x * b.x + b.y * b.y;
                }
                load8<TI>(xk + lane * 8, k);
                load8<TI>(reinterpret_cast<const TI *>(st + E::KV + E::ROW) + lane * 8, val);
#pragma unroll
                for (int e = 0; e < 8; ++e) sk += k[e] * k[e];
                s0 += s1;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    if (o < 4) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
                    sk += __shfl_xor_sync(0xffffffffu, sk, o);
                }
                const float rs = h < G ? 1.f / sqrtf(s0 / GQA_HD + p.eps) : 0.f;    // heads past the group's: q = 0
                const float rk = 1.f / sqrtf(sk / GQA_HD + p.eps);
                __syncwarp();               // (fp32: the roped dims take the place of what has been read)
                float *y = reinterpret_cast<float *>(st + E::Y);
                for (int j = lane; j < half; j += 32) {
                    const float c = cs[j], sv = sn[j];
#pragma unroll 3
                    for (int row = 0; row < GQA_GRP + 1; ++row) {               // the heads, then k
                        const TI *in = reinterpret_cast<const TI *>(st + row * E::ROW);
                        const float *w = sm.w1[row == GQA_GRP];
                        const float a = to_f32(in[j]) * w[j], b = to_f32(in[j + half]) * w[j + half];
                        y[row * E::YROW + j] = a * c - b * sv;
                        y[row * E::YROW + j + half] = b * c + a * sv;
                    }
                }
                __syncwarp();
#pragma unroll
                for (int kk = 0; kk < 16; ++kk)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int d = 16 * kk + 8 * e + d0;
                        float2 v;
                        if (d < p.rot) {
                            v = *reinterpret_cast<const float2 *>(y + h * E::YROW + d);
                        } else {
                            const float2 w = *reinterpret_cast<const float2 *>(&sm.w1[0][d]);
                            v = pair_of(x + d);
                            v.x *= w.x;
                            v.y *= w.y;
                        }
                        uint32_t parts[PARTS];
                        split_bf16<PARTS>(h < G ? v.x * rs : 0.f, h < G ? v.y * rs : 0.f, parts);
#pragma unroll
                        for (int q = 0; q < PARTS; ++q) qf[q][kk][e] = parts[q];
                    }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = lane * 8 + e;
                    k[e] = (d < p.rot ? y[GQA_GRP * E::YROW + d] : k[e] * sm.w1[1][d]) * rk;
                }
                new_k = make_uint4(pack_bf16(k[0], k[1]), pack_bf16(k[2], k[3]), pack_bf16(k[4], k[5]), pack_bf16(k[6], k[7]));
                new_vb = make_uint4(pack_bf16(val[0], val[1]), pack_bf16(val[2], val[3]), pack_bf16(val[4], val[5]), pack_bf16(val[6], val[7]));
#pragma unroll
                for (int mt = 0; mt < 16; ++mt) acc[mt][0] = acc[mt][1] = acc[mt][2] = acc[mt][3] = 0.f;
                m0 = m1 = -INFINITY;
                l0 = l1 = 0.f;
                at = AT_TILE;
            } else if (at == AT_TILE) {
                uint8_t *vt = st + GQA_TILE_BYTES;
                const uint32_t kb = smem_u32(st), vb = kb + GQA_TILE_BYTES;
                const int tok0 = tile * GQA_TILE, valid = min(GQA_TILE, pos + 1 - tok0);
                if (tile == nt - 1) {
                    // position pos: into the page and over the loaded tile (whose row is the page's old contents)
                    const int row = pos - tok0, off = (row >> 3) * 4096 + (lane >> 3) * 1024 + (row & 7) * 128 + (((lane & 7) ^ (row & 7)) << 4);
                    *reinterpret_cast<uint4 *>(st + off) = new_k;
                    *reinterpret_cast<uint4 *>(vt + off) = new_vb;
                    const long long to = pages_row(p.pv, r, kh, pos);
                    if (to >= 0) {
                        *reinterpret_cast<uint4 *>(p.pv.k + to * GQA_HD + lane * 8) = new_k;
                        *reinterpret_cast<uint4 *>(p.pv.v + to * GQA_HD + lane * 8) = new_vb;
                    }
                    // rows past the end are never weighted; cleared so that stale
                    // non-finite cache contents cannot come through as 0 * inf
                    for (int j = lane; j < (GQA_TILE - valid) * 32; j += 32) {
                        const int dead = valid + (j >> 5), c = (j & 31) >> 3, ch = j & 7;
                        *reinterpret_cast<uint4 *>(vt + (dead >> 3) * 4096 + c * 1024 + (dead & 7) * 128 + ch * 16) = make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                }
                // S^T[16 tok x 8 heads] = K[16 x 256] . Q^T[256 x 8]
                // in 2 PARTS independent sums, so that no MMA waits for the one before
                float part_s[2][PARTS][4] = {};
                {
                    const uint32_t base = kb + (mi & 1) * 4096 + r8 * 128;
#pragma unroll
                    for (int kk = 0; kk < 16; ++kk) {
                        const int chunk = (kk & 3) * 2 + (mi >> 1);
                        uint32_t a0, a1, a2, a3;
                        ldsm_x4(base + (kk >> 2) * 1024 + ((chunk ^ r8) << 4), a0, a1, a2, a3);
#pragma unroll
                        for (int q = 0; q < PARTS; ++q) mma_bf16_16816(part_s[kk & 1][q], a0, a1, a2, a3, qf[q][kk][0], qf[q][kk][1]);
                    }
                }
                float sc[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[e] = 0.f;
#pragma unroll
                    for (int q = PARTS - 1; q >= 0; --q) sc[e] += part_s[0][q][e] + part_s[1][q][e];
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
                uint32_t pa[PARTS], pb[PARTS];
                split_bf16<PARTS>(p0, p1, pa);
                split_bf16<PARTS>(p2, p3, pb);
#pragma unroll
                for (int q = 0; q < PARTS; ++q) { pa[q] = movmatrix_t(pa[q]); pb[q] = movmatrix_t(pb[q]); }
                // O^T[256 dims x 8 heads] += V^T[256 x 16 tok] . P^T[16 tok x 8 heads]
                {
                    const uint32_t base = vb + (mi >> 1) * 4096 + r8 * 128;
#pragma unroll
                    for (int mt = 0; mt < 16; ++mt) {
                        const int chunk = (mt & 3) * 2 + (mi & 1);
                        uint32_t a0, a1, a2, a3;
                        ldsm_x4_t(base + (mt >> 2) * 1024 + ((chunk ^ r8) << 4), a0, a1, a2, a3);
#pragma unroll
                        for (int q = PARTS - 1; q >= 0; --q) mma_bf16_16816(acc[mt], a0, a1, a2, a3, pa[q], pb[q]);
                    }
                }
                if (++tile == end_tile) {
#pragma unroll
                    for (int o = 4; o <= 16; o <<= 1) {
                        l0 += __shfl_xor_sync(0xffffffffu, l0, o);
                        l1 += __shfl_xor_sync(0xffffffffu, l1, o);
                    }
                    at = AT_GATE;
                    if (!(begins && ends)) {
                        // ---- a piece: to the CTA's merge below, through shared memory if it is
                        // the range's last (its loads have all landed), else parked in the workspace
                        at = AT_Q;
                        const int kind = begins ? 1 : 0;
                        const bool last = next_v >= v1;
                        if (lane == 0) {
                            if (begins) sm.open[warp] = make_int4(1, r, kh, (u0 + nt) / per / PD_WARPS);
                            else sm.cont[warp] = make_int4(ends ? 3 : 1, r, kh, last ? 0 : 1);
                        }
                        if (lane < 4) { sm.ml[warp][kind][h0] = make_float2(m0, l0); sm.ml[warp][kind][h0 + 1] = make_float2(m1, l1); }
                        float4 *o = last ? reinterpret_cast<float4 *>(sm.ring[warp][0])
                                         : part.park + (size_t)(cta * PD_WARPS + warp) * 512;
                        if (last) __syncwarp();       // this stage may be the one: other lanes have read it
#pragma unroll
                        for (int mt = 0; mt < 16; ++mt) o[mt * 32 + lane] = make_float4(acc[mt][0], acc[mt][1], acc[mt][2], acc[mt][3]);
                    }
                }
            } else {
                // ---- the whole unit: ctx = O / l * sigmoid(gate), turned to rows behind the gate rows, half the dims at a time
                const float i0 = 1.f / l0, i1 = 1.f / l1;
                float *o_ = reinterpret_cast<float *>(st + E::O);
                const uint8_t *gate = st + 4 * lane * sizeof(TI);
                TI *out = static_cast<TI *>(p.ctx) + ((size_t)r * p.H + kh * G) * GQA_HD + 4 * lane;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int mt = 0; mt < 8; ++mt) {
                        const float (&a)[4] = acc[half * 8 + mt];
                        float *o = o_ + h0 * PD_OROW + mt * 16 + dr;
                        o[0] = a[0] * i0; o[PD_OROW] = a[1] * i1; o[8] = a[2] * i0; o[PD_OROW + 8] = a[3] * i1;
                    }
                    __syncwarp();
#pragma unroll 4
                    for (int h = 0; h < GQA_GRP; ++h) {
                        float o[4], g[4];
                        load4(reinterpret_cast<const TI *>(gate + h * E::ROW) + half * 128, g);
                        load4(o_ + h * PD_OROW + 4 * lane, o);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] *= sigmoidf_(g[e]);
                        if (h < G) store4(out + (size_t)h * GQA_HD + half * 128, o);
                    }
                    __syncwarp();
                }
                at = AT_Q;
            }
            __syncwarp();
            fence_proxy_async();
        }
        issue_next();
    }
    // ---- the runs of pieces of one unit, added up by the whole CTA
    __syncthreads();
    int from = 0, n = 0;                    // the run: n pieces, warp `from`'s first
    bool opened = false;                    // .. which was opened there
    int4 unit = make_int4(-1, 0, 0, -1);
#pragma unroll 1
    for (int step = 0; step < 2 * PD_WARPS + 1; ++step) {
        const int w = step >> 1;
        bool whole = false;
        if (step == 2 * PD_WARPS) {         // what goes on in the next CTA
            if (n == 0) break;
        } else if (step & 1) {
            if (sm.open[w].x) { from = w; n = 1; opened = true; unit = sm.open[w]; }
            continue;
        } else {
            const int4 c = sm.cont[w];
            if (!c.x) continue;
            if (n++ == 0) from = w;
            if (!(c.x & 2)) continue;
            whole = opened;
        }
        // pieces: warps from .. from + n - 1, none of those between empty
        float f0[PD_WARPS], f1[PD_WARPS], M0 = -INFINITY, M1 = -INFINITY, L0 = 0.f, L1 = 0.f;
#pragma unroll
        for (int j = 0; j < PD_WARPS; ++j) {
            if (j >= n) continue;
            M0 = fmaxf(M0, sm.ml[from + j][opened && j == 0][h0].x);
            M1 = fmaxf(M1, sm.ml[from + j][opened && j == 0][h0 + 1].x);
        }
#pragma unroll
        for (int j = 0; j < PD_WARPS; ++j) {
            f0[j] = f1[j] = 0.f;
            if (j >= n) continue;
            const float2 a = sm.ml[from + j][opened && j == 0][h0], b = sm.ml[from + j][opened && j == 0][h0 + 1];
            f0[j] = a.x == -INFINITY ? 0.f : exp2f(a.x - M0);
            f1[j] = b.x == -INFINITY ? 0.f : exp2f(b.x - M1);
            L0 += a.y * f0[j];
            L1 += b.y * f1[j];
        }
        const int slot = 2 * cta + (opened ? 1 : 0);
        const float i0 = 1.f / L0, i1 = 1.f / L1;
        if (!whole && warp == 0 && lane < 4) {
            float2 *ml = part.ml + (size_t)slot * GQA_GRP + h0;
            ml[0] = make_float2(M0, L0);
            ml[1] = make_float2(M1, L1);
        }
#pragma unroll
        for (int u = 0; u < 16 / PD_WARPS; ++u) {
            const int mt = warp + PD_WARPS * u, d = mt * 16 + dr;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < PD_WARPS; ++j) {
                if (j >= n) continue;
                const bool parked = !(opened && j == 0) && sm.cont[from + j].w;
                const float4 a = parked ? part.park[(size_t)(cta * PD_WARPS + from + j) * 512 + mt * 32 + lane]
                                        : reinterpret_cast<const float4 *>(sm.ring[from + j][0])[mt * 32 + lane];
                o.x += a.x * f0[j]; o.y += a.y * f1[j]; o.z += a.z * f0[j]; o.w += a.w * f1[j];
            }
            if (whole) {
                const size_t row = (size_t)unit.y * p.H + unit.z * G + h0;
                TI *out = static_cast<TI *>(p.ctx) + row * GQA_HD + d;
                const TI *g = static_cast<const TI *>(p.qg) + row * 2 * GQA_HD + GQA_HD + d;
                if (h0 < G) {
                    out[0] = from_f32<TI>(o.x * i0 * sigmoidf_(to_f32(g[0])));
                    out[8] = from_f32<TI>(o.z * i0 * sigmoidf_(to_f32(g[8])));
                }
                if (h0 + 1 < G) {
                    out[GQA_HD] = from_f32<TI>(o.y * i1 * sigmoidf_(to_f32(g[2 * GQA_HD])));
                    out[GQA_HD + 8] = from_f32<TI>(o.w * i1 * sigmoidf_(to_f32(g[2 * GQA_HD + 8])));
                }
            } else {
                float *out = part.o + ((size_t)slot * GQA_GRP + h0) * GQA_HD + d;
                out[0] = o.x; out[8] = o.z;
                out[GQA_HD] = o.y; out[GQA_HD + 8] = o.w;
            }
        }
        if (step == 2 * PD_WARPS) break;
        n = 0;
        opened = false;
    }
    // a unit that begins in this CTA and goes on: its pieces are this CTA's last and the firsts of cta + 1 .. unit.w
    if (tid == 0) part.units[cta] = make_int4(n > 0 && opened ? unit.w : -1, unit.y, unit.z, 0);
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
    const int smem = (int)sizeof(PdSmem) + 1024;
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
    pages_rope_table(cs[warp], sn[warp], pos, p.rot, f.turn, lane, 32);
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
    pages_rope_table(cs[warp], sn[warp], pos, p.rot, f.turn, lane, 32);
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
