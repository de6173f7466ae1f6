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
// bad one raises g_dev_errors.pages, is left out, and touches no memory.
#include "common.cuh"
#include "kernels.h"
#include "tc05.cuh"

namespace coli {

// Argument errors found on the device (first one wins, read by every
// coli_cuda_sync, so that replayed graphs report theirs, and cleared there): the
// backend stays usable.
enum { PAGES_OK = 0, PAGES_BAD_ID = 1, PAGES_BAD_POS = 2, PAGES_BAD_ROWS = 3, PAGES_CONFLICT = 4, PAGES_BAD_REQ = 5 };
__device__ __forceinline__ void pages_error(int code) { atomicCAS(&g_dev_errors.pages, 0, code); }

// Angle table of position pos, entries [0, rot / 2): the angle in turns is the
// fraction of an exact 64-bit product, so far positions lose nothing.
__device__ __forceinline__ void pages_rope_entry(float *cs, float *sn, int pos, unsigned long long turn)
{
    const int top = (int)(((unsigned long long)pos * turn) >> 32);             // 2^-32 turns, [-1/2, 1/2)
    sincospif((float)top * 4.656612873077393e-10f, sn, cs);                    // 2^-31: in half turns
}
__device__ __forceinline__ void pages_rope_table(float *cs, float *sn, int pos, int rot, const unsigned long long *turn,
                                                 int tid0, int nthr)
{
    for (int j = tid0; j < (rot >> 1); j += nthr) pages_rope_entry(cs + j, sn + j, pos, turn[j]);
}

// Scalars of these kernels. The IEEE division and square root are long
// branchy sequences (a sigmoid with one took 150 cycles per element, a third of a
// short call); these use the approximate instructions, relative error about
// 2^-22, which neither bf16 nor the fp32 outputs' own sums resolve.
__device__ __forceinline__ float rcp_approx(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float gate_of(float x) { return rcp_approx(1.f + ex2_approx(x * -1.4426950408889634f)); }   // sigmoid
// o *= sigmoid(g) for four elements, e^g / (1 + e^g) with one reciprocal of the
// product of the four 1 + e^g: 5 special-function instructions instead of 8, which
// bound the epilogues. Above 20 a sigmoid is 1 in fp32; held there, the product
// stays below 6e34. A NaN gate is kept out of it, so that it is its own element's only.
__device__ __forceinline__ void gate4(float *o, const float *g)
{
    float e[4], d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        e[i] = ex2_approx(fminf(g[i], 20.f) * 1.4426950408889634f);       // fminf(NaN, 20) = 20
        d[i] = 1.f + e[i];
    }
    const float d01 = d[0] * d[1], d23 = d[2] * d[3], r = rcp_approx(d01 * d23), r01 = r * d23, r23 = r * d01;
    const float s[4] = {e[0] * d[1] * r01, e[1] * d[0] * r01, e[2] * d[3] * r23, e[3] * d[2] * r23};
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= g[i] == g[i] ? s[i] : g[i];
}
// 1 / sqrt(s2 / hd + eps), one Newton step; 0 where s2 is infinite (its row has an infinity)
__device__ __forceinline__ float rms_factor(float s2, float eps)
{
    const float a = fmaf(s2, 1.f / GQA_HD, eps), r = rsqrtf(a);
    return r * fmaf(-0.5f * fminf(a, 3.402823466e38f) * r, r, 1.5f);
}
// Squares are summed in fp32. Where that leaves the type's range (elements of 1e18 and
// more, or, without an eps, below 2^-48), the row's sum is formed once more of up * x, and the
// factor is up / sqrt(sum / hd + up^2 eps): rows of any normal numbers have one.
__device__ __forceinline__ float rms_rescale(float s2, float eps)    // 1: none needed
{
    return !(s2 <= 3.402823466e38f) ? 0x1p-72f : fmaf(s2, 1.f / GQA_HD, eps) < 0x1p-96f ? 0x1p72f : 1.f;
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

// One q or k row in the registers of a warp, lane = 8 dims: x raw in, normed
// and roped out; sums in fp32. w1 is the lane's 1 + w, w the whole row's 1 + w and
// `raw` the raw row (both read only where the rotation's half width is no
// multiple of 8, so that a dim's partner is not one other lane's).
template <typename TI>
__device__ __forceinline__ void pages_norm_rope(float (&x)[8], const float (&w1)[8], float eps, int rot, const float *cs,
                                                const float *sn, const TI *raw, const float *w, int lane)
{
    float s2 = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s2 = fmaf(x[i], x[i], s2);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    const float up = rms_rescale(s2, eps);
    if (__builtin_expect(up != 1.f, 0)) {   // (the same in all lanes)
        s2 = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s2 = fmaf(x[i] * up, x[i] * up, s2);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    }
    const float rs = up * rms_factor(s2, eps * up * up);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= rs * w1[i];
    const int half = rot >> 1, d0 = lane * 8;
    if ((half & 7) == 0) {                  // no branch inside: dims behind rot turn by angle 0
        const int hl = half >> 3, from = lane < hl ? lane + hl : lane - hl, j = d0 < half ? d0 : d0 < rot ? d0 - half : 0;
        const float sign = d0 < half ? -1.f : d0 < rot ? 1.f : 0.f;
        float c[8], sv[8];
        load8<float>(cs + j, c);
        load8<float>(sn + j, sv);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float z = __shfl_sync(0xffffffffu, x[i], from);
            x[i] = x[i] * (d0 < rot ? c[i] : 1.f) + z * (sign * sv[i]);
        }
    } else {
#pragma unroll 1
        for (int d = d0; d < min(d0 + 8, rot); ++d) {
            const bool lo = d < half;
            const int j = lo ? d : d - half, o = lo ? d + half : j;
            const float z = to_f32(raw[o]) * rs * w[o], v = to_f32(raw[d]) * rs * w[d];
            const float t = lo ? v * cs[j] - z * sn[j] : v * cs[j] + z * sn[j];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (d - d0 == i) x[i] = t;
        }
    }
}

// 32 / LANES rows at once, LANES lanes (q = lane % LANES) each: norm and partial
// RoPE of rows in shared memory, in place. A row gives its 8-dim chunk c (load /
// store) and single dims (load1 / store1); chunks go round the row's lanes, and a
// rotated pair of chunks is one lane's, so nothing is overwritten before it is
// read. A row on all 32 lanes takes 13 shuffles in a chain, 850 cycles; eight rows
// on four lanes each take about 2000 together. Rolled loops: code that runs once is
// bound by instruction fetch.
template <int LANES, typename Row>
__device__ __forceinline__ void pages_norm_rope_rows(const Row &row, int q, const float *w1, float eps, int rot, const float *cs,
                                                     const float *sn)
{
    float s0 = 0.f, s1 = 0.f;
#pragma unroll 2
    for (int k = 0; k < GQA_HD / 8 / LANES; ++k) {
        float x[8];
        row.load(LANES * k + q, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) { s0 = fmaf(x[i], x[i], s0); s1 = fmaf(x[4 + i], x[4 + i], s1); }
    }
    s0 += s1;
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
    const float up = rms_rescale(s0, eps);
    if (__builtin_expect(__any_sync(0xffffffffu, up != 1.f), 0)) {
        s0 = 0.f;
#pragma unroll 1
        for (int k = 0; k < GQA_HD / LANES; ++k) {
            const float x = row.load1(LANES * k + q) * up;
            s0 = fmaf(x, x, s0);
        }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) s0 += __shfl_xor_sync(0xffffffffu, s0, o);
    }
    const float rs = up * rms_factor(s0, eps * up * up);
    __syncwarp();
    const int half = rot >> 1;
    if ((half & 7) == 0) {
        const int hc = half >> 3;
#pragma unroll 1
        for (int c = q; c < hc; c += LANES) {
            float a[8], b[8], wa[8], wb[8], co[8], si[8];
            row.load(c, a);
            row.load(c + hc, b);
            load8<float>(w1 + 8 * c, wa);
            load8<float>(w1 + 8 * (c + hc), wb);
            load8<float>(cs + 8 * c, co);
            load8<float>(sn + 8 * c, si);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = a[i] * rs * wa[i], y = b[i] * rs * wb[i];   // the factor first: a * wa can overflow
                a[i] = x * co[i] - y * si[i];
                b[i] = y * co[i] + x * si[i];
            }
            row.store(c, a);
            row.store(c + hc, b);
        }
#pragma unroll 1
        for (int c = (rot >> 3) + q; c < GQA_HD / 8; c += LANES) {
            float a[8], wa[8];
            row.load(c, a);
            load8<float>(w1 + 8 * c, wa);
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = a[i] * rs * wa[i];
            row.store(c, a);
        }
    } else {
#pragma unroll 1
        for (int j = q; j < half; j += LANES) {
            const float x = row.load1(j) * rs * w1[j], y = row.load1(j + half) * rs * w1[j + half];
            row.store1(j, x * cs[j] - y * sn[j]);
            row.store1(j + half, y * cs[j] + x * sn[j]);
        }
#pragma unroll 1
        for (int d = rot + q; d < GQA_HD; d += LANES) row.store1(d, row.load1(d) * rs * w1[d]);
    }
    __syncwarp();
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
// unit waits for its own loads: a tile's K and V as one TMA box, q and gate rows
// as bulk copies. 32 entries are looked up at once by the 32 lanes, a
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
// numerators are not rounded to one bf16 but enter as PARTS of them (two, good to
// 2^-16, for bf16 activations; three, all 24 bits, for fp32 ones), one MMA
// for each.
//
// The new token's K and V rows are normed, roped and appended by the warp that
// owns the unit's last tile: to the page, and over the tile's copy in shared
// memory, so no tile load waits for an append.
//
// Short calls are bound by latency, instruction fetch a large part of it: what
// runs once per unit is kept in rolled loops over heads.
//
// Measured with the join (H / KH = 8, KH = 2 unless said): 64 requests at 32k tokens,
// 4.25 GB, 651 us from a graph, 660-670 a call, 6.35-6.53 TB/s (the device's copies: 6.56); 48
// ragged requests of up to 8k tokens, fp32, KH = 4, 305 MB, 73 us from a graph, 47 at the copy
// rate; one request of 4k tokens, 15 us from a graph, 17 a call: the join's launch, 4 us, and one
// pass through cold instructions.
constexpr int PD_WARPS = 4, PD_THREADS = 32 * PD_WARPS, PD_STAGES = 3, PD_STAGE = 2 * GQA_TILE_BYTES;
// Entries that a unit counts more than it has when the list is cut. A warp pays for the q of
// every piece; one that starts and ends in its range it also finishes and writes by itself. So a
// unit longer than a range counts PD_EXTRA more (0, 1, 2, 3, 4: 64 requests of 512 tokens 21.8, 22.5,
// 20.9, 22.3, 24.5 us) and one that fits into a range PD_WHOLE (48 requests of 1 to 8191 tokens,
// spread over the logarithm: 40 us with 8 or 12, 45 with 4, 52 with PD_EXTRA for all; fp32 43, 51,
// 61). Where a range has less than PD_WHOLE entries it rarely holds a whole unit, and all count alike.
constexpr int PD_EXTRA = 2, PD_WHOLE = 8;
constexpr int PD_OROW = 132;                 // floats between heads of O: 8 banks apart for the writers' heads
template <typename TI> struct PdEntry {      // layout of the q entry and of the gate entry in a stage
    static constexpr bool F32 = sizeof(TI) == 4;
    static constexpr int PARTS = F32 ? 3 : 2;
    static constexpr int BYTES = GQA_HD * (int)sizeof(TI);    // a head's q (or gate), the new k, the new v
    // rows of the q entry: fp32, or bf16 with room for the second part; 4 banks (fp32: 8, for pairs of words) apart
    static constexpr int ROW = 1024 + (F32 ? 32 : 16);
    static constexpr int KV = GQA_GRP * ROW;
    static constexpr int GROW = BYTES + 8 * (int)sizeof(TI);  // rows of the gate entry
    static constexpr int O = GQA_GRP * GROW;                  // gate entry: half of O, fp32, behind the gate rows
    static_assert((GQA_GRP + 2) * ROW <= PD_STAGE && O + GQA_GRP * PD_OROW * 4 <= PD_STAGE && GROW % 16 == 0, "");
};
// (x, y) as PARTS bf16 pairs whose sum is (x, y): all parts but the last cut off (one byte
// permutation), the last rounded, so two leave 2^-16 of it at most and three 2^-31. Every part has
// the sign of the whole and is not 0 unless it is, since 2^-32 of the whole is added to what a cut
// leaves (down to numbers of 2^-101): an infinity in the other operand stays that infinity, where
// rounded parts would make inf - inf or 0 * inf of it. (Rounded ones: 0.2 us less of the 15 of a
// request of 4k, nothing in the longer cases.)
template <int PARTS>
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t (&out)[PARTS])
{
    const float x0 = x, y0 = y;
#pragma unroll
    for (int i = 0; i < PARTS - 1; ++i) {
        out[i] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
        x = fmaf(x0, 0x1p-32f, x - __uint_as_float(out[i] << 16));
        y = fmaf(y0, 0x1p-32f, y - __uint_as_float(out[i] & 0xffff0000u));
    }
    out[PARTS - 1] = pack_bf16(x, y);
}

// A head's row in the q entry, normed and roped in place: bf16 as its parts (hi, and lo 512 bytes behind), fp32 as it is.
template <typename TI> struct PdRow;
template <> struct PdRow<__nv_bfloat16> {
    uint8_t *at;
    __device__ __forceinline__ void load(int c, float (&x)[8]) const { load8<__nv_bfloat16>(reinterpret_cast<__nv_bfloat16 *>(at) + 8 * c, x); }
    __device__ __forceinline__ void store(int c, const float (&x)[8]) const
    {
        uint32_t y[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_bf16<2>(x[2 * i], x[2 * i + 1], y[i]);
        *reinterpret_cast<uint4 *>(at + 16 * c) = make_uint4(y[0][0], y[1][0], y[2][0], y[3][0]);
        *reinterpret_cast<uint4 *>(at + 512 + 16 * c) = make_uint4(y[0][1], y[1][1], y[2][1], y[3][1]);
    }
    __device__ __forceinline__ float load1(int d) const { return __bfloat162float(reinterpret_cast<__nv_bfloat16 *>(at)[d]); }
    __device__ __forceinline__ void store1(int d, float x) const
    {
        uint32_t y[2];
        split_bf16<2>(x, 0.f, y);
        reinterpret_cast<uint16_t *>(at)[d] = (uint16_t)y[0];
        reinterpret_cast<uint16_t *>(at + 512)[d] = (uint16_t)y[1];
    }
};
template <> struct PdRow<float> {
    uint8_t *at;
    __device__ __forceinline__ void load(int c, float (&x)[8]) const { load8<float>(reinterpret_cast<float *>(at) + 8 * c, x); }
    __device__ __forceinline__ void store(int c, const float (&x)[8]) const
    {
        float4 *to = reinterpret_cast<float4 *>(at + 32 * c);
        to[0] = make_float4(x[0], x[1], x[2], x[3]);
        to[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
    __device__ __forceinline__ float load1(int d) const { return reinterpret_cast<float *>(at)[d]; }
    __device__ __forceinline__ void store1(int d, float x) const { reinterpret_cast<float *>(at)[d] = x; }
};
struct PdSmem {
    uint8_t ring[PD_WARPS][PD_STAGES][PD_STAGE];
    alignas(16) float w1[2][GQA_HD];        // 1 + q / k norm weights
    alignas(16) float cs[PD_WARPS][GQA_HD / 2], sn[PD_WARPS][GQA_HD / 2];
    unsigned long long turn[GQA_HD / 2];
    double2 turned[PD_WARPS][GQA_HD / 2];   // (cos, sin) of the row to append (fp32 activations)
    float2 ml[PD_WARPS][2][GQA_GRP];        // (max, sum) of a warp's continued / opened piece
    int4 cont[PD_WARPS], open[PD_WARPS];    // (there: 1, and ends here: 2; request; KV head; parked / last CTA)
    int pre[1024 + 4];                      // entries (of one KV head) before each request
    uint32_t cut[32];                       // a bit per request: its units are longer than a range
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
template <typename TI>
__global__ void __launch_bounds__(PD_THREADS, 1)
pages_decode_kernel(GqaPagesArgs p, PagesPart part, const __grid_constant__ CUtensorMap tmKV, const __grid_constant__ RopeFreq f)
{
    using E = PdEntry<TI>;
    constexpr int PARTS = E::PARTS;
    extern __shared__ uint8_t smem_raw[];
    PdSmem &sm = *reinterpret_cast<PdSmem *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
    const int KH = p.pv.KH, G = p.H / KH, page = p.pv.page;
    griddep_launch();                       // the join may be scheduled; it waits for this grid
    // entries before each request: its tiles, a q and a gate entry. Up to 32
    // requests every warp counts for itself (all write the same), with no barrier.
    auto tiles = [&](int r) {               // 0: idle
        int row0, pos0;
        return pages_rows_of(p, r, row0, pos0) ? pos0 / GQA_TILE + 1 : 0;
    };
    const int workers = gridDim.x * PD_WARPS;
    int whole = 0;                          // tiles of a unit that a range can hold
    auto entries = [&](int nt) { return nt == 0 ? 0 : nt + 2 + (nt <= whole ? PD_WHOLE : PD_EXTRA); };
    // the norm weights and rotary frequencies: loads in flight until the first
    // tiles are, then every warp writes the same
    float4 w_in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w_in[j] = reinterpret_cast<const float4 *>(p.qnw)[lane + 32 * j];   // knw follows qnw
    {
        const int each = (p.n_req + PD_THREADS - 1) / PD_THREADS, small = p.n_req <= 32;
        const int r0 = min(p.n_req, small ? lane : tid * each), r1 = min(p.n_req, small ? lane + 1 : r0 + each);
        int nt = 0, sum = 0;                // (the last of r0 .. r1 - 1, the only one where small)
#pragma unroll 1
        for (int r = r0; r < r1; ++r) { nt = tiles(r); sum += entries(nt); }
        if (lane == 0) {
            for (int s = 0; s < PD_STAGES; ++s) mbar_init(&sm.full[warp][s], 1);
            fence_mbar_init();
            sm.cont[warp] = sm.open[warp] = make_int4(0, 0, 0, 0);
        }
        if (p.n_req > 1) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (!small) {
                if (lane == 0) sm.part[warp] = sum;
                if (tid < 32) sm.cut[tid] = 0;
                __syncthreads();
                sum = 0;
                for (int w = 0; w < PD_WARPS; ++w) sum += sm.part[w];
                __syncthreads();            // read before it is written again
            }
            whole = (sum * KH + workers - 1) / workers;
            if (whole < PD_WHOLE) whole = 0;
        }
        int mine = entries(nt);
        if (!small) {
            mine = 0;
#pragma unroll 1
            for (int r = r0; r < r1; ++r) {
                nt = tiles(r);
                mine += entries(nt);
                if (nt > whole) atomicOr(&sm.cut[r >> 5], 1u << (r & 31));
            }
        }
        int inc = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += y;
        }
        int at = inc - mine;
        if (small) {
            const unsigned cut = __ballot_sync(0xffffffffu, nt > whole);
            if (lane < p.n_req) sm.pre[lane] = at;
            if (lane == 31) { sm.pre[p.n_req] = inc; sm.cut[0] = cut; }
            __syncwarp();
        } else {
            if (lane == 31) sm.part[warp] = inc;
            __syncthreads();
            for (int w = 0; w < warp; ++w) at += sm.part[w];
#pragma unroll 1
            for (int r = r0; r < r1; ++r) { sm.pre[r] = at; at += entries(tiles(r)); }
            if (tid == PD_THREADS - 1) sm.pre[p.n_req] = at;
            __syncthreads();
        }
    }
    auto extra = [&](int r) { return sm.cut[r >> 5] >> (r & 31) & 1 ? PD_EXTRA : PD_WHOLE; };
    const int total = sm.pre[p.n_req] * KH;
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
        const int ex = extra(r), rel = rel0 - kh * n - ex, nt = n - 2 - ex;    // 0: q, 1 ..: tiles, nt + 1: gate
        const bool begins = at - rel + 1 >= v0;                 // the unit's first tile is in the range
        if (v < v0) ahead = rel >= 1 && rel <= nt ? 1 : -1;
        else if (v == v1) ahead = rel == nt && begins ? 2 : -1;
        else if (rel == 0) ahead = v + 1 < v1 ? 1 : -1;
        else if (rel <= nt) ahead = rel < 0 ? -1 : 0;
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
                tma_load_5d(to, &tmKV, 0, 0, 0, e, 0, bar);
            }
        } else {                            // rows of unit `u`, a bulk copy per lane
            const int u = (-1 - e) >> 1, is_q = (-1 - e) & 1, r = p.pv.heads_div(u), n = is_q ? G + 2 : G;
            if (lane == 0) mbar_expect_tx(bar, n * E::BYTES);
            __syncwarp();
            const TI *from = static_cast<const TI *>(p.qg) + ((size_t)r * p.H + (u - r * KH) * G + lane) * 2 * GQA_HD + (is_q ? 0 : GQA_HD);
            if (lane == G) from = static_cast<const TI *>(p.k) + (size_t)u * GQA_HD;
            if (lane == G + 1) from = static_cast<const TI *>(p.v) + (size_t)u * GQA_HD;
            if (lane < n) bulk_load(to + (!is_q ? lane * E::GROW : lane < G ? lane * E::ROW : E::KV + (lane - G) * E::ROW), from, E::BYTES, bar);
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
        if (i == -1) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                reinterpret_cast<float4 *>(sm.w1[0])[lane + 32 * j] =
                    make_float4(1.f + w_in[j].x, 1.f + w_in[j].y, 1.f + w_in[j].z, 1.f + w_in[j].w);
            for (int j = lane; j < p.rot / 2; j += 32) sm.turn[j] = f.turn[j];
            __syncwarp();
        }
        if (i >= 0) {
            if (at == AT_Q) {
                // ---- the next unit with tiles in the range
                for (;;) {
                    if (next_v >= v1) break;
                    r = next_r; kh = next_kh;
                    const int n = sm.pre[r + 1] - sm.pre[r];
                    const int ex = extra(r);
                    nt = n - 2 - ex;
                    u0 = sm.pre[r] * KH + kh * n + ex;      // its q entry
                    tile = max(next_v - u0 - 1, 0);
                    end_tile = min(v1 - u0 - 1, nt);
                    next_v = min(v1, u0 + nt + 2);
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
                float val[8];
                load8<TI>(reinterpret_cast<const TI *>(st + E::KV + E::ROW) + lane * 8, val);
                new_vb = make_uint4(pack_bf16(val[0], val[1]), pack_bf16(val[2], val[3]), pack_bf16(val[4], val[5]), pack_bf16(val[6], val[7]));
                if (ends) {                 // the row to append
                    const TI *raw = reinterpret_cast<const TI *>(st + E::KV);
                    float x[8], w1[8];
                    load8<TI>(raw + lane * 8, x);
                    if constexpr (E::F32) {
                        // in double up to its rounding: fp32 outputs show it where an element of
                        // the cached row falls to the other side of a bf16 border
                        double s2 = 0.0;
#pragma unroll
                        for (int e = 0; e < 8; ++e) s2 += (double)x[e] * x[e];
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) s2 += __shfl_xor_sync(0xffffffffu, s2, o);
                        const double r = rsqrt(s2 * (1.0 / GQA_HD) + p.eps);
                        const int half = p.rot >> 1;
#pragma unroll 1
                        for (int j = lane; j < half; j += 32) {
                            double2 t;
                            sincospi((double)(long long)((unsigned long long)pos * sm.turn[j]) * 0x1p-63, &t.y, &t.x);
                            sm.turned[warp][j] = t;
                        }
                        __syncwarp();
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int d = lane * 8 + e;
                            double y = x[e] * r * (1.0 + p.knw[d]);
                            if (d < p.rot) {
                                const bool low = d < half;
                                const int o = low ? d + half : d - half;
                                const double2 t = sm.turned[warp][low ? d : o];
                                const double z = raw[o] * r * (1.0 + p.knw[o]);
                                y = low ? y * t.x - z * t.y : y * t.x + z * t.y;
                            }
                            x[e] = (float)y;
                        }
                    } else {
                        load8<float>(sm.w1[1] + lane * 8, w1);
                        pages_norm_rope(x, w1, p.eps, p.rot, cs, sn, raw, sm.w1[1], lane);
                    }
                    new_k = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
                }
                // heads past the group's: q = 0 (what lies there is finite or not: cleared, not scaled)
                for (int j = G * (E::ROW / 16) + lane; j < GQA_GRP * (E::ROW / 16); j += 32)
                    reinterpret_cast<uint4 *>(st)[j] = make_uint4(0, 0, 0, 0);
                __syncwarp();
                pages_norm_rope_rows<4>(PdRow<TI>{st + (lane >> 2) * E::ROW}, lane & 3, sm.w1[0], p.eps, p.rot, cs, sn);
#pragma unroll
                for (int kk = 0; kk < 16; ++kk)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint8_t *from = st + (lane >> 2) * E::ROW + (16 * kk + 8 * e + 2 * (lane & 3)) * (int)sizeof(TI);
                        if constexpr (E::F32) {
                            const float2 x = *reinterpret_cast<const float2 *>(from);
                            uint32_t parts[PARTS];
                            split_bf16<PARTS>(x.x, x.y, parts);
#pragma unroll
                            for (int q = 0; q < PARTS; ++q) qf[q][kk][e] = parts[q];
                        } else {
                            qf[0][kk][e] = *reinterpret_cast<const uint32_t *>(from);
                            qf[1][kk][e] = *reinterpret_cast<const uint32_t *>(from + 512);
                        }
                    }
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
                const float p0 = ex2_approx(x0 - b0), p1 = ex2_approx(x1 - b1), p2 = ex2_approx(x2 - b0), p3 = ex2_approx(x3 - b1);
                if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
                    const float al0 = ex2_approx(m0 - b0), al1 = ex2_approx(m1 - b1);
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
                        load4(reinterpret_cast<const TI *>(gate + h * E::GROW) + half * 128, g);
                        load4(o_ + h * PD_OROW + 4 * lane, o);
                        gate4(o, g);
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
        float M0 = -INFINITY, M1 = -INFINITY, L0 = 0.f, L1 = 0.f, o[4][4] = {};
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            const float2 *ml = sm.ml[from + j][opened && j == 0];
            M0 = fmaxf(M0, ml[h0].x);
            M1 = fmaxf(M1, ml[h0 + 1].x);
        }
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            const bool open = opened && j == 0;
            const float2 a = sm.ml[from + j][open][h0], b = sm.ml[from + j][open][h0 + 1];
            const float f0 = a.x == -INFINITY ? 0.f : ex2_approx(a.x - M0), f1 = b.x == -INFINITY ? 0.f : ex2_approx(b.x - M1);
            L0 += a.y * f0;
            L1 += b.y * f1;
            float4 x[4];
            if (!open && sm.cont[from + j].w) {
#pragma unroll
                for (int u = 0; u < 4; ++u) x[u] = part.park[(size_t)(cta * PD_WARPS + from + j) * 512 + (warp + PD_WARPS * u) * 32 + lane];
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u) x[u] = reinterpret_cast<const float4 *>(sm.ring[from + j][0])[(warp + PD_WARPS * u) * 32 + lane];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) { o[u][0] += x[u].x * f0; o[u][1] += x[u].y * f1; o[u][2] += x[u].z * f0; o[u][3] += x[u].w * f1; }
        }
        const int slot = 2 * cta + (opened ? 1 : 0);
        if (whole) {
            const float i0 = rcp_approx(L0), i1 = rcp_approx(L1);
            const size_t row = (size_t)unit.y * p.H + unit.z * G + h0;
            TI *out = static_cast<TI *>(p.ctx) + row * GQA_HD + warp * 16 + dr;
            const TI *g = static_cast<const TI *>(p.qg) + row * 2 * GQA_HD + GQA_HD + warp * 16 + dr;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)     // (head h0 + e % 2, dim + 8 (e / 2))
                    if (h0 + (e & 1) < G) {
                        const int d = 16 * PD_WARPS * u + 8 * (e >> 1);
                        out[(e & 1) * GQA_HD + d] = from_f32<TI>(o[u][e] * (e & 1 ? i1 : i0) * gate_of(to_f32(g[(e & 1) * 2 * GQA_HD + d])));
                    }
        } else {
            if (warp == 0 && lane < 4) {
                float2 *ml = part.ml + (size_t)slot * GQA_GRP + h0;
                ml[0] = make_float2(M0, L0);
                ml[1] = make_float2(M1, L1);
            }
            float *out = part.o + ((size_t)slot * GQA_GRP + h0) * GQA_HD + warp * 16 + dr;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) out[(e & 1) * GQA_HD + 16 * PD_WARPS * u + 8 * (e >> 1)] = o[u][e];
        }
        if (step == 2 * PD_WARPS) break;
        n = 0;
        opened = false;
    }
    // a unit that begins in this CTA and goes on: its pieces are this CTA's last and the firsts of cta + 1 .. unit.w
    if (tid == 0) part.units[cta] = make_int4(n > 0 && opened ? unit.w : -1, unit.y, unit.z, 0);
}

// A piece (max, sum) that weighs nothing: all its keys are masked, or their scores -infinity. Scores
// that are all NaN leave the maximum at -infinity as well (fmaxf passes NaN over), but not the sum at
// 0: such a piece's NaN is the result's.
__device__ __forceinline__ bool piece_empty(const float2 &ml) { return ml.x == -INFINITY && ml.y == 0.f; }

// One CTA of four warps per (CTA of the kernel before, query head): merges the
// pieces of the unit that begins there and goes on. Warp w takes pieces w, w + 4,
// .. with a running maximum, lane = 8 dims; then thread d merges the four results
// of dims d and d + 128. Small enough that all of them, most with nothing to do,
// are resident at once; one CTA for all heads of a unit had one SM read all pieces
// of a long single request (5 us of 20).
constexpr int PJ_WARPS = 4;
template <typename TI>
__global__ void __launch_bounds__(PJ_WARPS * 32)
pages_join_kernel(GqaPagesArgs p, PagesPart part)
{
    __shared__ float sm_ml[PJ_WARPS][2];
    __shared__ __align__(16) float sm_o[PJ_WARPS][GQA_HD];
    const int a = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();                         // a programmatic dependent of the decode kernel
    const int4 unit = part.units[a];
    if (unit.x < 0) return;
    const int n = unit.x - a + 1;
    const size_t row = (size_t)unit.y * p.H + unit.z * (p.H / p.pv.KH) + h;
    float gate[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) gate[e] = to_f32(static_cast<const TI *>(p.qg)[row * 2 * GQA_HD + GQA_HD + tid + 128 * e]);
    float m = -INFINITY, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    constexpr int U = 4;                    // pieces whose loads a warp issues together
    for (int s0 = warp; s0 < n; s0 += U * PJ_WARPS) {
        float2 ml[U];
        float4 x[U], y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * PJ_WARPS;
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
            if (piece_empty(ml[u])) continue;
            const float mn = fmaxf(m, ml[u].x);
            const float fo = m == -INFINITY ? 0.f : ex2_approx(m - mn), fs = ex2_approx(ml[u].x - mn);
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
    float M = -INFINITY, O[2] = {0.f, 0.f}, L = 0.f;
#pragma unroll
    for (int w = 0; w < PJ_WARPS; ++w) M = fmaxf(M, sm_ml[w][0]);
#pragma unroll
    for (int w = 0; w < PJ_WARPS; ++w) {
        const float f = sm_ml[w][0] == -INFINITY ? 0.f : ex2_approx(sm_ml[w][0] - M);
        O[0] += sm_o[w][tid] * f;
        O[1] += sm_o[w][tid + 128] * f;
        L += sm_ml[w][1] * f;
    }
    const float inv = rcp_approx(L);
#pragma unroll
    for (int e = 0; e < 2; ++e)
        static_cast<TI *>(p.ctx)[row * GQA_HD + tid + 128 * e] = from_f32<TI>(O[e] * inv * gate_of(gate[e]));
}

template <typename TI>
static cudaError_t pages_decode_run(const CUtensorMap &tkv, const GqaPagesArgs &a, const PagesPart &part,
                                    const RopeFreq &f, int ctas, cudaStream_t st)
{
    const int smem = (int)sizeof(PdSmem) + 1024;
    cudaError_t e = cudaFuncSetAttribute(pages_decode_kernel<TI>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    pages_decode_kernel<TI><<<ctas, PD_THREADS, smem, st>>>(a, part, tkv, f);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, a.H / a.pv.KH); cfg.blockDim = dim3(PJ_WARPS * 32); cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, pages_join_kernel<TI>, a, part);
}

cudaError_t launch_pages_decode(const CUtensorMap &tkv, const GqaPagesArgs &a, const PagesPart &part,
                                const RopeFreq &f, int in_bf16, int ctas, cudaStream_t st)
{
    return in_bf16 ? pages_decode_run<__nv_bfloat16>(tkv, a, part, f, ctas, st)
                   : pages_decode_run<float>(tkv, a, part, f, ctas, st);
}

// ------------------------------------------------------------------ prefill
// A unit is 128 query rows of one request and KV head: 128 / group tokens x
// the group's heads, so all heads of the group share each K / V tile and a
// tile of rows spans few positions (little of it is masked). Its work is its
// 128-key tiles plus PP_SETUP. The units of all requests, end to end, are cut into
// equal ranges, one per CTA (one CTA per SM): no tail wave, and few rows on a
// long context are spread over the GPU. A piece of a unit leaves its O, max and sum in the
// workspace, and pages_prefill_join_kernel merges them (two at most per CTA).
//
//   pages_append_kernel   k normed, roped and appended with v, a warp per (row, KV
//                         head); the next kernel starts beside it, and its loads of
//                         tiles that hold new rows wait for it
//   pages_prefill_kernel  each CTA lays out its range from the chunks' sizes; tcgen05,
//                         352 threads:
//     warp 0      K tiles into a 2-stage ring, up to 8 TMA boxes of whole pages
//                 each (a lane per box, its page id looked up there), and the gate
//                 tile into the stage that the piece's last K tile leaves
//     warp 1      V tiles, one buffer (which first stages Q)
//     warp 2      MMA issuer, TMEM owner: S = Q K^T (M = N = 128, A = Q from
//                 TMEM), O += P V (N = 256); S(j + 1) is issued before PV(j)
//     warps 3..10 q norm + RoPE and Q into TMEM; softmax, 16 rows per warp
//                 through the 16x256b TMEM shape, log2 domain, O corrected only
//                 where the running maximum grew by more than 2^8; epilogue
//   A page is a run of whole row groups, so one box of its rows lands as
//   [8-row group][64-column block][8 rows][128 B]: groups 4 KiB apart, column blocks
//   1 KiB, for K (K-major) and V (MN-major) alike, whatever the page size.
//   Keys behind the request's end: K scores are masked, V rows read as zeros
//   (boxes outside the pool; the last few rows of a group cleared in shared memory),
//   so non-finite stale rows cannot come through as 0 * inf. New v rows that are not finite are
//   flagged by the append (a word in the workspace, reset by the join); only then the V loader looks
//   through tiles that hide keys from some row, and clears what would reach it.
// TMEM (512 columns): scores 128 | O 256 | Q 128 (bf16 pairs). Q and P are
// rounded to bf16 (2^-9 of each element on average): a second part of either would double
// its MMAs, and the tensor pipe is the bound here.
// Measured, H / KH = 8, KH = 2: 4096 rows after 28672, 2.06 TFLOP of causal products, 1.82 ms
// under the power cap (1.13 PFLOP/s, 0.70 of the GPU's 8192^3 product), 1.55 before it sets in; nine
// chunks of up to 1023 rows after up to 4096, 155 GFLOP, 185 us from a graph (0.84 PFLOP/s; the
// rest are units' starts and ends, 15500 cycles each where a tile takes 2750, masked halves of
// diagonal tiles and the join of units cut at CTAs' ends); three short prompts 20 us, latency of
// three launches. In a tile's cycles shared memory is read for about 2500 (K and V by the MMAs, P
// written and read): next to the tensor pipe the second bound.
constexpr int PP_BM = 128, PP_BN = 128;
constexpr int PP_TILE = PP_BN * GQA_HD * 2, PP_P = PP_BM * PP_BN * 2;
constexpr int PP_SOFTMAX = 256, PP_THREADS = 96 + PP_SOFTMAX;
constexpr int PP_SETUP = 7;                 // a unit's start and end in tiles' time (4: 5-15 % slower, 9 and 12: 1-4 %)
constexpr int PP_MIN = 4;                   // least work of a CTA
struct PpBars {
    uint64_t q_tmem, k_full[2], k_empty[2], v_full, v_raw, v_empty, s_full, s_free, p_full, pv_done, g_full, epi_done;
    unsigned long long turn[GQA_HD / 2];
    alignas(16) float w1[GQA_HD];           // 1 + q norm weights
    int4 range[2];
    uint32_t tmem_base;
    int clean_from[2];                      // of the piece in work and the next: first key whose V tile was cleaned, or -1
    float lsum[PP_BM];
};
constexpr int PP_SMEM = 3 * PP_TILE + PP_P + (int)sizeof(PpBars);
static_assert(offsetof(PpBars, w1) % 16 == 0 && (3 * PP_TILE + PP_P) % 16 == 0, "16-byte loads");
static_assert(PP_SMEM <= 232448, "prefill shared memory exceeds the 227 KiB per-CTA limit");

// Tiles of query tile qt of a chunk of n rows at position b.
__device__ __forceinline__ int pp_tiles(int n, int b, int qt, int tokens)
{
    return (b + min(n, (qt + 1) * tokens) - 1) / PP_BN + 1;
}
// Work of its query tiles before qt (all of them whole): sum over j < qt of
// floor((a + j) / group) + 1 + PP_SETUP with a = floor((b - 1 + tokens) / tokens),
// group = 1 << gs, tokens = 128 >> gs.
__device__ __forceinline__ long long pp_work(int b, int qt, int gs)
{
    auto below = [&](long long m) {         // sum over i < m of floor(i / group)
        const long long k = m >> gs;
        return ((k * (k - 1) / 2) << gs) + k * (m - (k << gs));
    };
    const long long a = (b - 1 + (PP_BM >> gs)) >> (7 - gs);
    return below(a + qt) - below(a) + (long long)qt * (1 + PP_SETUP);
}

// Work of request r's chunk for one KV head.
__device__ __forceinline__ long long pp_chunk_work(const GqaPagesArgs &p, int r, int gs)
{
    int row0, b;
    const int n = pages_rows_of(p, r, row0, b);
    if (n == 0) return 0;
    const int last = (n - 1) >> (7 - gs);
    return pp_work(b, last, gs) + pp_tiles(n, b, last, PP_BM >> gs) + PP_SETUP;
}

// Where the ranges of CTAs cta and cta + 1 start, (request, KV head, query
// tile, key tile), into range[0] and range[1]; `scratch` 8 KiB + 256 of shared
// memory, all threads of the CTA.
__device__ __forceinline__ void pp_plan(const GqaPagesArgs &p, int cta, int ctas, int gs, void *scratch, int4 *range)
{
    long long *pre = static_cast<long long *>(scratch), *sums = pre + 1024 + 8;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, KH = p.pv.KH;
    const int each = (p.n_req + PP_THREADS - 1) / PP_THREADS, r0 = min(p.n_req, tid * each), r1 = min(p.n_req, r0 + each);
    long long mine = 0;
#pragma unroll 1
    for (int r = r0; r < r1; ++r) mine += pp_chunk_work(p, r, gs);
    long long inc = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += y;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    long long at = inc - mine;
    for (int w = 0; w < warp; ++w) at += sums[w];
#pragma unroll 1
    for (int r = r0; r < r1; ++r) { pre[r] = at; at += r + 1 < r1 || r > r0 ? pp_chunk_work(p, r, gs) : mine; }
    if (tid == PP_THREADS - 1) pre[p.n_req] = at;
    __syncthreads();
    if (warp < 2) {                         // a warp per range, 32 places looked at at a time
        const long long all = pre[p.n_req] * KH, per = max((long long)PP_MIN, (all + ctas - 1) / ctas), v = (cta + warp) * per;
        int4 u = make_int4(p.n_req, 0, 0, 0);
        if (v < all) {
            int lo = -1;                    // the last request that starts at or before v
            for (int r = lane; r - lane < p.n_req; r += 32) lo += __popc(__ballot_sync(0xffffffffu, r < p.n_req && pre[r] * KH <= v));
            const long long head = pre[lo + 1] - pre[lo];
            long long rel = v - pre[lo] * KH;
            u.x = lo;
            while (rel >= head) { rel -= head; ++u.y; }
            int row0, b, q0 = 0;
            const int n = pages_rows_of(p, lo, row0, b);
            for (int left = ((n - 1) >> (7 - gs)) + 1; left > 1;) {           // .. and query tile, of the `left` from q0 on
                const int step = (left + 31) / 32, k = __popc(__ballot_sync(0xffffffffu, lane * step < left && pp_work(b, q0 + lane * step, gs) <= rel)) - 1;
                q0 += k * step;
                left = min(step, left - k * step);
            }
            u.z = q0;
            u.w = max(0, (int)(rel - pp_work(b, q0, gs)) - PP_SETUP);
        }
        if (lane == 0) range[warp] = u;
    }
    __syncthreads();
}

// One pass over the new rows, bound by HBM for long chunks (4096 rows, KH = 2: 16.8 MB moved) and hidden
// behind the tiles of earlier rows; a chunk at position 0 waits for it, about 4 us.
constexpr int PA_WARPS = 8;
__global__ void __launch_bounds__(PA_WARPS * 32)
pages_append_kernel(GqaPagesArgs p, const __grid_constant__ RopeFreq f, int *odd)
{
    __shared__ __align__(16) float cs[PA_WARPS][GQA_HD / 2], sn[PA_WARPS][GQA_HD / 2], w1s[GQA_HD];
    griddep_launch();                       // the attention starts now; what reads appended rows waits
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, KH = p.pv.KH;
    w1s[tid] = 1.f + p.knw[tid];
    __syncthreads();
    const int item = blockIdx.x * PA_WARPS + warp, row = p.pv.heads_div(item), kh = item - row * KH;
    if (row >= p.S) return;
    const __nv_bfloat16 *k = static_cast<const __nv_bfloat16 *>(p.k) + (size_t)item * GQA_HD;
    float x[8], v[8], w1[8];
    load8<__nv_bfloat16>(k + lane * 8, x);
    load8<__nv_bfloat16>(static_cast<const __nv_bfloat16 *>(p.v) + (size_t)item * GQA_HD + lane * 8, v);
    int lo = -1, row0, b;                   // the request whose chunk holds the row, whatever the other offsets say
    for (int r = lane; lo < 0 && r - lane < p.n_req; r += 32) {
        const unsigned in = __ballot_sync(0xffffffffu, r < p.n_req && p.cu[r] <= row && row < p.cu[r + 1]);
        if (in) lo = r - lane + __ffs(in) - 1;
    }
    if (lo < 0 || pages_rows_of(p, lo, row0, b) == 0) return;
    const int pos = b + row - row0;
    const long long at = pages_row(p.pv, lo, kh, pos);
    pages_rope_table(cs[warp], sn[warp], pos, p.rot, f.turn, lane, 32);
    __syncwarp();
    load8<float>(w1s + lane * 8, w1);
    pages_norm_rope(x, w1, p.eps, p.rot, cs[warp], sn[warp], k, w1s, lane);
    if (at < 0) return;
    store8(p.pv.k + at * GQA_HD + lane * 8, x);
    store8(p.pv.v + at * GQA_HD + lane * 8, v);
    float zero = 0.f;                       // of finite values; NaN with any other
#pragma unroll
    for (int i = 0; i < 8; ++i) zero = fmaf(v[i], 0.f, zero);
    if (zero != 0.f) *odd = 1;
}

// A CTA's pieces, one after the other.
struct PpWalk {
    int4 at, stop;
    int n, row0, base, nt, t1;              // of the piece in work: rows, first row, first position, tiles, end tile
    bool ends;
    __device__ __forceinline__ PpWalk(const GqaPagesArgs &p, const int4 *range)
    {
        at = range[0];
        stop = range[1];
        n = at.x < p.n_req ? pages_rows_of(p, at.x, row0, base) : 0;
    }
    __device__ __forceinline__ bool piece(int tokens)
    {
        const bool last = at.x == stop.x && at.y == stop.y && at.z == stop.z;
        if (n == 0 || (last && at.w >= stop.w)) return false;
        nt = pp_tiles(n, base, at.z, tokens);
        t1 = last ? stop.w : nt;
        ends = t1 == nt;
        return true;
    }
    __device__ __forceinline__ void next(const GqaPagesArgs &p, int tokens)
    {
        if (!ends) { n = 0; return; }       // the rest is the next CTA's
        at.w = 0;
        if (++at.z * tokens < n) return;
        at.z = 0;
        if (++at.y < p.pv.KH) return;
        at.y = 0;
        n = 0;
        while (n == 0 && ++at.x < p.n_req && at.x <= stop.x) n = pages_rows_of(p, at.x, row0, base);
    }
};

// Sums of the infinities and NaN among the values in dims d .. d + 7 that position pos sees, from key
// `from` to the end of the piece; 0: there are none. Only for tiles that were cleaned of them.
__device__ __forceinline__ void pp_cleared(const GqaPagesArgs &p, const PpWalk &w, int from, int pos, int d, float (&sum)[8])
{
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.f;
    const int last = min(pos, min(w.base + w.n, w.t1 * PP_BN) - 1);
#pragma unroll 1
    for (int key = from; key <= last; ++key) {
        const long long at = pages_row(p.pv, w.at.x, w.at.y, key);
        if (at < 0) continue;
        float v[8];
        load8v(p.pv.v + at * GQA_HD + d, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += fabsf(v[e]) <= 3.4e38f ? 0.f : v[e];
    }
}

// K-major 128B-swizzled operand whose 8-row groups are 4 KiB apart.
__device__ __forceinline__ uint64_t pp_desc_k(uint32_t addr)
{
    return (tc::desc_k_sw128(addr) & ~((uint64_t)0x3FFF << 32)) | (uint64_t)(4096 >> 4) << 32;
}

// A q row in the V buffer: 16-byte chunk c of row r in 64-column block c / 8, at chunk (c % 8) ^ (r % 8).
struct PpRow {
    uint8_t *at;
    int swz;
    bool on;                                // off: this pass leaves the row alone
    __device__ __forceinline__ __nv_bfloat16 *chunk(int c) const
    {
        return reinterpret_cast<__nv_bfloat16 *>(at + (c >> 3) * (PP_BM * 128) + (((c & 7) ^ swz) << 4));
    }
    __device__ __forceinline__ void load(int c, float (&x)[8]) const { load8<__nv_bfloat16>(chunk(c), x); }
    __device__ __forceinline__ void store(int c, const float (&x)[8]) const { if (on) store8(chunk(c), x); }
    __device__ __forceinline__ float load1(int d) const { return __bfloat162float(chunk(d >> 3)[d & 7]); }
    __device__ __forceinline__ void store1(int d, float x) const { if (on) chunk(d >> 3)[d & 7] = __float2bfloat16_rn(x); }
};

// A V tile on its way to v_raw, without its infinities and NaN, to v_full (a whole warp; false: timed
// out). Not inlined: rare, and its code in the loader's loop cost three short prompts 0.2 us of 20 (the
// epilogue's part as functions 0.2 less, too, but 4096 rows 2 of 169 more).
__device__ __noinline__ bool pp_clean(uint8_t *v, PpBars *bars, int raws, int pc, int tile)
{
    const int lane = threadIdx.x & 31;
    const bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->v_raw, raws & 1));
    bool found = false;
#pragma unroll 4
    for (int c = lane; c < PP_TILE / 4; c += 32) {
        uint32_t *y = reinterpret_cast<uint32_t *>(v) + c, was = *y, is = was;
        if ((is & 0x7f80u) == 0x7f80u) is &= 0xffff0000u;
        if ((is & 0x7f800000u) == 0x7f800000u) is &= 0xffffu;
        if (is != was) { *y = is; found = true; }
    }
    fence_proxy_async();
    found = __any_sync(0xffffffffu, found);
    if (lane == 0) {
        if (found && bars->clean_from[pc & 1] < 0) bars->clean_from[pc & 1] = tile * PP_BN;
        if (ok) mbar_arrive(&bars->v_full);
    }
    __syncwarp();
    return ok;
}

__global__ void __launch_bounds__(PP_THREADS, 1)
pages_prefill_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const __grid_constant__ CUtensorMap tmV8, const __grid_constant__ CUtensorMap tmG, GqaPagesArgs p,
                     PagesPart part, const __grid_constant__ RopeFreq f)
{
    // all shared memory is dynamic, so the window starts 1024-byte aligned as
    // the swizzled boxes and descriptors need (checked: the budget leaves no padding)
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *sK = smem_raw, *sV = sK + 2 * PP_TILE, *sP = sV + PP_TILE;
    PpBars &bars = *reinterpret_cast<PpBars *>(sP + PP_P);
    if (smem_u32(smem_raw) & 1023) {        // uniform across the CTA: nothing has started yet
        if (threadIdx.x == 0) raise_error(2);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
    const int KH = p.pv.KH, group = p.H / KH, gs = __ffs(group) - 1, tokens = PP_BM / group;
    griddep_launch();
    if (threadIdx.x == 0) {
        mbar_init(&bars.q_tmem, PP_SOFTMAX);
        for (int i = 0; i < 2; ++i) { mbar_init(&bars.k_full[i], 1); mbar_init(&bars.k_empty[i], 1); }
        mbar_init(&bars.v_full, 1); mbar_init(&bars.v_raw, 1); mbar_init(&bars.v_empty, 1);
        mbar_init(&bars.s_full, 1); mbar_init(&bars.s_free, PP_SOFTMAX);
        mbar_init(&bars.p_full, PP_SOFTMAX); mbar_init(&bars.pv_done, 1);
        mbar_init(&bars.g_full, 1); mbar_init(&bars.epi_done, PP_SOFTMAX);
        fence_mbar_init();
    }
    if (threadIdx.x < p.rot / 2) bars.turn[threadIdx.x] = f.turn[threadIdx.x];
    if (threadIdx.x < GQA_HD) bars.w1[threadIdx.x] = 1.f + p.qnw[threadIdx.x];
    if (warp == 2) tc::alloc(&bars.tmem_base, 512);
    pp_plan(p, cta, gridDim.x, gs, sP, bars.range);   // (its barriers order the set-up above, too)
    if (threadIdx.x < 2) part.plan[cta + threadIdx.x] = bars.range[threadIdx.x];   // for the join
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tbase = bars.tmem_base;
    const uint32_t tS = tbase, tO = tbase + 128, tQ = tbase + 384;
    PpWalk w(p, bars.range);
    int jj = 0;                             // key tiles of this CTA so far

    if (warp < 2) {
        // ------------------------------------------------ TMA producers (a lane per box)
        if (lane == 0) { tma_prefetch_desc(warp ? &tmV : &tmK); tma_prefetch_desc(warp ? &tmV8 : &tmG); }
        const int box = p.box_rows, boxes = PP_BN / box, beyond = (int)((long long)p.pv.n_pages * KH * p.pv.page >> 3);
        bool ok = true;
        bool appended = false;              // .. the rows that the kernel before appends are visible
        int odd = 0, raws = 0;              // *part.odd; tiles cleaned so far
        int gate_in = -1, wholes = 0, pc = 0;   // the stage of the last gate tile, until its epilogue is known to be done
        for (; ok && w.piece(tokens); w.next(p, tokens), ++pc) {
            const int end = w.base + w.n;   // the request's rows
            if (warp == 1) {
                ok = mbar_wait(&bars.q_tmem, pc & 1);           // Q has left the V buffer
                if (lane == 0) bars.clean_from[pc & 1] = -1;
            }
            for (int j = w.at.w; ok && j < w.t1; ++j, ++jj) {
                const int s = jj & 1;
                // a lane's box: `rows` of them from key `key`; 8-row boxes where V ends inside the tile
                if (!appended && (j + 1) * PP_BN > w.base) {
                    griddep_wait();
                    fence_proxy_async_global();     // written by plain stores, read through the async proxy
                    appended = true;
                    if (warp == 1) odd = *(volatile int *)part.odd;
                }
                // a V tile that hides keys from some row of the unit: hidden keys weigh 0, and 0 * inf would
                // reach the rows before them, so infinities and NaN are cleared; the epilogue adds them to the
                // rows that see them
                const bool clean = warp == 1 && odd != 0 && (j + 1) * PP_BN - 1 > w.base + w.at.z * tokens;
                const bool tail = warp == 1 && (j + 1) * PP_BN > end;
                const int rows = tail ? 8 : box, key = j * PP_BN + lane * rows, n_box = tail ? PP_BN / 8 : boxes;
                int at = beyond;
                if (lane < n_box && key < end) {
                    const long long row = pages_row(p.pv, w.at.x, w.at.y, key);
                    if (row >= 0) at = (int)(row >> 3);
                }
                if (warp == 0) {
                    if (jj >= 2) ok = mbar_wait(&bars.k_empty[s], ((jj >> 1) - 1) & 1);
                    if (ok && gate_in == s) { ok = mbar_wait(&bars.epi_done, (wholes - 1) & 1); gate_in = -1; }
                } else if (jj >= 1) {
                    ok = mbar_wait(&bars.v_empty, (jj - 1) & 1);
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                uint64_t *bar = warp == 0 ? &bars.k_full[s] : clean ? &bars.v_raw : &bars.v_full;
                uint8_t *to = warp == 0 ? sK + s * PP_TILE : sV;
                if (lane == 0) mbar_expect_tx(bar, PP_TILE);
                __syncwarp();
                if (lane < n_box) tma_load_4d(to + lane * rows * 512, warp == 0 ? &tmK : tail ? &tmV8 : &tmV, 0, 0, 0, at, bar);
                __syncwarp();
                if (__builtin_expect(clean, 0)) {
                    ok = pp_clean(sV, &bars, raws++, pc, j);
                }
            }
            if (warp == 0 && ok && w.ends && w.at.w == 0) {
                // the gate tile, into the stage of the last K tile once S has read it, and once the
                // gate before is used up: g_full is one barrier for all of them, and where this unit is a
                // single tile no K load has waited for that. The epilogue before needs nothing that
                // this warp does from here on. One gate is unfinished at a time, so the parities are plain.
                const int s = (jj - 1) & 1;
                ok = mbar_wait(&bars.k_empty[s], ((jj - 1) >> 1) & 1);
                if (ok && gate_in >= 0) ok = mbar_wait(&bars.epi_done, (wholes - 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (ok && lane == 0) {
                    mbar_expect_tx(&bars.g_full, PP_TILE);
                    for (int c = 0; c < 4; ++c)
                        tma_load_3d(sK + s * PP_TILE + c * (PP_BM * 128), &tmG, GQA_HD + 64 * c, w.at.y * group,
                                    w.row0 + w.at.z * tokens, &bars.g_full);
                }
                gate_in = s;
                ++wholes;
            }
        }
    } else if (warp == 2) {
        // ------------------------------------------------ MMA issuer
        if (lane == 0) {
            constexpr uint32_t ID_QK = tc::idesc_bf16(PP_BM, PP_BN, 0, 0);
            constexpr uint32_t ID_PV = tc::idesc_bf16(PP_BM, GQA_HD, 0, 1);
            const uint32_t aK = smem_u32(sK), aV = smem_u32(sV), aP = smem_u32(sP);
            auto issue_s = [&](int j) -> bool {
                const int s = j & 1;
                if (!mbar_wait(&bars.k_full[s], (j >> 1) & 1)) return false;
                if (j >= 1 && !mbar_wait(&bars.s_free, (j - 1) & 1)) return false;   // S(j-1) read out
                tc::fence_after();
#pragma unroll
                for (int kk = 0; kk < GQA_HD / 16; ++kk)
                    tc::mma_bf16_ts(tS, tQ + kk * 8, pp_desc_k(aK + s * PP_TILE + (kk >> 2) * 1024 + (kk & 3) * 32), ID_QK,
                                    kk > 0 ? 1u : 0u);
                tc::commit(&bars.s_full);
                tc::commit(&bars.k_empty[s]);
                return true;
            };
            auto issue_pv = [&](int j, bool fresh) -> bool {
                if (!mbar_wait(&bars.p_full, j & 1)) return false;
                if (!mbar_wait(&bars.v_full, j & 1)) return false;
                tc::fence_after();
#pragma unroll
                for (int kk = 0; kk < PP_BN / 16; ++kk) {
                    const uint64_t da = tc::desc_k_sw128(aP + (kk >> 2) * (PP_BM * 128) + (kk & 3) * 32);
                    const uint64_t db = tc::desc_mn_sw128(aV + kk * 8192, 1024, 4096);
                    tc::mma_bf16(tO, da, db, ID_PV, (!fresh || kk > 0) ? 1u : 0u);
                }
                tc::commit(&bars.pv_done);
                tc::commit(&bars.v_empty);
                return true;
            };
            bool ok = true;
            for (int pc = 0; ok && w.piece(tokens); w.next(p, tokens), ++pc) {
                ok = mbar_wait(&bars.q_tmem, pc & 1);
                tc::fence_after();
                if (ok) ok = issue_s(jj);
                for (int j = w.at.w; ok && j < w.t1; ++j, ++jj) {
                    if (j + 1 < w.t1) ok = issue_s(jj + 1);
                    if (ok) ok = issue_pv(jj, j == w.at.w);
                }
            }
        }
    } else {
        // ------------------------------------------------ q, softmax, epilogue
        // Waits never break out of the loops here (a time-out raises the error
        // word and they run on): all 256 threads meet at the named barrier.
        const int quarter = warp & 3, sw = warp - 3, u = sw >> 2;
        const int g = lane >> 2, tq = lane & 3;
        const int rbase = 32 * quarter + 16 * u;
        const uint32_t lane_off = (uint32_t)rbase << 16;
        const int row0 = rbase + g, row1 = row0 + 8;
        const float sl2 = p.scale_log2;
        const __nv_bfloat16 *qg = static_cast<const __nv_bfloat16 *>(p.qg);
        int wholes = 0;
        int pc = 0;
        // ---- q of piece x: a warp copies its 16 rows (row = token * group + head) into the V buffer, in
        // 128B-swizzled 64-column blocks, norms and ropes them there, and they go to TMEM as bf16
        // pairs. The V buffer and Q's columns are free: the piece before has done its last product.
        auto load_q = [&](const PpWalk &x) {
            const int t_first = x.at.z * tokens;
#pragma unroll 4
            for (int r = 16 * sw; r < 16 * sw + 16; ++r) {
                const int t = min(t_first + (r >> gs), x.n - 1);
                copy16_async(sV + (lane >> 3) * (PP_BM * 128) + r * 128 + (((lane & 7) ^ (r & 7)) << 4),
                             qg + ((size_t)(x.row0 + t) * p.H + x.at.y * group + (r & (group - 1))) * 2 * GQA_HD + lane * 8);
            }
            // the angles of the warp's 16 / group (at least one) tokens in the P buffer, `fit` tokens at a time
            const int half = p.rot >> 1, many = max(1, 16 >> gs), fit = min(many, 1024 / p.rot);
            float *cs = reinterpret_cast<float *>(sP + sw * 4096), *sn = cs + fit * half;
            const int r = 16 * sw + (lane >> 4) * 8 + ((lane >> 3) & 1) + 2 * ((lane >> 1) & 3);   // lanes of a phase: all banks
#pragma unroll 1
            for (int t0 = 0; t0 < many; t0 += fit) {
                const int first = t_first + ((16 * sw) >> gs) + t0;
                __syncwarp();
#pragma unroll 1
                for (int i = lane; i < fit * half; i += 32) {
                    const int t = i / half;
                    pages_rope_entry(cs + i, sn + i, x.base + first + t, bars.turn[i - t * half]);
                }
                if (t0 == 0) copies_wait();
                __syncwarp();
                const int mine = t_first + (r >> gs) - first;
                PpRow row{sV + r * 128, r & 7, mine >= 0 && mine < fit};
                const int at = row.on ? mine * half : 0;
                pages_norm_rope_rows<2>(row, lane & 1, bars.w1, p.eps, p.rot, cs + at, sn + at);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(PP_SOFTMAX) : "memory");
            const int tr = 32 * quarter + lane;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                float v[32];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int d = 128 * u + 64 * hh + 8 * c;
                    const uint4 y = *reinterpret_cast<const uint4 *>(
                        sV + (d >> 6) * (PP_BM * 128) + tr * 128 + ((((d & 63) >> 3) ^ (tr & 7)) << 4));
                    v[4 * c] = __uint_as_float(y.x); v[4 * c + 1] = __uint_as_float(y.y);
                    v[4 * c + 2] = __uint_as_float(y.z); v[4 * c + 3] = __uint_as_float(y.w);
                }
                tc::st32(tQ + 64 * u + 32 * hh + ((uint32_t)(32 * quarter) << 16), v);
            }
            tc::wait_st();
            tc::fence_before();
            fence_proxy_async();            // what was written and read here before V tiles land in its place
            mbar_arrive(&bars.q_tmem);
        };
        bool more = w.piece(tokens);
        if (more) load_q(w);
        while (more) {
            const int tok0 = w.at.z * tokens, end = w.base + w.n;
            const int qpos0 = w.base + tok0 + (row0 >> gs), qpos1 = w.base + tok0 + (row1 >> gs);
            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
            for (int i = w.at.w; i < w.t1; ++i, ++jj) {
                mbar_wait(&bars.s_full, jj & 1);
                tc::fence_after();
                float x[64];
                {
                    float xa[32], xb[32];
                    tc::ld16x256_x8(tS + lane_off, xa);
                    tc::ld16x256_x8(tS + 64 + lane_off, xb);
                    tc::wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; ++e) { x[e] = xa[e]; x[32 + e] = xb[e]; }
                }
                tc::fence_before();
                mbar_arrive(&bars.s_free);
                // x[4j + 0/1]: row0, keys 8j + 2tq, +1; x[4j + 2/3]: row1. Raw scores; the
                // scale is applied inside the exponent (it is positive: the maximum commutes)
                const int key0 = i * PP_BN;
                if (key0 + PP_BN - 1 > qpos0) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int k = key0 + 8 * j + 2 * tq;
                        if (k > qpos0) x[4 * j] = -INFINITY;
                        if (k + 1 > qpos0) x[4 * j + 1] = -INFINITY;
                        if (k > qpos1) x[4 * j + 2] = -INFINITY;
                        if (k + 1 > qpos1) x[4 * j + 3] = -INFINITY;
                    }
                }
                float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    mx0 = fmaxf(mx0, fmaxf(x[4 * j], x[4 * j + 1]));
                    mx1 = fmaxf(mx1, fmaxf(x[4 * j + 2], x[4 * j + 3]));
                }
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
                mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2)) * sl2;
                mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2)) * sl2;
                const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
                if (i == w.at.w) {
                    m0 = mn0; m1 = mn1;
                } else {
                    const bool need0 = mn0 > m0 + PF_RESCALE_LOG2, need1 = mn1 > m1 + PF_RESCALE_LOG2;
                    if (__any_sync(0xffffffffu, need0 || need1)) {
                        mbar_wait(&bars.pv_done, (jj - 1) & 1);        // O complete up to the tile before
                        tc::fence_after();
                        const float a0 = need0 ? ex2_approx(m0 - mn0) : 1.f, a1 = need1 ? ex2_approx(m1 - mn1) : 1.f;
#pragma unroll 1
                        for (int c = 0; c < GQA_HD / 64; ++c) {
                            float o[32];
                            tc::ld16x256_x8(tO + 64 * c + lane_off, o);
                            tc::wait_ld();
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                o[4 * j] *= a0; o[4 * j + 1] *= a0; o[4 * j + 2] *= a1; o[4 * j + 3] *= a1;
                            }
                            tc::st16x256_x8(tO + 64 * c + lane_off, o);
                        }
                        tc::wait_st();
                        if (need0) { l0 *= a0; m0 = mn0; }
                        if (need1) { l1 *= a1; m1 = mn1; }
                    }
                }
                const float mu0 = (m0 == -INFINITY) ? 0.f : m0, mu1 = (m1 == -INFINITY) ? 0.f : m1;
                uint32_t pk0[16], pk1[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float p00 = ex2_approx(fmaf(x[4 * j], sl2, -mu0)), p01 = ex2_approx(fmaf(x[4 * j + 1], sl2, -mu0));
                    const float p10 = ex2_approx(fmaf(x[4 * j + 2], sl2, -mu1)), p11 = ex2_approx(fmaf(x[4 * j + 3], sl2, -mu1));
                    l0 += p00 + p01;
                    l1 += p10 + p11;
                    pk0[j] = pack_bf16(p00, p01);
                    pk1[j] = pack_bf16(p10, p11);
                }
                if (i > w.at.w) mbar_wait(&bars.pv_done, (jj - 1) & 1);   // the P buffer's last reader
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int at = (j >> 3) * (PP_BM * 128);
                    *reinterpret_cast<uint32_t *>(sP + at + row0 * 128 + (((j & 7) ^ (row0 & 7)) << 4) + 4 * tq) = pk0[j];
                    *reinterpret_cast<uint32_t *>(sP + at + row1 * 128 + (((j & 7) ^ (row1 & 7)) << 4) + 4 * tq) = pk1[j];
                }
                if (key0 + PP_BN > end && (end & 7) && end > key0 && sw == 0) {
                    // V rows end .. end | 7 of the tile's last group hold what the page held before
                    mbar_wait(&bars.v_full, jj & 1);
                    const int from = end - key0, n = 8 - (end & 7);
                    for (int j = lane; j < n * 32; j += 32) {
                        const int r = from + (j >> 5), c = (j & 31) >> 3;
                        *reinterpret_cast<uint4 *>(sV + (r >> 3) * 4096 + c * 1024 + (r & 7) * 128 + (j & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                }
                fence_proxy_async();
                mbar_arrive(&bars.p_full);
            }
            l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
            l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
            const bool whole = w.ends && w.at.w == 0;
            const size_t slot = 2 * cta + (w.at.w == 0 ? 1 : 0);
            if (tq == 0) {
                bars.lsum[row0] = l0; bars.lsum[row1] = l1;
                if (!whole) {
                    part.ml[slot * PP_BM + row0] = make_float2(m0, l0);
                    part.ml[slot * PP_BM + row1] = make_float2(m1, l1);
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(PP_SOFTMAX) : "memory");
            mbar_wait(&bars.pv_done, (jj - 1) & 1);
            tc::fence_after();
            // completed before pv_done, and the next V tile waits for the next piece's q: never false; it orders
            // the read behind the V loader's write
            mbar_try_wait(&bars.v_full, (jj - 1) & 1);
            const int clean_from = bars.clean_from[pc++ & 1];
            // the next piece's q first: its S runs during this epilogue
            PpWalk nx = w;
            nx.next(p, tokens);
            more = nx.piece(tokens);
            if (more) load_q(nx);
            const int row = 32 * quarter + lane;
            const uint32_t qoff = (uint32_t)(32 * quarter) << 16;
            if (whole) {
                // thread = tile row, O columns 128 u ..; ctx takes the gate's place in its
                // 128B-swizzled 64 x 128 boxes; then a warp per row to memory
                const float inv_l = 1.f / bars.lsum[row];
                uint8_t *gt = sK + ((jj - 1) & 1) * PP_TILE;
                mbar_wait(&bars.g_full, wholes++ & 1);
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    float o[32];
                    const int d0 = 128 * u + 32 * c;
                    tc::ld32(tO + d0 + qoff, o);
                    tc::wait_ld();
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int chunk = ((d0 & 63) >> 3) + k;
                        const uint32_t off = (d0 >> 6) * (PP_BM * 128) + row * 128 + ((chunk ^ (row & 7)) << 4);
                        float gv[8], y[8];
                        load8v(reinterpret_cast<const __nv_bfloat16 *>(gt + off), gv);
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = o[8 * k + e] * inv_l;
                        gate4(y, gv);
                        gate4(y + 4, gv + 4);
                        store8v(reinterpret_cast<__nv_bfloat16 *>(gt + off), y);
                    }
                }
                asm volatile("bar.sync 1, %0;" ::"n"(PP_SOFTMAX) : "memory");
#pragma unroll 4
                for (int i = 0; i < 16; ++i) {
                    const int r = 16 * sw + i, t = tok0 + (r >> gs);
                    if (t >= w.n) break;
                    const uint4 x = *reinterpret_cast<const uint4 *>(gt + (lane >> 3) * (PP_BM * 128) + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                    *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.ctx) +
                                               ((size_t)(w.row0 + t) * p.H + w.at.y * group + (r & (group - 1))) * GQA_HD + lane * 8) = x;
                }
                if (__builtin_expect(clean_from >= 0, 0)) {
                    // what was cleared of v, to the rows that see it: the thread's 8 dims of the warp's rows
                    float v[8];
#pragma unroll 1
                    for (int r = 16 * sw; r < 16 * sw + 16; ++r) {
                        const int t = tok0 + (r >> gs);
                        if (t >= w.n) break;
                        if (r == 16 * sw || (r & (group - 1)) == 0) pp_cleared(p, w, clean_from, w.base + t, lane * 8, v);
                        const size_t at = (size_t)(w.row0 + t) * p.H + w.at.y * group + (r & (group - 1));
                        __nv_bfloat16 *y = static_cast<__nv_bfloat16 *>(p.ctx) + at * GQA_HD + lane * 8;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (v[e] != 0.f) {
                                const float g = __bfloat162float(qg[at * 2 * GQA_HD + GQA_HD + lane * 8 + e]);
                                y[e] = __float2bfloat16_rn(__bfloat162float(y[e]) + v[e] * gate_of(g));
                            }
                    }
                }
                fence_proxy_async();        // read out: the stage takes K tiles again
                mbar_arrive(&bars.epi_done);
            } else {
                // O as it is, [16-byte column chunk][row]: a warp writes 512 bytes at a time
                float4 *out = reinterpret_cast<float4 *>(part.o) + slot * (PP_BM * GQA_HD / 4) + quarter * 32 + lane;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    float o[32];
                    tc::ld32(tO + 128 * u + 32 * c + qoff, o);
                    tc::wait_ld();
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        out[(32 * u + 8 * c + j) * PP_BM] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                }
                if (__builtin_expect(clean_from >= 0, 0)) {
                    float v[8];
#pragma unroll 1
                    for (int d = 128 * u; d < 128 * u + 128; d += 8) {
                        pp_cleared(p, w, clean_from, w.base + tok0 + (row >> gs), d, v);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (v[e] != 0.f) reinterpret_cast<float *>(out + (d >> 2) * PP_BM)[(e >> 2) * PP_BM * 4 + (e & 3)] += v[e];
                    }
                }
            }
            tc::fence_before();             // O read: the next piece's products overwrite it (behind p_full)
            w = nx;
        }
    }
    tc::fence_before();
    __syncthreads();
    if (warp == 2) {
        tc::fence_after();
        tc::dealloc(tbase, 512);
    }
    griddep_wait();                         // this grid ends after the one before, also where no tile waited for it
}

// The unit that begins in CTA a and goes on, and the number of its pieces; false
// where there is none. A whole CTA of at least `ctas` threads.
__device__ __forceinline__ bool pp_split_unit(const PagesPart &part, int a, int ctas, int4 &unit, int &n)
{
    const int4 first = part.plan[a];
    unit = part.plan[a + 1];
    const int4 u = unit;
    auto same = [&](const int4 &x) { return x.x == u.x && x.y == u.y && x.z == u.z && x.w > 0; };
    if (u.w == 0 || same(first)) return false;
    const int at = a + 1 + (int)threadIdx.x;
    n = 1 + __syncthreads_count(at <= ctas && same(part.plan[at]));
    return true;
}

// Two joins. Many units on the GPU: few pieces each, and one CTA per (unit, 32
// rows, 128 dims) adds them up, lane = row, a warp 4 x 4 dims whose loads go out
// together, then turns the block to write 256-byte runs. Few units (a quarter of
// the CTAs or less): many pieces each, and one CTA per (unit, 32 rows, 32 dims) has
// its warps take every eighth of them. A call with 16 rows
// after 28672 takes 50 us with the second and 93 with the first, one row after 4096 24 and 29; 1024
// rows (128 units) 45 with the second and 38 with the first, nine mixed chunks 195 and 183.
constexpr int PJ_THREADS = 256, PJ_DIMS = 128;
__global__ void __launch_bounds__(PJ_THREADS)
pages_prefill_join_kernel(GqaPagesArgs p, PagesPart part)
{
    __shared__ __align__(16) float turned[32][PJ_DIMS + 4];
    const int a = blockIdx.x, quarter = blockIdx.y & 3, block = blockIdx.y >> 2, tid = threadIdx.x, j = tid >> 5, lane = tid & 31;
    griddep_wait();
    if (blockIdx.x + blockIdx.y + tid == 0 && *part.odd != 0) *part.odd = 0;    // for the next call (a store holds up the grid's end)
    int4 unit;
    int n;
    if (!pp_split_unit(part, a, gridDim.x, unit, n)) return;
    const int row = quarter * 32 + lane;
    float m = -INFINITY, l = 0.f, o[4][4] = {};
#pragma unroll 2
    for (int s = 0; s < n; ++s) {
        const size_t slot = s ? 2 * (a + s) : 2 * a + 1;
        const float2 ml = part.ml[slot * PP_BM + row];
        float4 x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            x[c] = reinterpret_cast<const float4 *>(part.o)[slot * (PP_BM * GQA_HD / 4) + (block * (PJ_DIMS / 4) + 8 * c + j) * PP_BM + row];
        if (piece_empty(ml)) continue;
        const float mn = fmaxf(m, ml.x), fo = m == -INFINITY ? 0.f : ex2_approx(m - mn), fs = ex2_approx(ml.x - mn);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            o[c][0] = o[c][0] * fo + x[c].x * fs; o[c][1] = o[c][1] * fo + x[c].y * fs;
            o[c][2] = o[c][2] * fo + x[c].z * fs; o[c][3] = o[c][3] * fo + x[c].w * fs;
        }
        l = l * fo + ml.y * fs;
        m = mn;
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        *reinterpret_cast<float4 *>(&turned[lane][32 * c + 4 * j]) = make_float4(o[c][0] * inv, o[c][1] * inv, o[c][2] * inv, o[c][3] * inv);
    __syncthreads();
    int row0, base;
    const int rows = pages_rows_of(p, unit.x, row0, base);
    const int group = p.H / p.pv.KH, gs = __ffs(group) - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {           // a warp per row, 4 dims to a lane
        const int r = 8 * i + j, tile_row = quarter * 32 + r, t = (unit.z * PP_BM + tile_row) >> gs;
        if (t >= rows) continue;
        const size_t at = (size_t)(row0 + t) * p.H + unit.y * group + (tile_row & (group - 1));
        float g[4], y[4];
        load4(static_cast<const __nv_bfloat16 *>(p.qg) + at * 2 * GQA_HD + GQA_HD + block * PJ_DIMS + 4 * lane, g);
        load4(&turned[r][4 * lane], y);
        gate4(y, g);
        store4(static_cast<__nv_bfloat16 *>(p.ctx) + at * GQA_HD + block * PJ_DIMS + 4 * lane, y);
    }
}

constexpr int PJ_DEEP = 32;
__global__ void __launch_bounds__(PJ_THREADS)
pages_prefill_join_deep_kernel(GqaPagesArgs p, PagesPart part)
{
    __shared__ __align__(16) float acc[PJ_THREADS / 32][32][PJ_DEEP + 4];
    __shared__ float2 mls[PJ_THREADS / 32][32];
    const int a = blockIdx.x, quarter = blockIdx.y & 3, block = blockIdx.y >> 2, tid = threadIdx.x, j = tid >> 5, lane = tid & 31;
    griddep_wait();
    if (blockIdx.x + blockIdx.y + tid == 0 && *part.odd != 0) *part.odd = 0;    // for the next call (a store holds up the grid's end)
    int4 unit;
    int n;
    if (!pp_split_unit(part, a, gridDim.x, unit, n)) return;
    const int row = quarter * 32 + lane;
    float m = -INFINITY, l = 0.f, o[8][4] = {};
    for (int s = j; s < n; s += PJ_THREADS / 32) {
        const size_t slot = s ? 2 * (a + s) : 2 * a + 1;
        const float2 ml = part.ml[slot * PP_BM + row];
        float4 x[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
            x[c] = reinterpret_cast<const float4 *>(part.o)[slot * (PP_BM * GQA_HD / 4) + (block * (PJ_DEEP / 4) + c) * PP_BM + row];
        if (piece_empty(ml)) continue;
        const float mn = fmaxf(m, ml.x), fo = m == -INFINITY ? 0.f : ex2_approx(m - mn), fs = ex2_approx(ml.x - mn);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            o[c][0] = o[c][0] * fo + x[c].x * fs; o[c][1] = o[c][1] * fo + x[c].y * fs;
            o[c][2] = o[c][2] * fo + x[c].z * fs; o[c][3] = o[c][3] * fo + x[c].w * fs;
        }
        l = l * fo + ml.y * fs;
        m = mn;
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) *reinterpret_cast<float4 *>(&acc[j][lane][4 * c]) = make_float4(o[c][0], o[c][1], o[c][2], o[c][3]);
    mls[j][lane] = make_float2(m, l);
    __syncthreads();
    int row0, base;
    const int rows = pages_rows_of(p, unit.x, row0, base);
    const int group = p.H / p.pv.KH, gs = __ffs(group) - 1, r = tid >> 3, c = (tid & 7) * 4;
    const int tile_row = quarter * 32 + r, t = (unit.z * PP_BM + tile_row) >> gs;
    if (t >= rows) return;
    const size_t at = (size_t)(row0 + t) * p.H + unit.y * group + (tile_row & (group - 1));
    float g[4], y[4] = {}, M = -INFINITY, L = 0.f;
    load4(static_cast<const __nv_bfloat16 *>(p.qg) + at * 2 * GQA_HD + GQA_HD + block * PJ_DEEP + c, g);
#pragma unroll
    for (int w = 0; w < PJ_THREADS / 32; ++w) M = fmaxf(M, mls[w][r].x);
#pragma unroll
    for (int w = 0; w < PJ_THREADS / 32; ++w) {
        const float f = mls[w][r].x == -INFINITY ? 0.f : ex2_approx(mls[w][r].x - M);
        L += mls[w][r].y * f;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] += acc[w][r][c + e] * f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= 1.f / L;
    gate4(y, g);
    store4(static_cast<__nv_bfloat16 *>(p.ctx) + at * GQA_HD + block * PJ_DEEP + c, y);
}

cudaError_t launch_pages_prefill(const CUtensorMap &tk, const CUtensorMap &tv, const CUtensorMap &tv8, const CUtensorMap &tg,
                                 const GqaPagesArgs &a, const PagesPart &part, const RopeFreq &f, int ctas, cudaStream_t st)
{
    cudaError_t e = cudaFuncSetAttribute(pages_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PP_SMEM);
    if (e != cudaSuccess) return e;
    // at most that many units, and CTAs with work; the join looks at those only
    const int tokens = PP_BM / (a.H / a.pv.KH);
    const long long units = (long long)a.pv.KH * ((a.S + tokens - 1) / tokens + a.n_req);
    const long long work = units * (((long long)a.pv.max_pages * a.pv.page + PP_BN - 1) / PP_BN + PP_SETUP);
    const int used = (int)std::min<long long>(ctas, (work + PP_MIN - 1) / PP_MIN);
    pages_append_kernel<<<(int)(((long long)a.S * a.pv.KH + PA_WARPS - 1) / PA_WARPS), PA_WARPS * 32, 0, st>>>(a, f, part.odd);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 1;
    cfg.gridDim = dim3(used); cfg.blockDim = dim3(PP_THREADS); cfg.dynamicSmemBytes = PP_SMEM;
    if ((e = cudaLaunchKernelEx(&cfg, pages_prefill_kernel, tk, tv, tv8, tg, a, part, f)) != cudaSuccess) return e;
    const bool deep = 4 * units <= ctas;
    cfg.gridDim = dim3(used, 4 * GQA_HD / (deep ? PJ_DEEP : PJ_DIMS)); cfg.blockDim = dim3(PJ_THREADS); cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, deep ? pages_prefill_join_deep_kernel : pages_prefill_join_kernel, a, part);
}

}  // namespace coli
