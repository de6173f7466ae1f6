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
