// Moving pages of the paged KV cache: copies of whole pages, forks of
// requests, and compaction. One launch moves every layer's K and V; the
// kernels are plain copies, bound by HBM (each moved byte read and written).
//
// Page ids, request indices and lengths are checked on the device; what is
// out of range or in conflict raises g_dev_errors.pages and is left out.
#include "common.cuh"
#include "kernels.h"

namespace coli {

constexpr int MV_THREADS = 256, MV_CTAS = 148 * 128;

// Page `id` of plane y = 2 * layer + (0 K, 1 V).
__device__ __forceinline__ uint4 *page_at(const PageMoveArgs &m, int plane, int id)
{
    return reinterpret_cast<uint4 *>(m.base + ((size_t)plane * m.n_pages + id) * m.page_bytes);
}

// `words` 16-byte words by the CTA's threads, four loads in flight each.
__device__ __forceinline__ void copy_words(uint4 *to, const uint4 *from, int words)
{
    int j = threadIdx.x;
    for (; j + 3 * MV_THREADS < words; j += 4 * MV_THREADS) {
        uint4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __ldcs(from + j + i * MV_THREADS);
#pragma unroll
        for (int i = 0; i < 4; ++i) __stcs(to + j + i * MV_THREADS, x[i]);
    }
    for (; j < words; j += MV_THREADS) to[j] = from[j];
}

// ------------------------------------------------------------------ copy
// A CTA per pair and as many planes as leave MV_CTAS of them: each looks through all
// pairs first, which for many pairs and planes would otherwise cost more than the copies
// (45000 of 8 planes of 16 KiB: 2.98 ms, with a CTA per plane 10.6; 800 of 20 planes of 64 KiB:
// 319 us, 6.57 TB/s, either way, 327-336 with a quarter and a 16th of the CTAs). 8 pages of
// 20 planes of 16 KiB: 2.6 us in a graph, the latency of a launch and two dependent loads. A
// pair is left out when its destination is named by another pair too, or when its source is
// another pair's destination: either would make the result a matter of timing. A page onto
// itself is written by nobody, so other pairs may read it.
__global__ void __launch_bounds__(MV_THREADS)
pages_copy_kernel(PageMoveArgs m, int n, const int *src, const int *dst)
{
    const int i = blockIdx.x, s = src[i], d = dst[i];
    if ((unsigned)s >= (unsigned)m.n_pages || (unsigned)d >= (unsigned)m.n_pages) {
        pages_error(PAGES_BAD_ID);
        return;
    }
    int bad = 0;
    for (int j = threadIdx.x; j < n; j += MV_THREADS)
        if (j != i && (dst[j] == d || (dst[j] == s && src[j] != s))) bad = 1;
    if (__syncthreads_or(bad)) {
        pages_error(PAGES_CONFLICT);
        return;
    }
    if (s == d) return;
    for (int y = blockIdx.y; y < 2 * m.layers; y += gridDim.y)
        copy_words(page_at(m, y, d), page_at(m, y, s), (int)(m.page_bytes / 16));
}

// CTAs for n items in y, so that x * y come to about MV_CTAS.
static int mv_rows(const PageMoveArgs &m, int n) { return std::max(1, std::min(2 * m.layers, (MV_CTAS + n - 1) / n)); }

cudaError_t launch_pages_copy(const PageMoveArgs &m, int n, const int *src, const int *dst, cudaStream_t st)
{
    pages_copy_kernel<<<dim3(n, mv_rows(m, n)), MV_THREADS, 0, st>>>(m, n, src, dst);
    return cudaGetLastError();
}

// ------------------------------------------------------------------ fork
// CTAs as in a copy, per fork: the parent's started page is copied as far as it
// is filled; the CTAs of plane 0 write the child's table row and length. 256 forks of a
// page of 20 planes of 64 KiB: 43 us (359 MB; parents' pages are shared by 8 forks and read
// from L2); 4 forks: 4.5 us, the chain of dependent loads parent -> length -> page id -> rows.
// Every CTA looks through all forks for conflicts, as a copy's do: 1000 forks of short tails
// (4 layers, pages of 16 rows) take 42 us, 32 without the look at the other forks' started pages.
__global__ void __launch_bounds__(MV_THREADS)
pages_fork_kernel(PageMoveArgs m, PageForkArgs f)
{
    const int i = blockIdx.x, a = f.parent[i], c = f.child[i];
    if ((unsigned)a >= (unsigned)f.n_req || (unsigned)c >= (unsigned)f.n_req) {
        pages_error(PAGES_BAD_REQ);
        return;
    }
    const int len = f.len[a];
    if (len < 0 || (long long)len > (long long)f.max_pages * m.page) {
        pages_error(PAGES_BAD_POS);
        return;
    }
    const int full = len / m.page, tail = len - full * m.page;
    const int *row = f.table + (size_t)a * f.max_pages;
    const int to_id = f.fresh[i], from_id = tail ? row[full] : -1;
    if (tail && ((unsigned)to_id >= (unsigned)m.n_pages || (unsigned)from_id >= (unsigned)m.n_pages)) {
        pages_error(PAGES_BAD_ID);
        return;
    }
    // A child named twice, one that is also a parent, or a fresh page that another fork
    // uses too, as its own fresh one or as the started page that it copies: left out. The fresh
    // page of a parent that ends with a page is not used, whatever it says. (A parent's length and
    // row are written by no fork: its child would be a parent.)
    int bad = a == c;
    for (int j = threadIdx.x; j < f.n; j += MV_THREADS) {
        const int pj = f.parent[j], cj = f.child[j];
        if (pj == c || (j != i && (cj == c || cj == a))) bad = 1;
        if (tail && (unsigned)pj < (unsigned)f.n_req) {
            const int lj = max(f.len[pj], 0), fj = f.page_div(lj);
            if (fj < f.max_pages && lj - fj * m.page > 0 &&
                ((j != i && f.fresh[j] == to_id) || f.table[(size_t)pj * f.max_pages + fj] == to_id)) bad = 1;
        }
    }
    if (__syncthreads_or(bad)) {
        pages_error(PAGES_CONFLICT);
        return;
    }
    if (blockIdx.y == 0) {
        int *out = f.table + (size_t)c * f.max_pages;
        for (int j = threadIdx.x; j < full; j += MV_THREADS) out[j] = row[j];
        if (threadIdx.x == 0) {
            if (tail) out[full] = to_id;
            f.len[c] = len;
        }
    }
    if (tail == 0) return;
    const size_t per = (size_t)m.page * 32;      // 16-byte words of one head's rows in a page
    for (int y = blockIdx.y; y < 2 * m.layers; y += gridDim.y) {
        const uint4 *from = page_at(m, y, from_id);
        uint4 *to = page_at(m, y, to_id);
        for (int kh = 0; kh < m.KH; ++kh) copy_words(to + kh * per, from + kh * per, tail * 32);
    }
}

cudaError_t launch_pages_fork(const PageMoveArgs &m, const PageForkArgs &f, cudaStream_t st)
{
    pages_fork_kernel<<<dim3(f.n, mv_rows(m, f.n)), MV_THREADS, 0, st>>>(m, f);
    return cudaGetLastError();
}

// ------------------------------------------------------------------ compact
constexpr int CP_THREADS = 1024, CP_PIECE = 8 * MV_THREADS, CP_CTAS = 148 * 32;

// Exclusive prefix sums over the CTA's threads of two counts at once (low and
// high half); `total` is every thread's sums.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long x, unsigned long long &total)
{
    __shared__ unsigned long long part[CP_THREADS / 32 + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto scan = [&](unsigned long long v) {
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += y;
        }
        return v;
    };
    const unsigned long long inc = scan(x);
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    if (warp == 0) {                        // CP_THREADS / 32 = 32 warps
        const unsigned long long mine = part[lane], all = scan(mine);
        __syncwarp();
        part[lane] = all - mine;
        if (lane == 31) part[32] = all;
    }
    __syncthreads();
    total = part[32];
    const unsigned long long before = part[warp];
    __syncthreads();                        // the next scan writes here
    return before + inc - x;
}

// Pages that request r holds, 0 where its length is impossible.
__device__ __forceinline__ int pages_held(const PageMoveArgs &m, const PageCompactArgs &c, int r)
{
    const int len = c.len[r];
    if (len <= 0) return 0;
    if ((long long)len > (long long)c.max_pages * m.page) { pages_error(PAGES_BAD_POS); return 0; }
    return (len + m.page - 1) / m.page;
}

// One CTA, a bit per page in shared memory: mark what a request holds, count
// the live pages, then pair the k-th live page behind the count (a mover)
// with the k-th dead page before it (a hole). As many of the one as of the
// other: dead pages before n_live = n_live - (live pages before it). Latency alone: it and the
// move of 2.6 GB (half of 4000 pages of 20 planes of 64 KiB) take 414 us, 6.3 TB/s; with the
// 79 MB of half of 500 pages of 16 KiB 15.7 us in a graph, 12.1 of them the copy's.
__global__ void __launch_bounds__(CP_THREADS, 1)
pages_compact_plan_kernel(PageMoveArgs m, PageCompactArgs c)
{
    extern __shared__ uint32_t bits[];
    griddep_launch();
    const int words = (m.n_pages + 31) / 32, tid = threadIdx.x;
    for (int w = tid; w < words; w += CP_THREADS) bits[w] = 0;
    __syncthreads();
    for (int r = tid >> 5; r < c.n_req; r += CP_THREADS / 32) {
        const int held = pages_held(m, c, r);
        for (int j = tid & 31; j < held; j += 32) {
            const int id = c.table[(size_t)r * c.max_pages + j];
            if ((unsigned)id < (unsigned)m.n_pages) atomicOr(&bits[id >> 5], 1u << (id & 31));
            else pages_error(PAGES_BAD_ID);
        }
    }
    __syncthreads();
    const int per = (words + CP_THREADS - 1) / CP_THREADS, w0 = min(words, tid * per), w1 = min(words, w0 + per);
    unsigned long long mine = 0, total;
    for (int w = w0; w < w1; ++w) mine += __popc(bits[w]);
    block_scan(mine, total);
    const int live = (int)total;
    // of word w: the dead pages before `live`, and the live ones from there on
    auto low = [&](int w) { return w * 32 + 32 <= live ? ~0u : w * 32 >= live ? 0u : (1u << (live - w * 32)) - 1; };
    mine = 0;
    for (int w = w0; w < w1; ++w) mine += __popc(~bits[w] & low(w)) + ((unsigned long long)__popc(bits[w] & ~low(w)) << 32);
    const unsigned long long at = block_scan(mine, total);
    int h = (int)at, v = (int)(at >> 32);
    for (int w = w0; w < w1; ++w) {
        for (uint32_t x = ~bits[w] & low(w); x; x &= x - 1) c.dst[h++] = w * 32 + __ffs(x) - 1;
        for (uint32_t x = bits[w] & ~low(w); x; x &= x - 1) {
            const int id = w * 32 + __ffs(x) - 1;
            c.remap[id] = v;
            c.src[v++] = id;
        }
    }
    if (tid == 0) { *c.count = (int)(total >> 32); *c.live = live; }
}

// Moves the pages and writes the new table: every entry, those behind a
// request's length as they are. A page goes in pieces of 32 KiB, so that a few movers
// fill the GPU as many do.
__global__ void __launch_bounds__(MV_THREADS)
pages_compact_move_kernel(PageMoveArgs m, PageCompactArgs c, int piece)
{
    griddep_wait();                         // a programmatic dependent of the plan
    const int movers = *c.count, live = *c.live, words = (int)(m.page_bytes / 16);
    // blockIdx.y: a plane and a piece of the page; blockIdx.x and on: the movers, the next one's ids ahead
    const int pieces = (words + piece - 1) / piece, plane = blockIdx.y / pieces, at = (blockIdx.y - plane * pieces) * piece;
    int k = blockIdx.x, from = k < movers ? c.src[k] : 0, to = k < movers ? c.dst[k] : 0;
    while (k < movers) {
        k += gridDim.x;
        const int next_from = k < movers ? c.src[k] : 0, next_to = k < movers ? c.dst[k] : 0;
        copy_words(page_at(m, plane, to) + at, page_at(m, plane, from) + at, min(piece, words - at));
        from = next_from;
        to = next_to;
    }
    const long long cells = (long long)c.n_req * c.max_pages;
    const long long first = (blockIdx.y * (long long)gridDim.x + blockIdx.x) * MV_THREADS + threadIdx.x;
    for (long long i = first; i < cells; i += (long long)gridDim.x * gridDim.y * MV_THREADS) {
        const int r = (int)(i / c.max_pages), j = (int)(i - (long long)r * c.max_pages);
        int id = c.table[i];
        if (j < pages_held(m, c, r) && id >= live && id < m.n_pages) id = c.dst[c.remap[id]];
        c.table_out[i] = id;
    }
}

cudaError_t launch_pages_compact(const PageMoveArgs &m, const PageCompactArgs &c, cudaStream_t st)
{
    const size_t smem = (size_t)(m.n_pages + 31) / 32 * 4;     // 128 KiB at 2^20 pages
    cudaError_t e = cudaFuncSetAttribute(pages_compact_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 128 << 10);
    if (e != cudaSuccess) return e;
    pages_compact_plan_kernel<<<1, CP_THREADS, smem, st>>>(m, c);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    // pieces of a page: small enough that few pages fill the GPU, few enough for the grid's y
    const int words = (int)(m.page_bytes / 16), most = 65535 / (2 * m.layers), piece = std::max(CP_PIECE, (words + most - 1) / most);
    const int rows = 2 * m.layers * ((words + piece - 1) / piece);
    cfg.gridDim = dim3(std::max(1, std::min(m.n_pages, (CP_CTAS + rows - 1) / rows)), rows); cfg.blockDim = dim3(MV_THREADS); cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, pages_compact_move_kernel, m, c, piece);
}

}  // namespace coli
