// Host side of the paged KV cache: the handle, its argument checks and the
// launches of gqa_pages.cu and page_moves.cu.
//
// A handle names one pool of pages for all its layers, [layers][K, V]
// [n_pages][KH][page][256] bf16, in the caller's device memory or its own, the
// layers' q/k norm weights, and one workspace of a fixed size, so that no
// call after coli_cuda_pages_create allocates, frees or waits: every call can
// be captured into a graph.
//
// Included by backend.cu (one translation unit), after the backend state.
#include <cmath>
#include <new>

struct ColiCudaPages {
    uintptr_t handle;         // what the caller holds in its place
    int layers, n_pages, page, KH;
    uint8_t *base;
    bool own_base;
    float *norm_w;            // [layers][2][256]
    unsigned char *norm_set;  // [layers] (host)
    uint8_t *ws, *own_ws;
    CUtensorMap *maps;        // [layers][4] K and V in one box of 16 rows each; K, V in boxes of box_rows, V of 8
    int box_rows;
    int rot;                  // rotary frequencies as last used
    float theta;
    RopeFreq freq;
};

namespace {

constexpr int PAGES_MAX_LAYERS = MAX_LAYERS, PAGES_MAX_REQ = 1024, PAGES_MAX_PAGES = 1 << 20;
constexpr int PAGES_MAX_HANDLES = 256;
// Live pools. A caller's handle is no address but a count of pools made * 256 + slot, so that one
// kept past its pool's end (coli_cuda_pages_free, a shutdown) never names a later pool.
ColiCudaPages *g_pages[PAGES_MAX_HANDLES] = {};
uintptr_t g_pages_made = 0;

size_t pages_page_bytes(int KH, int page) { return (size_t)KH * page * GQA_HD * 2; }
size_t pages_norm_bytes(int layers) { return (size_t)layers * 2 * GQA_HD * 4; }
size_t pages_list_bytes(int n_pages) { return ((size_t)n_pages * 4 + 255) & ~size_t(255); }
// the workspace serves one call at a time: a compaction's lists, or an attention call's pieces
size_t pages_part_rows() { return (size_t)2 * G.num_sms * PP_BM; }   // decode: 8 rows to a piece, prefill: 128
size_t pages_part_bytes() { return pages_part_rows() * (GQA_HD * 4 + 8) + (size_t)G.num_sms * (4 * 512 + 2) * 16 + 32; }
size_t pages_ws_bytes(int n_pages)
{
    return (std::max(3 * pages_list_bytes(n_pages) + 256, pages_part_bytes()) + 255) & ~size_t(255);
}
PagesPart pages_part(uint8_t *ws)
{
    PagesPart t{};
    t.o = (float *)ws;
    t.ml = (float2 *)(ws + pages_part_rows() * GQA_HD * 4);
    t.park = (float4 *)(t.ml + pages_part_rows());
    t.units = (int4 *)(t.park + (size_t)G.num_sms * 4 * 512);
    t.plan = t.units + G.num_sms;
    t.odd = (int *)(t.plan + G.num_sms + 1);
    return t;
}

// Rows of 256 bf16 as (64 columns, 8 rows, 4 column blocks, groups of 8 rows), and
// `planes` such arrays `plane` bytes apart: one box is a run of whole row groups of
// every plane, [plane][group][block][8 rows][128 B] in shared memory, 128B-swizzled.
int make_pages_tmap(CUtensorMap *m, void *base, long long rows, int box_rows, int planes, size_t plane)
{
    cuuint64_t dims[5] = {64, 8, 4, (cuuint64_t)(rows / 8), (cuuint64_t)planes};
    cuuint64_t strides[4] = {GQA_HD * 2, 128, 8 * GQA_HD * 2, (cuuint64_t)plane};
    cuuint32_t box[5] = {64, 8, 4, (cuuint32_t)(box_rows / 8), (cuuint32_t)planes};
    cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    CUresult r = G.encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, planes > 1 ? 5 : 4, base, dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("cuTensorMapEncodeTiled (pages) failed (%d)", (int)r);
    return 1;
}

int pages_geometry(int layers, int n_pages, int page, int KH, int hd)
{
    if (layers < 1 || layers > PAGES_MAX_LAYERS) return fail("pages: layers %d out of 1..%d", layers, PAGES_MAX_LAYERS);
    if (n_pages < 1 || n_pages > PAGES_MAX_PAGES) return fail("pages: n_pages %d out of 1..%d", n_pages, PAGES_MAX_PAGES);
    if (page < 16 || page > 1024 || page % 16) return fail("pages: page %d is not a multiple of 16 up to 1024", page);
    if (KH < 1 || KH > 64 || hd != GQA_HD) return fail("pages: unsupported shape KH=%d hd=%d (needs KH 1..64, hd=256)", KH, hd);
    if ((long long)n_pages * page * KH > 0x7fffffffLL) return fail("pages: %d pages of %d x %d rows pass 2^31 rows", n_pages, page, KH);
    return 1;
}

ColiCudaPages *pages_find(const ColiCudaPages *handle)
{
    ColiCudaPages *p = g_pages[(uintptr_t)handle % PAGES_MAX_HANDLES];
    return p && p->handle == (uintptr_t)handle ? p : nullptr;
}
int pages_usable(ColiCudaPages **p, const ColiCudaPages *handle)
{
    READY();
    *p = pages_find(handle);
    if (!*p) return fail("pages: not a live handle (coli_cuda_pages_create)");
    int dev = -1;
    CK(cudaGetDevice(&dev));
    if (dev != G.device) return fail("pages: device %d is current, the backend runs on device %d", dev, G.device);
    return 1;
}

void pages_release(ColiCudaPages *p)
{
    if (p->own_base) dev_free(p->base, (size_t)p->layers * 2 * p->n_pages * pages_page_bytes(p->KH, p->page));
    dev_free(p->norm_w, pages_norm_bytes(p->layers));
    dev_free(p->own_ws, pages_ws_bytes(p->n_pages));
    delete[] p->norm_set;
    delete[] p->maps;
    delete p;
}

// Handles freed while the backend stream was capturing: waiting for it there
// would end the capture, so that is left to the next call that may.
ColiCudaPages *g_pages_freed[PAGES_MAX_HANDLES] = {};
bool pages_capturing()
{
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(stream(), &st) != cudaSuccess) {
        cudaGetLastError();                // the legacy stream, which cannot be used while a blocking stream captures
        return true;
    }
    return st != cudaStreamCaptureStatusNone;
}
// A pool may be freed at any time (the Python object's is by garbage collection), so also while a
// stream other than the backend's captures in the global mode, in which this thread's cudaFree would
// end that capture: the memory is none of the capture's business, and the relaxed mode says so.
struct RelaxedCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};
void pages_release_freed()
{
    RelaxedCapture relaxed;
    for (int i = 0; i < PAGES_MAX_HANDLES; ++i) {
        if (!g_pages_freed[i]) continue;
        cudaStreamSynchronize(stream());   // queued calls may still use the pool and the workspace
        pages_release(g_pages_freed[i]);
        g_pages_freed[i] = nullptr;
    }
}

void pages_shutdown()
{
    pages_release_freed();
    for (int i = 0; i < PAGES_MAX_HANDLES; ++i) {
        if (g_pages[i]) pages_release(g_pages[i]);
        g_pages[i] = nullptr;
    }
}

// The word as coli_cuda_sync read it: 1, or cleared and reported.
int pages_error_ok(int h)
{
    if (h == PAGES_OK) return 1;
    const int zero = 0;
    CK(cudaMemcpyToSymbolAsync(g_dev_errors, &zero, sizeof(int), offsetof(DevErrors, pages), cudaMemcpyHostToDevice, stream()));
    CK(cudaStreamSynchronize(stream()));
    static const char *const what[] = {"", "a page id outside the pool", "a position or length beyond the page table",
                                       "row offsets that do not ascend within the rows given",
                                       "pages or requests named twice, or both read and written",
                                       "a request index out of range"};
    return fail("pages: a call met %s (error %d); what it names was left out", h >= 1 && h <= 5 ? what[h] : "an error", h);
}

PageMoveArgs pages_move_args(const ColiCudaPages *p)
{
    PageMoveArgs m{};
    m.base = p->base; m.page_bytes = pages_page_bytes(p->KH, p->page);
    m.layers = p->layers; m.n_pages = p->n_pages; m.page = p->page; m.KH = p->KH;
    return m;
}

// The checks that the two attention calls share, and their kernel arguments.
int pages_attend_args(GqaPagesArgs &a, ColiCudaPages *p, int layer, const void *qg, const void *k, const void *v,
                      const int *base, const int *table, int max_pages, void *ctx, int H, int KH, int hd, int rot,
                      float eps, float theta)
{
    if (layer < 0 || layer >= p->layers) return fail("pages: layer %d out of range", layer);
    const int group = KH > 0 ? H / KH : 0;
    if (hd != GQA_HD || KH != p->KH || H != group * KH || (group != 1 && group != 2 && group != 4 && group != 8))
        return fail("pages: unsupported GQA shape H=%d KH=%d hd=%d (needs hd=256, KH=%d, H / KH 1, 2, 4 or 8)", H, KH, hd, p->KH);
    if (!p->norm_set[layer]) return fail("pages: q/k norm weights of layer %d not set (coli_cuda_pages_norm_weight)", layer);
    if (rot < 2 || rot > hd || (rot & 1)) return fail("pages: bad rot %d", rot);
    if (!(eps >= 0.f) || !(theta > 0.f) || std::isinf(eps) || std::isinf(theta)) return fail("pages: bad eps or theta");
    if (max_pages < 1 || (long long)max_pages * p->page > 1 << 30) return fail("pages: bad max_pages %d (max_pages * page up to 2^30)", max_pages);
    if (!qg || !k || !v || !base || !table || !ctx) return fail("pages: a null pointer among the arguments");
    if (((uintptr_t)qg | (uintptr_t)k | (uintptr_t)v | (uintptr_t)ctx) & 15)
        return fail("pages: qg, k, v and ctx must be 16-byte aligned");
    if (((uintptr_t)base | (uintptr_t)table) & 3) return fail("pages: index arrays must be 4-byte aligned");
    if (p->rot != rot || p->theta != theta) {
        for (int j = 0; j < rot / 2; ++j) {
            const double t = std::pow((double)theta, -2.0 * j / rot) / 6.283185307179586476925286766559;
            p->freq.turn[j] = (unsigned long long)((t - std::floor(t)) * 18446744073709551616.0);
        }
        p->rot = rot;
        p->theta = theta;
    }
    const size_t plane = (size_t)p->n_pages * pages_page_bytes(p->KH, p->page);
    a.pv.k = (__nv_bfloat16 *)(p->base + 2 * layer * plane);
    a.pv.v = (__nv_bfloat16 *)(p->base + (2 * layer + 1) * plane);
    a.pv.table = table; a.pv.n_pages = p->n_pages; a.pv.page = p->page; a.pv.KH = KH; a.pv.max_pages = max_pages;
    a.pv.tiles_div = FastDiv::of(p->page / GQA_TILE); a.pv.heads_div = FastDiv::of(KH);
    a.qg = qg; a.k = k; a.v = v; a.ctx = ctx; a.base = base;
    a.qnw = p->norm_w + (size_t)layer * 2 * GQA_HD; a.knw = a.qnw + GQA_HD;
    a.H = H; a.rot = rot; a.eps = eps;
    a.scale_log2 = (1.f / sqrtf((float)hd)) * 1.4426950408889634f;
    return 1;
}

// The gate halves of q|gate [S][H][2 hd] in boxes of 64 columns x the group's heads x 128 / group tokens.
int make_pages_gate_tmap(CUtensorMap *m, const void *qg, int S, int H, int group)
{
    cuuint64_t dims[3] = {2 * GQA_HD, (cuuint64_t)H, (cuuint64_t)S};
    cuuint64_t strides[2] = {2 * GQA_HD * 2, (cuuint64_t)H * 2 * GQA_HD * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)(PP_BM / group)};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = G.encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(qg), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail("cuTensorMapEncodeTiled (gate) failed (%d)", (int)r);
    return 1;
}

}  // namespace

extern "C" {

size_t coli_cuda_pages_bytes(int layers, int n_pages, int page, int KH, int hd)
{
    if (!pages_geometry(layers, n_pages, page, KH, hd)) return 0;
    return (size_t)layers * 2 * n_pages * pages_page_bytes(KH, page);
}

int coli_cuda_pages_create(ColiCudaPages **pages, int layers, int n_pages, int page, int KH, int hd, void *kv_dev)
{
    READY();
    if (!pages) return fail("pages: null handle");
    if (!pages_geometry(layers, n_pages, page, KH, hd)) return 0;
    if ((uintptr_t)kv_dev & 127) return fail("pages: kv_dev must be 128-byte aligned");
    if (pages_capturing()) return fail("pages: a pool cannot be made while the backend stream is capturing");
    pages_release_freed();
    int slot = 0;
    while (slot < PAGES_MAX_HANDLES && g_pages[slot]) ++slot;
    if (slot == PAGES_MAX_HANDLES) return fail("pages: %d handles are alive already", PAGES_MAX_HANDLES);
    ColiCudaPages *p = new (std::nothrow) ColiCudaPages();
    if (!p) return fail("pages: out of host memory");
    p->layers = layers; p->n_pages = n_pages; p->page = page; p->KH = KH;
    p->base = (uint8_t *)kv_dev;
    p->norm_set = new (std::nothrow) unsigned char[layers]();
    p->maps = new (std::nothrow) CUtensorMap[4 * layers];
    const size_t bytes = (size_t)layers * 2 * n_pages * pages_page_bytes(KH, page);
    int ok = p->norm_set && p->maps;
    if (!ok) fail("pages: out of host memory");
    if (ok && !kv_dev) {
        ok = dev_alloc((void **)&p->base, bytes);
        p->own_base = ok;
        if (ok && cudaMemsetAsync(p->base, 0, bytes, stream()) != cudaSuccess) ok = cuda_fail(cudaGetLastError(), "pages memset");
    }
    ok = ok && dev_alloc((void **)&p->norm_w, pages_norm_bytes(layers)) && dev_alloc((void **)&p->own_ws, pages_ws_bytes(n_pages));
    if (ok && cudaMemsetAsync(pages_part(p->own_ws).odd, 0, 16, stream()) != cudaSuccess) ok = cuda_fail(cudaGetLastError(), "pages memset");
    p->ws = p->own_ws;
    p->box_rows = std::min(PP_BN, page & -page);
    for (int i = 0; ok && i < layers; ++i) {
        uint8_t *k = p->base + (size_t)i * (bytes / layers), *v = k + bytes / layers / 2;
        const long long rows = (long long)n_pages * KH * page;
        CUtensorMap *m = p->maps + 4 * i;
        ok = make_pages_tmap(m, k, rows, GQA_TILE, 2, v - k) && make_pages_tmap(m + 1, k, rows, p->box_rows, 1, 0) &&
             make_pages_tmap(m + 2, v, rows, p->box_rows, 1, 0) && make_pages_tmap(m + 3, v, rows, 8, 1, 0);
    }
    if (!ok) { pages_release(p); return 0; }
    p->handle = ++g_pages_made * PAGES_MAX_HANDLES + slot;
    g_pages[slot] = p;
    *pages = (ColiCudaPages *)p->handle;
    return 1;
}

void coli_cuda_pages_free(ColiCudaPages *handle)
{
    ColiCudaPages *p = pages_find(handle);
    if (!p) return;
    const int slot = (int)(p->handle % PAGES_MAX_HANDLES);
    if (g_pages_freed[slot]) return;       // as many are waiting for a capture to end as there can be handles
    g_pages[slot] = nullptr;
    g_pages_freed[slot] = p;
    if (!pages_capturing()) pages_release_freed();
}

int coli_cuda_pages_device_ptr(const ColiCudaPages *handle, int layer, void **k, void **v)
{
    ColiCudaPages *pages;
    if (!pages_usable(&pages, handle)) return 0;
    if (layer < 0 || layer >= pages->layers) return fail("pages: layer %d out of range", layer);
    const size_t plane = (size_t)pages->n_pages * pages_page_bytes(pages->KH, pages->page);
    if (k) *k = pages->base + 2 * layer * plane;
    if (v) *v = pages->base + (2 * layer + 1) * plane;
    return 1;
}

int coli_cuda_pages_norm_weight(ColiCudaPages *handle, int layer, const float *qnw, const float *knw, int hd)
{
    ColiCudaPages *pages;
    if (!pages_usable(&pages, handle)) return 0;
    if (layer < 0 || layer >= pages->layers) return fail("pages: layer %d out of range", layer);
    if (hd != GQA_HD || !qnw || !knw) return fail("pages: bad norm weights (hd=%d)", hd);
    if (pages_capturing()) return fail("pages: norm weights cannot be set while the backend stream is capturing");
    float *d = pages->norm_w + (size_t)layer * 2 * GQA_HD;
    CK(cudaMemcpyAsync(d, qnw, GQA_HD * 4, cudaMemcpyHostToDevice, stream()));
    CK(cudaMemcpyAsync(d + GQA_HD, knw, GQA_HD * 4, cudaMemcpyHostToDevice, stream()));
    CK(cudaStreamSynchronize(stream()));
    pages->norm_set[layer] = 1;
    return 1;
}

size_t coli_cuda_pages_workspace_bytes(const ColiCudaPages *handle)
{
    ColiCudaPages *pages;
    return pages_usable(&pages, handle) ? pages_ws_bytes(pages->n_pages) : 0;
}

int coli_cuda_pages_set_workspace(ColiCudaPages *handle, void *ws, size_t bytes)
{
    ColiCudaPages *pages;
    if (!pages_usable(&pages, handle)) return 0;
    if (ws && (bytes < pages_ws_bytes(pages->n_pages) || ((uintptr_t)ws & 255)))
        return fail("pages: the workspace needs %zu bytes, 256-byte aligned", pages_ws_bytes(pages->n_pages));
    pages->ws = ws ? (uint8_t *)ws : pages->own_ws;
    return 1;
}

int coli_cuda_gqa_decode_pages_dev(ColiCudaPages *handle, int layer, int B, const void *qg, const void *k, const void *v,
                                   const int *pos_dev, const int *table, int max_pages, void *ctx, int H, int KH, int hd,
                                   int rot, float eps, float theta, int dtype)
{
    ColiCudaPages *pages;
    if (!pages_usable(&pages, handle)) return 0;
    if (dtype != 0 && dtype != 1) return fail("dtype must be 0 (fp32) or 1 (bf16)");
    if (B < 0 || B > PAGES_MAX_REQ) return fail("pages: batch %d out of 0..%d", B, PAGES_MAX_REQ);
    if (B == 0) return 1;
    GqaPagesArgs a{};
    if (!pages_attend_args(a, pages, layer, qg, k, v, pos_dev, table, max_pages, ctx, H, KH, hd, rot, eps, theta)) return 0;
    if (((long long)max_pages * (pages->page / GQA_TILE) + PD_WHOLE + 3) * B * pages->KH > 1 << 30)
        return fail("pages: a table of %d x %d pages passes 2^30 tiles", B, max_pages);
    a.n_req = a.S = B;
    CK(launch_pages_decode(pages->maps[4 * layer], a, pages_part(pages->ws), pages->freq, dtype,
                           G.num_sms, stream()));
    g_launches += 2;
    return 1;
}

int coli_cuda_gqa_prefill_pages_dev(ColiCudaPages *handle, int layer, int n_seq, int S, const int *cu, const int *pos_base,
                                    const void *qg, const void *k, const void *v, const int *table, int max_pages,
                                    void *ctx, int H, int KH, int hd, int rot, float eps, float theta, int dtype)
{
    ColiCudaPages *pages;
    if (!pages_usable(&pages, handle)) return 0;
    if (dtype != 1) return fail("pages: prefill takes bf16 activations (dtype 1)");
    if (n_seq < 0 || n_seq > PAGES_MAX_REQ) return fail("pages: %d sequences out of 0..%d", n_seq, PAGES_MAX_REQ);
    if (S < 0 || S > 1 << 24) return fail("pages: %d rows out of 0..2^24", S);
    if (n_seq == 0 || S == 0) return 1;
    if (!cu) return fail("pages: a null pointer among the arguments");
    if ((uintptr_t)cu & 3) return fail("pages: index arrays must be 4-byte aligned");
    GqaPagesArgs a{};
    if (!pages_attend_args(a, pages, layer, qg, k, v, pos_base, table, max_pages, ctx, H, KH, hd, rot, eps, theta)) return 0;
    a.cu = cu;
    a.n_req = n_seq; a.S = S;
    const CUtensorMap *m = pages->maps + 4 * layer;
    CUtensorMap gate;
    if (!make_pages_gate_tmap(&gate, qg, S, H, H / KH)) return 0;
    a.box_rows = pages->box_rows;
    CK(launch_pages_prefill(m[1], m[2], m[3], gate, a, pages_part(pages->ws), pages->freq, G.num_sms, stream()));
    g_launches += 3;
    return 1;
}

int coli_cuda_pages_copy_dev(ColiCudaPages *handle, int n, const int *src, const int *dst)
{
    ColiCudaPages *pages;
    if (!pages_usable(&pages, handle)) return 0;
    if (n < 0 || n > pages->n_pages) return fail("pages: %d pairs for %d pages", n, pages->n_pages);
    if (n == 0) return 1;
    if (!src || !dst) return fail("pages: a null pointer among the arguments");
    if (((uintptr_t)src | (uintptr_t)dst) & 3) return fail("pages: index arrays must be 4-byte aligned");
    CK(launch_pages_copy(pages_move_args(pages), n, src, dst, stream()));
    g_launches += 1;
    return 1;
}

int coli_cuda_pages_fork_dev(ColiCudaPages *handle, int n, const int *parent, const int *child, const int *fresh, int *len,
                             int *table, int n_req, int max_pages)
{
    ColiCudaPages *pages;
    if (!pages_usable(&pages, handle)) return 0;
    if (n_req < 1 || max_pages < 1 || (long long)max_pages * pages->page > 1 << 30)
        return fail("pages: bad table %d x %d", n_req, max_pages);
    if (n < 0 || n >= n_req) return fail("pages: %d forks among %d requests", n, n_req);
    if (n == 0) return 1;
    if (!parent || !child || !fresh || !len || !table) return fail("pages: a null pointer among the arguments");
    if (((uintptr_t)parent | (uintptr_t)child | (uintptr_t)fresh | (uintptr_t)len | (uintptr_t)table) & 3)
        return fail("pages: index arrays must be 4-byte aligned");
    PageForkArgs f{};
    f.parent = parent; f.child = child; f.fresh = fresh; f.len = len; f.table = table;
    f.n = n; f.n_req = n_req; f.max_pages = max_pages; f.page_div = FastDiv::of(pages->page);
    CK(launch_pages_fork(pages_move_args(pages), f, stream()));
    g_launches += 1;
    return 1;
}

int coli_cuda_pages_compact_dev(ColiCudaPages *handle, int n_req, const int *len, const int *table, int max_pages,
                                int *table_out, int *live)
{
    ColiCudaPages *pages;
    if (!pages_usable(&pages, handle)) return 0;
    if (n_req < 1 || max_pages < 1 || (long long)max_pages * pages->page > 1 << 30)
        return fail("pages: bad table %d x %d", n_req, max_pages);
    if (!len || !table || !table_out || !live) return fail("pages: a null pointer among the arguments");
    if (((uintptr_t)len | (uintptr_t)table | (uintptr_t)table_out | (uintptr_t)live) & 3)
        return fail("pages: index arrays must be 4-byte aligned");
    PageCompactArgs c{};
    const size_t list = pages_list_bytes(pages->n_pages);
    c.len = len; c.table = table; c.table_out = table_out; c.live = live;
    c.src = (int *)pages->ws; c.dst = (int *)(pages->ws + list); c.remap = (int *)(pages->ws + 2 * list);
    c.count = (int *)(pages->ws + 3 * list);
    c.n_req = n_req; c.max_pages = max_pages;
    CK(launch_pages_compact(pages_move_args(pages), c, stream()));
    g_launches += 2;
    return 1;
}

}  // extern "C"
