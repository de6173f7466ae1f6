"""The paged KV cache on the GPU: decode and ragged prefill over pages, page
copies, forks and compaction, against a 64-bit restatement (pages_ref)."""
import numpy as np
import pytest

import pages_ref as ref
from conftest import load_pkg
from helpers import assert_close

pytestmark = pytest.mark.gpu

HD, ROT, EPS, THETA = 256, 64, 1e-6, 1e7


@pytest.fixture(scope="module")
def be():
    import torch
    pkg = load_pkg()
    pkg.build()
    b = pkg.Backend(0)
    b.set_stream(torch.cuda.current_stream().cuda_stream or 1)   # 1: the legacy default stream
    yield b
    b.shutdown()


def ints(x):
    import torch
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


class Pool:
    """A paged cache over a torch tensor, with norm weights per layer."""

    def __init__(self, be, n_pages, page, KH, layers=1, seed=0):
        import torch
        self.torch, self.be, self.page, self.KH = torch, be, page, KH
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.kv = self.randn(layers, 2, n_pages, KH, page, HD, dtype=torch.bfloat16)
        self.cache = load_pkg().PagedCache(be, layers, n_pages, page, KH, kv=self.kv.data_ptr())
        self.qnw, self.knw = ((self.randn(HD) * 0.1).cpu().numpy() for _ in range(2))
        for layer in range(layers):
            self.cache.norm_weight(layer, self.qnw, self.knw)

    def randn(self, *shape, dtype=None):
        return self.torch.randn(shape, generator=self.g, device="cuda").to(dtype or self.torch.float32)

    def inputs(self, rows, H, dtype):
        t = self.torch.bfloat16 if dtype else self.torch.float32
        qg, k, v = (self.randn(rows, n, w, dtype=t) for n, w in ((H, 2 * HD), (self.KH, HD), (self.KH, HD)))
        return qg, k, v, self.torch.full((rows, H, HD), 7.0, dtype=t, device="cuda")

    def host(self, layer=0):
        return self.kv[layer].float().cpu().numpy().astype(np.float64)


def pages_for(lens, page, n_pages, seed, spare=0):
    """A random table with pages of their own for each length; behind them, ids that must not be used."""
    rng = np.random.default_rng(seed)
    counts = [max(0, -(-int(n) // page)) for n in lens]
    ids = rng.permutation(n_pages)
    table = np.full((len(lens), max(1, max(counts)) + spare), 1 << 30, np.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = ids[at:at + c]
        at += c
    assert at <= n_pages
    return table


def poison(P, table, lens):
    """NaN and infinities in every cache row that no request holds."""
    t = P.torch
    held = t.zeros(P.kv.shape[2], P.page, dtype=t.bool, device="cuda")
    for r, n in enumerate(lens):
        at = t.arange(max(0, int(n)), device="cuda")
        held[ints(table[r]).long()[at // P.page], at % P.page] = True
    junk = t.where(P.randn(*P.kv.shape) > 0, float("nan"), float("inf")).bfloat16()
    P.kv.copy_(t.where(held[None, None, :, None, :, None], P.kv, junk))


def check_rows(P, before, qg, k, v, ctx, table, placed, group, dtype, rot=ROT, theta=THETA, parts=None):
    """placed: (row, request, position) of every row the call was to compute, in cache order;
    parts: bf16 parts of q and the probabilities (None: a decode call's)."""
    after = P.host()
    u, u_out = 2.0 ** (-8 * (parts or (2 if dtype else 3))) + 2.0 ** -19, 2.0 ** -8 if dtype else 2.0 ** -24
    qg64, k64, v64 = (x.double().cpu().numpy() for x in (qg, k, v))
    got = ctx.double().cpu().numpy()
    row, req, pos = (np.array(x) for x in zip(*placed))
    kn = ref.norm_rope(k64[row], P.knw, pos, rot, EPS, theta)
    at = table[req, pos // P.page], pos % P.page
    # the appended rows: rounded to bf16 from values good to about 2^-20
    np.testing.assert_allclose(after[0][at[0], :, at[1]], kn, rtol=2.0 ** -8 + 2.0 ** -16, atol=1e-4)
    np.testing.assert_array_equal(after[1][at[0], :, at[1]], ref.bf16(v64[row]))
    # no other row changed, bit for bit
    want = before.copy()
    for which in (0, 1):
        want[which][at[0], :, at[1]] = after[which][at[0], :, at[1]]
    np.testing.assert_array_equal(after, want)
    q = ref.norm_rope(qg64[row][..., :HD], P.qnw, pos, rot, EPS, theta)
    outs, refs = [], []
    for i, (n, r, t) in enumerate(placed):
        o, tol = ref.attend(q[i], qg64[n][..., HD:], ref.rows_of(after, table[r], P.page, t + 1), group, u, u_out)
        assert np.all(np.abs(got[n] - o) <= tol), f"row {n} request {r} position {t}: {np.max(np.abs(got[n] - o) / tol)}"
        outs.append(got[n]); refs.append(o)
    assert_close(np.array(outs), np.array(refs), max_abs=2e-2 if dtype else 2e-4, what="ctx")


DECODE = [
    # lengths (0: an idle slot), page, KH, group, dtype
    ([1], 16, 2, 8, 1),
    ([16, 17, 15, 1], 16, 2, 8, 1),
    ([64, 65, 0, 63, 1, 128], 64, 2, 8, 1),
    ([300, 0, 0, 4093], 48, 2, 8, 1),
    ([5000], 256, 1, 8, 1),
    ([257, 31, 1000], 32, 4, 4, 0),
    ([1, 2, 777], 16, 2, 8, 0),
    ([129, 500], 128, 3, 1, 1),
    ([129, 500], 1024, 2, 2, 0),
    (list(range(1, 66)), 16, 1, 4, 1),
    ([20000, 3], 64, 2, 8, 1),
]


@pytest.mark.parametrize("lens,page,KH,group,dtype", DECODE)
def test_decode(be, lens, page, KH, group, dtype):
    n_pages = sum(-(-n // page) for n in lens) + 3
    P = Pool(be, n_pages, page, KH, seed=len(lens) * 131 + lens[0])
    table = pages_for(lens, page, n_pages, seed=lens[0], spare=2)
    poison(P, table, lens)
    before = P.host()
    qg, k, v, ctx = P.inputs(len(lens), KH * group, dtype)
    pos = ints([n - 1 for n in lens])
    td = ints(table)
    P.cache.decode_dev(0, len(lens), qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), table.shape[1],
                       ctx.data_ptr(), H=KH * group, rot=ROT, eps=EPS, theta=THETA, dtype=dtype)
    be.sync()
    placed = [(r, r, n - 1) for r, n in enumerate(lens) if n]
    check_rows(P, before, qg, k, v, ctx, table, placed, group, dtype)
    for r, n in enumerate(lens):
        if not n:
            assert (ctx[r] == 7).all(), "an idle slot's row was written"


@pytest.mark.parametrize("rot,theta", [(256, 1e7), (2, 1e4), (36, 5e5)])
def test_decode_rotary_widths(be, rot, theta):
    lens, page, KH, group = [900, 33], 32, 2, 8
    P = Pool(be, 40, page, KH, seed=rot)
    table = pages_for(lens, page, 40, seed=1)
    before = P.host()
    qg, k, v, ctx = P.inputs(2, 16, 1)
    pos, td = ints([n - 1 for n in lens]), ints(table)
    P.cache.decode_dev(0, 2, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), table.shape[1],
                       ctx.data_ptr(), rot=rot, eps=EPS, theta=theta)
    be.sync()
    check_rows(P, before, qg, k, v, ctx, table, [(0, 0, 899), (1, 1, 32)], group, 1, rot, theta)


PREFILL = [
    # rows and context of each chunk, page, KH, group, rows behind the last chunk
    ([(1, 0)], 16, 2, 8, 0),
    ([(16, 0)], 16, 2, 8, 3),
    ([(17, 0), (0, 50), (1, 127), (1, 128), (33, 100)], 16, 2, 8, 5),
    ([(130, 0)], 64, 2, 8, 0),
    ([(200, 300), (3, 1000), (1, 0)], 48, 2, 8, 1),
    ([(70, 59), (129, 1)], 128, 1, 1, 2),
    ([(70, 59), (129, 1)], 32, 3, 2, 0),
    ([(65, 190), (64, 64), (1, 31)], 1024, 2, 4, 0),
    ([(300, 2100)], 256, 2, 8, 0),
    ([(1, n) for n in range(0, 600, 7)], 16, 1, 8, 0),
    ([(2, 9000)], 64, 2, 8, 0),
]


@pytest.mark.parametrize("chunks,page,KH,group,behind", PREFILL)
def test_prefill(be, chunks, page, KH, group, behind):
    total = [n + c if n else 0 for n, c in chunks]
    n_pages = sum(-(-n // page) for n in total) + 2
    P = Pool(be, n_pages, page, KH, seed=chunks[0][0] * 7 + len(chunks))
    table = pages_for(total, page, n_pages, seed=3, spare=1)
    poison(P, table, total)
    before = P.host()
    cu = np.concatenate([[0], np.cumsum([n for n, _ in chunks])])
    S = int(cu[-1]) + behind
    qg, k, v, ctx = P.inputs(S, KH * group, 1)
    cu_d, base, td = ints(cu), ints([c for _, c in chunks]), ints(table)
    P.cache.prefill_dev(0, len(chunks), S, cu_d.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(),
                        td.data_ptr(), table.shape[1], ctx.data_ptr(), H=KH * group, rot=ROT, eps=EPS, theta=THETA)
    be.sync()
    placed = [(int(cu[r]) + i, r, c + i) for r, (n, c) in enumerate(chunks) for i in range(n)]
    check_rows(P, before, qg, k, v, ctx, table, placed, group, 1, parts=1)
    assert (ctx[int(cu[-1]):] == 7).all(), "rows behind the last chunk were written"


def test_bad_ids_and_positions_are_reported_and_left_out(be):
    """A page id outside the pool, a position beyond the table, offsets that
    descend: reported once by the next sync, the other requests computed."""
    BackendError = load_pkg().BackendError
    P = Pool(be, 8, 16, 2, seed=5)
    table = np.array([[0, 1], [8, 2], [3, -1], [4, 5]], np.int32)
    pos = [20, 3, 30, 32]                      # ok, bad id, bad id, beyond 2 pages
    before = P.host()
    qg, k, v, ctx = P.inputs(4, 16, 1)
    pd, td = ints(pos), ints(table)
    P.cache.decode_dev(0, 4, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pd.data_ptr(), td.data_ptr(), 2, ctx.data_ptr())
    with pytest.raises(BackendError, match="page id outside|beyond the page table"):
        be.sync()
    be.sync()                                  # reported once, still usable
    check_rows(P, before, qg, k, v, ctx, table, [(0, 0, 20)], 8, 1)
    assert (ctx[3] == 7).all()
    before = P.host()
    cu, base = ints([0, 3, 1, 4, 9]), ints([0, 0, 2, 0])
    qg, k, v, ctx = P.inputs(4, 16, 1)
    table = np.array([[0, 1], [2, 3], [4, 5], [6, 7]], np.int32)
    td = ints(table)
    P.cache.prefill_dev(0, 4, 4, cu.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(), td.data_ptr(), 2,
                        ctx.data_ptr())
    with pytest.raises(BackendError, match="offsets"):
        be.sync()
    be.sync()


# ------------------------------------------------------------------ page moves
@pytest.mark.parametrize("n,page,KH,layers", [(1, 16, 1, 1), (3, 48, 2, 3), (7, 1024, 1, 2), (60, 16, 2, 10), (1000, 16, 1, 3), (5000, 16, 1, 2)])
def test_copy(be, n, page, KH, layers):
    P = Pool(be, 2 * n + 3, page, KH, layers, seed=n)
    ids = np.random.default_rng(n).permutation(2 * n + 3)
    src, dst = ids[:n].copy(), ids[n:2 * n]
    src[-1] = src[0]                           # one source, two destinations
    want = P.kv.clone()
    want[:, :, dst] = P.kv[:, :, src]
    s, d = ints(src), ints(dst)
    P.cache.copy_dev(n, s.data_ptr(), d.data_ptr())
    be.sync()
    assert P.torch.equal(P.kv.view(P.torch.int16), want.view(P.torch.int16))


def test_copy_leaves_out_conflicts(be):
    BackendError = load_pkg().BackendError
    P = Pool(be, 16, 16, 2, 2, seed=2)
    #        ok  dup  dup  chain reads 5 -> left out; 4 -> 5 stays; out of the pool; onto itself
    src, dst = [0, 1, 2, 5, 4, 6, 16, 9], [8, 3, 3, 7, 5, 99, 10, 9]
    want = P.kv.clone()
    want[:, :, [8, 5]] = P.kv[:, :, [0, 4]]
    s, d = ints(src), ints(dst)
    P.cache.copy_dev(8, s.data_ptr(), d.data_ptr())
    with pytest.raises(BackendError, match="named twice|page id outside"):
        be.sync()
    be.sync()
    assert P.torch.equal(P.kv.view(P.torch.int16), want.view(P.torch.int16))


def fork_want(P, table, lens, parent, child, fresh):
    kv, table, lens = P.kv.clone(), table.copy(), list(lens)
    for a, c, f in zip(parent, child, fresh):
        full, tail = divmod(lens[a], P.page)
        table[c, :full] = table[a, :full]
        if tail:
            table[c, full] = f
            kv[:, :, f, :, :tail] = P.kv[:, :, table[a, full], :, :tail]
        lens[c] = lens[a]
    return kv, table, lens


@pytest.mark.parametrize("page,KH,layers,lens", [(16, 2, 2, [0, 1, 15, 16, 17, 100]), (64, 1, 10, [63, 64, 65, 640]), (1024, 2, 1, [1023, 1]),
                                                 (16, 1, 3, [n % 40 for n in range(1200)])])
def test_fork(be, page, KH, layers, lens):
    kids = 2 * len(lens)
    held = sum(-(-n // page) for n in lens)
    P = Pool(be, held + kids, page, KH, layers, seed=page)
    table = np.full((len(lens) + kids, max(-(-n // page) for n in lens)), -5, np.int32)
    ids = np.random.default_rng(0).permutation(held + kids)
    at = 0
    for r, n in enumerate(lens):
        c = -(-n // page)
        table[r, :c] = ids[at:at + c]
        at += c
    parent = [i % len(lens) for i in range(kids)]
    child, fresh = list(range(len(lens), len(lens) + kids)), ids[at:]
    all_lens = lens + [0] * kids
    kv, want_table, want_lens = fork_want(P, table, all_lens, parent, child, fresh)
    p, c, f, td, ld = ints(parent), ints(child), ints(fresh), ints(table), ints(all_lens)
    P.cache.fork_dev(kids, p.data_ptr(), c.data_ptr(), f.data_ptr(), ld.data_ptr(), td.data_ptr(), len(all_lens), table.shape[1])
    be.sync()
    np.testing.assert_array_equal(td.cpu().numpy(), want_table)
    assert ld.tolist() == want_lens
    assert P.torch.equal(P.kv.view(P.torch.int16), kv.view(P.torch.int16))


def test_fork_leaves_out_conflicts(be):
    BackendError = load_pkg().BackendError
    P = Pool(be, 12, 16, 1, 1, seed=4)
    lens = [20, 5, 0, 0, 0, 0, 0, 0]
    table = np.array([[0, 1], [2, 9]] + [[-1, -1]] * 6, np.int32)
    # ok; child twice (both out); child that is a parent (both out); fresh page twice (both out); request 8; length beyond
    parent, child, fresh = [0, 1, 1, 4, 1, 0], [2, 3, 3, 6, 4, 8], [5, 6, 7, 8, 10, 11]
    want_kv, want_table, want_lens = fork_want(P, table, lens, [0], [2], [5])
    p, c, f, td, ld = ints(parent), ints(child), ints(fresh), ints(table), ints(lens)
    P.cache.fork_dev(6, p.data_ptr(), c.data_ptr(), f.data_ptr(), ld.data_ptr(), td.data_ptr(), 8, 2)
    with pytest.raises(BackendError, match="named twice|request index"):
        be.sync()
    be.sync()
    np.testing.assert_array_equal(td.cpu().numpy(), want_table)
    assert ld.tolist() == want_lens
    assert P.torch.equal(P.kv.view(P.torch.int16), want_kv.view(P.torch.int16))


@pytest.mark.parametrize("n_pages,page,lens,shared", [
    (1, 16, [1], False), (33, 16, [0, 100, -3, 17], False), (64, 48, [400, 1000, 48, 47], True),
    (200, 16, [3200], False), (90, 16, [0, 0], False), (1100, 16, [500] * 12, True)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(be, n_pages, page, lens, shared, in_place):
    P = Pool(be, n_pages, page, 2, 2, seed=n_pages)
    table = pages_for(lens, page, n_pages, seed=n_pages, spare=1)
    table[table == 1 << 30] = -1
    if shared:                                 # a forked request's pages count once
        table[-1, 0] = table[0, 0]
    want_table, live, moves = ref.compact(table, lens, page, n_pages)
    want = P.kv.clone()
    if moves:
        src, dst = (list(x) for x in zip(*moves))
        want[:, :, dst] = P.kv[:, :, src]
    ld, td, lv = ints(lens), ints(table), ints([-1])
    out = td if in_place else ints(np.zeros_like(table))
    P.cache.compact_dev(len(lens), ld.data_ptr(), td.data_ptr(), table.shape[1], out.data_ptr(), lv.data_ptr())
    be.sync()
    assert lv.item() == live
    np.testing.assert_array_equal(out.cpu().numpy(), want_table)
    assert P.torch.equal(P.kv.view(P.torch.int16), want.view(P.torch.int16))


def test_zero_sized_calls_do_nothing(be):
    P = Pool(be, 4, 16, 2, seed=1)
    want = P.kv.clone()
    P.cache.decode_dev(0, 0, 0, 0, 0, 0, 0, 1, 0)
    P.cache.prefill_dev(0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 0)
    P.cache.copy_dev(0, 0, 0)
    P.cache.fork_dev(0, 0, 0, 0, 0, 0, 1, 1)
    be.sync()
    assert P.torch.equal(P.kv, want)


def test_refusals(be):
    pkg = load_pkg()
    BackendError = pkg.BackendError
    import torch
    P = Pool(be, 4, 16, 2, seed=1)
    c = P.cache
    x = torch.zeros(1 << 16, dtype=torch.float32, device="cuda")
    p = x.data_ptr()
    ok = dict(H=16)
    with pytest.raises(BackendError, match="layer"):
        c.decode_dev(1, 1, p, p, p, p, p, 1, p, **ok)
    with pytest.raises(BackendError, match="shape"):
        c.decode_dev(0, 1, p, p, p, p, p, 1, p, H=12)
    with pytest.raises(BackendError, match="shape"):
        c.decode_dev(0, 1, p, p, p, p, p, 1, p, H=32)
    with pytest.raises(BackendError, match="batch"):
        c.decode_dev(0, 1025, p, p, p, p, p, 1, p, **ok)
    with pytest.raises(BackendError, match="batch"):
        c.decode_dev(0, -1, p, p, p, p, p, 1, p, **ok)
    with pytest.raises(BackendError, match="rot"):
        c.decode_dev(0, 1, p, p, p, p, p, 1, p, rot=7, **ok)
    with pytest.raises(BackendError, match="dtype"):
        c.decode_dev(0, 1, p, p, p, p, p, 1, p, dtype=2, **ok)
    with pytest.raises(BackendError, match="eps or theta"):
        c.decode_dev(0, 1, p, p, p, p, p, 1, p, theta=0.0, **ok)
    with pytest.raises(BackendError, match="aligned"):
        c.decode_dev(0, 1, p + 2, p, p, p, p, 1, p, **ok)
    with pytest.raises(BackendError, match="null"):
        c.decode_dev(0, 1, p, p, p, 0, p, 1, p, **ok)
    with pytest.raises(BackendError, match="max_pages"):
        c.decode_dev(0, 1, p, p, p, p, p, 1 << 30, p, **ok)
    with pytest.raises(BackendError, match="bf16"):
        c.prefill_dev(0, 1, 1, p, p, p, p, p, p, 1, p, dtype=0, **ok)
    with pytest.raises(BackendError, match="sequences"):
        c.prefill_dev(0, 1025, 1, p, p, p, p, p, p, 1, p, **ok)
    with pytest.raises(BackendError, match="pairs"):
        c.copy_dev(5, p, p)
    with pytest.raises(BackendError, match="forks"):
        c.fork_dev(2, p, p, p, p, p, 2, 1)
    with pytest.raises(BackendError, match="workspace"):
        c.set_workspace(p, 16)
    bare = pkg.PagedCache(be, 1, 4, 16, 2)
    with pytest.raises(BackendError, match="norm weights"):
        bare.decode_dev(0, 1, p, p, p, p, p, 1, p, **ok)
    bare.free()
    with pytest.raises(BackendError, match="live handle"):
        bare.copy_dev(1, p, p)
    for bad in (dict(page=24), dict(page=8), dict(n_pages=0), dict(KH=0), dict(hd=128), dict(layers=0), dict(n_pages=1 << 21)):
        with pytest.raises(BackendError, match="pages"):
            pkg.PagedCache(be, **{**dict(layers=1, n_pages=4, page=16, KH=2), **bad})
    be.sync()


# ------------------------------------------------------------------ as used together
def test_serving_run_matches_contiguous_cache(be):
    """Two prompts prefilled together in two chunks, one forked into three
    samples, six steps decoded from a captured graph, a request dropped and the
    pool compacted, three more steps: each step equals the contiguous cache's
    decode of the same tokens."""
    import torch
    page, KH, H, layers, R = 16, 2, 16, 2, 6
    P = Pool(be, 64, page, KH, layers, seed=9)
    st = torch.cuda.Stream()
    lens = [45, 80]
    ids = list(np.random.default_rng(1).permutation(64))
    table = np.full((R, 8), -1, np.int32)
    for r, n in enumerate(lens):
        for j in range(-(-(n + 12) // page)):
            table[r, j] = ids.pop()
    td = ints(table)
    tokens = {r: [P.inputs(n, H, 1)[:3] for _ in range(layers)] for r, n in enumerate(lens)}   # per layer q|gate, k, v
    for lo, hi in ((0, 30), (30, 80)):
        part = [(max(0, min(n, hi) - lo)) for n in lens]
        cu, base = ints(np.concatenate([[0], np.cumsum(part)])), ints([lo if p else 0 for p in part])
        for layer in range(layers):
            x = [torch.cat([tokens[r][layer][i][lo:lo + p] for r, p in enumerate(part)]) for i in range(3)]
            ctx = torch.zeros(sum(part), H, HD, dtype=torch.bfloat16, device="cuda")
            P.cache.prefill_dev(layer, 2, sum(part), cu.data_ptr(), base.data_ptr(), *(t.data_ptr() for t in x), td.data_ptr(),
                                8, ctx.data_ptr())
            be.sync()
    # the contiguous cache, fed with the same prompts
    be.kv_reset()
    for layer in range(layers):
        be.kv_ensure(layer, R, KH, 128)
        be.gqa_norm_weight(layer, P.qnw, P.knw)
    heir = {0: 0, 1: 1, 2: 0, 3: 0, 4: 0}
    for r, a in heir.items():
        for layer in range(layers):
            x = tokens[a][layer]
            out = torch.zeros(lens[a], H, HD, dtype=torch.bfloat16, device="cuda")
            be.gqa_step_dev(layer, r, lens[a], 0, *(t.data_ptr() for t in x), out.data_ptr())
            be.sync()
    # fork request 0 into 2, 3 and 4
    ld = ints(lens + [0] * 4)
    for r in (2, 3, 4):
        for j in range(2, 4):
            table[r, j] = ids.pop()
    td[2:5, 3] = ints(table[2:5, 3])
    parent, child, fresh = ints([0, 0, 0]), ints([2, 3, 4]), ints(table[2:5, 2])
    P.cache.fork_dev(3, parent.data_ptr(), child.data_ptr(), fresh.data_ptr(), ld.data_ptr(), td.data_ptr(), R, 8)
    be.sync()
    assert ld.tolist() == [45, 80, 45, 45, 45, 0]
    pos = torch.where(ld > 0, ld, -1).int()
    x = [[t.clone() for t in P.inputs(R, H, 1)] for _ in range(layers)]

    def step():
        for layer in range(layers):
            qg, k, v, ctx = (t.data_ptr() for t in x[layer])
            P.cache.decode_dev(layer, R, qg, k, v, pos.data_ptr(), td.data_ptr(), 8, ctx)

    def contiguous(layer):
        qg, k, v, _ = x[layer]
        out = torch.zeros(R, H, HD, dtype=torch.bfloat16, device="cuda")
        at = pos.clamp(min=0)
        be.gqa_decode_dev(layer, R, qg.data_ptr(), k.data_ptr(), v.data_ptr(), at.data_ptr(), out.data_ptr())
        be.sync()
        return out

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    be.set_stream(st.cuda_stream)
    with torch.cuda.graph(graph, stream=st, capture_error_mode="thread_local"):
        step()
    be.set_stream(torch.cuda.current_stream().cuda_stream or 1)

    def steps(n):
        for _ in range(n):
            for layer in range(layers):
                for t, new in zip(x[layer][:3], P.inputs(R, H, 1)[:3]):
                    t.copy_(new)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            be.sync()
            live = pos >= 0
            for layer in range(layers):
                want = contiguous(layer)
                # both round q, p and the output to bf16: 2 x 2^-8 of the values on average well below the bound
                assert_close(x[layer][3][live].float().cpu().numpy(), want[live].float().cpu().numpy(), what=f"layer {layer}")
            pos.copy_(torch.where(live, pos + 1, pos))

    steps(6)
    pos[1] = -1                                # request 1 ends
    ld.copy_(pos.clamp(min=0))
    want_table, live, _ = ref.compact(td.cpu().numpy(), ld.tolist(), page, 64)
    lv = ints([0])
    # the next token's pages are part of what a request holds
    hold = torch.where(pos >= 0, pos + 4, 0).int()
    want_table, live, _ = ref.compact(td.cpu().numpy(), hold.tolist(), page, 64)
    P.cache.compact_dev(R, hold.data_ptr(), td.data_ptr(), 8, td.data_ptr(), lv.data_ptr())
    be.sync()
    assert lv.item() == live
    np.testing.assert_array_equal(td.cpu().numpy(), want_table)
    steps(3)
    be.kv_reset()


def test_compact_twice_is_the_identity(be):
    """A compacted pool has nothing to move: the table stays, no page changes."""
    P = Pool(be, 120, 16, 1, 3, seed=7)
    lens = [100, 0, 333, 16, 5]
    table = pages_for(lens, 16, 120, seed=2)
    table[table == 1 << 30] = -1
    ld, td, lv = ints(lens), ints(table), ints([0])
    for _ in range(2):
        P.cache.compact_dev(5, ld.data_ptr(), td.data_ptr(), table.shape[1], td.data_ptr(), lv.data_ptr())
    be.sync()
    want, live, _ = ref.compact(table, lens, 16, 120)
    np.testing.assert_array_equal(td.cpu().numpy(), want)
    again, live2, moves = ref.compact(want, lens, 16, 120)
    assert lv.item() == live == live2 and not moves and np.array_equal(again, want)


# lengths over the whole range, enough of them that some units fit into a warp's range and some are cut
@pytest.mark.parametrize("B,KH,group,dtype", [(30, 4, 2, 1), (60, 2, 8, 0)])
def test_decode_short_beside_long(be, B, KH, group, dtype):
    rng = np.random.default_rng(B)
    lens = [0, 6000, 6000] + [int(n) for n in np.exp(rng.uniform(0, np.log(6000), size=B - 3))]
    page = 32
    n_pages = sum(-(-n // page) for n in lens) + 1
    P = Pool(be, n_pages, page, KH, seed=B)
    table = pages_for(lens, page, n_pages, seed=B)
    poison(P, table, lens)
    before = P.host()
    qg, k, v, ctx = P.inputs(B, KH * group, dtype)
    pos, td = ints([n - 1 for n in lens]), ints(table)
    P.cache.decode_dev(0, B, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), table.shape[1],
                       ctx.data_ptr(), H=KH * group, rot=ROT, eps=EPS, theta=THETA, dtype=dtype)
    be.sync()
    check_rows(P, before, qg, k, v, ctx, table, [(r, r, n - 1) for r, n in enumerate(lens) if n], group, dtype)
    assert (ctx[0] == 7).all()


# the most requests of a call, some idle, and more of them than a warp counts alone
@pytest.mark.parametrize("B,KH,group,dtype", [(1024, 1, 2, 1), (33, 2, 8, 0), (200, 3, 4, 1)])
def test_decode_many_requests(be, B, KH, group, dtype):
    rng = np.random.default_rng(B)
    lens = [int(n) for n in rng.integers(0, 70, size=B)]
    page = 16
    n_pages = sum(-(-n // page) for n in lens) + 1
    P = Pool(be, n_pages, page, KH, seed=B)
    table = pages_for(lens, page, n_pages, seed=B)
    poison(P, table, lens)
    before = P.host()
    qg, k, v, ctx = P.inputs(B, KH * group, dtype)
    pos, td = ints([n - 1 for n in lens]), ints(table)
    P.cache.decode_dev(0, B, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), table.shape[1],
                       ctx.data_ptr(), H=KH * group, rot=ROT, eps=EPS, theta=THETA, dtype=dtype)
    be.sync()
    check_rows(P, before, qg, k, v, ctx, table, [(r, r, n - 1) for r, n in enumerate(lens) if n], group, dtype)
    for r, n in enumerate(lens):
        if not n:
            assert (ctx[r] == 7).all()


def test_all_slots_idle(be):
    P = Pool(be, 4, 16, 2, seed=1)
    before = P.kv.clone()
    qg, k, v, ctx = P.inputs(3, 16, 1)
    pos, td = ints([-1, -1, -7]), ints([[0], [1], [2]])
    P.cache.decode_dev(0, 3, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), 1, ctx.data_ptr())
    cu, base = ints([0, 0, 0, 0]), ints([5, -1, 0])
    P.cache.prefill_dev(0, 3, 3, cu.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(), td.data_ptr(), 1,
                        ctx.data_ptr())
    be.sync()
    assert (ctx == 7).all() and P.torch.equal(P.kv, before)


def test_prefill_many_chunks(be):
    """The most chunks of a call, most of them empty or a token long."""
    rng = np.random.default_rng(3)
    chunks = [(int(n), int(c)) for n, c in zip(rng.integers(0, 3, size=1024), rng.integers(0, 40, size=1024))]
    page, KH, group = 16, 1, 8
    total = [n + c if n else 0 for n, c in chunks]
    n_pages = sum(-(-n // page) for n in total) + 1
    P = Pool(be, n_pages, page, KH, seed=4)
    table = pages_for(total, page, n_pages, seed=4)
    poison(P, table, total)
    before = P.host()
    cu = np.concatenate([[0], np.cumsum([n for n, _ in chunks])])
    qg, k, v, ctx = P.inputs(int(cu[-1]), KH * group, 1)
    cu_d, base, td = ints(cu), ints([c for _, c in chunks]), ints(table)
    P.cache.prefill_dev(0, 1024, int(cu[-1]), cu_d.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(),
                        td.data_ptr(), table.shape[1], ctx.data_ptr(), H=KH * group)
    be.sync()
    check_rows(P, before, qg, k, v, ctx, table, [(int(cu[r]) + i, r, c + i) for r, (n, c) in enumerate(chunks) for i in range(n)],
               group, 1, parts=1)


@pytest.mark.parametrize("rot,group", [(256, 1), (256, 8), (36, 2), (2, 4)])
def test_prefill_rotary_widths(be, rot, group):
    page, KH = 32, 2
    chunks = [(150, 10), (9, 77)]
    total = [n + c for n, c in chunks]
    P = Pool(be, 12, page, KH, seed=rot + group)
    table = pages_for(total, page, 12, seed=1)
    before = P.host()
    qg, k, v, ctx = P.inputs(159, KH * group, 1)
    cu, base, td = ints([0, 150, 159]), ints([10, 77]), ints(table)
    P.cache.prefill_dev(0, 2, 159, cu.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(), td.data_ptr(),
                        table.shape[1], ctx.data_ptr(), H=KH * group, rot=rot, theta=5e5)
    be.sync()
    placed = [(i, 0, 10 + i) for i in range(150)] + [(150 + i, 1, 77 + i) for i in range(9)]
    check_rows(P, before, qg, k, v, ctx, table, placed, group, 1, rot, 5e5, parts=1)


def test_gate_extremes(be):
    """Gates of +-infinity, the type's lowest and highest values, NaN: 0, 1, 0, 1 and NaN times the attention."""
    import torch
    P = Pool(be, 8, 16, 1, seed=3)
    edge = [float("-inf"), float("inf"), -3.38e38, 3.38e38, -100.0, 100.0, 20.5, float("nan")]
    for dtype in (0, 1):
        qg, k, v, ctx = P.inputs(2, 8, dtype)
        qg[:, :, HD:HD + 8] = torch.tensor(edge, device="cuda").to(qg.dtype)
        table, td = np.array([[0, 1, 2], [3, 4, 5]], np.int32), ints([[0, 1, 2], [3, 4, 5]])
        pos = ints([0, 40])
        P.cache.decode_dev(0, 2, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), 3, ctx.data_ptr(),
                           H=8, dtype=dtype)
        be.sync()
        got = ctx[0, :, :8].double().cpu().numpy()       # one key: the attention is its v row
        want = v[0, 0, :8].bfloat16().double().cpu().numpy()
        assert np.isnan(got[:, 7]).all()
        np.testing.assert_array_equal(got[:, [0, 2]], 0)
        np.testing.assert_allclose(got[:, [1, 3, 5, 6]], np.tile(want[[1, 3, 5, 6]], (8, 1)), rtol=2.0 ** -8 + 1e-6)
        assert (np.abs(got[:, 4]) < 1e-37).all()


def test_offsets_beyond_32_bits(be):
    """Pages whose elements lie past 2^31 and whose bytes lie past 2^32: decode, prefill, copy, fork and compaction there."""
    import torch
    page, KH, n_pages = 64, 2, 70000                     # 2.3e9 elements, 4.6 GB, to a plane
    kv = torch.empty(1, 2, n_pages, KH, page, HD, dtype=torch.bfloat16, device="cuda")
    far = list(range(n_pages - 12, n_pages))
    kv[:, :, far] = torch.randn(1, 2, 12, KH, page, HD, device="cuda").bfloat16()
    kv[:, :, :4] = 0
    cache = load_pkg().PagedCache(be, 1, n_pages, page, KH, kv=kv.data_ptr())
    zero = np.zeros(HD, np.float32)
    cache.norm_weight(0, zero, zero)

    class View:                                          # what check_rows looks at: the far pages as pages 0 .. 11
        knw = qnw = zero

        def host(self):
            return kv[0][:, far].float().cpu().numpy().astype(np.float64)

    View.page = page
    P = View()
    near = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    td = ints(near + n_pages - 12)
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()   # noqa: E731
    qg, k, v, ctx = rnd(2, 16, 2 * HD), rnd(2, KH, HD), rnd(2, KH, HD), torch.zeros(2, 16, HD, dtype=torch.bfloat16, device="cuda")
    before = P.host()
    pos = ints([190, 100])
    cache.decode_dev(0, 2, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), 3, ctx.data_ptr())
    be.sync()
    check_rows(P, before, qg, k, v, ctx, near, [(0, 0, 190), (1, 1, 100)], 8, 1)
    qg, k, v, ctx = rnd(40, 16, 2 * HD), rnd(40, KH, HD), rnd(40, KH, HD), torch.zeros(40, 16, HD, dtype=torch.bfloat16, device="cuda")
    before = P.host()
    cu, base = ints([0, 30, 40]), ints([150, 101])
    cache.prefill_dev(0, 2, 40, cu.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(), td.data_ptr(), 3, ctx.data_ptr())
    be.sync()
    check_rows(P, before, qg, k, v, ctx, near, [(i, 0, 150 + i) for i in range(30)] + [(30 + i, 1, 101 + i) for i in range(10)], 8, 1, parts=1)
    src, dst = ints([n_pages - 12]), ints([n_pages - 1])
    cache.copy_dev(1, src.data_ptr(), dst.data_ptr())
    table, ln = ints([[n_pages - 12, n_pages - 11], [0, 0]]), ints([100, 0])
    par, chi, fre = ints([0]), ints([1]), ints([n_pages - 2])
    cache.fork_dev(1, par.data_ptr(), chi.data_ptr(), fre.data_ptr(), ln.data_ptr(), table.data_ptr(), 2, 2)
    be.sync()
    assert torch.equal(kv[:, :, n_pages - 1], kv[:, :, n_pages - 12])
    assert table.tolist() == [[n_pages - 12, n_pages - 11], [n_pages - 12, n_pages - 2]] and ln.tolist() == [100, 100]
    assert torch.equal(kv[:, :, n_pages - 2, :, :36], kv[:, :, n_pages - 11, :, :36])
    live = ints([0])
    want = [kv[:, :, i].clone() for i in (n_pages - 12, n_pages - 11, n_pages - 2)]
    cache.compact_dev(2, ln.data_ptr(), table.data_ptr(), 2, table.data_ptr(), live.data_ptr())
    be.sync()
    assert live.item() == 3 and table.tolist() == [[0, 1], [0, 2]]
    for i, w in enumerate(want):
        assert torch.equal(kv[:, :, i], w)
    cache.free()


def test_two_graphs_in_flight_with_their_own_workspaces(be):
    """Two captured steps of one handle on two streams, split units in both, replayed together many times."""
    import torch
    P = Pool(be, 1100, 16, 2, 2, seed=8)
    R = 4
    lens = [[4000, 33, 700, 3000], [2500, 4000, 1, 90]]
    ids = np.random.default_rng(4).permutation(1100)
    tables, at = [], 0
    for group_lens in lens:
        t = np.full((R, 256), 1 << 30, np.int32)
        for r, n in enumerate(group_lens):
            c = -(-n // 16)
            t[r, :c] = ids[at:at + c]
            at += c
        tables.append(ints(t))
    pos = [ints([n - 1 for n in group_lens]) for group_lens in lens]
    x = [P.inputs(R, 16, 1) for _ in lens]
    chunk = [P.inputs(20, 16, 1) for _ in lens]
    cu, base = ints([0, 20]), [ints([lens[i][1] - 1]) for i in (0, 1)]
    ws = [None, torch.empty(P.cache.workspace_bytes(), dtype=torch.uint8, device="cuda")]
    streams, graphs = [torch.cuda.Stream() for _ in lens], []

    def step(i):
        qg, k, v, ctx = (t.data_ptr() for t in x[i])
        P.cache.decode_dev(i, R, qg, k, v, pos[i].data_ptr(), tables[i].data_ptr(), 256, ctx)
        qg, k, v, ctx = (t.data_ptr() for t in chunk[i])
        # the second request goes on with 20 rows
        P.cache.prefill_dev(i, 1, 20, cu.data_ptr(), base[i].data_ptr(), qg, k, v, tables[i][1].data_ptr(), 256, ctx)

    # room for the 20 rows
    for i in (0, 1):
        c = -(-lens[i][1] // 16)
        extra = min(256, c + 2) - c
        tables[i][1, c:c + extra] = ints(ids[at:at + extra])
        at += extra
        base[i].clamp_(max=256 * 16 - 20)
    want = []
    for i in (0, 1):
        step(i)
        be.sync()
        want.append((x[i][3].clone(), chunk[i][3].clone()))
    torch.cuda.synchronize()
    for i in (0, 1):
        if ws[i] is not None:
            P.cache.set_workspace(ws[i].data_ptr(), ws[i].numel())
        be.set_stream(streams[i].cuda_stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i], capture_error_mode="thread_local"):
            step(i)
        graphs.append(g)
    P.cache.set_workspace()
    be.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    for i in (0, 1):
        x[i][3].zero_()
        chunk[i][3].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    be.sync()
    for i in (0, 1):
        assert torch.equal(x[i][3], want[i][0]) and torch.equal(chunk[i][3], want[i][1])


def test_moves_replay_from_a_graph(be):
    """Copy, fork and compaction captured once and replayed on new contents."""
    import torch
    P = Pool(be, 40, 16, 2, 2, seed=6)
    table = np.full((4, 4), -1, np.int32)
    table[0, :3], table[1, :1] = [30, 7, 21], [12]
    td0, ln0 = ints(table), ints([40, 9, 0, 0])
    td, ln, lv = td0.clone(), ln0.clone(), ints([0])
    src, dst = ints([30]), ints([33])
    par, chi, fre = ints([0, 1]), ints([2, 3]), ints([25, 26])
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    be.set_stream(st.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
        P.cache.copy_dev(1, src.data_ptr(), dst.data_ptr())
        P.cache.fork_dev(2, par.data_ptr(), chi.data_ptr(), fre.data_ptr(), ln.data_ptr(), td.data_ptr(), 4, 4)
        P.cache.compact_dev(4, ln.data_ptr(), td.data_ptr(), 4, td.data_ptr(), lv.data_ptr())
    be.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    for _ in range(3):
        P.kv.copy_(P.randn(*P.kv.shape).bfloat16())
        td.copy_(td0)
        ln.copy_(ln0)
        kv = P.kv.clone()
        kv[:, :, 33] = kv[:, :, 30]
        Q = type("Q", (), dict(kv=kv, page=16))
        kv, t1, l1 = fork_want(Q, table, [40, 9, 0, 0], [0, 1], [2, 3], [25, 26])
        want, live, moves = ref.compact(t1, l1, 16, 40)
        s, d = (list(z) for z in zip(*moves))
        after = kv.clone()
        after[:, :, d] = kv[:, :, s]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        be.sync()
        np.testing.assert_array_equal(td.cpu().numpy(), want)
        assert lv.item() == live and ln.tolist() == l1
        assert torch.equal(P.kv.view(torch.int16), after.view(torch.int16))


def test_a_pool_of_its_own_and_handles_that_end(be):
    """Library-owned memory: zeroed, counted, given back; the most handles; a handle freed while its stream captures."""
    import torch
    pkg = load_pkg()
    before = be.mem_info()
    c = pkg.PagedCache(be, 2, 8, 16, 1)
    assert pkg.PagedCache.nbytes_for(be, 2, 8, 16, 1) == 2 * 2 * 8 * 16 * 512
    k0, v0 = c.device_ptr(0)
    k1, _ = c.device_ptr(1)
    assert v0 - k0 == 8 * 16 * 512 and k1 - k0 == 2 * 8 * 16 * 512
    be.sync()
    c.free()
    assert be.mem_info() == before
    many = [pkg.PagedCache(be, 1, 1, 16, 1) for _ in range(8)]
    st = torch.cuda.Stream()
    x = ints([0])
    y = ints([0])
    torch.cuda.synchronize()
    be.set_stream(st.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
        many[0].copy_dev(1, x.data_ptr(), y.data_ptr())
        many[1].free()
        with pytest.raises(pkg.BackendError, match="capturing"):
            pkg.PagedCache(be, 1, 1, 16, 1)
    be.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    g.replay()
    torch.cuda.synchronize()
    del g
    for m in many:
        m.free()
    be.sync()
    assert be.mem_info() == before


def test_a_handle_ends_with_its_pool(be):
    """A handle kept past its pool's end names no later pool, in calls or in a second free."""
    pkg = load_pkg()
    P = Pool(be, 4, 16, 1)
    x, y = ints([0]), ints([1])
    old = [P.cache.h]
    P.cache.free()
    for _ in range(5):
        c = pkg.PagedCache(be, 1, 4, 16, 1, kv=P.kv.data_ptr())
        assert c.h not in old
        for h in old:
            be.lib.coli_cuda_pages_free(h)
            assert be.lib.coli_cuda_pages_copy_dev(h, 1, x.data_ptr(), y.data_ptr()) == 0
            assert b"live handle" in be.lib.coli_cuda_last_error()
        c.copy_dev(1, x.data_ptr(), y.data_ptr())
        be.sync()
        assert P.torch.equal(P.kv[:, :, 0].view(P.torch.int16), P.kv[:, :, 1].view(P.torch.int16))
        old.append(c.h)
        c.free()


def test_prefill_many_whole_units_of_one_tile(be):
    """Prompts that end inside their first 128 positions, so many that every CTA works through whole units of one key
    tile each, one behind the other; repeated calls give the same bits."""
    rng = np.random.default_rng(11)
    chunks = [(int(n), int(c)) for n, c in zip(rng.integers(17, 41, size=256), rng.integers(0, 80, size=256))]
    page, KH, group = 64, 2, 8
    total = [n + c for n, c in chunks]
    n_pages = sum(-(-n // page) for n in total) + 1
    P = Pool(be, n_pages, page, KH, seed=12)
    table = pages_for(total, page, n_pages, seed=12)
    poison(P, table, total)
    before = P.host()
    cu = np.concatenate([[0], np.cumsum([n for n, _ in chunks])])
    S = int(cu[-1])
    qg, k, v, ctx = P.inputs(S, KH * group, 1)
    cu_d, base, td = ints(cu), ints([c for _, c in chunks]), ints(table)

    def call():
        P.cache.prefill_dev(0, len(chunks), S, cu_d.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(),
                            td.data_ptr(), table.shape[1], ctx.data_ptr(), H=KH * group)
        be.sync()

    call()
    check_rows(P, before, qg, k, v, ctx, table, [(int(cu[r]) + i, r, c + i) for r, (n, c) in enumerate(chunks) for i in range(n)],
               group, 1, parts=1)
    first, rows = ctx.clone(), P.kv.clone()
    for _ in range(20):
        ctx.fill_(7.0)
        call()
        assert P.torch.equal(ctx, first) and P.torch.equal(P.kv.view(P.torch.int16), rows.view(P.torch.int16))


# rows from where the squares leave fp32 (2^128) downwards; without eps also rows whose squares vanish
@pytest.mark.parametrize("scales,eps", [([1e18, 3e19, 1.1e38, 1.0, 1e-30], 1e-6), ([1e-18, 1e-25, 1e-35, 1e30, 1.0], 0.0)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_decode_rows_of_any_finite_scale(be, monkeypatch, scales, eps, dtype):
    monkeypatch.setitem(globals(), "EPS", eps)      # what check_rows norms with
    lens, page, KH, group = [40, 17, 700, 33, 64], 16, 2, 4
    n_pages = sum(-(-n // page) for n in lens)
    P = Pool(be, n_pages, page, KH, seed=21)
    table = pages_for(lens, page, n_pages, seed=21)
    before = P.host()
    qg, k, v, ctx = P.inputs(5, KH * group, dtype)
    by = P.torch.tensor(scales, device="cuda")[:, None, None]
    qg[..., :HD] = (qg[..., :HD].float().clamp(-3, 3) * by).to(qg.dtype)
    k = (k.float().clamp(-3, 3) * by).to(k.dtype)
    pos, td = ints([n - 1 for n in lens]), ints(table)
    P.cache.decode_dev(0, 5, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), table.shape[1],
                       ctx.data_ptr(), H=KH * group, eps=eps, dtype=dtype)
    be.sync()
    check_rows(P, before, qg, k, v, ctx, table, [(r, r, n - 1) for r, n in enumerate(lens)], group, dtype)


@pytest.mark.parametrize("scale,eps,rot", [(2e19, 1e-6, 64), (1.1e38, 1e-6, 64), (1.1e38, 1e-6, 36), (1e-25, 0.0, 64), (1e-25, 0.0, 36)])
def test_prefill_rows_of_any_finite_scale(be, monkeypatch, scale, eps, rot):
    """Rows of 1 and of `scale` in turn, whose norms a warp takes together."""
    monkeypatch.setitem(globals(), "EPS", eps)
    page, KH, group = 32, 2, 8
    P = Pool(be, 4, page, KH, seed=22)
    table = pages_for([70], page, 4, seed=22)
    before = P.host()
    qg, k, v, ctx = P.inputs(50, KH * group, 1)
    by = P.torch.tensor([1.0, scale] * 25, device="cuda")[:, None, None]
    qg[..., :HD] = (qg[..., :HD].float().clamp(-3, 3) * by).bfloat16()
    k = (k.float().clamp(-3, 3) * by).bfloat16()
    cu, base, td = ints([0, 50]), ints([20]), ints(table)
    P.cache.prefill_dev(0, 1, 50, cu.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(), td.data_ptr(),
                        table.shape[1], ctx.data_ptr(), H=KH * group, rot=rot, eps=eps)
    be.sync()
    check_rows(P, before, qg, k, v, ctx, table, [(i, 0, 20 + i) for i in range(50)], group, 1, rot=rot, parts=1)


def test_rows_with_an_infinity(be):
    """x / rms(x) of a row with an infinity: 0 for its finite elements, NaN for the infinite ones, so NaN as an output."""
    P = Pool(be, 8, 16, 1, seed=23)
    for dtype in (0, 1):
        qg, k, v, ctx = P.inputs(2, 8, dtype)
        qg[0, 3, 100] = float("inf")
        pos, td = ints([20, 20]), ints([[0, 1], [2, 3]])
        P.cache.decode_dev(0, 2, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), 2, ctx.data_ptr(),
                           H=8, dtype=dtype)
        be.sync()
        bad = P.torch.zeros(2, 8, dtype=P.torch.bool, device="cuda")
        bad[0, 3] = True
        assert ctx[bad].isnan().all() and ctx[~bad].isfinite().all()


def test_fork_ignores_fresh_pages_that_are_not_used(be):
    """Parents that end with a page need no fresh one: what stands in its place may repeat another's or be no page at all."""
    P = Pool(be, 14, 16, 2, 2, seed=31)
    lens = [32, 20, 16, 0, 0, 0, 0, 0, 0, 0]
    table = np.array([[0, 1], [2, 3], [4, -1]] + [[-1, -1]] * 7, np.int32)
    parent, child, fresh = [0, 1, 2, 0, 1, 2], [3, 4, 5, 6, 7, 8], [9, 9, 9, -1, 10, 3]
    want_kv, want_table, want_lens = fork_want(P, table, lens, parent, child, fresh)
    p, c, f, td, ld = ints(parent), ints(child), ints(fresh), ints(table), ints(lens)
    P.cache.fork_dev(6, p.data_ptr(), c.data_ptr(), f.data_ptr(), ld.data_ptr(), td.data_ptr(), 10, 2)
    be.sync()
    np.testing.assert_array_equal(td.cpu().numpy(), want_table)
    assert ld.tolist() == want_lens
    assert P.torch.equal(P.kv.view(P.torch.int16), want_kv.view(P.torch.int16))


@pytest.mark.parametrize("extra", [0, 400])
def test_fork_leaves_out_a_fresh_page_that_another_fork_copies(be, extra):
    """Page 3 is request 1's started page: a fork that would write to it is left out, the one that reads it is not."""
    BackendError = load_pkg().BackendError
    n = 4 + 2 * (3 + extra)
    P = Pool(be, 8 + extra, 16, 1, 2, seed=32)
    lens = [5, 20, 9] + [0] * (n - 3)
    table = np.full((n, 2), -1, np.int32)
    table[0, 0], table[1], table[2, 0] = 0, [2, 3], 4
    parent, child, fresh = [0, 1, 2], [3, 4, 5], [3, 5, 6]
    for i in range(extra):                     # many more, so that the two stand far apart
        parent.insert(1, 2)
        child.insert(1, 6 + i)
        fresh.insert(1, 8 + i)
    keep = [i for i in range(len(parent)) if i != 0]
    want_kv, want_table, want_lens = fork_want(P, table, lens, *([x[i] for i in keep] for x in (parent, child, fresh)))
    p, c, f, td, ld = ints(parent), ints(child), ints(fresh), ints(table), ints(lens)
    P.cache.fork_dev(len(parent), p.data_ptr(), c.data_ptr(), f.data_ptr(), ld.data_ptr(), td.data_ptr(), n, 2)
    with pytest.raises(BackendError, match="named twice"):
        be.sync()
    be.sync()
    np.testing.assert_array_equal(td.cpu().numpy(), want_table)
    assert ld.tolist() == want_lens
    assert P.torch.equal(P.kv.view(P.torch.int16), want_kv.view(P.torch.int16))


def test_copy_of_a_page_onto_itself_stands_beside_its_copies(be):
    """A page onto itself writes nothing, so pairs that read it are copied; one that writes to it is still left out."""
    BackendError = load_pkg().BackendError
    P = Pool(be, 12, 16, 2, 2, seed=33)
    want = P.kv.clone()
    src, dst = [3, 3, 3, 5], [3, 4, 6, 5]
    want[:, :, [4, 6]] = P.kv[:, :, [3, 3]]
    s, d = ints(src), ints(dst)
    P.cache.copy_dev(4, s.data_ptr(), d.data_ptr())
    be.sync()
    assert P.torch.equal(P.kv.view(P.torch.int16), want.view(P.torch.int16))
    s, d = ints([7, 8, 9]), ints([7, 7, 10])     # 8 over the page that another pair names
    want[:, :, 10] = P.kv[:, :, 9]
    P.cache.copy_dev(3, s.data_ptr(), d.data_ptr())
    with pytest.raises(BackendError, match="named twice"):
        be.sync()
    be.sync()
    assert P.torch.equal(P.kv.view(P.torch.int16), want.view(P.torch.int16))


@pytest.mark.parametrize("dtype", [0, 1])
def test_decode_keeps_nan_keys_of_a_cut_request(be, dtype):
    """K rows of NaN inside a request's length make its ctx NaN however its tiles are cut: a run of them at every offset
    from where the cuts are, so that in some of the calls it fills whole pieces and no other."""
    page, KH, group, n = 16, 1, 8, 5000
    n_pages = -(-n // page)
    P = Pool(be, n_pages, page, KH, seed=41)
    table = pages_for([n], page, n_pages, seed=41)
    kv = P.kv.clone()
    qg, k, v, ctx = P.inputs(1, KH * group, dtype)
    pos, td = ints([n - 1]), ints(table)
    for first in range(100, 108):
        P.kv.copy_(kv)
        P.kv[0, 0, ints(table[0, first:first + 40]).long()] = float("nan")
        ctx.zero_()
        P.cache.decode_dev(0, 1, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), table.shape[1],
                           ctx.data_ptr(), H=KH * group, dtype=dtype)
        be.sync()
        assert ctx.isnan().all(), f"tiles {first} .. {first + 39} were left out"


# few units (many pieces each, the deep join) and many (a few pieces)
@pytest.mark.parametrize("rows,before,runs", [(2, 9000, [(8 + o, 24 + o) for o in range(8)]), (700, 3000, [(0, n) for n in range(1, 23)])])
def test_prefill_keeps_nan_keys_of_a_cut_unit(be, rows, before, runs):
    page, KH, group = 128, 2, 8
    n_pages = -(-(rows + before) // page)
    P = Pool(be, n_pages, page, KH, seed=42)
    table = pages_for([rows + before], page, n_pages, seed=42)
    kv = P.kv.clone()
    qg, k, v, ctx = P.inputs(rows, KH * group, 1)
    cu, base, td = ints([0, rows]), ints([before]), ints(table)
    for first, last in runs:                             # key tiles, here a page each, of NaN in KV head 0
        P.kv.copy_(kv)
        P.kv[0, 0, ints(table[0, first:last]).long(), 0] = float("nan")
        ctx.zero_()
        P.cache.prefill_dev(0, 1, rows, cu.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(),
                            td.data_ptr(), table.shape[1], ctx.data_ptr(), H=KH * group)
        be.sync()
        assert ctx[:, :group].isnan().all() and ctx[:, group:].isfinite().all(), f"tiles {first} .. {last - 1}"


def test_offsets_that_descend_leave_the_good_chunks(be):
    """Rows named by offsets that descend or pass the rows given belong to no chunk; the chunks before are computed."""
    BackendError = load_pkg().BackendError
    P = Pool(be, 8, 16, 2, seed=53)
    table = np.array([[0, 1], [2, 3], [4, 5], [6, 7]], np.int32)
    for cu in ([0, 3, 3, 9, 9], [0, 3, 2, 2, 2], [0, 3, 3, -5, -5]):
        before = P.host()
        qg, k, v, ctx = P.inputs(4, 16, 1)
        cu_d, base, td = ints(cu), ints([2, 0, 2, 0]), ints(table)
        P.cache.prefill_dev(0, 4, 4, cu_d.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(),
                            td.data_ptr(), 2, ctx.data_ptr())
        with pytest.raises(BackendError, match="offsets"):
            be.sync()
        be.sync()
        check_rows(P, before, qg, k, v, ctx, table, [(i, 0, 2 + i) for i in range(3)], 8, 1, parts=1)
        assert (ctx[3] == 7).all()


def test_an_argument_error_ends_with_its_session(be):
    """A bad page id met before a shutdown is not reported to what runs after the next init."""
    import torch
    pkg = load_pkg()
    P = Pool(be, 4, 16, 1)
    bad, x, y = ints([99]), ints([0]), ints([1])
    P.cache.copy_dev(1, bad.data_ptr(), x.data_ptr())
    be.shutdown()
    assert be.lib.coli_cuda_init(0) == 1
    be.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    be.sync()
    c = pkg.PagedCache(be, 1, 4, 16, 1, kv=P.kv.data_ptr())
    c.copy_dev(1, x.data_ptr(), y.data_ptr())
    be.sync()
    assert torch.equal(P.kv[:, :, 0].view(torch.int16), P.kv[:, :, 1].view(torch.int16))
    c.copy_dev(1, bad.data_ptr(), x.data_ptr())
    with pytest.raises(pkg.BackendError, match="page id outside"):
        be.sync()
    be.sync()


def test_a_handle_freed_while_another_stream_captures(be):
    """Freeing a pool (as garbage collection may at any time) leaves a capture on a stream that is not the backend's
    alone, with the backend on a stream of its own as on the legacy stream, which a blocking stream's capture makes
    unusable until it ends."""
    import gc

    import torch
    pkg = load_pkg()
    gc.collect()
    before = be.mem_info()
    x = torch.zeros(64, device="cuda")
    side, own_stream = torch.cuda.Stream(), torch.cuda.Stream()
    caches = [pkg.PagedCache(be, 1, 4, 16, 1) for _ in range(2)]
    torch.cuda.synchronize()
    be.set_stream(own_stream.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):     # the global mode
        x += 1
        caches.pop().free()
    g.replay()
    torch.cuda.synchronize()
    assert (x == 1).all()
    from cuda.bindings import runtime as cudart
    err, blocking = cudart.cudaStreamCreate()
    assert err == cudart.cudaError_t.cudaSuccess
    be.set_stream(1)
    err, = cudart.cudaStreamBeginCapture(blocking, cudart.cudaStreamCaptureMode.cudaStreamCaptureModeThreadLocal)
    assert err == cudart.cudaError_t.cudaSuccess
    caches.pop().free()
    with pytest.raises(pkg.BackendError, match="capturing"):
        pkg.PagedCache(be, 1, 4, 16, 1)
    err, graph = cudart.cudaStreamEndCapture(blocking)
    assert err == cudart.cudaError_t.cudaSuccess, "the capture was ended from outside"
    cudart.cudaGraphDestroy(graph)
    cudart.cudaStreamDestroy(blocking)
    be.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    pkg.PagedCache(be, 1, 4, 16, 1).free()
    be.sync()
    assert be.mem_info() == before


def test_moves_report_bad_lengths_and_ids_and_leave_them_out(be):
    """Fork of a parent whose length passes its table; compaction of such a length and of ids outside the pool: the good
    requests are served, and every other row of the pool, the table and the lengths is left alone."""
    BackendError = load_pkg().BackendError
    P = Pool(be, 12, 16, 1, 2, seed=51)
    lens = [20, 33, -4, 5, 0, 0, 0, 0, 0]      # of 2 pages: ok, beyond, negative, its started page is no page
    table = np.array([[0, 1], [2, 3], [4, 5], [12, -1]] + [[-1, -1]] * 5, np.int32)
    parent, child, fresh = [0, 1, 2, 3, 0], [4, 5, 6, 7, 8], [8, 9, 10, 11, -1]
    want_kv, want_table, want_lens = fork_want(P, table, lens, [0], [4], [8])
    p, c, f, td, ld = ints(parent), ints(child), ints(fresh), ints(table), ints(lens)
    P.cache.fork_dev(5, p.data_ptr(), c.data_ptr(), f.data_ptr(), ld.data_ptr(), td.data_ptr(), 9, 2)
    with pytest.raises(BackendError, match="beyond the page table|page id outside"):
        be.sync()
    be.sync()
    np.testing.assert_array_equal(td.cpu().numpy(), want_table)
    assert ld.tolist() == want_lens
    assert P.torch.equal(P.kv.view(P.torch.int16), want_kv.view(P.torch.int16))

    lens = [33, 20, 32, 16]                    # beyond (holds nothing), ok, one id below and one behind the pool, ok
    table = np.array([[0, 1], [11, 9], [-1, 12], [7, 12]], np.int32)
    good = np.array([[0, 1], [11, 9], [-1, 12], [7, 12]], np.int32)
    want_table, live, moves = ref.compact(good, [0, 20, 0, 16], 16, 12)
    assert live == 3
    want_kv = P.kv.clone()
    s, d = (list(x) for x in zip(*moves))
    want_kv[:, :, d] = P.kv[:, :, s]
    ld, td, lv = ints(lens), ints(table), ints([-1])
    P.cache.compact_dev(4, ld.data_ptr(), td.data_ptr(), 2, td.data_ptr(), lv.data_ptr())
    with pytest.raises(BackendError, match="beyond the page table|page id outside"):
        be.sync()
    be.sync()
    assert lv.item() == live
    np.testing.assert_array_equal(td.cpu().numpy(), want_table)
    assert P.torch.equal(P.kv.view(P.torch.int16), want_kv.view(P.torch.int16))


@pytest.mark.parametrize("bad", [-1, 14, 1 << 30, -(1 << 31)])
def test_prefill_leaves_out_bad_ids_and_positions(be, bad):
    """A chunk with an id outside the pool, one that passes its table and one with a negative start beside two good
    ones: those are computed, the bad ones append only where their own rows have a page, nothing else changes."""
    BackendError = load_pkg().BackendError
    page, KH, group = 16, 2, 8
    P = Pool(be, 14, page, KH, seed=52)
    chunks = [(20, 12), (17, 15), (9, 24), (5, -1), (3, 7)]     # the third: 33 rows in 2 pages
    table = np.array([[0, 1], [2, bad], [4, 5], [6, 7], [8, bad]], np.int32)
    cu = np.concatenate([[0], np.cumsum([n for n, _ in chunks])])
    before = P.host()
    qg, k, v, ctx = P.inputs(int(cu[-1]), KH * group, 1)
    cu_d, base, td = ints(cu), ints([c for _, c in chunks]), ints(table)
    P.cache.prefill_dev(0, 5, int(cu[-1]), cu_d.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(),
                        td.data_ptr(), 2, ctx.data_ptr(), H=KH * group)
    with pytest.raises(BackendError, match="page id outside|beyond the page table"):
        be.sync()
    be.sync()
    # request 1's row at position 15 is in its good page; those from 16 on have none
    one = P.host()[:, 2, :, 15]
    before[:, 2, :, 15] = one
    np.testing.assert_array_equal(one[1], ref.bf16(v[20].double().cpu().numpy()))
    placed = [(i, 0, 12 + i) for i in range(20)] + [(int(cu[4]) + i, 4, 7 + i) for i in range(3)]
    check_rows(P, before, qg, k, v, ctx, table, placed, group, 1, parts=1)
    assert (ctx[int(cu[2]):int(cu[4])] == 7).all(), "a chunk that was left out was written"


@pytest.mark.parametrize("dtype", [0, 1])
def test_decode_infinite_values_and_keys(be, dtype):
    """Infinities in live rows come out as the formula says: a value's in its own dim, those of both signs as NaN, a key's
    that makes the score -infinity as a token without weight; whole units and cut ones."""
    import torch
    lens, page, KH, group = [40, 5000], 16, 1, 8
    n_pages = sum(-(-n // page) for n in lens)
    P = Pool(be, n_pages, page, KH, seed=61)
    table = pages_for(lens, page, n_pages, seed=61)
    qg, k, v, ctx = P.inputs(2, 8, dtype)
    pos, td = ints([n - 1 for n in lens]), ints(table)
    inf = float("inf")
    qg[:, :, HD:].clamp_(-4, 4)

    def call():
        P.cache.decode_dev(0, 2, qg.data_ptr(), k.data_ptr(), v.data_ptr(), pos.data_ptr(), td.data_ptr(), table.shape[1],
                           ctx.data_ptr(), H=8, dtype=dtype)
        be.sync()
        return ctx.clone()

    def row(which, r, t):
        return P.kv[0, which, int(table[r, t // page]), 0, t % page]

    plain = call()
    for r, ts in ((0, (7, 30)), (1, (2000, 4990))):
        row(1, r, ts[0])[5] = inf
        row(1, r, ts[1])[9] = -inf
        row(1, r, ts[0])[11] = inf
        row(1, r, ts[1])[11] = -inf
    v[:, :, 13] = inf
    got = call()
    assert (got[..., 5] == inf).all() and (got[..., 9] == -inf).all() and got[..., 11].isnan().all() and (got[..., 13] == inf).all()
    rest = [d for d in range(HD) if d not in (5, 9, 11, 13)]
    assert torch.equal(got[..., rest], plain[..., rest])

    for r, t in ((0, 7), (1, 2000)):
        row(1, r, t)[:] = 0
    v[:, :, 13] = 0
    for r, t in ((0, 30), (1, 4990)):
        row(1, r, t)[:] = 0
    for r, t in ((0, 7), (1, 2000)):
        row(0, r, t)[200] = -inf               # behind the rotated dims: q keeps its sign there
    got = call().double().cpu().numpy()
    after, qg64 = P.host(), qg.double().cpu().numpy()
    for r, t in ((0, 7), (1, 2000)):
        rows = np.delete(ref.rows_of(after, table[r], page, lens[r]), t, axis=2)
        q = ref.norm_rope(qg64[r:r + 1, :, :HD], P.qnw, np.array([lens[r] - 1]), ROT, EPS, THETA)[0]
        u = 2.0 ** (-16 if dtype else -24) + 2.0 ** -19
        o, tol = ref.attend(q, qg64[r, :, HD:], rows, group, u, 2.0 ** -8 if dtype else 2.0 ** -24)
        seen = qg64[r, :, 200] < 0             # .. the score is +infinity: no softmax
        assert 0 < seen.sum() < 8
        assert np.isnan(got[r][seen]).all()
        assert (np.abs(got[r] - o) <= tol)[~seen].all()


def test_repeated_calls_give_the_same_bits(be):
    """Cut and whole units, merged and joined: a call gives the same bits each time, decode and prefill."""
    P = Pool(be, 700, 16, 2, seed=71)
    lens = [4000, 33, 700, 3000, 1, 129]
    table = pages_for([n + 40 for n in lens], 16, 700, seed=71)
    td, cu = ints(table), ints([0, 40, 57, 58, 90, 90, 99])
    pos, base = ints([n - 1 for n in lens]), ints(lens)
    d, p = P.inputs(6, 16, 1), P.inputs(99, 16, 1)
    d32 = P.inputs(6, 16, 0)
    kept = None
    for _ in range(30):
        for x, dtype in ((d, 1), (d32, 0)):
            x[3].zero_()
            P.cache.decode_dev(0, 6, *(t.data_ptr() for t in x[:3]), pos.data_ptr(), td.data_ptr(), table.shape[1], x[3].data_ptr(),
                               dtype=dtype)
        p[3].zero_()
        P.cache.prefill_dev(0, 6, 99, cu.data_ptr(), base.data_ptr(), *(t.data_ptr() for t in p[:3]), td.data_ptr(),
                            table.shape[1], p[3].data_ptr())
        be.sync()
        got = [t.clone() for t in (d[3], d32[3], p[3], P.kv)]
        kept = kept or got
        for a, b in zip(got, kept):
            assert P.torch.equal(a, b)


# chunks whose rows share 128-key tiles with later ones: whole units, cut ones, one query head a group, a start inside a page
@pytest.mark.parametrize("chunks,page,KH,group", [
    ([(60, 0), (40, 100), (3, 5)], 16, 2, 8), ([(200, 70)], 64, 1, 1), ([(300, 2100), (9, 0)], 128, 2, 4), ([(24, 9000)], 64, 1, 8)])
def test_prefill_non_finite_values_reach_no_earlier_row(be, chunks, page, KH, group):
    """Infinite and NaN values of new rows: rows that do not see them are bit for bit what they are without them, rows that
    do have the infinity or NaN in its dim and no other; in the call after, nothing is left of them."""
    import torch
    total = [n + c for n, c in chunks]
    n_pages = sum(-(-n // page) for n in total) + 1
    P = Pool(be, n_pages, page, KH, seed=81)
    table = pages_for(total, page, n_pages, seed=81)
    poison(P, table, total)
    cu = np.concatenate([[0], np.cumsum([n for n, _ in chunks])])
    S = int(cu[-1])
    qg, k, v, ctx = P.inputs(S, KH * group, 1)
    qg[:, :, HD:].clamp_(-4, 4)
    cu_d, base, td = ints(cu), ints([c for _, c in chunks]), ints(table)

    def call(v):
        ctx.fill_(7.0)
        P.cache.prefill_dev(0, len(chunks), S, cu_d.data_ptr(), base.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(),
                            td.data_ptr(), table.shape[1], ctx.data_ptr(), H=KH * group)
        be.sync()
        return ctx.clone()

    plain = call(v)
    want, odd = plain.clone(), v.clone()
    for r, (n, _) in enumerate(chunks):
        mine = slice(int(cu[r]), int(cu[r + 1]))
        for i, d, x in ((n // 3, 3, float("inf")), (n // 2, 130, float("-inf")), (2 * n // 3, 77, float("nan")), (n - 1, 255, float("inf")),
                        (n // 3, 200, float("inf")), (n // 2, 200, float("-inf"))):
            odd[int(cu[r]) + i, KH - 1, d] = x
        seen = torch.where(odd[mine].isfinite(), 0.0, odd[mine].float()).cumsum(0)   # inf - inf: NaN
        want[mine] = (plain[mine].float() + seen.repeat_interleave(group, 1)).bfloat16()
    for _ in range(2):
        assert torch.equal(call(odd).nan_to_num(nan=1e30), want.nan_to_num(nan=1e30))
    assert torch.equal(call(v), plain)


@pytest.mark.parametrize("rows,dtype", [(0, 1), (0, 0), (5, 1)])
def test_contexts_of_a_million_tokens(be, rows, dtype):
    """A decode step (rows 0) and a chunk at position 10^6, over a table that names a few pages again and again; KV heads
    and lengths odd."""
    import torch
    page, KH, group, T, n_pages = 48, 3, 4, 1000003, 40
    P = Pool(be, n_pages, page, KH, seed=91)
    P.kv.mul_(0.25)
    rng = np.random.default_rng(91)
    table = rng.integers(0, n_pages - 2, size=(1, -(-T // page)))
    n = max(rows, 1)
    table[0, (T - n) // page:] = [n_pages - 2, n_pages - 1][-(table.shape[1] - (T - n) // page):]    # its own
    qg, k, v, ctx = P.inputs(n, KH * group, dtype)
    td, at = ints(table), ints([T - n])
    if rows:
        cu = ints([0, n])
        P.cache.prefill_dev(0, 1, n, cu.data_ptr(), at.data_ptr(), qg.data_ptr(), k.data_ptr(), v.data_ptr(), td.data_ptr(),
                            table.shape[1], ctx.data_ptr(), H=KH * group)
    else:
        P.cache.decode_dev(0, 1, qg.data_ptr(), k.data_ptr(), v.data_ptr(), at.data_ptr(), td.data_ptr(), table.shape[1],
                           ctx.data_ptr(), H=KH * group, dtype=dtype)
    be.sync()
    pos = np.arange(T - n, T)
    q = torch.tensor(ref.norm_rope(qg[..., :HD].double().cpu().numpy(), P.qnw, pos, ROT, EPS, THETA), device="cuda")
    where = ints(table[0, pos // page]).long(), ints(pos % page).long()
    kn = torch.tensor(ref.norm_rope(k.double().cpu().numpy(), P.knw, pos, ROT, EPS, THETA), device="cuda")
    assert ((P.kv[0, 0][where[0], :, where[1]].double() - kn).abs() <= (2.0 ** -8 + 2.0 ** -16) * kn.abs() + 1e-4).all()
    u, u_out = 2.0 ** (-8 if rows else -16 if dtype else -24) + 2.0 ** -19, 2.0 ** -8 if dtype else 2.0 ** -24
    for h in range(KH * group):
        K, V = (P.kv[0, w][td[0].long(), h // group].reshape(-1, HD)[:T].double() for w in (0, 1))
        s, a = q[:, h] @ K.T / 16, q[:, h].abs() @ K.abs().T / 16
        s = s.masked_fill(torch.arange(T, device="cuda") > ints(pos)[:, None], -float("inf"))
        p, gate = s.softmax(-1), torch.sigmoid(qg[:, h, HD:].double())
        o = p @ V * gate
        # as in pages_ref; a 32-bit sum takes at most 62500 x 3 / 592 tiles in a warp (8 x 7800 / 148 in a prefill's CTA) and
        # 592 pieces in the joins, each off by 2^-24 of it: below 2^-14, beside pages_ref's own
        tol = (torch.expm1(2 * u * a.amax(1, keepdim=True)) + u + 2.0 ** -13) * (p @ V.abs() * gate)
        assert ((ctx[:, h].double() - o).abs() <= tol + u_out * (o.abs() + tol) + 1e-30).all(), h
