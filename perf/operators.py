"""The paged key-value cache's operators: cases, plain forms and 64-bit values.

Operators (each on a pool [layers][K, V][n_pages][KH][page][256] of bf16 rows and a page table [requests][max_pages]):
  decode   one new token per request: q/k norm, RoPE, append, attention over the pages, sigmoid gate
  prefill  chunks of several prompts in one call, each continuing its request's pages
  copy     page src[i] -> page dst[i] in every layer
  fork     child requests that share the parent's full pages and get a copy of the started one
  compact  live pages renumbered to 0 .. n_live - 1, tables rewritten
"""
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

HD, ROT, EPS, THETA = 256, 64, 1e-6, 1e7
PAGES = (16, 32, 48, 64, 128, 256)
TOKENS = 64 * 32768 * 2          # cached tokens x KV heads of the largest decode case
SCORES = 16 * 4096 * 32768       # padded scores of the largest prefill case
MOVED = 1 << 30                  # bytes of one side of the largest page move


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one chat request in the middle of an answer, small pages: latency
        dict(name="decode 1 x 4k", op="decode", B=1, low=4093, high=4093, page=16, KH=2, group=8, f32=False, mix=1),
        # a server's batch of very different lengths, fp32 activations, four query heads to a KV head
        dict(name="decode 48 ragged f32", op="decode", B=48, low=1, high=8191, page=32, KH=4, group=4, f32=True, mix=2),
        # the full batch at full context
        dict(name="decode 64 x 32k", op="decode", B=64, low=32000, high=32768, page=64, KH=2, group=8, f32=False, mix=3),
        # three short prompts that start together
        dict(name="prefill 3 short", op="prefill", n=3, low=1, high=101, ctx=0, page=16, KH=2, group=8, mix=4),
        # chunks of nine requests at different depths, some of a single row
        dict(name="prefill 9 mixed", op="prefill", n=9, low=1, high=1023, ctx=4096, page=64, KH=2, group=8, mix=5),
        # the last chunk of a 32k prompt
        dict(name="prefill 4k after 28k", op="prefill", n=1, low=4096, high=4096, ctx=28672, page=128, KH=2, group=8, mix=6),
        # a request's started pages before it writes to them
        dict(name="copy 8", op="copy", n=8, pages=64, page=16, layers=10, KH=2, mix=7),
        # a prefix taken over as a whole
        dict(name="copy 800", op="copy", n=800, pages=2000, page=64, layers=10, KH=2, mix=8),
        # four samples of one prompt
        dict(name="fork 4", op="fork", n=4, parents=1, high=499, page=64, layers=10, KH=2, mix=9),
        # eight samples each of 32 prompts
        dict(name="fork 256", op="fork", n=256, parents=32, high=8191, page=64, layers=10, KH=2, mix=10),
        # a small pool after some requests ended
        dict(name="compact 500", op="compact", B=20, pages=500, live=290, page=16, layers=10, KH=2, mix=11),
        # a large pool, half of it free
        dict(name="compact 4000", op="compact", B=64, pages=4000, live=2000, page=64, layers=10, KH=2, mix=12),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("decode", "decode", "prefill", "prefill", "copy", "fork", "compact"))
    page, KH, mix = rng.choice(PAGES), rng.choice((1, 2, 2, 4)), rng.randrange(1 << 20)
    if op == "decode":
        B = _log(rng, 1, 64)
        high = _log(rng, 1, min(32768, TOKENS // (B * KH)))
        return dict(op=op, B=B, low=rng.choice((1, max(1, high // 2), high)), high=high, page=page, KH=KH,
                    group=rng.choice((1, 2, 4, 8, 8)), f32=rng.random() < 0.3, mix=mix)
    if op == "prefill":
        n, group = _log(rng, 1, 16), rng.choice((1, 2, 4, 8, 8))
        high = _log(rng, 1, 4096)
        room = SCORES // (n * KH * group * high) - high
        while room < 0:
            n, high = max(1, n // 2), max(1, high // 2)
            room = SCORES // (n * KH * group * high) - high
        return dict(op=op, n=n, low=rng.choice((1, max(1, high // 2), high)), high=high,
                    ctx=rng.choice((0, _log(rng, 1, max(1, min(28672, room))))), page=page, KH=KH, group=group, mix=mix)
    layers = rng.choice((1, 4, 10))
    most = MOVED // (layers * 4 * KH * page * HD)
    if op == "copy":
        n = _log(rng, 1, min(2000, most))
        return dict(op=op, n=n, pages=2 * n + rng.randrange(1, 200), page=page, layers=layers, KH=KH, mix=mix)
    if op == "fork":
        n = _log(rng, 1, min(256, most))
        return dict(op=op, n=n, parents=rng.randint(1, min(n, 32)), high=_log(rng, 1, min(8192, page * 128)), page=page,
                    layers=layers, KH=KH, mix=mix)
    pages = _log(rng, 16, min(6000, 2 * most))
    return dict(op=op, B=rng.randint(1, 64), pages=pages, live=max(1, int(pages * rng.uniform(0.1, 0.95))), page=page,
                layers=layers, KH=KH, mix=mix)


def _lengths(case):
    """The requests' lengths: spread over the logarithm from low to high, the longest one among them."""
    rng, n = random.Random(case["mix"]), case.get("B") or case["n"]
    got = [_log(rng, case["low"], case["high"]) for _ in range(n)]
    got[rng.randrange(n)] = case["high"]
    return got


def _contexts(case):
    """The tokens that each request of a prefill holds already."""
    rng, n = random.Random(case["mix"] + 1), case["n"]
    got = [rng.randint(0, case["ctx"]) for _ in range(n)]
    got[rng.randrange(n)] = case["ctx"]
    return got


def _parents(case):
    rng = random.Random(case["mix"])
    lens = [rng.randint(1, case["high"]) for _ in range(case["parents"])]
    return lens, [i % case["parents"] for i in range(case["n"])]


def work(case):
    op, KH, page = case["op"], case["KH"], case["page"]
    row = HD * 2 * 2                      # a token's K and V rows of one KV head
    if op == "decode":
        T, B, H, act = sum(_lengths(case)), case["B"], KH * case["group"], 4 if case["f32"] else 2
        inout = B * (3 * H + 2 * KH) * HD * act
        return {"bytes": T * KH * row + inout + 4 * B * (1 + case["high"] // page), "flops": 4.0 * HD * H * T}
    if op == "prefill":
        lens, ctx, H = _lengths(case), _contexts(case), KH * case["group"]
        S, T = sum(lens), sum(lens) + sum(ctx)
        seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(lens, ctx))
        return {"bytes": T * KH * row + S * (3 * H + 2 * KH) * HD * 2, "flops": 4.0 * HD * H * seen}
    moved = case["layers"] * KH * row * 2  # a token's rows, read and written, in every layer
    if op == "copy":
        return {"bytes": moved * page * case["n"] + 8 * case["n"], "flops": 0}
    if op == "fork":
        lens, parent = _parents(case)
        return {"bytes": sum(moved * (lens[p] % page) + 8 * (1 + lens[p] // page) for p in parent), "flops": 0}
    L, P = case["live"], case["pages"]
    return {"bytes": moved * page * (L * (P - L) // P) + 8 * L, "flops": 0}


# ---------------------------------------------------------------- inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed * 1000003 + case["mix"])
    op, page, KH = case["op"], case["page"], case["KH"]

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def tables(counts, rows, n_pages, fill=0):
        """`counts[r]` pages of their own for request r, anywhere in the pool."""
        width = max(counts)
        ids = rng.sample(range(n_pages), sum(counts))
        table, at = np.full((rows, width), fill, np.int32), 0
        for r, c in enumerate(counts):
            table[r, :c] = ids[at:at + c]
            at += c
        return table, set(range(n_pages)) - set(ids)

    if op in ("decode", "prefill"):
        lens = _lengths(case)
        ctx = [n - 1 for n in lens] if op == "decode" else _contexts(case)
        total = lens if op == "decode" else [n + c for n, c in zip(lens, ctx)]
        counts = [-(-t // page) for t in total]
        n_pages = sum(counts) + 3
        table, _ = tables(counts, len(counts), n_pages)
        rows, H = len(lens) if op == "decode" else sum(lens), KH * case["group"]
        act = torch.float32 if case.get("f32") else torch.bfloat16
        s = dict(pool=normal(1, 2, n_pages, KH, page, HD), table=ints(table), width=max(counts), longest=max(total),
                 qg=normal(rows, H, 2 * HD, dtype=act), k=normal(rows, KH, HD, dtype=act), v=normal(rows, KH, HD, dtype=act),
                 qnw=normal(HD, dtype=torch.float32) * 0.1, knw=normal(HD, dtype=torch.float32) * 0.1,
                 ctx=torch.zeros(rows, H, HD, dtype=act, device="cuda"), H=H)
        if op == "decode":
            s["pos"] = ints(ctx)
        else:
            s["most"] = max(lens)
            s["base"], s["cu"] = ints(ctx), ints(np.concatenate([[0], np.cumsum(lens)]))
        return s
    layers = case["layers"]
    if op == "copy":
        n_pages, n = case["pages"], case["n"]
        ids = rng.sample(range(n_pages), 2 * n)
        return dict(pool=normal(layers, 2, n_pages, KH, page, HD), src=ints(ids[:n]), dst=ints(ids[n:]))
    if op == "fork":
        lens, parent = _parents(case)
        n, counts = case["n"], [-(-t // page) for t in lens]
        n_pages = sum(counts) + n + 2
        table, free = tables(counts, len(lens) + n, n_pages)
        return dict(pool=normal(layers, 2, n_pages, KH, page, HD), table=ints(table), width=table.shape[1],
                    parent=ints(parent), child=ints([len(lens) + i for i in range(n)]),
                    fresh=ints(sorted(free)[:n]), len=ints(lens + [0] * n))
    B, L, n_pages = case["B"], case["live"], case["pages"]
    counts = [L // B + (r < L % B) for r in range(B)]
    lens = [max(0, c * page - rng.randrange(page)) for c in counts]
    table, _ = tables(counts, B, n_pages, fill=-1)
    return dict(pool=normal(layers, 2, n_pages, KH, page, HD), table=ints(table), width=table.shape[1], len=ints(lens),
                table_out=torch.zeros_like(ints(table)), live=torch.zeros(1, dtype=torch.int32, device="cuda"))


_BE, _STREAM = None, None


def _backend():
    """The backend, on the stream that torch uses now (1 names the legacy default stream, whose torch handle is 0)."""
    global _BE, _STREAM
    if _BE is None:
        d = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3.c_b200")
        spec = importlib.util.spec_from_file_location("qwen3c_b200", os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        sys.modules["qwen3c_b200"] = pkg = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(pkg)
        _BE = pkg, pkg.Backend(0)
    stream = torch._C._cuda_getCurrentRawStream(0) or 1    # (without the Stream object, 3 us of a 5 us call)
    if stream != _STREAM:
        _BE[1].set_stream(stream)
        _STREAM = stream
    return _BE


def prepare(case, seed):
    s = _inputs(case, seed)
    s["op"], s["page"] = case["op"], case["page"]
    if own:
        pkg, be = _backend()
        layers, _, n_pages, KH, page, _ = s["pool"].shape
        s["cache"] = pkg.PagedCache(be, layers, n_pages, page, KH, kv=s["pool"].data_ptr())
        if "qnw" in s:
            s["cache"].norm_weight(0, s["qnw"].cpu().numpy(), s["knw"].cpu().numpy())
    return s


# ---------------------------------------------------------------- plain forms
def _norm_rope(x, w, pos):
    """Zero-centred RMSNorm over a head, then the half-split rotation of its first ROT dims at `pos`."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w)
    j = torch.arange(ROT // 2, device=x.device, dtype=torch.float64)
    angle = pos.double()[..., None] * torch.pow(torch.tensor(THETA, dtype=torch.float64, device=x.device), -2 * j / ROT)
    cos, sin = angle.cos().float(), angle.sin().float()
    lo, hi, rest = x[..., :ROT // 2], x[..., ROT // 2:ROT], x[..., ROT:]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, rest], -1)


def _append(s, k, v, req, pos):
    at = s["table"][req, pos // s["page"]].long()
    s["pool"][0, 0, at, :, pos % s["page"]] = k.bfloat16()
    s["pool"][0, 1, at, :, pos % s["page"]] = v.bfloat16()


def _gathered(s, which):
    """K or V of every request, [requests][KH][longest][HD] in 32 bits."""
    x = s["pool"][0, which][s["table"].long()].transpose(1, 2)      # [requests][KH][pages][page][HD]
    return x.reshape(x.shape[0], x.shape[1], -1, HD)[:, :, :s["longest"]].float()


def _attend(q, keys, values, seen):
    """q [n][KH][m][HD], keys and values [n][KH][T][HD], seen [n][1][m][T]."""
    x = (q @ keys.transpose(-1, -2)) * HD ** -0.5
    x = x.masked_fill_(~seen, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True)).exp_()
    return (x @ values) / x.sum(-1, keepdim=True)


def _plain_decode(s):
    B, H = s["pos"].shape[0], s["H"]
    KH, pos = s["k"].shape[1], s["pos"].long()
    q = _norm_rope(s["qg"][..., :HD].float(), s["qnw"], pos[:, None])
    k = _norm_rope(s["k"].float(), s["knw"], pos[:, None])
    _append(s, k, s["v"], torch.arange(B, device=pos.device), pos)
    seen = torch.arange(s["longest"], device=pos.device) <= pos[:, None, None, None]
    o = _attend(q.view(B, KH, -1, HD), _gathered(s, 0), _gathered(s, 1), seen).reshape(B, H, HD)
    s["ctx"].copy_(o * torch.sigmoid(s["qg"][..., HD:].float()))
    return {"ctx": s["ctx"], "pool": s["pool"]}


def _plain_prefill(s):
    (S, KH), H, n, most = s["k"].shape[:2], s["H"], s["base"].shape[0], s["most"]
    rows = torch.arange(S, device="cuda")
    req = torch.searchsorted(s["cu"][1:].long(), rows, right=True)
    at = rows - s["cu"].long()[req]
    pos = s["base"].long()[req] + at
    q = _norm_rope(s["qg"][..., :HD].float(), s["qnw"], pos[:, None])
    k = _norm_rope(s["k"].float(), s["knw"], pos[:, None])
    _append(s, k, s["v"], req, pos)
    padded = torch.zeros(n, most, H, HD, device="cuda")
    padded[req, at] = q
    padded = padded.view(n, most, KH, -1, HD).permute(0, 2, 3, 1, 4).reshape(n, KH, -1, HD)
    last = s["base"].long()[:, None] + torch.arange(most, device="cuda")
    seen = torch.arange(s["longest"], device="cuda") <= last.repeat(1, H // KH)[:, None, :, None]
    o = _attend(padded, _gathered(s, 0), _gathered(s, 1), seen)
    o = o.view(n, KH, H // KH, most, HD).permute(0, 3, 1, 2, 4).reshape(n, most, H, HD)[req, at]
    s["ctx"].copy_(o * torch.sigmoid(s["qg"][..., HD:].float()))
    return {"ctx": s["ctx"], "pool": s["pool"]}


def _plain_copy(s):
    s["pool"][:, :, s["dst"].long()] = s["pool"][:, :, s["src"].long()]
    return {"pool": s["pool"].view(torch.int16)}


def _plain_fork(s):
    table, parent, child, page = s["table"], s["parent"].long(), s["child"].long(), s["page"]
    length = s["len"][parent].long()
    full, tail = length // page, length % page
    col = torch.arange(s["width"], device="cuda")
    rows = torch.where(col < full[:, None], table[parent], table[child])
    rows = torch.where((col == full[:, None]) & (tail > 0)[:, None], s["fresh"][:, None], rows)
    src, dst = table[parent, full.clamp(max=s["width"] - 1)].long(), s["fresh"].long()
    held = torch.arange(page, device="cuda")[:, None] < tail[:, None, None, None]
    s["pool"][:, :, dst] = torch.where(held, s["pool"][:, :, src], s["pool"][:, :, dst])
    table[child] = rows
    s["len"][child] = length.int()
    return {"pool": s["pool"].view(torch.int16), "table": table, "len": s["len"]}


def _plain_compact(s):
    n_pages, table = s["pool"].shape[2], s["table"].long()
    used = torch.arange(s["width"], device="cuda") < -(-s["len"].long() // s["page"])[:, None]
    live = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
    live[table[used]] = True
    count, ids = live.sum(), torch.arange(n_pages, device="cuda")
    dst, src = ids[~live & (ids < count)], ids[live & (ids >= count)]
    s["pool"][:, :, dst] = s["pool"][:, :, src]
    ids[src] = dst
    s["table_out"].copy_(torch.where(used, ids[table.clamp(min=0)], table))
    s["live"].copy_(count.view(1))
    return {"pool": s["pool"].view(torch.int16), "table": s["table_out"], "live": s["live"]}


# ---------------------------------------------------------------- one pass
def run(state):
    s = state
    if not own:
        return {"decode": _plain_decode, "prefill": _plain_prefill, "copy": _plain_copy, "fork": _plain_fork,
                "compact": _plain_compact}[s["op"]](s)
    _backend()
    c, p = s["cache"], torch.Tensor.data_ptr
    if s["op"] == "decode":
        c.decode_dev(0, s["pos"].shape[0], p(s["qg"]), p(s["k"]), p(s["v"]), p(s["pos"]), p(s["table"]), s["width"], p(s["ctx"]),
                     H=s["H"], rot=ROT, eps=EPS, theta=THETA, dtype=int(s["qg"].dtype == torch.bfloat16))
        return {"ctx": s["ctx"], "pool": s["pool"]}
    if s["op"] == "prefill":
        c.prefill_dev(0, s["base"].shape[0], s["qg"].shape[0], p(s["cu"]), p(s["base"]), p(s["qg"]), p(s["k"]), p(s["v"]),
                      p(s["table"]), s["width"], p(s["ctx"]), H=s["H"], rot=ROT, eps=EPS, theta=THETA)
        return {"ctx": s["ctx"], "pool": s["pool"]}
    if s["op"] == "copy":
        c.copy_dev(s["src"].shape[0], p(s["src"]), p(s["dst"]))
        return {"pool": s["pool"].view(torch.int16)}
    if s["op"] == "fork":
        c.fork_dev(s["parent"].shape[0], p(s["parent"]), p(s["child"]), p(s["fresh"]), p(s["len"]), p(s["table"]),
                   s["len"].shape[0], s["width"])
        return {"pool": s["pool"].view(torch.int16), "table": s["table"], "len": s["len"]}
    c.compact_dev(s["len"].shape[0], p(s["len"]), p(s["table"]), s["width"], p(s["table_out"]), p(s["live"]))
    return {"pool": s["pool"].view(torch.int16), "table": s["table_out"], "live": s["live"]}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    """ctx and the appended rows from the definition, request by request; page moves are whole numbers and need none."""
    if case["op"] not in ("decode", "prefill"):
        return None
    s = _inputs(case, seed)
    KH, page, H, group = case["KH"], case["page"], s["H"], case["group"]
    lens = [1] * case["B"] if case["op"] == "decode" else _lengths(case)
    base = s["pos"].tolist() if case["op"] == "decode" else s["base"].tolist()
    freq = torch.tensor([THETA ** (-2.0 * j / ROT) for j in range(ROT // 2)], dtype=torch.float64, device="cuda")

    def head(x, w, at):                                  # x [rows][heads][HD], at [rows]
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / HD + EPS).sqrt() * (1.0 + w.double())
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), at.double()[:, None, None] * freq)
        z = torch.complex(x[..., :ROT // 2].contiguous(), x[..., ROT // 2:ROT].contiguous()) * turn
        return torch.cat((z.real, z.imag, x[..., ROT:]), -1)

    pool = s["pool"][0]
    fresh, ctx, row = pool.float(), torch.zeros(s["ctx"].shape, dtype=torch.float64, device="cuda"), 0
    for r, n in enumerate(lens):
        at = torch.arange(base[r], base[r] + n, device="cuda")
        T = base[r] + n
        ids = s["table"][r, :-(-T // page)].long()
        mine = slice(row, row + n)
        k = head(s["k"][mine], s["knw"], at)
        v = s["v"][mine].double()
        where = ids[at // page], at % page
        for which, new in ((0, k), (1, v)):
            fresh[which][where[0], :, where[1]] = new.float()
            pool[which][where[0], :, where[1]] = new.bfloat16()
        q = head(s["qg"][mine, :, :HD], s["qnw"], at)
        keys, values = (pool[w][ids].transpose(0, 1).reshape(KH, -1, HD)[:, :T] for w in (0, 1))
        for h in range(H):
            K, V = keys[h // group].double(), values[h // group].double()
            x = q[:, h] @ K.t() / math.sqrt(HD)
            x = x + torch.zeros_like(x).masked_fill_(torch.arange(T, device="cuda")[None] > at[:, None], -math.inf)
            gate = 1.0 / (1.0 + torch.exp(-s["qg"][mine, h, HD:].double()))
            ctx[mine, h] = torch.softmax(x, -1) @ V * gate
        row += n
    return {"ctx": ctx, "pool": fresh[None]}
