"""64-bit restatement of the paged-cache operators for the tests (CPU, numpy).

Rounding a value to bf16 is off by at most 2^-8 of it (half a step), so where
q and the softmax's numerators are rounded to parts of relative error u, an
output differs from the exact one by at most
    (exp(2 d) - 1 + u) * sum_t p_t |v_t| * gate,   d = u * max_t sum_i |q_i k_ti| / 16
(every score is off by at most d, the numerators by u more), plus the rounding
of the output itself. A bf16 part leaves 2^-8 of what it rounds, so u is 2^-8
with one (prefill), 2^-16 with two (decode, bf16 activations) and 2^-24 with three
(decode, fp32 activations), plus 2^-19 for the 32-bit norm, rotation, products and
exponentials; the 32-bit sums add less than 2^-14 of the same terms.
"""
import numpy as np

HD = 256


def bf16(x):
    """Round to nearest even bf16, as float64."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint32) << 16
    return r.astype(np.uint32).view(np.float32).astype(np.float64)


def norm_rope(x, w, pos, rot, eps, theta):
    """x [..., heads, 256] float64, pos [...] -> normed and roped."""
    x = np.asarray(x, np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + np.asarray(w, np.float64))
    half = rot // 2
    ang = np.asarray(pos, np.float64)[..., None, None] * np.float64(theta) ** (-2.0 * np.arange(half) / rot)
    c, s = np.cos(ang), np.sin(ang)
    lo, hi = x[..., :half].copy(), x[..., half:rot].copy()
    x[..., :half] = lo * c - hi * s
    x[..., half:rot] = hi * c + lo * s
    return x


def rows_of(pool, table, page, T):
    """K and V rows 0..T-1 of a request, [2][KH][T][256]; pool [2][n_pages][KH][page][256]."""
    ids = table[:-(-T // page)]
    x = pool[:, ids].swapaxes(1, 2)
    return x.reshape(2, pool.shape[2], -1, HD)[:, :, :T]


def attend(q, gate, rows, group, u, u_out):
    """One query row: q, gate [H][256], rows [2][KH][T][256] -> (ctx, bound)."""
    K, V = rows[0].repeat(group, 0), rows[1].repeat(group, 0)
    s = np.einsum("hd,htd->ht", q, K) / 16.0
    a = np.einsum("hd,htd->ht", np.abs(q), np.abs(K)).max(1, keepdims=True) / 16.0
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    g = 1.0 / (1.0 + np.exp(-gate))
    o = np.einsum("ht,htd->hd", p, V) * g
    spread = np.einsum("ht,htd->hd", p, np.abs(V)) * g
    tol = (np.expm1(2 * u * a) + u + 2.0 ** -14) * spread
    return o, tol + u_out * (np.abs(o) + tol) + 1e-30


def compact(table, lens, page, n_pages):
    """(new table, live, [(src, dst)])."""
    held = [max(0, -(-int(n) // page)) for n in lens]
    live_ids = sorted({int(i) for r, n in enumerate(held) for i in table[r, :n]})
    live = len(live_ids)
    holes = sorted(set(range(live)) - set(live_ids))
    movers = [i for i in live_ids if i >= live]
    to = dict(zip(movers, holes))
    out = table.copy()
    for r, n in enumerate(held):
        for j in range(n):
            out[r, j] = to.get(int(table[r, j]), table[r, j])
    return out, live, list(zip(movers, holes))
