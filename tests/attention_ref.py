"""Float64 references of the window attention, its gradients and the 4-bit KV
cache, and the bounds that their bf16 results are held to.

Bounds count the roundings to bf16, each at most u = 2^-8 of its value, and
u / 4 of the terms' magnitudes for everything done in f32 (scores, exponentials,
sums: thousands of roundings of 2^-24 each).
"""
import numpy as np

U = 2.0 ** -8
HD = 128


def visible(i, j, window, sinks):
    ok = j <= i
    if window:
        ok &= (i - j < window) | (j < sinks)
    return ok


def attention(q, k, v, window, sinks, first=0, d_out=None, keep=None):
    """One query head: q / d_out [n, 128] at positions first .., k / v [L, 128]
    (float64).  keep: bool [L], keys that exist.  Returns a dict of out, lse and
    (with d_out) dq, dk, dv, and the bound of each under e_out, e_lse, ..."""
    n, L = len(q), len(k)
    scale = 1 / np.sqrt(HD)
    i, j = first + np.arange(n)[:, None], np.arange(L)[None]
    ok = visible(i, j, window, sinks)
    if keep is not None:
        ok &= keep[None]
    s = np.where(ok, q @ k.T * scale, -np.inf)
    empty = ~ok.any(1)
    m = np.where(empty, 0, s.max(1, initial=-np.inf))
    e = np.exp(s - m[:, None])
    total = e.sum(1)
    p = e / np.where(empty, 1, total)[:, None]
    out = p @ v
    mag = p @ np.abs(v)
    r = dict(out=out, lse=np.where(empty, -np.inf, m + np.log(np.where(empty, 1, total))))
    # p rounded in the numerator, the sum of rounded p in the denominator, then
    # the output itself.
    r["e_out"] = U * (mag + 2 * np.abs(out)) * (1 + U) + U / 4 * mag
    r["e_lse"] = np.full(n, U + U / 4)
    if d_out is None:
        return r
    dp = d_out @ v.T
    delta = (d_out * out).sum(1, keepdims=True)
    ds = p * (dp - delta) * scale
    r["dv"] = p.T @ d_out
    r["dq"] = ds @ k
    r["dk"] = ds.T @ q
    # p has the error of lse and its own rounding; delta that of the output.
    e_p = (2 * U + U / 2) * p
    e_delta = (np.abs(d_out) * r["e_out"]).sum(1, keepdims=True)
    mag_dp = np.abs(d_out) @ np.abs(v).T
    mag_delta = (np.abs(d_out) * np.abs(out)).sum(1, keepdims=True)
    e_ds = scale * (p * e_delta * (1 + 4 * U) + e_p * np.abs(dp - delta)
                    + U / 4 * p * (mag_dp + mag_delta))
    for name, err, x, res in (("dv", e_p.T, d_out, r["dv"]), ("dq", e_ds, k, r["dq"]),
                              ("dk", e_ds.T, q, r["dk"])):
        r["e_" + name] = err @ np.abs(x) * (1 + U) + U * np.abs(res)
    return r


def batch_attention(q, k, v, batch, seq_len, heads, kv, window, sinks, lens=None, d_out=None):
    """q / d_out [batch * seq_len, heads * 128], k / v [.., kv * 128] float64:
    the dict of ``attention`` in these layouts (lse [batch, heads, seq_len])."""
    names = ["out"] + (["dq", "dk", "dv"] if d_out is not None else [])
    width = dict(out=heads, dq=heads, dk=kv, dv=kv)
    r = {e + n: np.zeros((batch * seq_len, width[n] * HD)) for n in names for e in ("", "e_")}
    r["lse"] = np.full((batch, heads, seq_len), -np.inf)
    r["e_lse"] = np.zeros((batch, heads, seq_len))
    for b in range(batch):
        L = seq_len if lens is None else min(max(lens[b], 0), seq_len)
        if L == 0:
            continue
        rows = slice(b * seq_len, b * seq_len + L)
        for h in range(heads):
            c = slice(h * HD, (h + 1) * HD)
            ck = slice(h // (heads // kv) * HD, (h // (heads // kv) + 1) * HD)
            one = attention(q[rows, c], k[rows, ck], v[rows, ck], window, sinks,
                            d_out=None if d_out is None else d_out[rows, c])
            for n in names:
                for e in ("", "e_"):
                    r[e + n][rows, c if n in ("out", "dq") else ck] += one[e + n]
            r["lse"][b, h, :L], r["e_lse"][b, h, :L] = one["lse"], one["e_lse"]
    return r


# ------------------------------------------------------------- 4-bit values --
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def cached_values(x):
    """What the cache holds of x [..., 128]: per group of 32 the least scale 2^s, -126
    <= s <= 125, with max|x| <= 7 * 2^s; nearest level, ties to the even code."""
    g = np.asarray(x, dtype=np.float64).reshape(-1, 32)
    bad = ~np.isfinite(g).all(1)
    top = np.abs(np.where(bad[:, None], 0, g)).max(1)
    s = np.full(len(g), -126)
    for e in range(-125, 126):
        s[top > 7 * 2.0 ** (e - 1)] = e
    y = np.abs(g) / 2.0 ** s[:, None]
    # The nearest level; a value in the middle of two goes to the even code.
    code = np.zeros(g.shape, dtype=int)
    for c in range(7):
        mid = (LEVELS[c] + LEVELS[c + 1]) / 2
        code += (y > mid) | ((y == mid) & (c % 2 == 1))
    out = np.sign(g) * LEVELS[code] * 2.0 ** s[:, None]
    out[bad] = np.nan
    return out.reshape(np.shape(x))
