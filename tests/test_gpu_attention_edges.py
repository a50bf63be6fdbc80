"""Window attention and cache attention where their edges meet: the longest sequence, the
workspace of a batch whose first blocks of keys are cut, the log-sum-exp against its f32
bound, keys that are not finite beside padding, and long sequences dealt by die with
sinks."""
import numpy as np
import pytest
import torch

import attention_ref as R
from prichs_amd import _lib as L
from prichs_amd import ops, synth

pytestmark = pytest.mark.gpu
HD, PAGE = 128, L.KV_PAGE


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to("cuda").bfloat16()


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def say(*a):
    print(*a, flush=True)


def near(got, want, bound, name):
    err = np.abs(host(got) - want)
    worst = np.argmax(err - bound)
    assert (err <= bound).all(), (name, err.flat[worst], bound.flat[worst])


def inputs(B, S, H, K, seed):
    rng = np.random.default_rng(seed)
    return [synth.round_bf16(rng.standard_normal((B * S, n * HD))) for n in (H, K, K, H)]


def piece(q, k, v, d_out, a, z, W, sinks):
    """R.attention of the rows a .. z - 1 of one head (window W > 0) and the keys that
    they see, and those keys.  The sinks before the window take the places right before
    it, which leaves the mask as it is."""
    lo = max(0, a - W + 1)
    s = min(sinks, lo)
    keys = np.concatenate([np.arange(s), np.arange(lo, z)])
    return R.attention(q[a:z], k[keys], v[keys], W, s if lo > s else sinks, first=a - lo + s,
                       d_out=d_out[a:z]), keys


def by_pieces(q, k, v, d_out, B, S, H, K, W, sinks, lens):
    """R.batch_attention from pieces of 1000 rows.  A key's gradients are sums over the
    pieces, and so are their bounds."""
    r = {e + n: np.zeros((B * S, (H if n in ("out", "dq") else K) * HD))
         for n in ("out", "dq", "dk", "dv") for e in ("", "e_")}
    for b, n in enumerate(lens):
        for a in range(0, n, 1000):
            z = min(a + 1000, n)
            for h in range(H):
                c = slice(h * HD, (h + 1) * HD)
                ck = slice(h // (H // K) * HD, (h // (H // K) + 1) * HD)
                seq = slice(b * S, b * S + n)
                one, keys = piece(q[seq, c], k[seq, ck], v[seq, ck], d_out[seq, c], a, z, W, sinks)
                for e in ("", "e_"):
                    for name in ("out", "dq"):
                        r[e + name][b * S + a:b * S + z, c] = one[e + name]
                    for name in ("dk", "dv"):
                        r[e + name][b * S + keys, ck] += one[e + name]
    return r


@pytest.mark.parametrize("spans", [[(0, 200), ((1 << 20) - 100, (1 << 20) + 100),
                                    ((1 << 21) - 300, 1 << 21)]])
def test_the_longest_sequence(cuda, spans):
    """2^21 rows: the first, some in the middle and the last, in both directions."""
    S, H, K, W = 1 << 21, 4, 1, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv, d_o = (torch.randn((S, n * HD), generator=g, device="cuda", dtype=torch.bfloat16)
                for n in (H + 2 * K, H))
    q, k, v = qkv[:, :H * HD], qkv[:, H * HD:(H + K) * HD], qkv[:, (H + K) * HD:]
    out, lse = ops.window_attention(q, k, v, 1, S, H, K, W, want_lse=True)
    dq, dk, dv = ops.window_attention_backward(d_o, q, k, v, out, lse, 1, S, H, K, W)
    for a, z in spans:
        say("rows:", a, z)
        lo, end = max(0, a - W), min(S, z + W)  # and what sees their keys
        rows = slice(lo, end)
        x = [host(t[rows]) for t in (q, k, v, d_o)]
        for h in range(H):
            c = slice(h * HD, (h + 1) * HD)
            # Rows from max(lo, a) on see nothing before lo.
            one, keys = piece(x[0][:, c], x[1], x[2], x[3][:, c], a - lo, end - lo, W, 0)
            for name, t in (("out", out), ("dq", dq)):
                near(t[a:z, c], one[name][:z - a], one["e_" + name][:z - a], name)
            if h == 0:
                sums = {e + n: 0 for n in ("dk", "dv") for e in ("", "e_")}
            for name in sums:
                sums[name] = sums[name] + one[name][keys >= a - lo][:z - a]
        for name, t in (("dk", dk), ("dv", dv)):
            near(t[a:z], sums[name], sums["e_" + name], name)


@pytest.mark.parametrize("B,S,H,K,W,sinks,lens", [
    (6, 1500, 4, 4, 60, 4, [1500, 3, 0, 1400, 129, 700]), (10, 1100, 8, 4, 60, 200, [1100] * 9 + [64])])
def test_a_workspace_of_the_size_asked_for_is_enough(cuda, B, S, H, K, W, sinks, lens):
    """Batches whose partial sums are of the cut blocks only: the right gradients, and
    nothing written behind the workspace."""
    say("case:", B, S, H, K, W, sinks)
    x = inputs(B, S, H, K, 5)
    ref = by_pieces(*x, B, S, H, K, W, sinks, lens)
    q, k, v, d_o = (dev(a) for a in x)
    sl = i32(lens)
    out, lse = ops.window_attention(q, k, v, B, S, H, K, W, sinks, sl, want_lse=True)
    lib = L.load()
    need = lib.prichs_window_attention_backward_workspace(B, S, H, K, W, sinks)
    ws = torch.full((need + (4 << 20),), 0xff, dtype=torch.uint8, device="cuda")
    grads = [torch.empty_like(t) for t in (q, k, v)]
    args = [a for t in (d_o, q, k, v, out) for a in (t.data_ptr(), t.stride(0))]
    to = [a for t in grads for a in (t.data_ptr(), t.stride(0))]
    L.check(lib.prichs_window_attention_backward(
        *args, lse.data_ptr(), sl.data_ptr(), *to, B, S, H, K, HD, W, sinks, L.DTYPE_BF16,
        ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    for t, name in zip(grads, ("dq", "dk", "dv")):
        near(t, ref[name], ref["e_" + name], name)
    assert (ws[need:] == 0xff).all()


# ------------------------------------------------------------ log-sum-exp --
def lse_and_bound(q, k, first, W, sinks):
    """lse of query rows q [n, 128] at positions first .. over keys k [L, 128], and how
    far one formed in f32 may be off.  With ulp = 2^-23, which is also what a sum that
    cuts off instead of rounding loses:
      a score      128 additions, each of at most the terms' magnitudes;
      an exponent  up to 8 roundings of the largest score (scale, product, maximum);
      the sum      an addition for each visible key, and for each 64 keys a rescaling
                   by a power that is off by its exponent's rounding, and a join;
      the logarithm and what is added to it: 4 of the result and of the sum's."""
    i, j = first + np.arange(len(q))[:, None], np.arange(len(k))[None]
    ok = R.visible(i, j, W, sinks)
    scale = 1 / np.sqrt(HD)
    s = np.where(ok, q @ k.T * scale, -np.inf)
    m = s.max(1)
    lse = m + np.log(np.exp(s - m[:, None]).sum(1))
    terms = np.where(ok, np.abs(q) @ np.abs(k).T * scale, 0).max(1)
    top = np.where(ok, np.abs(s), 0).max(1)
    n = ok.sum(1)
    blocks = n // 64 + 2 + sinks // 64
    return lse, 2.0 ** -23 * (128 * terms + 8 * top + n + 8 * blocks * (1 + top)
                              + 4 * (np.abs(lse) + np.log(n) + 1))


@pytest.mark.parametrize("S,H,K,W,sinks,lens", [
    (1, 1, 1, 0, 0, None), (70, 4, 1, 2, 0, None), (70, 4, 2, 3, 1, None), (300, 6, 3, 0, 0, None),
    (200, 2, 2, 17, 70, [133]), (2600, 4, 1, 300, 4, None), (1700, 48, 12, 5, 0, None)])
def test_lse_is_formed_in_f32(cuda, S, H, K, W, sinks, lens):
    """Of the unrounded exponentials, though the output's sum is of rounded ones."""
    say("case:", S, H, K, W, sinks, lens)
    q, k, v, _ = inputs(1, S, H, K, S + W)
    _, lse = ops.window_attention(dev(q), dev(k), dev(v), 1, S, H, K, W, sinks,
                                  None if lens is None else i32(lens), want_lse=True)
    n = S if lens is None else lens[0]
    for h in range(H):
        c, ck = slice(h * HD, (h + 1) * HD), slice(h // (H // K) * HD, (h // (H // K) + 1) * HD)
        want, bound = lse_and_bound(q[:n, c], k[:n, ck], 0, W, sinks)
        near(lse[0, h, :n], want, bound, h)
        assert torch.isneginf(lse[0, h, n:]).all()


# 4, 2 and 1 heads that share tiles; few workgroups, many, and dealt by die.
WITHOUT_LSE = [
    (2, 200, 4, 1, 17, 3), (1, 300, 6, 3, 100, 70), (1, 257, 3, 3, 0, 0), (3, 330, 48, 12, 100, 4),
    (6, 330, 24, 12, 90, 0), (6, 330, 24, 24, 0, 0), (1, 8200, 8, 2, 150, 4), (1, 8195, 6, 3, 70, 0),
    (2, 8193, 3, 3, 100, 0)]


@pytest.mark.parametrize("B,S,H,K,W,sinks", WITHOUT_LSE)
def test_the_output_does_not_depend_on_whether_lse_is_wanted(cuda, B, S, H, K, W, sinks):
    say("case:", B, S, H, K, W, sinks)
    q, k, v = (dev(x) for x in inputs(B, S, H, K, S)[:3])
    for lens in (None, i32([S - 70] * B)):
        out, lse = ops.window_attention(q, k, v, B, S, H, K, W, sinks, lens, want_lse=True)
        assert torch.isfinite(out).all() and torch.isfinite(lse[:, :, :S - 70]).all()
        assert torch.equal(out, ops.window_attention(q, k, v, B, S, H, K, W, sinks, lens)[0])


@pytest.mark.parametrize("n_q,lens,H,K,W,sinks", [
    (1, [1, 2, 3, 60], 4, 1, 0, 0), (1, [300, 129], 4, 2, 0, 0), (5, [900, 70], 6, 2, 3, 1),
    (1, [5000], 4, 1, 0, 0), (2, [1300, 1500], 4, 2, 0, 0), (40, [1500], 8, 2, 2, 0),
    (300, [700], 12, 3, 100, 4)])
def test_lse_over_the_cache_is_formed_in_f32(cuda, n_q, lens, H, K, W, sinks):
    """By one workgroup a tile, and joined from parts."""
    say("case:", n_q, lens, H, K, W, sinks)
    rng = np.random.default_rng(sum(lens) + W)
    batch, top = len(lens), max(lens)
    pages = -(-top // PAGE)
    table = i32(rng.permutation(batch * pages).reshape(batch, pages))
    cache = ops.kv_cache_pages(batch * pages, K)
    cache.fill_(255)
    k, v = (synth.round_bf16(rng.standard_normal((batch * top, K * HD))) for _ in range(2))
    q = synth.round_bf16(rng.standard_normal((batch * n_q, H * HD)))
    ops.kv_cache_write(cache, table, i32([0] * batch), dev(k), dev(v), batch, top, K,
                       counts=i32(lens))
    out, lse = ops.kv_cache_attention(dev(q), cache, table, i32(lens), batch, n_q, H, K, W, sinks,
                                      want_lse=True)
    # The output is the same bits with and without it.
    assert torch.equal(out, ops.kv_cache_attention(dev(q), cache, table, i32(lens), batch, n_q, H, K,
                                                   W, sinks)[0])
    kc = R.cached_values(k.reshape(-1, HD)).reshape(batch, top, K, HD)
    for b, n in enumerate(lens):
        for h in range(H):
            want, bound = lse_and_bound(q[b * n_q:(b + 1) * n_q, h * HD:(h + 1) * HD],
                                        kc[b, :n, h // (H // K)], n - n_q, W, sinks)
            near(lse[b, h], want, bound, (b, h))


# ------------------------------------------------- keys that are not finite --
def weightless(S, H, K, at, seed):
    """Inputs where key `at` holds an infinity that gives it a score of -inf with every
    query, and no weight."""
    q, k, v, g = inputs(1, S, H, K, seed)
    q[:, ::HD], k[:, ::HD] = -1, 0
    k[at, ::HD] = np.inf
    return q, k, v, g


def without_key(q, k, v, g, H, K, W, sinks, at):
    """R.batch_attention of whole sequences without key `at` (row `at` sees others)."""
    S = len(q)
    keep = np.ones(S, bool)
    keep[at] = False
    k = np.where(np.isfinite(k), k, 0)
    r = {e + n: np.zeros((S, (H if n in ("out", "dq") else K) * HD))
         for n in ("out", "dq", "dk", "dv") for e in ("", "e_")}
    for h in range(H):
        c, ck = slice(h * HD, (h + 1) * HD), slice(h // (H // K) * HD, (h // (H // K) + 1) * HD)
        one = R.attention(q[:, c], k[:, ck], v[:, ck], W, sinks, d_out=g[:, c], keep=keep)
        for n in ("out", "dq", "dk", "dv"):
            for e in ("", "e_"):
                r[e + n][:, c if n in ("out", "dq") else ck] += one[e + n]
    return r


@pytest.mark.parametrize("S,n,at", [(40, 40, 3), (40, 40, 33), (64, 40, 3), (96, 70, 66),
                                    (400, 333, 200), (400, 333, 325)])
def test_padding_does_not_reach_a_key_that_is_not_finite(cuda, S, n, at):
    """Rows past a sequence's end are in the tiles of its last rows: a key without any
    weight keeps gradients of zero, as it has without such rows."""
    H, K, W, sinks = 4, 2, 100, 2
    say("case:", S, n, at)
    q, k, v, g = (x for x in weightless(n, H, K, at, 3))
    ref = without_key(q, k, v, g, H, K, W, sinks, at)
    t = []
    for x in (q, k, v, g):
        pad = torch.full((S, x.shape[1]), float("nan"), dtype=torch.bfloat16, device="cuda")
        pad[:n] = dev(x)
        t.append(pad)
    sl = i32([n]) if S != n else None
    out, lse = ops.window_attention(*t[:3], 1, S, H, K, W, sinks, sl, want_lse=True)
    near(out[:n], ref["out"], ref["e_out"], "out")
    _, dk, dv = ops.window_attention_backward(t[3], *t[:3], out, lse, 1, S, H, K, W, sinks, sl)
    assert not host(dk[at]).any() and not host(dv[at]).any()
    near(dk[:n], ref["dk"], ref["e_dk"], "dk")
    near(dv[:n], ref["dv"], ref["e_dv"], "dv")
    assert not host(dk[n:]).any() and not host(dv[n:]).any()


@pytest.mark.parametrize("S,W,at", [(40, 0, 3), (300, 0, 70), (300, 100, 130), (900, 500, 310),
                                    (900, 0, 5)])
def test_d_q_of_a_row_that_sees_an_infinite_key(cuda, S, W, at):
    """d_q = scale sum dS k: 0 times an infinity is NaN in that element, whether or not
    the rows of the tile all see the key, and nothing elsewhere."""
    H, K = 4, 2
    q, k, v, g = weightless(S, H, K, at, 4)
    ref = without_key(q, k, v, g, H, K, W, 0, at)
    t = [dev(x) for x in (q, k, v, g)]
    out, lse = ops.window_attention(*t[:3], 1, S, H, K, W, want_lse=True)
    dq = ops.window_attention_backward(t[3], *t[:3], out, lse, 1, S, H, K, W)[0]
    sees = (np.arange(S) >= at) & ((W == 0) | (np.arange(S) < at + W))
    h = host(dq)
    nan = np.zeros(h.shape, bool)
    nan[sees, ::HD] = True
    assert np.array_equal(np.isnan(h), nan)
    dq[torch.from_numpy(nan).cuda()] = 0
    ref["dq"][nan] = 0
    near(dq, ref["dq"], ref["e_dq"], "dq")


# ------------------------------------------------------------- dealt by die --
# (batch, seq_len, heads, kv heads, window, sinks, lens): every one deals its rows and
# its key blocks, and joins the blocks that the sinks cut (tests/test_attention_limits.py
# checks that).
DEALT = [(1, 8200, 8, 2, 150, 4, [8200]), (1, 8195, 6, 3, 70, 130, [8190]),
         (2, 8193, 3, 3, 100, 9, [8193, 1200])]


@pytest.mark.parametrize("B,S,H,K,W,sinks,lens", DEALT)
def test_sinks_of_long_sequences_dealt_by_die(cuda, B, S, H, K, W, sinks, lens):
    say("case:", B, S, H, K, W, sinks, lens)
    x = inputs(B, S, H, K, S + W)
    ref = by_pieces(*x, B, S, H, K, W, sinks, lens)
    sl = i32(lens)
    q, k, v, g = (dev(a) for a in x)
    out, lse = ops.window_attention(q, k, v, B, S, H, K, W, sinks, sl, want_lse=True)
    near(out, ref["out"], ref["e_out"], "out")
    d = ops.window_attention_backward(g, q, k, v, out, lse, B, S, H, K, W, sinks, sl)
    for t, name in zip(d, ("dq", "dk", "dv")):
        near(t, ref[name], ref["e_" + name], name)
