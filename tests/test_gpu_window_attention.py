"""Window attention with sinks and its gradients against float64 references of
the same bf16 inputs, through the C ABI.  The bounds of every element are
attention_ref's: the roundings to bf16 that the kernels make, counted."""
import numpy as np
import pytest
import torch

import attention_ref as R
from prichs_amd import _lib as L
from prichs_amd import ops, synth

pytestmark = pytest.mark.gpu
HD = 128


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to("cuda").bfloat16()


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def say(*a):
    print(*a, flush=True)


def near(got, ref, name):
    err, bound = np.abs(host(got) - ref[name]), ref["e_" + name]
    worst = np.argmax(err - bound)
    assert (err <= bound).all(), (name, err.flat[worst], bound.flat[worst])


def inputs(B, S, H, K, seed, q_scale=1.0):
    rng = np.random.default_rng(seed)
    x = [synth.round_bf16(rng.standard_normal((B * S, n * HD))) for n in (H, K, K, H)]
    return synth.round_bf16(x[0] * q_scale), x[1], x[2], x[3]


# (batch, seq_len, heads, kv heads, window, sinks, lens): one token; a window of
# one; sizes around a tile; sinks past a tile, past the window and past the
# sequence; groups of 1 to 8 heads; empty, short, full and overlong sequences.
CASES = [
    (1, 1, 1, 1, 0, 0, None), (1, 1, 2, 1, 1, 3, None), (2, 63, 2, 1, 1, 0, None),
    (1, 64, 2, 2, 64, 0, None), (1, 65, 4, 1, 64, 1, None), (2, 200, 4, 2, 17, 3, None),
    (1, 333, 12, 3, 64, 4, None), (1, 300, 3, 3, 100, 70, None), (1, 257, 8, 1, 128, 200, None),
    (1, 129, 6, 2, 1000, 4, None), (1, 700, 4, 1, 0, 0, None), (1, 520, 5, 1, 450, 0, None),
    (1, 450, 2, 1, 65, 500, None), (1, 900, 4, 1, 130, 5, None),
    (3, 130, 6, 2, 50, 1, [0, 130, 77]), (4, 90, 2, 1, 0, 0, [1, 64, 500, -3]),
    (2, 400, 4, 1, 100, 4, [399, 130]),
    # More workgroups than the short-row variants take, for 4, 2 and 1 heads that
    # share a workgroup's tiles.
    (3, 330, 48, 12, 100, 4, [330, 200, 17]), (6, 330, 24, 12, 90, 0, None),
    (6, 330, 24, 24, 0, 0, [330, 1, 0, 129, 300, 64]),
]


@pytest.mark.parametrize("B,S,H,K,W,sinks,lens", CASES)
def test_forward_and_backward(cuda, B, S, H, K, W, sinks, lens):
    say("case:", B, S, H, K, W, sinks, lens)
    q, k, v, g = inputs(B, S, H, K, B + S + W)
    ref = R.batch_attention(q, k, v, B, S, H, K, W, sinks, lens, d_out=g)
    sl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    # q, k, v as column slices of one buffer, gradients into slices of another;
    # rows past the batch stay as they were.
    n = (H + 2 * K) * HD
    qkv = torch.full((B * S + 3, n + 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    cols = [slice(32, 32 + H * HD), slice(32 + H * HD, 32 + (H + K) * HD),
            slice(32 + (H + K) * HD, 32 + n)]
    for c, x in zip(cols, (q, k, v)):
        qkv[:B * S, c] = dev(x)
    out = torch.full((B * S + 2, H * HD), 7.0, dtype=torch.bfloat16, device="cuda")
    got, lse = ops.window_attention(*(qkv[:, c] for c in cols), B, S, H, K, W, sinks, sl, out=out,
                                    want_lse=True)
    assert got is out
    near(out[:B * S], ref, "out")
    assert (out[B * S:] == 7.0).all()
    hl = host(lse)
    assert np.array_equal(np.isinf(hl), np.isinf(ref["lse"]))
    fin = np.isfinite(hl)
    assert (np.abs(hl[fin] - ref["lse"][fin]) <= ref["e_lse"][fin]).all()
    dqkv = torch.full((B * S + 1, n + 64), 7.0, dtype=torch.bfloat16, device="cuda")
    args = (dev(g), *(qkv[:, c] for c in cols), out, lse, B, S, H, K, W, sinks, sl)
    ops.window_attention_backward(*args, d_q=dqkv[:, cols[0]], d_k=dqkv[:, cols[1]],
                                  d_v=dqkv[:, cols[2]])
    for c, name in zip(cols, ("dq", "dk", "dv")):
        near(dqkv[:B * S, c], ref, name)
    h = host(dqkv)
    assert (h[:, :32] == 7).all() and (h[:, 32 + n:] == 7).all() and (h[B * S:] == 7).all()
    # The same bits again, into tensors of its own.
    again = ops.window_attention_backward(*args)
    for t, c in zip(again, cols):
        assert torch.equal(t, dqkv[:B * S, c].contiguous())


@pytest.mark.parametrize("q_scale", [0.0, 30.0, -200.0])
def test_steep_and_flat_scores(cuda, q_scale):
    B, S, H, K, W, sinks = 1, 210, 4, 2, 90, 5
    q, k, v, g = inputs(B, S, H, K, 3, q_scale)
    ref = R.batch_attention(q, k, v, B, S, H, K, W, sinks, d_out=g)
    # A score's f32 error is 128 roundings of 2^-24 of its terms' magnitudes; its
    # exponential is off by that much more of itself.
    mag = np.abs(q_scale) * 16 * HD ** 0.5 * 128 * 2.0 ** -24
    out, lse = ops.window_attention(dev(q), dev(k), dev(v), B, S, H, K, W, sinks, want_lse=True)
    for key in [n for n in ref if n.startswith("e_")]:
        ref[key] = ref[key] * (1 + 2 * mag / R.U)
    near(out, ref, "out")
    d = ops.window_attention_backward(dev(g), dev(q), dev(k), dev(v), out, lse, B, S, H, K, W,
                                      sinks)
    for t, name in zip(d, ("dq", "dk", "dv")):
        near(t, ref, name)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_does_not_reach_it(cuda, bad):
    # No seq_lens: the keys past row n are garbage, and so are the first keys,
    # which the rows from 40 + W on do not see (no sinks).
    B, S, H, K, W, n = 1, 320, 4, 2, 100, 250
    q, k, v, _ = inputs(B, S, H, K, 5)
    clean = ops.window_attention(dev(q), dev(k), dev(v), B, S, H, K, W)[0]
    k2, v2 = k.copy(), v.copy()
    for x in (k2, v2):
        x[n:] = bad
        x[:40:3, ::5] = bad
    got = ops.window_attention(dev(q), dev(k2), dev(v2), B, S, H, K, W)[0]
    rows = slice(39 + W, n)
    assert torch.equal(got[rows], clean[rows])
    # Rows that do see them have no finite output where v is not finite.
    assert not torch.isfinite(got[n:]).any()
    assert not torch.isfinite(got[:40, ::5][0:1]).any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gradients_of_what_is_not_seen(cuda, bad):
    # Rows 200.. of q and d_out are garbage: keys that only earlier rows see keep
    # their gradients; the keys below 30 are garbage: so do later rows.
    B, S, H, K, W = 1, 300, 4, 2, 60
    q, k, v, g = inputs(B, S, H, K, 6)
    t = [dev(x) for x in (q, k, v, g)]
    out, lse = ops.window_attention(*t[:3], B, S, H, K, W, want_lse=True)
    clean = ops.window_attention_backward(t[3], *t[:3], out, lse, B, S, H, K, W)
    q2, g2, k2, v2 = q.copy(), g.copy(), k.copy(), v.copy()
    q2[200:, ::3] = bad
    g2[200:] = bad
    k2[:30, ::7] = bad
    v2[:30] = bad
    t = [dev(x) for x in (q2, k2, v2, g2)]
    out, lse = ops.window_attention(*t[:3], B, S, H, K, W, want_lse=True)
    dq, dk, dv = ops.window_attention_backward(t[3], *t[:3], out, lse, B, S, H, K, W)
    assert torch.equal(dq[29 + W:200], clean[0][29 + W:200])
    # Keys that neither garbage row nor a row that sees a garbage key sees.
    keys = slice(29 + W, 201 - W)
    assert torch.equal(dk[keys], clean[1][keys]) and torch.equal(dv[keys], clean[2][keys])


def test_padding_of_a_batch_is_not_used(cuda):
    B, S, H, K, W, lens = 3, 150, 4, 1, 70, [150, 3, 65]
    q, k, v, g = inputs(B, S, H, K, 8)
    ref = R.batch_attention(q, k, v, B, S, H, K, W, 2, lens, d_out=g)
    pad = np.concatenate([np.arange(S) >= n for n in lens])
    t = [dev(x) for x in (q, k, v, g)]
    for x in t:
        x[torch.from_numpy(pad).cuda()] = float("nan")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = ops.window_attention(*t[:3], B, S, H, K, W, 2, sl, want_lse=True)
    near(out, ref, "out")
    for x, name in zip(ops.window_attention_backward(t[3], *t[:3], out, lse, B, S, H, K, W, 2, sl),
                       ("dq", "dk", "dv")):
        near(x, ref, name)
        assert not host(x)[pad].any()


def test_agrees_with_the_whole_causal_attention(cuda):
    B, S, H, K = 2, 300, 12, 3
    q, k, v, _ = inputs(B, S, H, K, 9)
    ref = R.batch_attention(q, k, v, B, S, H, K, 0, 0)
    t = [dev(x) for x in (q, k, v)]
    near(ops.attention(*t, B, S, H, K), ref, "out")
    near(ops.window_attention(*t, B, S, H, K, 0)[0], ref, "out")


def test_other_stream_and_graph(cuda):
    """A step captured into a graph replays on new inputs, next to eager calls, and
    gives the eager bits; so does a call on a stream of its own."""
    B, S, H, K, W, sinks = 2, 190, 4, 2, 80, 3
    sets = [[dev(x) for x in inputs(B, S, H, K, s)] for s in (11, 12, 13)]

    def step(t, stream=None):
        out, lse = ops.window_attention(*t[:3], B, S, H, K, W, sinks, want_lse=True, stream=stream)
        return (out, *ops.window_attention_backward(t[3], *t[:3], out, lse, B, S, H, K, W, sinks,
                                                    stream=stream))

    want = [[x.clone() for x in step(t)] for t in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = step(sets[1], side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    buf = [x.clone() for x in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = step(buf)
    for i in (1, 2, 0, 2):
        for b, x in zip(buf, sets[i]):
            b.copy_(x)
        eager = step(sets[(i + 1) % 3])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(cap, want[i])), i
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3])), i


def test_wrapper_refusals(cuda):
    q, k, v, g = (dev(x) for x in inputs(1, 8, 2, 1, 1))
    ok = (1, 8, 2, 1, 4)
    with pytest.raises(ValueError):
        ops.window_attention(q, k, v, 2, 8, 2, 1, 4)  # fewer rows than batch * seq_len
    with pytest.raises(ValueError):
        ops.window_attention(q.t().contiguous().t(), k, v, *ok)
    with pytest.raises(TypeError):
        ops.window_attention(q.float(), k, v, *ok)
    with pytest.raises(ValueError):
        ops.window_attention(q, k, v, 1, 8, 2, 1, -1)
    with pytest.raises(ValueError):
        ops.window_attention(q.cpu(), k, v, *ok)
    with pytest.raises(ValueError):
        ops.window_attention(q, k, v, *ok, seq_lens=torch.tensor([8], device="cuda"))
    with pytest.raises(L.PrichsError):
        ops.window_attention(q, k, v, 1, 8, 2, 1, 4, out=torch.empty(
            (8, 256 + 4), dtype=torch.bfloat16, device="cuda")[:, :256])
    out, lse = ops.window_attention(q, k, v, *ok, want_lse=True)
    with pytest.raises(ValueError):
        ops.window_attention_backward(g, q, k, v, out, None, *ok)
    with pytest.raises(ValueError):
        ops.window_attention_backward(g, q, k, v, out, lse[:, :1], *ok)
    out, lse = ops.window_attention(q[:0], k[:0], v[:0], 0, 8, 2, 1, 4, want_lse=True)
    assert out.shape == (0, 256) and lse.shape == (0, 2, 8)


@pytest.mark.parametrize("S,H,K", [(10, 4, 1), (777, 8, 2), (33, 2, 1), (16, 3, 3)])
def test_what_the_workspace_held_does_not_matter(cuda, S, H, K):
    """NaN everywhere in it, sequences that end in the first half of a 32-row tile
    among the cases."""
    W, sinks = 40, 3
    x = inputs(1, S, H, K, 7)
    ref = R.batch_attention(*x[:3], 1, S, H, K, W, sinks, d_out=x[3])
    q, k, v, d_o = (dev(a) for a in x)
    out, lse = ops.window_attention(q, k, v, 1, S, H, K, W, sinks, want_lse=True)
    lib = L.load()
    need = lib.prichs_window_attention_backward_workspace(1, S, H, K, W, sinks)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    grads = [torch.empty_like(t) for t in (q, k, v)]
    args = [a for t in (d_o, q, k, v, out) for a in (t.data_ptr(), t.stride(0))]
    to = [a for t in grads for a in (t.data_ptr(), t.stride(0))]
    L.check(lib.prichs_window_attention_backward(
        *args, lse.data_ptr(), None, *to, 1, S, H, K, HD, W, sinks, L.DTYPE_BF16, ws.data_ptr(),
        need, torch.cuda.current_stream().cuda_stream))
    for t, name in zip(grads, ("dq", "dk", "dv")):
        near(t, ref, name)


def test_offsets_past_32_bits(cuda):
    """All operands and gradients as columns of one buffer of 4.7 GB, with the largest
    leading dimension there is."""
    S, H, K, W, sinks, ld = 140, 2, 1, 60, 3, (1 << 24) - 8
    x = inputs(1, S, H, K, 9)
    ref = R.batch_attention(*x[:3], 1, S, H, K, W, sinks, d_out=x[3])
    buf = torch.empty((S, ld), dtype=torch.bfloat16, device="cuda")
    heads = [H, K, K, H, H, H, K, K]
    q, k, v, d_o, out, dq, dk, dv = (buf[:, (e - n) * HD:e * HD]
                                     for n, e in zip(heads, np.cumsum(heads)))
    for t, a in zip((q, k, v, d_o), x):
        t.copy_(dev(a))
    _, lse = ops.window_attention(q, k, v, 1, S, H, K, W, sinks, out=out, want_lse=True)
    ops.window_attention_backward(d_o, q, k, v, out, lse, 1, S, H, K, W, sinks, d_q=dq, d_k=dk,
                                  d_v=dv)
    for t, name in ((out, "out"), (dq, "dq"), (dk, "dk"), (dv, "dv")):
        near(t, ref, name)


def by_pieces(q, k, v, d_out, B, S, H, K, W, lens):
    """R.batch_attention without sinks, from pieces of rows and the keys they see."""
    r = {e + n: np.zeros((B * S, (H if n in ("out", "dq") else K) * HD))
         for n in ("out", "dq", "dk", "dv") for e in ("", "e_")}
    for b, n in enumerate(lens):
        for a in range(0, n, 1000):
            lo, mid, end = max(0, a - W + 1), min(a + 1000, n), min(a + 1000 + W, n)
            rows, keys, own = (slice(b * S + x, b * S + y) for x, y in ((a, end), (lo, end), (a, mid)))
            for h in range(H):
                c = slice(h * HD, (h + 1) * HD)
                ck = slice(h // (H // K) * HD, (h // (H // K) + 1) * HD)
                one = R.attention(q[rows, c], k[keys, ck], v[keys, ck], W, 0, first=a - lo,
                                  d_out=d_out[rows, c])
                for e in ("", "e_"):
                    for name in ("out", "dq"):
                        r[e + name][own, c] = one[e + name][:mid - a]
                    for name in ("dk", "dv"):
                        r[e + name][own, ck] += one[e + name][a - lo:mid - lo]
    return r


LONG = [(1, 8200, 8, 2, 150, [8200]), (1, 8195, 6, 3, 70, [8190]),
        (2, 8193, 3, 3, 100, [8193, 1200])]


@pytest.mark.parametrize("B,S,H,K,W,lens", LONG)
def test_long_sequences_dealt_by_die(cuda, B, S, H, K, W, lens):
    """Launches whose workgroups are dealt to the dies in runs, the last one ragged."""
    say("case:", B, S, H, K, W, lens)
    x = inputs(B, S, H, K, S + W)
    ref = by_pieces(*x, B, S, H, K, W, lens)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q, k, v, g = (dev(a) for a in x)
    out, lse = ops.window_attention(q, k, v, B, S, H, K, W, 0, sl, want_lse=True)
    near(out, ref, "out")
    d = ops.window_attention_backward(g, q, k, v, out, lse, B, S, H, K, W, 0, sl)
    for t, name in zip(d, ("dq", "dk", "dv")):
        near(t, ref, name)
