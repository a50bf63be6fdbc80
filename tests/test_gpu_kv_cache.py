"""The 4-bit KV cache (written, read back) and the attention over it, through the
C ABI: cached values exactly those of attention_ref.cached_values, attention
within the bounds of attention_ref for those values."""
import numpy as np
import pytest
import torch

import attention_ref as R
from prichs_amd import _lib as L
from prichs_amd import ops, synth

pytestmark = pytest.mark.gpu
HD, PAGE = 128, L.KV_PAGE


def dev(a, dtype=torch.bfloat16):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to("cuda").to(dtype)


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def say(*a):
    print(*a, flush=True)


def table_of(batch, pages, seed=0, spare=0):
    """Distinct pages in mixed order for every sequence, and how many there are."""
    rng = np.random.default_rng(seed)
    return i32(rng.permutation(batch * pages + spare)[:batch * pages].reshape(batch, pages)), \
        batch * pages + spare


def filled(n_pages, kv):
    """Pages of bytes that stand for NaN everywhere: no call may use what was not
    written."""
    cache = ops.kv_cache_pages(n_pages, kv)
    cache.fill_(255)
    return cache


def same(got, want):
    g = host(got)
    assert np.array_equal(g, want, equal_nan=True), np.argwhere(~((g == want) | (
        np.isnan(g) & np.isnan(want))))[:5]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,n,kv,start", [
    (1, 1, 1, [0]), (3, 1, 3, [63, 64, 5]), (2, 200, 2, [0, 100]), (1, 65, 5, [63]),
    (1, 130, 3, [1])])
def test_write_then_read(cuda, dtype, batch, n, kv, start):
    say("case:", dtype, batch, n, kv, start)
    rng = np.random.default_rng(n + kv)
    table, n_pages = table_of(batch, 5, n, spare=2)
    cache = filled(n_pages, kv)
    before = cache.clone()
    x = [rng.standard_normal((batch * n, kv * HD)) * 10.0 ** rng.integers(-4, 4, (batch * n, 1))
         for _ in range(2)]
    x = [synth.round_bf16(a) if dtype == torch.bfloat16 else a.astype(np.float32) for a in x]
    # Row views of wider buffers.
    wide = [torch.zeros((batch * n + 1, kv * HD + 16), dtype=dtype, device="cuda")
            for _ in range(2)]
    for w, a in zip(wide, x):
        w[:batch * n, 8:8 + kv * HD] = dev(a, dtype)
    views = [w[:, 8:8 + kv * HD] for w in wide]
    ops.kv_cache_write(cache, table, i32(start), *views, batch, n, kv)
    want = [R.cached_values(a.reshape(-1, HD)).reshape(a.shape) for a in x]
    got = ops.kv_cache_read(cache, table, i32(start), batch, n, kv, out_dtype=dtype)
    for g, w in zip(got, want):
        same(g, w)
    # In the other type too (both hold the values exactly), into views.
    other = torch.float32 if dtype == torch.bfloat16 else torch.bfloat16
    out = [torch.full((batch * n + 1, kv * HD + 8), 7.0, dtype=other, device="cuda")
           for _ in range(2)]
    ops.kv_cache_read(cache, table, i32(start), batch, n, kv, k=out[0][:, :kv * HD],
                      v=out[1][:, :kv * HD])
    for o, w in zip(out, want):
        same(o[:batch * n, :kv * HD], w)
        assert (o[batch * n:] == 7).all() and (o[:, kv * HD:] == 7).all()
    # Only what belongs to these positions changed: 136 bytes each at most.
    changed = (cache != before).sum().item()
    assert 0 < changed <= batch * n * kv * 136
    untouched = [p for p in range(n_pages) if p not in set(table.flatten().tolist())]
    assert torch.equal(cache[untouched], before[untouched])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_at_the_borders(cuda, dtype):
    """Zeros, ties, a maximum at and past seven scales, subnormals, the largest
    values, infinities and NaN, each in a group of its own."""
    rows = []
    for top in (0.0, 7.0, 7.03125, 6.0, 4.0, 3.5, 3.515625, 1e-38, 2.0 ** -130, 2.0 ** -126,
                3.0e38, 2.0 ** 127, -2.0 ** 100):
        r = np.zeros(32)
        r[0] = top
        r[1:8] = np.sign(top) * np.abs(top) / 7 * np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
        r[8:15] = -r[1:8]
        r[15] = -0.0
        rows.append(r)
    for bad in (np.inf, -np.inf, np.nan):
        r = np.linspace(-3, 3, 32)
        r[17] = bad
        rows.append(r)
    x = np.array(rows, dtype=np.float32).reshape(-1, HD)
    if dtype == torch.bfloat16:
        x = dev(x).float().cpu().numpy()
    n = len(x)
    table, n_pages = table_of(1, 2)
    cache = filled(n_pages, 1)
    start = i32([60])
    ops.kv_cache_write(cache, table, start, dev(x, dtype), dev(x[::-1], dtype), 1, n, 1)
    k, v = ops.kv_cache_read(cache, table, start, 1, n, 1, out_dtype=torch.float32)
    want = R.cached_values(x)
    same(k, want)
    same(v, want[::-1])


def test_appending_equals_writing_at_once(cuda):
    rng = np.random.default_rng(4)
    kv, n = 2, 150
    k, v = (dev(rng.standard_normal((n, kv * HD))) for _ in range(2))
    table, n_pages = table_of(1, 3)
    whole, steps = filled(n_pages, kv), filled(n_pages, kv)
    ops.kv_cache_write(whole, table, i32([0]), k, v, 1, n, kv)
    at = 0
    for m in (1, 1, 1, 60, 1, 2, 64, 20):
        ops.kv_cache_write(steps, table, i32([at]), k[at:at + m], v[at:at + m], 1, m, kv)
        at += m
    assert at == n and torch.equal(whole, steps)


def test_counts_and_positions_without_a_page(cuda):
    rng = np.random.default_rng(5)
    batch, n, kv = 4, 70, 2
    x = [synth.round_bf16(rng.standard_normal((batch * n, kv * HD))) for _ in range(2)]
    table, n_pages = table_of(batch, 2)
    table[1, 1] = n_pages       # one past the last page
    table[2, 0] = -1
    start, counts = i32([0, 0, 0, 100]), i32([10, 70, 70, 70])
    cache = filled(n_pages, kv)
    ops.kv_cache_write(cache, table, start, dev(x[0]), dev(x[1]), batch, n, kv, counts=counts)
    out = [torch.full((batch * n, kv * HD), 7.0, dtype=torch.bfloat16, device="cuda")
           for _ in range(2)]
    ops.kv_cache_read(cache, table, start, batch, n, kv, counts=counts, k=out[0], v=out[1])
    for o, a in zip(out, x):
        w = R.cached_values(a.reshape(-1, HD)).reshape(batch, n, kv * HD)
        w[0, 10:] = 7           # past its count: as it was
        w[1, 64:] = 0           # page past the last
        w[2, :64] = 0           # page -1
        w[3, 28:] = 0           # past the table
        same(o, w.reshape(batch * n, -1))
    # Allocated by the call: zeros past a count.
    k, _ = ops.kv_cache_read(cache, table, start, batch, n, kv, counts=counts)
    assert not host(k)[10:n].any()
    # Negative starts: rows before position 0 are dropped.
    cache2 = filled(n_pages, kv)
    t2, _ = table_of(batch, 2)
    ops.kv_cache_write(cache2, t2, i32([-3] * batch), dev(x[0]), dev(x[1]), batch, n, kv)
    k, _ = ops.kv_cache_read(cache2, t2, i32([0] * batch), batch, n - 3, kv)
    w = R.cached_values(x[0].reshape(-1, HD)).reshape(batch, n, -1)[:, 3:]
    same(k, w.reshape(batch * (n - 3), -1))


# ---------------------------------------------------------------- attention --
# (batch, n_q, lens, heads, kv, window, sinks): one token over one, over a page
# and one more, over many; sequences of length zero, or shorter than n_q; groups
# of 1 to 8; drafted tokens; chunks that cross row tiles; windows that end inside
# a page; sinks past a page.
ATTEND = [
    (1, 1, [1], 1, 1, 0, 0), (1, 1, [64], 4, 1, 0, 0), (1, 1, [65], 12, 3, 0, 0),
    (4, 1, [0, 1, 700, 129], 8, 2, 0, 0), (3, 1, [500, 64, 333], 12, 3, 100, 4),
    (1, 1, [3000], 4, 2, 0, 0), (2, 1, [2500, 1], 4, 4, 1, 0), (1, 1, [900], 6, 1, 64, 150),
    (2, 5, [300, 3], 12, 3, 0, 0), (2, 3, [130, 66], 8, 1, 20, 2), (1, 4, [70], 5, 1, 0, 0),
    (3, 17, [400, 17, 20], 4, 1, 33, 1), (1, 40, [40], 8, 2, 0, 0), (1, 130, [450], 12, 3, 96, 4),
    (2, 70, [500, 100], 3, 3, 0, 0), (1, 1, [5000], 12, 3, 4096, 4), (1, 33, [1000], 16, 2, 300, 70),
    # A few splits joined; more tiles than workgroups that fit at once.
    (1, 1, [1500], 8, 2, 0, 0), (2, 40, [1300, 60], 12, 3, 0, 0), (9, 40, [300] * 9, 12, 3, 0, 0),
    (2, 700, [750, 700], 12, 3, 200, 3),
]


def attend_case(batch, n_q, lens, heads, kv, seed, max_pages=None, q_scale=1.0):
    rng = np.random.default_rng(seed)
    top = max(max(lens), 1)
    pages = max_pages or -(-top // PAGE)
    table, n_pages = table_of(batch, pages, seed, spare=1)
    cache = filled(n_pages, kv)
    k, v = (synth.round_bf16(rng.standard_normal((batch * top, kv * HD))) for _ in range(2))
    q = synth.round_bf16(rng.standard_normal((batch * n_q, heads * HD)) * q_scale)
    ops.kv_cache_write(cache, table, i32([0] * batch), dev(k), dev(v), batch, top, kv,
                       counts=i32(lens))
    kc, vc = (R.cached_values(x.reshape(-1, HD)).reshape(batch, top, kv, HD) for x in (k, v))
    return table, cache, q, kc, vc


def attend_ref(q, kc, vc, lens, n_q, heads, kv, window, sinks, keep=None):
    batch = len(lens)
    r = {n: np.zeros((batch * n_q, heads * HD)) for n in ("out", "e_out")}
    r["lse"] = np.full((batch, heads, n_q), -np.inf)
    for b, n in enumerate(lens):
        rows = slice(b * n_q, (b + 1) * n_q)
        for h in range(heads):
            c, j = slice(h * HD, (h + 1) * HD), h // (heads // kv)
            if n == 0:
                continue
            one = R.attention(q[rows, c], kc[b, :n, j], vc[b, :n, j], window, sinks, first=n - n_q,
                              keep=None if keep is None else keep[b][:n])
            r["out"][rows, c], r["e_out"][rows, c] = one["out"], one["e_out"]
            r["lse"][b, h] = one["lse"]
    return r


def check(out, lse, ref):
    err = np.abs(host(out) - ref["out"])
    worst = np.argmax(err - ref["e_out"])
    assert (err <= ref["e_out"]).all(), (err.flat[worst], ref["e_out"].flat[worst], worst)
    if lse is not None:
        h = host(lse)
        assert np.array_equal(np.isneginf(h), np.isneginf(ref["lse"]))
        fin = np.isfinite(h)
        assert (np.abs(h[fin] - ref["lse"][fin]) <= 1.25 * R.U).all()


@pytest.mark.parametrize("batch,n_q,lens,heads,kv,window,sinks", ATTEND)
def test_attention_over_the_cache(cuda, batch, n_q, lens, heads, kv, window, sinks):
    say("case:", batch, n_q, lens, heads, kv, window, sinks)
    table, cache, q, kc, vc = attend_case(batch, n_q, lens, heads, kv, n_q + sum(lens))
    ref = attend_ref(q, kc, vc, lens, n_q, heads, kv, window, sinks)
    wide = torch.full((batch * n_q + 1, heads * HD + 8), float("nan"), dtype=torch.bfloat16,
                      device="cuda")
    wide[:batch * n_q, :heads * HD] = dev(q)
    out = torch.full((batch * n_q + 1, heads * HD + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    _, lse = ops.kv_cache_attention(wide[:, :heads * HD], cache, table, i32(lens), batch, n_q, heads,
                                    kv, window, sinks, out=out[:, 8:8 + heads * HD], want_lse=True)
    check(out[:batch * n_q, 8:8 + heads * HD], lse, ref)
    h = host(out)
    assert (h[batch * n_q:] == 7).all() and (h[:, :8] == 7).all() and \
        (h[:, 8 + heads * HD:] == 7).all()
    again, _ = ops.kv_cache_attention(dev(q), cache, table, i32(lens), batch, n_q, heads, kv, window,
                                      sinks)
    assert torch.equal(again, out[:batch * n_q, 8:8 + heads * HD].contiguous())


@pytest.mark.parametrize("n_q", [1, 6, 40])
def test_long_tables_lens_past_them_and_shared_pages(cuda, n_q):
    """A table far longer than the sequences; a length past the table counts as the
    table's; two sequences on the same pages."""
    lens = [100, 200]
    table, cache, q, kc, vc = attend_case(2, n_q, lens, 4, 2, 21, max_pages=300)
    ref = attend_ref(q, kc, vc, lens, n_q, 4, 2, 0, 0)
    check(*ops.kv_cache_attention(dev(q), cache, table, i32(lens), 2, n_q, 4, 2, want_lse=True), ref)
    short = table[:, :2].contiguous()
    vis = [100, 128]
    ref = attend_ref(q, kc, vc, vis, n_q, 4, 2, 0, 0)
    check(*ops.kv_cache_attention(dev(q), cache, short, i32([100, 1 << 30]), 2, n_q, 4, 2,
                                  want_lse=True), ref)
    both = table[1:].repeat(2, 1).contiguous()
    ref = attend_ref(q, np.stack([kc[1], kc[1]]), np.stack([vc[1], vc[1]]), [200, 150], n_q, 4, 2,
                     70, 3)
    check(*ops.kv_cache_attention(dev(q), cache, both, i32([200, 150]), 2, n_q, 4, 2, 70, 3,
                                  want_lse=True), ref)


@pytest.mark.parametrize("n_q", [1, 5, 30])
def test_pages_that_do_not_exist(cuda, n_q):
    lens = [300, 290, 60]
    table, cache, q, kc, vc = attend_case(3, n_q, lens, 4, 1, 22)
    table[0, 1] = cache.shape[0]
    table[1, 0], table[1, 4] = -1, 1 << 30
    table[2, 0] = -(1 << 31)
    keep = [np.ones(300, bool) for _ in range(3)]
    keep[0][64:128] = False
    keep[1][:64] = keep[1][256:] = False
    keep[2][:] = False
    for window, sinks in ((0, 0), (40, 4)):
        ref = attend_ref(q, kc, vc, lens, n_q, 4, 1, window, sinks, keep)
        check(*ops.kv_cache_attention(dev(q), cache, table, i32(lens), 3, n_q, 4, 1, window, sinks,
                                      want_lse=True), ref)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_query_does_not_see_does_not_reach_it(cuda, bad):
    """Positions that hold no finite value: queries that do not see them are as
    without them, queries that see them have no finite output there."""
    rng = np.random.default_rng(23)
    n, n_q, W = 260, 70, 40
    k, v = (synth.round_bf16(rng.standard_normal((n, HD))) for _ in range(2))
    q = synth.round_bf16(rng.standard_normal((n_q, 2 * HD)))
    table, n_pages = table_of(1, 5)
    clean, dirty = filled(n_pages, 1), filled(n_pages, 1)
    ops.kv_cache_write(clean, table, i32([0]), dev(k), dev(v), 1, n, 1)
    k2, v2 = k.copy(), v.copy()
    v2[200, 40] = bad            # seen by the queries at 200 .. 239
    k2[170, 3] = bad             # at 170 .. 209
    ops.kv_cache_write(dirty, table, i32([0]), dev(k2), dev(v2), 1, n, 1)
    a, b = (ops.kv_cache_attention(dev(q), c, table, i32([n]), 1, n_q, 2, 1, W)[0]
            for c in (clean, dirty))
    at = np.arange(n - n_q, n)
    unseen = torch.from_numpy((at < 170) | (at >= 240)).cuda()
    assert torch.equal(a[unseen], b[unseen])
    hb = host(b).reshape(n_q, 2, 4, 32)
    assert not np.isfinite(hb[(at >= 200) & (at < 240)][:, :, 1]).any()
    late = (at >= 210) & (at < 240)  # past the key: the other groups are finite
    assert np.isfinite(hb[late][:, :, [0, 2, 3]]).all()
    assert not np.isfinite(hb[(at >= 170) & (at < 210)]).any()


@pytest.mark.parametrize("q_scale", [0.0, 40.0])
def test_flat_and_steep_scores(cuda, q_scale):
    lens = [700, 64]
    table, cache, q, kc, vc = attend_case(2, 2, lens, 4, 2, 24, q_scale=q_scale)
    ref = attend_ref(q, kc, vc, lens, 2, 4, 2, 0, 0)
    # A score is off by 128 roundings of 2^-24 of its terms, and p by that.
    ref["e_out"] *= 1 + 2 * (q_scale * 16 * HD ** 0.5 * 128 * 2.0 ** -24) / R.U
    check(ops.kv_cache_attention(dev(q), cache, table, i32(lens), 2, 2, 4, 2)[0], None, ref)


@pytest.mark.parametrize("length", [50, 500, 3000])
def test_queries_without_finite_scores(cuda, length):
    """Scores of -inf have no weight; a row of nothing else, and one with a NaN or a
    +inf, has no softmax.  The keys' first dim is 1 from position 40 on and 0 before
    (0 times an infinity is NaN)."""
    k = np.zeros((length, HD), np.float32)
    v = synth.round_bf16(np.random.default_rng(1).standard_normal((length, HD)))
    k[40:, 0] = 1
    table, n_pages = table_of(1, -(-length // PAGE))
    cache = filled(n_pages, 1)
    ops.kv_cache_write(cache, table, i32([0]), dev(k), dev(v), 1, length, 1)
    q = np.zeros((1, 4 * HD), np.float32)
    q[0, 0], q[0, HD], q[0, 2 * HD] = -np.inf, np.inf, np.nan
    for window in (0, length - 45):  # with and without keys whose score is NaN
        out, lse = ops.kv_cache_attention(dev(q), cache, table, i32([length]), 1, 1, 4, 1, window,
                                          want_lse=True)
        h, hl = host(out).reshape(4, HD), host(lse).reshape(4)
        assert np.isnan(h[:3]).all() and np.isnan(hl[:3]).all(), window
        assert np.isfinite(h[3]).all() and np.isfinite(hl[3])


def test_prefill_then_decode_steps_in_a_graph(cuda):
    """As a program uses them together: a prompt's window attention, its keys and
    values into the cache, then decode steps -- one captured graph whose table,
    lengths and token change between replays -- against float64 over the values
    that the cache holds."""
    rng = np.random.default_rng(25)
    H, K, W, sinks, S, steps = 4, 2, 50, 3, 100, 30
    lens = [S, 61]
    batch, n = 2, S + steps
    k, v = (synth.round_bf16(rng.standard_normal((batch, n, K * HD))) for _ in range(2))
    q = synth.round_bf16(rng.standard_normal((batch, n, H * HD)))
    flat = lambda x: dev(x[:, :S].reshape(batch * S, -1))  # noqa: E731
    out, _ = ops.window_attention(flat(q), flat(k), flat(v), batch, S, H, K, W, sinks, i32(lens))
    ref = R.batch_attention(*(x[:, :S].reshape(batch * S, -1) for x in (q, k, v)), batch, S, H, K, W,
                            sinks, lens)
    assert (np.abs(host(out) - ref["out"]) <= ref["e_out"]).all()
    table, n_pages = table_of(batch, 3)
    cache = filled(n_pages, K)
    ops.kv_cache_write(cache, table, i32([0, 0]), flat(k), flat(v), batch, S, K, counts=i32(lens))
    # The step's own buffers.
    pos, length = i32(lens), i32([0, 0])
    bq, bk, bv = (torch.zeros((batch, w * HD), dtype=torch.bfloat16, device="cuda")
                  for w in (H, K, K))

    def step():
        torch.add(pos, 1, out=length)
        ops.kv_cache_write(cache, table, pos, bk, bv, batch, 1, K)
        o, _ = ops.kv_cache_attention(bq, cache, table, length, batch, 1, H, K, W, sinks)
        pos.add_(1)
        return o

    saved = pos.clone(), cache.clone()
    step()
    torch.cuda.synchronize()
    pos.copy_(saved[0]), cache.copy_(saved[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    pos.copy_(saved[0]), cache.copy_(saved[1])
    kc, vc = (np.concatenate([R.cached_values(x[b].reshape(-1, HD)).reshape(1, n, K, HD)
                              for b in range(batch)]) for x in (k, v))
    for s in range(steps):
        at = [x + s for x in lens]
        for buf, x in ((bq, q), (bk, k), (bv, v)):
            buf.copy_(dev(np.stack([x[b, at[b]] for b in range(batch)])))
        graph.replay()
        got = o.clone()
        # An eager call between the replays, on other lengths.
        ops.kv_cache_attention(bq, cache, table, i32([5, 9]), batch, 1, H, K)
        ref = attend_ref(np.stack([q[b, at[b]] for b in range(batch)]), kc, vc,
                         [x + 1 for x in at], 1, H, K, W, sinks)
        check(got, None, ref)


def test_wrapper_refusals(cuda):
    kv, n = 2, 4
    table, n_pages = table_of(1, 1)
    cache = filled(n_pages, kv)
    k = torch.zeros((n, kv * HD), dtype=torch.bfloat16, device="cuda")
    st = i32([0])
    w = lambda *a, **b: ops.kv_cache_write(*a, **b)  # noqa: E731
    with pytest.raises(ValueError):
        w(cache, table, st, k, k, 1, n, 1)             # pages of other heads
    with pytest.raises(ValueError):
        w(cache.cpu(), table, st, k, k, 1, n, kv)
    with pytest.raises(ValueError):
        w(cache, table.long(), st, k, k, 1, n, kv)
    with pytest.raises(ValueError):
        w(cache, table, i32([0, 0]), k, k, 1, n, kv)
    with pytest.raises(ValueError):
        w(cache, table, st, k, k, 1, n + 1, kv)
    with pytest.raises(TypeError):
        w(cache, table, st, k.half(), k.half(), 1, n, kv)
    with pytest.raises(TypeError):
        w(cache, table, st, k, k.float(), 1, n, kv)
    q = torch.zeros((1, 4 * HD), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(L.PrichsError):
        ops.kv_cache_attention(q[:, :3 * HD], cache, table, st, 1, 1, 3, kv)
    with pytest.raises(ValueError):
        ops.kv_cache_attention(q, cache, table, st, 1, 1, 4, kv, window=-1)
    with pytest.raises(TypeError):
        ops.kv_cache_attention(q.float(), cache, table, st, 1, 1, 4, kv)
    # Nothing to do: no rows, and a table without pages.
    assert ops.kv_cache_attention(q[:0], cache, table[:0], st[:0], 0, 1, 4, kv)[0].shape[0] == 0
    none = torch.empty((1, 0), dtype=torch.int32, device="cuda")
    out, lse = ops.kv_cache_attention(q, cache, none, i32([5]), 1, 1, 4, kv, want_lse=True)
    assert not host(out).any() and np.isneginf(host(lse)).all()


def test_without_pages_or_positions(cuda):
    """A cache of no pages and a table of no columns: nothing is written, zeros are
    read, and a query sees no key."""
    for n_pages, cols in ((0, 0), (0, 2), (3, 0)):
        say("case:", n_pages, cols)
        cache = ops.kv_cache_pages(n_pages, 2)
        cache.fill_(255)
        table = torch.zeros((2, cols), dtype=torch.int32, device="cuda")
        x = torch.ones((2 * 3, 2 * HD), dtype=torch.bfloat16, device="cuda")
        ops.kv_cache_write(cache, table, i32([0, 1]), x, x, 2, 3, 2)
        assert (cache == 255).all()
        k, v = ops.kv_cache_read(cache, table, i32([0, 1]), 2, 3, 2)
        assert (k == 0).all() and (v == 0).all()
        out, lse = ops.kv_cache_attention(torch.ones((6, 4 * HD), dtype=torch.bfloat16, device="cuda"),
                                          cache, table, i32([3, 70]), 2, 3, 4, 2, want_lse=True)
        assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("batch,n_q,lens,heads,kv,window", [
    (1, 1, [3000], 4, 1, 0), (3, 5, [1300, 0, 3], 6, 2, 0), (2, 40, [1500, 1100], 4, 2, 100)])
def test_what_the_workspace_held_does_not_matter(cuda, batch, n_q, lens, heads, kv, window):
    table, cache, q, kc, vc = attend_case(batch, n_q, lens, heads, kv, 11)
    ref = attend_ref(q, kc, vc, lens, n_q, heads, kv, window, 2)
    lib, pages, x = L.load(), table.shape[1], dev(q)
    need = lib.prichs_kv_cache_attention_workspace(batch, n_q, heads, kv, pages)
    assert need > 0
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    out, lens_d = torch.empty_like(x), i32(lens)
    lse = torch.empty((batch, heads, n_q), dtype=torch.float32, device="cuda")
    L.check(lib.prichs_kv_cache_attention(
        x.data_ptr(), heads * HD, cache.data_ptr(), cache.shape[0], table.data_ptr(), pages,
        lens_d.data_ptr(), out.data_ptr(), heads * HD, lse.data_ptr(), batch, n_q, heads, kv, HD,
        window, 2, L.DTYPE_BF16, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    check(out, lse, ref)


def test_pages_past_32_bits(cuda):
    """A cache of 4.7 GB whose used pages lie at its start and its end."""
    kv, lens, n_q, heads = 2, [150, 200], 3, 4
    n_pages = 270_000
    assert n_pages * kv * L.KV_PAGE_BYTES > 1 << 32
    cache = ops.kv_cache_pages(n_pages, kv)
    table = torch.tensor([[n_pages - 1, 0, n_pages - 5, 7], [n_pages - 2, n_pages - 3, 1, 2]],
                         dtype=torch.int32, device="cuda")
    cache[table.flatten().long()] = 255
    rng = np.random.default_rng(4)
    k, v = (synth.round_bf16(rng.standard_normal((2 * 200, kv * HD))) for _ in range(2))
    q = synth.round_bf16(rng.standard_normal((2 * n_q, heads * HD)))
    ops.kv_cache_write(cache, table, i32([0, 0]), dev(k), dev(v), 2, 200, kv, counts=i32(lens))
    kc, vc = (R.cached_values(x.reshape(-1, HD)).reshape(2, 200, kv * HD) for x in (k, v))
    back = ops.kv_cache_read(cache, table, i32([0, 0]), 2, 150, kv)
    for got, want in zip(back, (kc, vc)):
        same(got, want[:, :150].reshape(300, kv * HD))
    kc, vc = (x.reshape(2, 200, kv, HD) for x in (kc, vc))
    ref = attend_ref(q, kc, vc, lens, n_q, heads, kv, 0, 0)
    check(*ops.kv_cache_attention(dev(q), cache, table, i32(lens), 2, n_q, heads, kv,
                                  want_lse=True), ref)
