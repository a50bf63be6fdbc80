"""Attention over a cache whose sequences share pages in groups, through the C ABI, against
float64 over the values that the cache holds (attention_ref's bounds: the parts are f32)."""
import numpy as np
import pytest
import torch

import attention_ref as R
from prichs_amd import _lib as L
from prichs_amd import ops, synth
from tests.test_gpu_kv_cache import attend_ref, check, dev, filled, host, i32, say

pytestmark = pytest.mark.gpu
HD, PAGE = 128, L.KV_PAGE


class Scene:
    """groups: (sequences, shared positions) of each, in order from sequence `first` on.  A
    group's pages stand in its first sequence's row alone: the others' rows name no page
    there."""

    def __init__(self, groups, lens, n_q, heads, kv, seed, first=0, max_pages=None, q_scale=1.0):
        rng = np.random.default_rng(seed)
        batch, top = len(lens), max(max(lens), 1)
        self.lens, self.n_q, self.heads, self.kv, self.batch = lens, n_q, heads, kv, batch
        pages = max_pages or -(-top // PAGE)
        self.n_pages = batch * pages + 1
        table = rng.permutation(self.n_pages)[:batch * pages].reshape(batch, pages)
        k, v = (synth.round_bf16(rng.standard_normal((batch, top, kv * HD))) for _ in range(2))
        starts, b = [first], first
        for size, shared in groups:
            full = max(shared, 0) // PAGE
            for i in range(b + 1, min(b + size, batch)):
                k[i, :full * PAGE], v[i, :full * PAGE] = k[b, :full * PAGE], v[b, :full * PAGE]
                table[i, :full] = -1
            b += size
            starts.append(b)
        self.start, self.shared = i32(starts), i32([s for _, s in groups])
        self.table, self.cache = i32(table), filled(self.n_pages, kv)
        # Everything that a sequence holds, and the group's pages by whoever names them.
        held = [min(max(n, 0), pages * PAGE) for n in lens]
        b = first
        for size, shared in groups:
            if b < batch:
                held[b] = max([held[b]] + [min(shared, h) for h in held[b:b + size]])
            b += size
        ops.kv_cache_write(self.cache, self.table, i32([0] * batch), dev(k.reshape(-1, kv * HD)),
                           dev(v.reshape(-1, kv * HD)), batch, top, kv, counts=i32(held))
        self.kc, self.vc = (R.cached_values(x.reshape(-1, HD)).reshape(batch, top, kv, HD)
                            for x in (k, v))
        self.q = synth.round_bf16(rng.standard_normal((batch * n_q, heads * HD)) * q_scale)

    def ref(self, window=0, sinks=0, keep=None):
        pages = self.table.shape[1]
        seen = [min(max(n, 0), pages * PAGE) for n in self.lens]
        return attend_ref(self.q, self.kc, self.vc, seen, self.n_q, self.heads, self.kv, window,
                          sinks, keep)

    def run(self, window=0, sinks=0, **kw):
        kw = {**dict(want_lse=True, q=dev(self.q), table=self.table, cache=self.cache,
                     start=self.start, shared=self.shared), **kw}
        return ops.kv_cache_shared_attention(
            kw.pop("q"), kw.pop("cache"), kw.pop("table"), i32(self.lens), kw.pop("start"),
            kw.pop("shared"), self.batch, self.n_q, self.heads, self.kv, window, sinks, **kw)


# (groups, lengths, n_q, heads, kv, window, sinks): nothing shared; one group of few and of
# many rows; groups of one sequence, empty ones, shared positions that end inside a page or
# past the sequence; lengths of zero, shorter than n_q and than what is shared; windows that
# end in the shared pages, in the own ones, and sinks past either.
CASES = [
    ([], [70, 3], 1, 4, 2, 0, 0),
    ([(2, 64)], [65, 64], 1, 1, 1, 0, 0),
    ([(2, 63)], [65, 64], 1, 4, 1, 0, 0),
    ([(3, 200)], [300, 193, 640], 1, 12, 3, 0, 0),
    ([(1, 128), (4, 256), (0, 64), (2, 0)], [200, 300, 257, 256, 400, 90, 10], 1, 8, 2, 0, 0),
    ([(5, 500)], [700, 448, 100, 0, 3], 1, 12, 3, 0, 0),
    ([(3, 640)], [700, 650, 900], 5, 6, 2, 0, 0),
    ([(3, 640)], [700, 650, 641], 20, 4, 4, 0, 0),
    ([(4, 640)], [700, 650, 900, 1400], 1, 8, 1, 100, 0),
    ([(4, 640)], [700, 650, 900, 800], 3, 8, 2, 200, 70),
    ([(2, 320), (3, 320)], [400, 330, 700, 1000, 321], 2, 12, 3, 1, 700),
    ([(30, 1000)], [1000 + 7 * i for i in range(30)], 1, 12, 3, 0, 0),
    ([(64, 128)], [129 + i for i in range(64)], 1, 4, 1, 0, 0),
    ([(40, 640)], [641 + 3 * i for i in range(40)], 1, 10, 2, 300, 4),
    ([(17, 2048)], [2049 + 11 * i for i in range(17)], 4, 6, 1, 0, 0),
    ([(9, 3000)], [3000 + i for i in range(9)], 3, 5, 1, 0, 0),
    ([(2, 64)] * 70, [100] * 140, 1, 2, 1, 0, 0),
    ([(1, 64)] * 130 + [(20, 128)], [100] * 130 + [200] * 20, 1, 4, 2, 0, 0),
    ([(25, 192), (31, 128)], [250] * 25 + [129] * 31, 6, 3, 3, 0, 0),
    ([(70, 1280)], [1281 + 5 * i for i in range(70)], 2, 4, 2, 700, 130),
    ([(90, 640)], [650 + 2 * i for i in range(90)], 1, 6, 3, 200, 70),
    ([(130, 320), (140, 128)], [400 + i for i in range(130)] + [130 + i for i in range(140)], 1, 4,
     1, 64, 0),
    ([(30, 2000)], [1900 + 15 * i for i in range(30)], 2, 4, 2, 1600, 130),
]


def columns(batch, n_q, heads, kv):
    """Columns of a table with which a call has 4096 tiles of 16 rows times pages, from where
    on groups of 32 rows and more take tiles of 32."""
    return -(-4096 // (-(-batch * n_q * (heads // kv) // 16) * kv))


# A call of few pages has a workgroup for each tile of a sequence.  The same with tables so
# long that shared and own pages are taken apart, and so long that there are tiles of 32 rows
# (most entries of either nobody reaches).
LONG = [CASES[i] for i in (0, 1, 2, 3, 4, 5, 6, 7, 11, 12, 16)]
MANY = [CASES[i] for i in (3, 5, 6, 7, 8, 9, 10, 11, 13, 14, 18, 19, 20, 21, 22)]
FORMS = [(*c, form) for cases, form in ((CASES, 0), (LONG, 1), (MANY, 2)) for c in cases]


def pages_of(lens, n_q, heads, kv, form):
    """Columns of a case's table."""
    need = -(-max(lens) // PAGE)
    return (need, max(need, 25), max(need, columns(len(lens), n_q, heads, kv)))[form]


@pytest.mark.parametrize("groups,lens,n_q,heads,kv,window,sinks,form", FORMS)
def test_groups(cuda, groups, lens, n_q, heads, kv, window, sinks, form):
    say("case:", groups[:3], lens[:3], n_q, heads, kv, window, sinks, form)
    s = Scene(groups, lens, n_q, heads, kv, n_q + sum(lens),
              max_pages=pages_of(lens, n_q, heads, kv, form))
    ref = s.ref(window, sinks)
    wide = torch.full((s.batch * n_q + 1, heads * HD + 8), float("nan"), dtype=torch.bfloat16,
                      device="cuda")
    wide[:s.batch * n_q, :heads * HD] = dev(s.q)
    out = torch.full((s.batch * n_q + 1, heads * HD + 16), 7.0, dtype=torch.bfloat16,
                     device="cuda")
    rows = slice(0, s.batch * n_q), slice(8, 8 + heads * HD)
    _, lse = s.run(window, sinks, q=wide[:, :heads * HD], out=out[:, rows[1]])
    check(out[rows], lse, ref)
    h = host(out)
    assert (h[rows[0].stop:] == 7).all() and (h[:, :8] == 7).all() and \
        (h[:, rows[1].stop:] == 7).all()
    again, none = s.run(window, sinks, want_lse=False)
    assert none is None and torch.equal(again, out[rows].contiguous())


def wide(size, heads=8, kv=2):
    """Columns by the sequences of a group: shared and own pages apart with 4, tiles of 32 rows
    with 40 and 264."""
    return columns(size, 1, heads, kv) if size in (40, 264) else 30 if size == 4 else None


@pytest.mark.parametrize("max_pages", [None, 25])
def test_starts_of_every_kind(cuda, max_pages):
    """Starts below zero, past the batch, that fall, and sequences before and behind the
    groups: each counts as no less than those before it."""
    lens = [300, 280, 400, 350, 129, 200, 260]
    s = Scene([(2, 256), (3, 128)], lens, 1, 4, 2, 31, first=1, max_pages=max_pages)
    ref = s.ref()
    check(*s.run(), ref)
    kinds = [([1, 3, 6], [256, 128]), ([1, 3, 2, 6], [256, 1 << 30, 128]),
             ([-5, 1, 3, 6, 1 << 30], [-1, 256, 128, 0]), ([1, 1, 3, 6, 6], [999, 256, 128, 128]),
             ([1, 3, 6, -(1 << 31)], [256, 128, 64])]
    for start, shared in kinds:
        say("case:", start, shared)
        check(*s.run(start=i32(start), shared=i32(shared)), ref)


@pytest.mark.parametrize("n_q,window,max_pages", [(1, 0, None), (5, 100, None), (1, 0, 30)])
def test_no_groups_and_no_arrays_of_them(cuda, n_q, window, max_pages):
    """n_groups 0 with NULL for both arrays: every sequence shares nothing."""
    s = Scene([], [300, 1, 0, 129], n_q, 4, 2, 33, max_pages=max_pages)
    say("case:", n_q, window, max_pages)
    q, lens = dev(s.q), i32(s.lens)
    out = torch.full_like(q, 7)
    lse = torch.empty((4, 4, n_q), device="cuda")
    max_pages, lib = s.table.shape[1], L.load()
    need = lib.prichs_kv_cache_shared_attention_workspace(4, n_q, 4, 2, max_pages, 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    L.check(lib.prichs_kv_cache_shared_attention(
        q.data_ptr(), q.stride(0), s.cache.data_ptr(), s.n_pages, s.table.data_ptr(), max_pages,
        lens.data_ptr(), None, None, 0, out.data_ptr(), out.stride(0), lse.data_ptr(), 4, n_q, 4,
        2, HD, window, 0, L.DTYPE_BF16, ws.data_ptr(), need,
        torch.cuda.current_stream().cuda_stream))
    check(out, lse, s.ref(window))


def test_whole_table_shared_and_lens_past_it(cuda):
    """Sequences that hold nothing of their own, and lengths past the table."""
    s = Scene([(6, 256)], [256, 256, 255, 100, 200, 1], 1, 8, 2, 32, max_pages=4)
    check(*s.run(), s.ref())
    check(*s.run(shared=i32([1 << 30])), s.ref())  # no more than the table holds
    s.lens = [1 << 30, 256, 255, 100, 200, 1]
    check(*s.run(), s.ref())


@pytest.mark.parametrize("size", [3, 4, 40])
def test_pages_that_do_not_exist(cuda, size):
    s = Scene([(size, 320)], [400 + i for i in range(size)], 1, 8, 2, 33, max_pages=wide(size))
    s.table[0, 1], s.table[0, 4], s.table[1, 5] = s.n_pages, -1, 1 << 30
    keep = [np.ones(500, bool) for _ in range(size)]
    for k in keep:
        k[64:128] = k[256:320] = False
    keep[1][320:384] = False
    for window, sinks in ((0, 0), (150, 70)):
        check(*s.run(window, sinks), s.ref(window, sinks, keep))
    s.table.fill_(-1)
    out, lse = s.run()
    assert not host(out).any() and np.isneginf(host(lse)).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("size", [3, 260, 264])
def test_what_a_row_does_not_see_does_not_reach_it(cuda, size, bad):
    """Values that are not finite in a shared page: rows behind a window, and a sequence
    that ends before them, are as without them."""
    lens = [330 + 7 * (i % 40) for i in range(size)]
    lens[1] = 150
    W = 120
    s = Scene([(size, 320)], lens, 1, 4, 1, 34, max_pages=wide(size, 4, 1))
    x = synth.round_bf16(np.random.default_rng(1).standard_normal((2, HD)))
    k, v = x[:1].copy(), x[1:].copy()
    one = s.table[:1].contiguous()
    ops.kv_cache_write(s.cache, one, i32([301]), dev(k), dev(v), 1, 1, 1)
    clean = s.run(W)[0]
    v[0, 40] = bad
    ops.kv_cache_write(s.cache, one, i32([301]), dev(k), dev(v), 1, 1, 1)
    dirty = s.run(W)[0]
    pos = np.array(lens) - 1
    sees = (pos >= 301) & (pos - 301 < W)
    unseen = torch.from_numpy(~sees).cuda()
    assert sees.any() and not sees.all() and torch.equal(clean[unseen], dirty[unseen])
    h = host(dirty).reshape(size, 4, 4, 32)[sees]
    assert not np.isfinite(h[:, :, 1]).any() and np.isfinite(h[:, :, [0, 2, 3]]).all()


@pytest.mark.parametrize("size", [3, 4, 40])
@pytest.mark.parametrize("q_scale", [0.0, 40.0])
def test_flat_and_steep_scores(cuda, size, q_scale):
    s = Scene([(size, 640)], [700 + i for i in range(size)], 1, 4, 2, 35, q_scale=q_scale,
              max_pages=wide(size, 4))
    ref = s.ref()
    # A score is off by 128 roundings of 2^-24 of its terms, and p by that.
    ref["e_out"] *= 1 + 2 * (q_scale * 16 * HD ** 0.5 * 128 * 2.0 ** -24) / R.U
    # f32 has no p below 2^-126, the hardware's 2^x flushes it: where a dim's other values
    # are zeros (the cache has many), outputs of 1e-48 are all of such terms.
    ref["e_out"] += 2.0 ** -126 * max(s.lens) * np.abs(s.vc).max()
    check(s.run()[0], None, ref)


@pytest.mark.parametrize("size", [2, 4, 40])
def test_rows_without_finite_scores(cuda, size):
    """Scores of -inf alone, in the shared pages, in the own ones or in both, and a +inf or
    NaN: as for a sequence that shares nothing."""
    n, kv = 150, 1
    s = Scene([(size, 128)], [n] * size, 1, 4, kv, 36, max_pages=wide(size, 4, 1))
    k = np.zeros((n, HD), np.float32)
    v = synth.round_bf16(np.random.default_rng(1).standard_normal((n, HD)))
    k[:, 0], k[128:, 1], k[:128, 2] = 1, 1, 1
    for b in range(size):
        ops.kv_cache_write(s.cache, s.table[b:b + 1].contiguous(), i32([0]), dev(k), dev(v), 1, n,
                           kv)
    for dim in range(3):
        for x in (-np.inf, np.inf, np.nan):
            q = np.zeros((size, 4 * HD), np.float32)
            q[:, dim] = x               # of the first head; the others are flat
            out, lse = s.run(q=dev(q))
            t = s.table.clone()
            t[:, :2] = s.table[0, :2]
            want, want_lse = ops.kv_cache_attention(dev(q), s.cache, t, i32(s.lens), size, 1, 4, kv,
                                                    want_lse=True)
            h, w = host(out), host(want)
            assert np.array_equal(np.isnan(h), np.isnan(w)) and np.isnan(h[:, :HD]).all(), (dim, x)
            assert np.array_equal(np.isnan(host(lse)), np.isnan(host(want_lse)))


@pytest.mark.parametrize("size,n_q", [(3, 1), (4, 1), (4, 9), (40, 1), (12, 9)])
def test_what_the_workspace_held_does_not_matter(cuda, size, n_q):
    s = Scene([(size, 640), (2, 0)], [700 + i for i in range(size)] + [90, 0], n_q, 8, 2, 37,
              max_pages=wide(size))
    lib, pages, x, lens = L.load(), s.table.shape[1], dev(s.q), i32(s.lens)
    need = lib.prichs_kv_cache_shared_attention_workspace(s.batch, n_q, 8, 2, pages, 2)
    ws = torch.full((need + 64,), 0xff, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(x)
    lse = torch.empty((s.batch, 8, n_q), dtype=torch.float32, device="cuda")
    L.check(lib.prichs_kv_cache_shared_attention(
        x.data_ptr(), 8 * HD, s.cache.data_ptr(), s.n_pages, s.table.data_ptr(), pages,
        lens.data_ptr(), s.start.data_ptr(), s.shared.data_ptr(), 2, out.data_ptr(), 8 * HD,
        lse.data_ptr(), s.batch, n_q, 8, 2, HD, 0, 0, L.DTYPE_BF16, ws.data_ptr(), need,
        torch.cuda.current_stream().cuda_stream))
    check(out, lse, s.ref())
    assert (ws[need:] == 0xff).all()


def test_pages_past_32_bits(cuda):
    """A cache of 4.7 GB whose shared and own pages lie at its start and its end."""
    s = Scene([(40, 256)], [300 + i for i in range(40)], 1, 4, 2, 38, max_pages=wide(40, 4))
    n = 270_000
    far = ops.kv_cache_pages(n, 2)
    old = torch.arange(s.n_pages, dtype=torch.int32, device="cuda")
    new = torch.where(old % 2 == 0, old, n - 1 - old)
    ops.kv_cache_copy(far, s.cache, new, old, 2)
    table = torch.where(s.table >= 0, new[s.table.clamp(min=0).long()], s.table)
    check(*s.run(cache=far, table=table), s.ref())


def test_two_graphs_at_once_and_a_stream_of_its_own(cuda):
    """Two captured calls replayed at the same time on two streams, each with a workspace of
    its own; the page calls and the attention on a stream that is not the current one."""
    scenes = [Scene([(12, 1280)], [1290 + 70 * i for i in range(12)], 1, 12, 3, 40),
              Scene([(3, 640), (4, 256)], [700, 650, 900, 300, 260, 257, 400], 2, 8, 2, 41)]
    refs = [s.ref() for s in scenes]
    lens = [i32(s.lens) for s in scenes]
    qs = [dev(s.q) for s in scenes]

    def call(i, stream=None):
        s = scenes[i]
        return ops.kv_cache_shared_attention(qs[i], s.cache, s.table, lens[i], s.start, s.shared,
                                             s.batch, s.n_q, s.heads, s.kv, want_lse=True,
                                             stream=stream)

    graphs, outs = [], []
    for i in range(2):
        check(*call(i), refs[i])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for o, lse in outs:
            o.fill_(7), lse.fill_(7)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            check(*outs[i], refs[i])
    side = streams[0]
    side.wait_stream(torch.cuda.current_stream())
    got = [call(i, side) for i in range(2)]
    side.synchronize()
    for i in range(2):
        check(*got[i], refs[i])

    # Pages taken, shared, given back and moved on that stream.
    refs, table = ops.kv_pages_refs(20), torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    cache, held, short = ops.kv_cache_pages(20, 2), i32([0] * 3), i32([9])
    counts, now, kids, parents, first = (i32(x) for x in ([0, 130, 0], [0, 130, 0], [0, 2],
                                                         [1, 1], [1]))
    side.wait_stream(torch.cuda.current_stream())
    ops.kv_pages_reserve(refs, table, held, counts, shortfall=short, stream=side)
    with torch.cuda.stream(side):
        held.copy_(now)
    ops.kv_pages_fork(cache, refs, table, held, parents, kids, 2, stream=side)
    ops.kv_pages_release(refs, table, first, stream=side)
    n_live, new = ops.kv_pages_compact(cache, refs, table, 2, stream=side)
    side.synchronize()
    assert (short.item(), n_live.item(), held.tolist()) == (0, 4, [130] * 3)
    assert table.tolist() == [[0, 1, 3, -1], [-1] * 4, [0, 1, 2, -1]]
    assert refs.tolist() == [2, 2, 1, 1] + [0] * 16 and new.tolist()[:5] == [0, 1, -1, 3, 2]


def test_forked_continuations_in_a_graph(cuda):
    """As a program uses the calls together: prompts normed, rotated and cached, forked into
    continuations, and decode steps in one captured graph (pages reserved, the token's keys
    and values normed, rotated and cached, attention over shared and own pages), a round
    that starts anew and a compaction between them; against float64 at every step."""
    rng = np.random.default_rng(39)
    H, K, prompts, each, steps = 4, 2, 2, 3, 70
    P = [100, 128]
    batch, n = prompts * each, max(P) + steps
    angle = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, HD, 2) / HD)
    cos, sin = dev(np.cos(angle), torch.float32), dev(np.sin(angle), torch.float32)
    wq, wk = (dev(1 + 0.2 * rng.standard_normal(HD), torch.float32) for _ in range(2))
    width, n_pages = -(-n // PAGE), 40
    cache, refs = filled(n_pages, K), ops.kv_pages_refs(n_pages)
    refs[[0, 3, 7]] = 1                           # pages that another holder keeps
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    lens, short = i32([0] * batch), i32([0])
    first = [g * each for g in range(prompts)]
    raw_k, raw_v = (synth.round_bf16(rng.standard_normal((batch, n, K * HD))) for _ in range(2))
    raw_q = synth.round_bf16(rng.standard_normal((batch, n, H * HD)))
    for g, b in enumerate(first):
        raw_k[b:b + each, :P[g]], raw_v[b:b + each, :P[g]] = raw_k[b, :P[g]], raw_v[b, :P[g]]

    def rotated(x, w, heads, at):
        q, k = (dev(x), None) if heads == H else (None, dev(x))
        r = ops.qk_norm_rope(q, k, wq, wk, cos, sin, *((H, 0) if heads == H else (0, K)),
                             positions=at)
        return r[0] if heads == H else r[1]

    # What the cache will hold: of each position the rotated key as the kernel rounds it.
    kc = np.stack([R.cached_values(host(rotated(raw_k[b], wk, K, i32(range(n)))).reshape(-1, HD))
                   .reshape(n, K, HD) for b in range(batch)])
    vc = R.cached_values(raw_v.reshape(-1, HD)).reshape(batch, n, K, HD)
    qr = np.stack([host(rotated(raw_q[b], wq, H, i32(range(n)))) for b in range(batch)])

    counts = i32([P[b // each] if b in first else 0 for b in range(batch)])
    ops.kv_pages_reserve(refs, table, lens, counts, shortfall=short)
    top = max(P)
    _, k = ops.qk_norm_rope(None, dev(raw_k[:, :top].reshape(-1, K * HD)), wq, wk, cos, sin, 0, K,
                            seq_len=top)
    ops.kv_cache_write(cache, table, lens, k, dev(raw_v[:, :top].reshape(-1, K * HD)), batch, top,
                       K, counts=counts)
    lens.copy_(counts)
    kids = [b for b in range(batch) if b not in first]
    parents, children = i32([b // each * each for b in kids]), i32(kids)
    start, shared = i32([0, each, 2 * each]), i32([p // PAGE * PAGE for p in P])
    ones = i32([1] * batch)
    bq, bk, bv = (torch.zeros((batch, w * HD), dtype=torch.bfloat16, device="cuda")
                  for w in (H, K, K))

    def step():
        ops.kv_pages_reserve(refs, table, lens, ones, shortfall=short)
        q, k = ops.qk_norm_rope(bq, bk, wq, wk, cos, sin, H, K, positions=lens)
        ops.kv_cache_write(cache, table, lens, k, bv, batch, 1, K)
        lens.add_(1)
        return ops.kv_cache_shared_attention(q, cache, table, lens, start, shared, batch, 1, H,
                                             K)[0]

    def begin():
        ops.kv_pages_release(refs, table, children)
        ops.kv_pages_fork(cache, refs, table, lens, parents, children, K, shortfall=short)
        assert short.item() == 0

    begin()
    saved = [t.clone() for t in (cache, refs, table, lens)]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    for turn in range(2):
        for t, v in zip((cache, refs, table, lens), saved):
            t.copy_(v)
        for i in range(steps - max(P) + 100 if turn else steps):
            at = [P[b // each] + i for b in range(batch)]
            for buf, x in ((bq, raw_q), (bk, raw_k), (bv, raw_v)):
                buf.copy_(dev(np.stack([x[b, at[b]] for b in range(batch)])))
            graph.replay()
            got = o.clone()
            assert short.item() == 0
            ref = attend_ref(np.stack([qr[b, at[b]] for b in range(batch)]), kc, vc,
                             [a + 1 for a in at], 1, H, K, 0, 0)
            check(got, None, ref)
            if i % 20 == 7:                       # eager calls between the replays
                n_live, new = ops.kv_pages_compact(cache, refs, table, K)
                assert n_live.item() == int((refs > 0).sum())
                # The other holder follows the pages that moved.
                assert all(refs[int(new[p])] > 0 for p in range(n_pages) if int(new[p]) >= 0)
        # Everything but the prompts' pages is given back; a round starts anew.
        ops.kv_pages_release(refs, table, i32(range(batch)), counts)
        want = 3 + sum(-(-p // PAGE) for p in P)
        assert int((refs > 0).sum()) == want
        lens.copy_(counts)
        begin()
        saved = [t.clone() for t in (cache, refs, table, lens)]


def test_wrapper_refusals(cuda):
    s = Scene([(2, 64)], [70, 80], 1, 4, 2, 40)
    for change in (dict(start=i32([0, 1, 2])), dict(start=s.start.long()), dict(shared=i32([[64]])),
                   dict(start=s.start.cpu()), dict(cache=s.cache[:, :1].contiguous())):
        with pytest.raises(ValueError):
            s.run(**change)
    with pytest.raises(ValueError):
        s.run(window=-1)
    with pytest.raises(TypeError):
        s.run(q=dev(s.q).float())
    q = dev(s.q)
    none = i32(np.zeros(0))
    assert ops.kv_cache_shared_attention(q[:0], s.cache, s.table[:0], none, i32([0]), none, 0, 1, 4,
                                         2)[0].shape[0] == 0
    empty = torch.empty((2, 0), dtype=torch.int32, device="cuda")
    out, lse = s.run(table=empty)
    assert not host(out).any() and np.isneginf(host(lse)).all()
