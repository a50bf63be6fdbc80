"""Attention over shared pages where parts of a row have no softmax, where lse has to be a
number, and where calls over long tables run together and in a captured step."""
import numpy as np
import pytest
import torch

import attention_ref as R
from prichs_amd import _lib as L
from prichs_amd import ops, synth
from tests.test_gpu_kv_cache import ATTEND, attend_case, attend_ref, check, dev, filled, host, i32
from tests.test_gpu_kv_shared import FORMS, HD, PAGE, Scene, columns, pages_of

pytestmark = pytest.mark.gpu


def check_finite(out, lse, ref):
    """check, and that lse is a number wherever the reference's is."""
    h, w = host(lse), ref["lse"]
    fin = np.isfinite(w)
    assert np.isfinite(h[fin]).all(), (np.isnan(h).sum(), np.argwhere(fin & ~np.isfinite(h))[:5])
    assert np.array_equal(np.isneginf(h), np.isneginf(w))
    assert np.isfinite(host(out)).all()
    check(out, lse, ref)


# ------------------------------------------------------ parts without a softmax --
BIG = 1e30   # BIG * BIG is past the largest f32: such a score is -inf, of finite operands
P, TOP = 256, 450                                     # shared positions; a sequence's at most
# Keys whose score is -inf for the rows that ask for it: all shared ones, all own ones, the
# first and the last shared page, a page of the own ones, everything but one key of either.
LOST = [[(0, P)], [(P, TOP)], [(0, 64)], [(192, P)], [(0, P), (320, 384)], [(64, P), (P, TOP)],
        [(0, 200), (201, TOP)], [(0, 399), (400, TOP)]]
# (sequences of 8 + 2 heads, columns of their table, window): one launch, parts with tiles of
# 16 rows, with tiles of 32; a window that leaves few pages is taken in parts by many sequences.
TABLES = [(3, None, 0, "rows"), (4, 30, 0, "1"), (40, columns(40, 1, 8, 2), 0, "2"),
          (3, None, 300, "rows"), (129, None, 300, "1"), (129, columns(129, 1, 8, 2), 300, "2")]


@pytest.mark.parametrize("lost", LOST)
@pytest.mark.parametrize("size,max_pages,window,form", TABLES)
def test_parts_whose_scores_are_all_minus_infinity(cuda, size, max_pages, window, form, lost):
    """The softmax of a row is that of its other keys, whichever part holds them.  Odd heads
    have finite scores everywhere."""
    print("case:", size, max_pages, lost, window, flush=True)
    H, K = 8, 2
    lens = [TOP - i % 40 for i in range(size)]
    s = Scene([(size, P)], lens, 1, H, K, 50, max_pages=max_pages)
    rng = np.random.default_rng(51)
    k, v = (synth.round_bf16(rng.standard_normal((TOP, K * HD))) for _ in range(2))
    gone = np.zeros(TOP, bool)
    for a, b in lost:
        gone[a:b] = True
    k.reshape(TOP, K, HD)[:, :, 5] = np.where(gone, BIG, 0)[:, None]
    k = synth.round_bf16(k)
    for b in range(size):     # the first sequence's row of the table names the shared pages
        t = s.table[b:b + 1].clone()
        t[:, :P // PAGE] = s.table[0, :P // PAGE]
        ops.kv_cache_write(s.cache, t, i32([0]), dev(k), dev(v), 1, TOP, K, counts=i32([lens[b]]))
    q = synth.round_bf16(rng.standard_normal((size, H, HD)))
    q[:, ::2, 5], q[:, 1::2, 5] = -BIG, 0
    q = synth.round_bf16(q.reshape(size, H * HD))
    kc, vc = (R.cached_values(x.reshape(-1, HD)).reshape(1, TOP, K, HD).repeat(size, 0)
              for x in (k, v))
    assert (kc[0, gone, :, 5] > 1e29).all() and not kc[0, ~gone, :, 5].any()
    # In 64 bits a score of -1e59 is a number, and its exponential zero.
    ref = attend_ref(q, kc, vc, lens, 1, H, K, window, 0)
    alone = np.array([not (~gone[max(0, n - window) if window else 0:n]).any() for n in lens])
    for shared in (True, False):
        if shared:
            out, lse = s.run(window, q=dev(q))
        else:
            t = s.table.clone()
            t[:, :P // PAGE] = s.table[0, :P // PAGE]
            out, lse = ops.kv_cache_attention(dev(q), s.cache, t, i32(lens), size, 1, H, K, window,
                                              want_lse=True)
        # Rows that see such keys alone have no softmax: NaN.
        h, hl = host(out).reshape(size, H, HD), host(lse)[:, :, 0]
        none = alone[:, None] & (np.arange(H) % 2 == 0)
        assert np.isnan(h[none]).all() and np.isnan(hl[none]).all()
        assert np.isfinite(h[~none]).all() and np.isfinite(hl[~none]).all()
        bound = ref["e_out"].reshape(h.shape)
        err = np.abs(h - ref["out"].reshape(h.shape))
        assert (err[~none] <= bound[~none]).all(), (shared, (err - bound)[~none].max())
        assert (np.abs(hl - ref["lse"][:, :, 0])[~none] <= 1.25 * R.U).all()


# ------------------------------------------------------------------------ lse --
@pytest.mark.parametrize("groups,lens,n_q,heads,kv,window,sinks,form", FORMS[::2])
def test_lse_is_a_number_where_a_row_sees_keys(cuda, groups, lens, n_q, heads, kv, window, sinks,
                                               form):
    """Through the C ABI, with NaN in lse and in the workspace before the call."""
    print("case:", groups[:3], lens[:3], n_q, heads, kv, window, sinks, form, flush=True)
    pages = pages_of(lens, n_q, heads, kv, form)
    s = Scene(groups, lens, n_q, heads, kv, n_q + sum(lens), max_pages=pages)
    lib, x, L32 = L.load(), dev(s.q), i32(lens)
    need = lib.prichs_kv_cache_shared_attention_workspace(s.batch, n_q, heads, kv, pages,
                                                          len(groups))
    ws = torch.full((need + 16,), 0xff, dtype=torch.uint8, device="cuda")
    out = torch.full_like(x, float("nan"))
    lse = torch.full((s.batch, heads, n_q), float("nan"), device="cuda")
    L.check(lib.prichs_kv_cache_shared_attention(
        x.data_ptr(), heads * HD, s.cache.data_ptr(), s.n_pages, s.table.data_ptr(), pages,
        L32.data_ptr(), s.start.data_ptr(), s.shared.data_ptr(), len(groups), out.data_ptr(),
        heads * HD, lse.data_ptr(), s.batch, n_q, heads, kv, HD, window, sinks, L.DTYPE_BF16,
        ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    check_finite(out, lse, s.ref(window, sinks))


@pytest.mark.parametrize("batch,n_q,lens,heads,kv,window,sinks", ATTEND[::2])
def test_lse_of_each_sequence_by_itself(cuda, batch, n_q, lens, heads, kv, window, sinks):
    print("case:", batch, n_q, lens, heads, kv, window, sinks, flush=True)
    table, cache, q, kc, vc = attend_case(batch, n_q, lens, heads, kv, n_q + sum(lens))
    got = ops.kv_cache_attention(dev(q), cache, table, i32(lens), batch, n_q, heads, kv, window,
                                 sinks, want_lse=True)
    check_finite(*got, attend_ref(q, kc, vc, lens, n_q, heads, kv, window, sinks))


# ---------------------------------------------------------------- long tables --
FULL = [(6, 26, 1), (40, 60, 4)]  # (sequences, pages, tokens): tiles of 16 rows and of 32


@pytest.mark.parametrize("size,pages,n_q", FULL)
def test_a_table_full_of_shared_pages(cuda, size, pages, n_q):
    """Sequences that hold nothing of their own, shared positions and lengths past the
    table, in parts."""
    top = pages * PAGE
    lens = [top, top, top - 1, 100, 200, 1] + [top - 5 * i for i in range(size - 6)]
    s = Scene([(size, top)], lens, n_q, 8, 2, 52, max_pages=pages)
    check_finite(*s.run(), s.ref())
    check_finite(*s.run(shared=i32([1 << 30])), s.ref())    # no more than the table holds
    check_finite(*s.run(shared=i32([(1 << 31) - 1])), s.ref())
    s.lens = [1 << 30, (1 << 31) - 1] + lens[2:]
    check_finite(*s.run(), s.ref())
    check_finite(*s.run(300, 70), s.ref(300, 70))


# Scenes whose calls have workspaces, the second in tiles of 32 rows.
PAIR = [([(12, 1280)], [1290 + 70 * i for i in range(12)], 1, 12, 3, None),
        ([(30, 640), (10, 256)], [700 + 3 * i for i in range(30)] + [300 + i for i in range(10)],
         1, 8, 2, columns(40, 1, 8, 2))]


def test_two_graphs_with_workspaces_at_once(cuda):
    """Two captured calls in parts replayed at the same time on two streams, each with a
    workspace of its own."""
    scenes = [Scene(g, lens, n_q, h, k, 40 + i, max_pages=p)
              for i, (g, lens, n_q, h, k, p) in enumerate(PAIR)]
    lib = L.load()
    for s in scenes:
        assert lib.prichs_kv_cache_shared_attention_workspace(
            s.batch, s.n_q, s.heads, s.kv, s.table.shape[1], s.shared.numel()) > 0
    refs = [s.ref() for s in scenes]
    lens, qs = [i32(s.lens) for s in scenes], [dev(s.q) for s in scenes]

    def call(i):
        s = scenes[i]
        return ops.kv_cache_shared_attention(qs[i], s.cache, s.table, lens[i], s.start, s.shared,
                                             s.batch, s.n_q, s.heads, s.kv, want_lse=True)

    graphs, outs = [], []
    for i in range(2):
        check_finite(*call(i), refs[i])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(call(i))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for o, lse in outs:
            o.fill_(7), lse.fill_(7)
        torch.cuda.synchronize()
        for _ in range(20):
            for g, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            check_finite(*outs[i], refs[i])
            eager = call(i)
            assert torch.equal(eager[0], outs[i][0]) and torch.equal(eager[1], outs[i][1])


# A step over long tables: prompts of 26 and of 30 pages and a bit, (query, kv heads).
PROMPTS, EACH, STEP_HEADS, STEP_COLUMNS = [1700, 1920], 3, (4, 2), 33


def test_forked_continuations_over_long_tables_in_a_graph(cuda):
    """Prompts cached and forked, then captured decode steps (pages reserved, keys and values
    cached, attention in parts), with a compaction and a round that starts anew between the
    replays; every step against float64."""
    rng = np.random.default_rng(53)
    (H, K), each, steps = STEP_HEADS, EACH, 70
    batch = len(PROMPTS) * each
    n, n_pages = max(PROMPTS) + steps, 110
    assert -(-n // PAGE) <= STEP_COLUMNS
    k, v = (synth.round_bf16(rng.standard_normal((batch, n, K * HD))) for _ in range(2))
    q = synth.round_bf16(rng.standard_normal((steps, batch, H * HD)))
    first = [g * each for g in range(len(PROMPTS))]
    for g, b in enumerate(first):
        k[b:b + each, :PROMPTS[g]], v[b:b + each, :PROMPTS[g]] = k[b, :PROMPTS[g]], v[b, :PROMPTS[g]]
    kc, vc = (R.cached_values(x.reshape(-1, HD)).reshape(batch, n, K, HD) for x in (k, v))
    cache, refs = filled(n_pages, K), ops.kv_pages_refs(n_pages)
    refs[[1, 4, 9, 60]] = 1                               # pages that another holder keeps
    table = torch.full((batch, STEP_COLUMNS), -1, dtype=torch.int32, device="cuda")
    lens, short = i32([0] * batch), i32([0])
    counts = i32([PROMPTS[b // each] if b in first else 0 for b in range(batch)])
    ops.kv_pages_reserve(refs, table, lens, counts, shortfall=short)
    assert short.item() == 0
    top = max(PROMPTS)
    ops.kv_cache_write(cache, table, lens, dev(k[:, :top].reshape(-1, K * HD)),
                       dev(v[:, :top].reshape(-1, K * HD)), batch, top, K, counts=counts)
    lens.copy_(counts)
    kids = [b for b in range(batch) if b not in first]
    parents, children = i32([b // each * each for b in kids]), i32(kids)
    start = i32([0, each, 2 * each])
    shared = i32([p // PAGE * PAGE for p in PROMPTS])
    ones = i32([1] * batch)
    bq, bk, bv = (torch.zeros((batch, w * HD), dtype=torch.bfloat16, device="cuda")
                  for w in (H, K, K))

    def step():
        ops.kv_pages_reserve(refs, table, lens, ones, shortfall=short)
        ops.kv_cache_write(cache, table, lens, bk, bv, batch, 1, K)
        lens.add_(1)
        return ops.kv_cache_shared_attention(bq, cache, table, lens, start, shared, batch, 1, H, K,
                                             want_lse=True)

    def begin():
        ops.kv_pages_release(refs, table, children)
        ops.kv_pages_fork(cache, refs, table, lens, parents, children, K, shortfall=short)
        assert short.item() == 0
        return [t.clone() for t in (cache, refs, table, lens)]

    saved = begin()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(2):
        for t, x in zip((cache, refs, table, lens), saved):
            t.copy_(x)
        for i in range(steps if turn == 0 else 10):
            at = [PROMPTS[b // each] + i for b in range(batch)]
            bq.copy_(dev(q[i]))
            for buf, x in ((bk, k), (bv, v)):
                buf.copy_(dev(np.stack([x[b, at[b]] for b in range(batch)])))
            graph.replay()
            got = [t.clone() for t in held]
            assert short.item() == 0
            if i % 9 == 0 or i > steps - 4:
                check_finite(*got, attend_ref(q[i], kc, vc, [a + 1 for a in at], 1, H, K, 0, 0))
            if i % 30 == 7:                               # eager calls between the replays
                n_live, _ = ops.kv_pages_compact(cache, refs, table, K)
                assert n_live.item() == int((refs > 0).sum())
        ops.kv_pages_release(refs, table, i32(range(batch)), counts)
        assert int((refs > 0).sum()) == 4 + sum(-(-p // PAGE) for p in PROMPTS)
        lens.copy_(counts)
        saved = begin()
