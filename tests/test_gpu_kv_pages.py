"""Page bookkeeping of the KV cache on the device against pages_ref, exactly."""
import numpy as np
import pytest
import torch

from pages_ref import PAGE, Pages
from prichs_amd import _lib as L
from prichs_amd import ops

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def random_cache(rng, n_pages, kv):
    """Pages of random bytes."""
    g = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    return torch.randint(0, 256, (n_pages, kv, L.KV_PAGE_BYTES), generator=g, device="cuda",
                         dtype=torch.uint8)


def digest(cache):
    """A number for each page that stands for its bytes."""
    w = torch.arange(1, cache.shape[1] * cache.shape[2] + 1, device="cuda", dtype=torch.int64)
    return (cache.flatten(1).long() * (w * 2654435761 % 1000003)).sum(1).cpu().numpy() \
        if cache.shape[0] else np.zeros(0, np.int64)


def scene(seed, n_pages, batch, width, kv, used=0.6, shared=True):
    """A table whose rows hold random pages, some of them shared, and lengths that fit."""
    rng = np.random.default_rng(seed)
    order = list(rng.permutation(n_pages))
    lens = np.zeros(batch, int)
    table = np.full((batch, width), -1)
    budget = int(n_pages * used)
    for b in range(batch):
        n = int(min(rng.integers(0, width + 1), budget))
        budget -= n
        table[b, :n] = [order.pop() for _ in range(n)]
        if shared and b and rng.random() < 0.3:
            m = int(min(n, (table[b - 1] >= 0).sum()))
            table[b, :m] = table[b - 1, :m]
        lens[b] = rng.integers(0, n * PAGE + 1) if n else 0
    refs = np.bincount(table[table >= 0], minlength=n_pages) if n_pages else np.zeros(0, int)
    cache = random_cache(rng, n_pages, kv)
    ref = Pages(refs, table, lens, digest(cache))
    return rng, ref, cache, i32(refs), i32(table).view(batch, width), i32(lens)


def same(ref, cache, refs, table, lens):
    assert refs.tolist() == ref.refs
    assert table.tolist() == ref.table
    assert lens.tolist() == ref.lens
    assert np.array_equal(digest(cache), ref.data)


# (pages, rows, columns, kv heads): one page, less than a block of pages, several blocks;
# tables of one column and of more than a workgroup has threads; more pages than a workgroup
# takes in one round, and more pages or rows than one workgroup plans for.
SCENES = [(1, 1, 1, 1), (70, 6, 8, 3), (300, 40, 7, 1), (5000, 100, 40, 1), (9000, 17, 600, 1),
          (4096, 3, 1300, 1), (40, 9, 3, 5), (4097, 2100, 2, 1), (20000, 50, 300, 1),
          (16384, 30, 400, 1), (66000, 20, 3000, 1), (500, 4100, 2, 1), (70000, 4200, 9, 1)]


@pytest.mark.parametrize("n_pages,batch,width,kv", SCENES)
def test_reserve_fork_release_compact(cuda, n_pages, batch, width, kv):
    """Rounds of all four calls with rows, counts and items of every kind, shortages among
    them."""
    print("case:", n_pages, batch, width, kv, flush=True)
    rng, ref, cache, refs, table, lens = scene(n_pages + batch, n_pages, batch, width, kv)
    short = i32([77])
    for turn in range(4):
        counts = rng.integers(-3, 3 * PAGE, batch)
        counts[rng.random(batch) < 0.3] = 0
        ops.kv_pages_reserve(refs, table, lens, i32(counts), shortfall=short)
        assert short.item() == ref.reserve(counts), turn
        same(ref, cache, refs, table, lens)
        # Children: distinct rows as a rule, some named twice, parents or out of the table.
        n = int(rng.integers(1, batch + 2))
        kids = rng.permutation(batch)[:n]
        kids = np.concatenate([kids, rng.integers(-2, batch + 2, 2)])
        parents = rng.integers(-1, batch + 1, len(kids))
        ops.kv_pages_release(refs, table, i32(kids))
        ref.release(kids)
        same(ref, cache, refs, table, lens)
        ops.kv_pages_fork(cache, refs, table, lens, i32(parents), i32(kids), kv, shortfall=short)
        assert short.item() == ref.fork(parents, kids), turn
        same(ref, cache, refs, table, lens)
        rows = rng.integers(-1, batch + 1, max(1, batch // 3))
        keep = rng.integers(-5, width * PAGE, len(rows))
        ops.kv_pages_release(refs, table, i32(rows), i32(keep))
        ref.release(rows, keep)
        new_lens = [min(n, PAGE * sum(p >= 0 for p in row)) for n, row in zip(ref.lens, ref.table)]
        ref.lens = new_lens
        lens.copy_(i32(new_lens))
        same(ref, cache, refs, table, lens)
        n_live, new = ops.kv_pages_compact(cache, refs, table, kv)
        want_live, want = ref.compact()
        assert n_live.item() == want_live and new.tolist() == want
        same(ref, cache, refs, table, lens)


def test_forks_that_most_children_want(cuda):
    """One prompt forked into every other row; then again with pages for a part of them."""
    rng, ref, cache, refs, table, lens = scene(3, 400, 1, 6, 3, used=0.01)
    batch, width, kv = 300, 6, 3
    t = np.full((batch, width), -1)
    t[0, :5] = [399, 3, 250, 17, 8]
    refs_h = np.bincount(t[t >= 0], minlength=400)
    for length, missing in ((4 * PAGE + 5, 0), (4 * PAGE, 0), (1, 0), (0, 0), (5 * PAGE + 1, 0)):
        ref = Pages(refs_h, t, [length] + [9] * (batch - 1), digest(cache))
        refs, table, lens, short = i32(refs_h), i32(t), i32(ref.lens), i32([5])
        parents, kids = [0] * (batch - 1), list(range(1, batch))
        ops.kv_pages_fork(cache, refs, table, lens, i32(parents), i32(kids), kv, shortfall=short)
        assert short.item() == ref.fork(parents, kids) == missing
        same(ref, cache, refs, table, lens)
    refs_h[:200] += 1                       # pages that some other holder has
    ref = Pages(refs_h, t, [PAGE + 1] + [0] * (batch - 1), digest(cache))
    refs, table, lens = i32(refs_h), i32(t), i32(ref.lens)
    ops.kv_pages_fork(cache, refs, table, lens, i32(parents), i32(kids), kv, shortfall=short)
    assert short.item() == ref.fork(parents, kids) > 0
    same(ref, cache, refs, table, lens)


def test_rows_named_twice_and_counts_that_are_too_low(cuda):
    refs, table = i32([1, 0, -2, 5]), i32([[0, 1, 2, 3], [3, 3, 9, -7], [0, 0, 0, 0]])
    ref = Pages(refs.tolist(), table.tolist())
    rows, keep = [1, 1, 0, 0, 7, -1], [64, 65, 1, 200, 0, 0]
    ops.kv_pages_release(refs, table, i32(rows), i32(keep))
    ref.release(rows, keep)
    assert refs.tolist() == ref.refs == [1, 0, -2, 3] and table.tolist() == ref.table
    assert table.tolist() == [[0, -1, -1, -1], [3, -1, -1, -1], [0, 0, 0, 0]]


def test_reserve_past_the_table_and_of_long_rows(cuda):
    table = torch.full((3, 100), -1, dtype=torch.int32, device="cuda")
    refs, short = ops.kv_pages_refs(150), i32([0])
    table[1, 70] = 149
    refs[149] = 1
    last = (1 << 31) - 1                 # a length and a count: no entry in the table
    ref = Pages(refs.tolist(), table.tolist(), [0, 6300, last])
    counts = [6400 * 3, 6400, last]
    ops.kv_pages_reserve(refs, table, i32(ref.lens), i32(counts), shortfall=short)
    far = (2 * last - 1) // PAGE - last // PAGE + 1
    ref.lens[2], counts[2] = 0, 0
    assert short.item() == ref.reserve(counts) + far
    assert refs.tolist() == ref.refs and table.tolist() == ref.table


@pytest.mark.parametrize("n_pages,batch,width", [
    (9000, 40, 1100),     # one workgroup
    (9000, 1500, 70),     # more rows than its threads
    (66000, 33, 1100),    # many workgroups
])
def test_reserve_for_rows_of_every_length(cuda, n_pages, batch, width):
    """Rows that want one page beside rows that want hundreds, in tables with gaps; where there
    are many rows until the pages are all taken."""
    print("case:", n_pages, batch, width, flush=True)
    rng, ref, cache, refs, table, lens = scene(batch, n_pages, batch, width, 1, used=0.3)
    spans, short = [1, 2, 4, 5, 6, 63, 64, 65, 511, 512, 513, width], i32([0])
    for turn in range(3):
        for b in range(batch):  # gaps: entries that name no page behind a row's last position
            for e in range(ref.lens[b] // PAGE + 1, width):
                if ref.table[b][e] < 0 and rng.random() < 0.2:
                    ref.table[b][e] = int(rng.choice([-1, -7, n_pages, n_pages + 5]))
        table = i32(ref.table)
        counts = PAGE * rng.choice(spans, batch) - rng.integers(0, PAGE, batch)
        counts[rng.random(batch) < 0.5] = 0
        ops.kv_pages_reserve(refs, table, lens, i32(counts), shortfall=short)
        assert short.item() == ref.reserve(counts), turn
        same(ref, cache, refs, table, lens)


def test_compact_with_entries_that_name_free_pages(cuda):
    rng = np.random.default_rng(8)
    cache = random_cache(rng, 9, 2)
    refs_h, t = [0, 2, 0, 1, 0, 0, 1, 0, 1], [[8, 1, 5, -1, 99], [1, 3, 6, 0, -4]]
    ref = Pages(refs_h, t, [0, 0], digest(cache))
    refs, table = i32(refs_h), i32(t)
    n_live, new = ops.kv_pages_compact(cache, refs, table, 2)
    assert (n_live.item(), new.tolist()) == ref.compact() == (4, [-1, 1, -1, 3, -1, -1, 0, -1, 2])
    same(ref, cache, refs, table, i32([0, 0]))
    # All pages in use, and none.
    for value in (1, 0):
        refs = i32([value] * 9)
        before = cache.clone()
        n_live, new = ops.kv_pages_compact(cache, refs, table, 2)
        assert n_live.item() == 9 * value and torch.equal(cache, before)
        assert new.tolist() == (list(range(9)) if value else [-1] * 9)


def test_copy_to_another_cache_and_within_one(cuda):
    rng = np.random.default_rng(9)
    small, big = random_cache(rng, 6, 5), random_cache(rng, 20, 5)
    want = big.clone()
    to, from_ = [19, 0, 20, -1, 7, 3], [0, 5, 1, 2, 6, 3]
    for t, f in ((19, 0), (0, 5), (3, 3)):
        want[t] = small[f]
    ops.kv_cache_copy(big, small, i32(to), i32(from_), 5)
    assert torch.equal(big, want)
    want[1], want[2] = want[19], want[0]
    ops.kv_cache_copy(big, big, i32([1, 2]), i32([19, 0]), 5)
    assert torch.equal(big, want)
    n = 70_000  # more pairs than a grid has rows
    one = random_cache(rng, 3, 1)
    many = torch.zeros((n, 1, L.KV_PAGE_BYTES), dtype=torch.uint8, device="cuda")
    ops.kv_cache_copy(many, one, torch.arange(n, dtype=torch.int32, device="cuda"),
                      torch.arange(n, dtype=torch.int32, device="cuda") % 3, 1)
    assert all(torch.equal(many[i::3], one[i:i + 1].expand(len(many[i::3]), -1, -1))
               for i in range(3))


def test_pages_past_32_bits(cuda):
    """A cache of 4.7 GB: pages move from its end to its start, and a fork copies one there."""
    n_pages, kv = 270_000, 2
    cache = ops.kv_cache_pages(n_pages, kv)
    refs = torch.ones((n_pages,), dtype=torch.int32, device="cuda")
    refs[[5, 100_000, 269_000]] = 0
    table = i32([[269_999, 3], [-1, -1]])
    cache[269_999], cache[269_998], cache[269_997] = 11, 12, 13
    cache[5] = 0
    lens = i32([40, 0])
    ops.kv_pages_fork(cache, refs, table, lens, i32([0]), i32([1]), kv)
    assert table.tolist() == [[269_999, 3], [5, -1]] and (cache[5] == 11).all()
    n_live, new = ops.kv_pages_compact(cache, refs, table, kv)
    assert n_live.item() == 269_998 and table.tolist() == [[269_000, 3], [5, -1]]
    assert (cache[269_000] == 11).all() and (cache[100_000] == 12).all()
    assert new[269_998].item() == 100_000 and refs[269_998:].tolist() == [0, 0]


def test_a_graph_of_all_calls(cuda):
    """Release, fork and reserve captured once and replayed with other items, eager calls
    between the replays."""
    rng, ref, cache, refs, table, lens = scene(12, 500, 20, 9, 2, used=0.5, shared=False)
    parents, kids, counts, short = i32([0] * 6), i32([15] * 6), i32([0] * 20), i32([0])

    def step():
        ops.kv_pages_release(refs, table, kids)
        ops.kv_pages_fork(cache, refs, table, lens, parents, kids, 2)
        ops.kv_pages_reserve(refs, table, lens, counts, shortfall=short)
        return ops.kv_pages_compact(cache, refs, table, 2)

    saved = [t.clone() for t in (cache, refs, table, lens)]
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n_live, new = step()
    for t, s in zip((cache, refs, table, lens), saved):
        t.copy_(s)
    for turn in range(5):
        p, k = rng.integers(0, 10, 6), 10 + rng.permutation(10)[:6]
        c = rng.integers(0, 100, 20)
        parents.copy_(i32(p)), kids.copy_(i32(k)), counts.copy_(i32(c))
        graph.replay()
        torch.cuda.synchronize()
        ref.release(k), ref.fork(p, k)
        missing = ref.reserve(c)
        live, moved = ref.compact()
        assert (n_live.item(), new.tolist(), short.item()) == (live, moved, missing), turn
        same(ref, cache, refs, table, lens)
        other = i32(np.zeros(500))
        ops.kv_pages_reserve(other, torch.full_like(table, -1), lens * 0, counts)
        lens.copy_(lens + counts)
        ref.lens = [min(n + int(x), 9 * PAGE) for n, x in zip(ref.lens, c)]
        lens.clamp_(max=9 * PAGE)


def test_nothing_to_do(cuda):
    none = i32(np.zeros(0))
    refs, table = ops.kv_pages_refs(0), i32(np.full((2, 3), 5))
    cache = ops.kv_cache_pages(0, 1)
    short, lens = i32([9]), i32([0, 0])
    ops.kv_pages_reserve(refs, table, lens, i32([1, 100]), shortfall=short)
    assert short.item() == 3 and table.tolist() == [[-1, 5, 5], [-1, -1, 5]]
    n_live, new = ops.kv_pages_compact(cache, refs, table, 1)
    assert n_live.item() == 0 and new.numel() == 0
    short.fill_(9)
    ops.kv_pages_fork(cache, refs, table, lens, none, none, 1, shortfall=short)
    assert short.item() == 0
    ops.kv_pages_release(refs, table, none)
    ops.kv_cache_copy(cache, cache, none, none, 1)
    refs, empty = ops.kv_pages_refs(5), i32(np.zeros((0, 4)))
    ops.kv_pages_reserve(refs, empty, none, none, shortfall=short)
    ops.kv_pages_release(refs, empty, i32([0]))
    assert short.item() == 0 and refs.tolist() == [0] * 5
    wide = i32(np.zeros((2, 0)))
    ops.kv_pages_reserve(refs, wide, lens, i32([1, 65]), shortfall=short)
    assert short.item() == 3
    ops.kv_pages_fork(ops.kv_cache_pages(5, 1), refs, wide, i32([5, 6]), i32([0]), i32([1]), 1)


def test_wrapper_refusals(cuda):
    refs, table, lens = ops.kv_pages_refs(4), i32(np.zeros((2, 3))), i32([0, 0])
    cache = ops.kv_cache_pages(4, 2)
    with pytest.raises(ValueError):
        ops.kv_pages_reserve(refs.long(), table, lens, lens)
    with pytest.raises(ValueError):
        ops.kv_pages_reserve(refs, table, lens[:1], lens)
    with pytest.raises(ValueError):
        ops.kv_pages_reserve(refs, table.t(), lens, lens)
    with pytest.raises(ValueError):
        ops.kv_pages_reserve(refs, table, lens, lens.cpu())
    with pytest.raises(ValueError):
        ops.kv_pages_reserve(refs, table, lens, lens, shortfall=i32([0, 0]))
    with pytest.raises(ValueError):
        ops.kv_pages_fork(cache, refs, table, lens, i32([0]), i32([1, 0]), 2)
    with pytest.raises(ValueError):
        ops.kv_pages_fork(cache, refs, table, lens, i32([0]), i32([1]), 3)
    with pytest.raises(ValueError):
        ops.kv_pages_compact(cache[:3], refs, table, 2)
    with pytest.raises(ValueError):
        ops.kv_pages_release(refs, table, i32([[0]]))
    with pytest.raises(ValueError):
        ops.kv_cache_copy(cache, cache, i32([0, 1]), i32([2]), 2)
