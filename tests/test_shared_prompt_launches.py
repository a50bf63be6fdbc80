"""Which kernels the norms with rotation, the page calls and the attention over shared
pages launch, on the CPU (tests/launch_log.py), and that the GPU tests reach them all."""
import pytest

from tests import launch_log as ll


def attend(cases):
    """Launches for each (batch, n_q, max_pages, heads, kv heads, groups, with lse, window,
    sinks)."""
    rows = ll.run(f"""
result = []
for b, n, p, h, k, g, lse, window, sinks in {cases!r}:
    need = lib.prichs_kv_cache_shared_attention_workspace(b, n, h, k, p, g)
    L.check(lib.prichs_kv_cache_shared_attention(P, 128 * h, P, 1000, P, p, P, P, P, g, P, 128 * h,
                                                 P if lse else None, b, n, h, k, 128, window, sinks,
                                                 1, P,
                                                 need, None))
    result.append([need, launches()])
""")
    return [(need, ll.as_launches(x)) for need, x in rows]


# (case, blocks of 16 rows in a tile, tiles x splits over shared pages of a kv head, splits
# of own pages): nothing shared; few rows; many rows and few pages; many of both; more tiles
# than workgroups; groups that could each have a short tile; more groups than sequences.
@pytest.mark.parametrize("case,blocks,tiles,split_p,split_s", [
    ((4, 1, 40, 12, 3, 0), 1, 0, 0, 8), ((8, 1, 37, 12, 3, 1), 1, 2, 10, 8),
    ((24, 6, 133, 12, 3, 1), 2, 18, 4, 1), ((256, 1, 528, 12, 3, 1), 2, 32, 5, 1),
    ((64, 1, 136, 12, 3, 1), 2, 8, 10, 1), ((64, 1, 37, 12, 3, 16), 1, 31, 4, 2),
    ((200, 16, 8, 8, 2, 2), 2, 401, 1, 1), ((3, 1, 50, 4, 4, 100), 1, 3, 13, 8)])
def test_how_a_call_is_cut(case, blocks, tiles, split_p, split_s):
    b, n, p, h, k, g = case
    for lse in (0, 1):
        (need, got), = attend([(*case, lse, 0, 0)])
        own = b * k * -(-n * (h // k) // 16)
        flag = "true" if lse else "false"
        assert got[0].kernel == f"kv_shared_kernel<{blocks}, {flag}>"
        assert got[0].grid == [-(-k * tiles * split_p // 8) * 8 + own * split_s, 1, 1]
        parts = split_p + split_s
        wide = parts > 8
        assert got[1].kernel == f"kv_shared_join_kernel<{8 if wide else 1}, {flag}>"
        assert got[1].grid[0] == (b * n * h if wide else -(-b * n * h // 8)) and len(got) == 2
        assert need == b * n * h * parts * 131 * 4


# Few pages: of a table, or that a window leaves.
@pytest.mark.parametrize("case,window,sinks,rows", [
    ((8, 1, 24, 12, 3, 1), 0, 0, True), ((8, 1, 25, 12, 3, 1), 0, 0, False),
    ((85, 1, 4, 12, 3, 1), 0, 0, True), ((86, 1, 4, 12, 3, 1), 0, 0, False),
    ((1, 1, 0, 4, 4, 1), 0, 0, True), ((4, 20, 9, 8, 2, 0), 0, 0, True),
    ((8, 1, 500, 12, 3, 1), 1400, 4, True), ((8, 1, 500, 12, 3, 1), 1472, 64, False),
    ((8, 1, 500, 12, 3, 1), 1 << 20, 0, False)])
def test_few_pages_take_one_launch(case, window, sinks, rows):
    b, n, p, h, k, g = case
    for lse in (0, 1):
        (need, got), = attend([(*case, lse, window, sinks)])
        if rows:
            flag = "true" if lse else "false"
            assert [x.kernel for x in got] == [f"kv_shared_rows_kernel<{flag}>"]
            assert got[0].grid == [k * -(-n * (h // k) // 16), 1, b]
            assert (need == 0) == (window == 0)
        else:
            assert len(got) == 2


def test_a_launch_too_large_is_refused():
    out = ll.run("""
need = lib.prichs_kv_cache_shared_attention_workspace(65535, 1, 1024, 1024, 4, 1)
rc = lib.prichs_kv_cache_shared_attention(P, 1 << 17, P, 1000, P, 4, P, P, P, 1, P, 1 << 17, None,
                                          65535, 1, 1024, 1024, 128, 0, 0, 1, P, need, None)
result = [rc, launches()]
""")
    assert out == [-1, []]


def test_the_gpu_tests_reach_every_variant():
    from tests import test_gpu_kv_shared as t

    calls, forms = [], []
    for groups, lens, n_q, heads, kv, window, sinks, form in t.FORMS:
        pages = t.pages_of(lens, n_q, heads, kv, form)
        for lse in (0, 1):
            calls.append((len(lens), n_q, pages, heads, kv, len(groups), lse, window, sinks))
            forms.append((form, window))
    got = [{x.kernel for x in ls} for _, ls in attend(calls)]
    kinds = {f"kv_shared_{k}<{n}{f}>" for f in ("true", "false")
             for k, n in (("kernel", "1, "), ("kernel", "2, "), ("join_kernel", "1, "),
                          ("join_kernel", "8, "), ("rows_kernel", ""))}
    assert set.union(*got) == kinds
    # With a window as well.
    assert {x.split("<")[0] + x.split("<")[1][0] for g, (_, w) in zip(got, forms) if w for x in g} \
        >= {"kv_shared_kernel1", "kv_shared_kernel2", "kv_shared_rows_kernelt"}
    assert all(not any("rows" in x for x in g) for g, f in zip(got, forms) if f[0] == 1)

    def kernel(size, heads, kv, pages, window=0):
        (_, got), = attend([(size, 1, t.wide(size, heads, kv) or pages, heads, kv, 1, 0, window,
                             0)])
        return got[0].kernel
    assert kernel(3, 8, 2, 7) == "kv_shared_rows_kernel<false>"
    assert kernel(4, 8, 2, 7) == kernel(260, 4, 1, 10, 120) == "kv_shared_kernel<1, false>"
    assert kernel(40, 8, 2, 7) == kernel(264, 4, 1, 10, 120) == "kv_shared_kernel<2, false>"


def rotate(cases):
    """Launches of a forward and a backward for each (rows, heads, kv heads, head dim, dtype)."""
    return [ll.as_launches(x) for x in ll.run(f"""
result = []
for r, h, k, d, dt in {cases!r}:
    H, K = d * h, d * k
    L.check(lib.prichs_qk_norm_rope_forward(P, H, P, K, P, P, P, P, 9, P, 0, 0, P, H, P, K, r, h, k,
                                            d, 1e-5, dt, None))
    need = lib.prichs_qk_norm_rope_backward_workspace(r, h, k, d)
    L.check(lib.prichs_qk_norm_rope_backward(P, H, P, K, P, H, P, K, P, P, P, P, 9, P, 0, 0, P, H,
                                             P, K, P, P, 0, r, h, k, d, 1e-5, dt, P, need, None))
    result.append(launches())
""")]


def test_rotation_takes_the_lanes_that_a_head_needs():
    from tests.test_gpu_qk_norm_rope import SHAPES

    cases = [(*s, dt) for s in SHAPES for dt in (0, 1)]
    names = set()
    for (rows, h, k, d, dt), got in zip(cases, rotate(cases)):
        lanes = 4 if d <= 32 else 8 if d <= 64 else 16 if d <= 128 else 32
        t = "unsigned short" if dt else "float"
        fwd, bwd, dw = got
        assert fwd.kernel == f"qk_norm_rope_kernel<{t}, {lanes}>"
        assert bwd.kernel == f"qk_norm_rope_bwd_kernel<{t}, {lanes}>"
        assert dw.kernel == "qk_norm_dw_kernel" and dw.grid[0] == 2 * d // 8
        assert bwd.grid[0] <= 1024
        names |= {fwd.kernel, bwd.kernel}
    assert len(names) == 16


def pages(cases):
    """Names of the launches of a reserve, a fork and a compaction for each (pages, rows)."""
    return ll.run(f"""
result = []
for n, b in {cases!r}:
    one = []
    need = lib.prichs_kv_pages_workspace(n, b, b)
    L.check(lib.prichs_kv_pages_reserve(P, n, P, 9, P, P, b, None, P, need, None))
    one.append([x[0] for x in launches()])
    L.check(lib.prichs_kv_pages_fork(P, P, n, P, 9, P, b, P, P, b, 3, None, P, need, None))
    one.append([x[0] for x in launches()])
    L.check(lib.prichs_kv_pages_compact(P, P, n, P, 9, b, 3, P, P, P, need, None))
    one.append([x[0] for x in launches()])
    result.append(one)
""")


def test_one_workgroup_plans_for_few_pages_and_rows():
    from tests.test_gpu_kv_pages import SCENES

    few = [["reserve_small_kernel"], ["fork_small_kernel", "fork_apply_kernel"],
           ["compact_small_kernel", "compact_apply_kernel"]]
    many = [["reserve_count_kernel", "reserve_list_kernel", "reserve_apply_kernel"],
            ["count_kernel", "fork_list_kernel", "fork_apply_kernel"],
            ["count_kernel", "compact_list_kernel", "compact_apply_kernel"]]
    got = pages([(16384, 4096), (16385, 4), (4, 4097), (0, 4)])
    assert got == [few, many, many[:2] + few[2:], few[:2] + [few[2][:1]]]
    seen = {x for one in pages([s[:2] for s in SCENES]) for call in one for x in call}
    assert seen == {x for one in (few, many) for call in one for x in call}
