"""What the tests at the edges of the norms with rotation and of the attention over shared
pages reach, on the CPU (tests/launch_log.py), and the refusals of the norms whose padding
rows become zeros."""
import pytest

from prichs_amd import _lib as L
from tests import launch_log as ll
from tests import test_shared_prompt_abi as abi

ZEROS = [(c, s) for n, _, c, s in abi.BAD if n == "prichs_qk_norm_rope_forward"]


@pytest.mark.parametrize("change,status", ZEROS,
                         ids=[f"{'-'.join(map(str, c))}-{i}" for i, (c, _) in enumerate(ZEROS)])
def test_norms_with_zeros_refuse_what_those_without_do(change, status):
    lib = L.load()
    lib.prichs_clear_error()
    assert abi.call(lib, "prichs_qk_norm_rope_forward_zeros", {**abi.NORM, **change}) == status
    assert L.last_error().startswith("qk_norm_rope_forward_zeros")
    assert abi.call(lib, "prichs_qk_norm_rope_forward_zeros", {**abi.NORM, "rows": 0}) == L.PRICHS_OK


def test_zeros_are_written_where_rows_can_lie_outside_the_tables():
    """A kernel of its own for positions from memory; without them the host has checked that
    every row has one."""
    from tests.test_gpu_qk_norm_rope_edges import PADDED

    shapes = PADDED + [(9, 2, 1, 256)]
    got = ll.run(f"""
result = []
for r, h, k, d in {shapes!r}:
    for dt in (0, 1):
        H, K = d * h, d * k
        for pos, seq in ((P, 0), (None, 9)):
            L.check(lib.prichs_qk_norm_rope_forward_zeros(
                P, H, P, K, P, P, P, P, 9, pos, seq, 0, P, H, P, K, r, h, k, d, 1e-5, dt, None))
            result.append(launches())
""")
    at, names = iter(got), set()
    for _, _, _, d in shapes:
        lanes = 4 if d <= 32 else 8 if d <= 64 else 16 if d <= 128 else 32
        for t in ("float", "unsigned short"):
            for kind in ("_zeros", ""):
                (x,) = ll.as_launches(next(at))
                assert x.kernel == f"qk_norm_rope{kind}_kernel<{t}, {lanes}>"
                names.add(x.kernel)
    assert len(names) == 16


def test_long_backwards_take_more_blocks_than_workgroups():
    from tests.test_gpu_qk_norm_rope_edges import LONG
    from tests.test_shared_prompt_launches import rotate

    cases = [(*s, dt) for s in LONG for dt in (0, 1)]
    turns, lanes_seen = [], set()
    for (rows, h, k, d, _), (_, bwd, dw) in zip(cases, rotate(cases)):
        lanes = 4 if d <= 32 else 8 if d <= 64 else 16 if d <= 128 else 32
        blocks = -(-rows * -(-(h + k) // 3) // (256 // lanes))
        assert bwd.grid[0] == min(1024, blocks) and blocks > 1024 and blocks % 1024
        assert bwd.kernel.endswith(f", {lanes}>")
        turns.append(-(-blocks // 1024))
        lanes_seen.add(lanes)
    assert lanes_seen == {4, 8, 16, 32} and min(turns) == 2 and max(turns) >= 3


def attend(batch, n_q, pages, heads, kv, groups, window=0):
    from tests.test_shared_prompt_launches import attend as launches

    ((need, got),) = launches([(batch, n_q, pages, heads, kv, groups, 1, window, 0)])
    return need, got[0].kernel


def test_attention_over_long_tables_is_taken_in_parts():
    from tests import test_gpu_kv_shared_edges as t

    # Parts without a softmax: every form of a call, with a window too.
    for size, pages, window, form in t.TABLES:
        _, name = attend(size, 1, pages or -(-t.TOP // 64), 8, 2, 1, window)
        assert name == ("kv_shared_rows_kernel<true>" if form == "rows" else
                        f"kv_shared_kernel<{form}, true>")
    # Tables full of shared pages.
    got = [attend(size, n_q, pages, 8, 2, 1) for size, pages, n_q in t.FULL]
    assert [x for _, x in got] == ["kv_shared_kernel<1, true>", "kv_shared_kernel<2, true>"]
    # Both of two graphs at once have a workspace, in both heights of a tile.
    got = [attend(len(lens), n_q, p or -(-max(lens) // 64), h, k, len(groups))
           for groups, lens, n_q, h, k, p in t.PAIR]
    assert all(need > 0 for need, _ in got)
    assert [x for _, x in got] == ["kv_shared_kernel<1, true>", "kv_shared_kernel<2, true>"]
    # The captured step.
    need, name = attend(len(t.PROMPTS) * t.EACH, 1, t.STEP_COLUMNS, *t.STEP_HEADS, len(t.PROMPTS))
    assert need > 0 and name == "kv_shared_kernel<1, true>"
    # lse in every kernel that gives it.
    names = set()
    for groups, lens, n_q, heads, kv, window, _, form in t.FORMS[::2]:
        pages = t.pages_of(lens, n_q, heads, kv, form)
        names.add(attend(len(lens), n_q, pages, heads, kv, len(groups), window)[1])
    assert names == {"kv_shared_rows_kernel<true>", "kv_shared_kernel<1, true>",
                     "kv_shared_kernel<2, true>"}
