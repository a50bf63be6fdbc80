"""Which kernels the window attention and the cache attention launch, on the CPU
(tests/launch_log.py), and that the GPU tests' shapes reach every one of them."""
import pytest

from tests import launch_log as ll


def _run(body):
    return ll.as_launches(ll.run(body))


def window(cases):
    """Launches of a forward and a backward for each (batch, seq_len, heads, kv heads,
    window, sinks)."""
    rows = ll.run(f"""
result = []
for b, S, h, k, w, s in {cases!r}:
    H, K = 128 * h, 128 * k
    L.check(lib.prichs_window_attention_forward(P, H, P, K, P, K, P, H, P, None, b, S, h, k, 128,
                                                w, s, 1, None))
    need = lib.prichs_window_attention_backward_workspace(b, S, h, k, w, s)
    L.check(lib.prichs_window_attention_backward(P, H, P, H, P, K, P, K, P, H, P, None, P, H, P, K,
                                                 P, K, b, S, h, k, 128, w, s, 1, P, need, None))
    result.append([need, launches()])
""")
    return [(need, ll.as_launches(x)) for need, x in rows]


def attend(cases):
    """Launches for each (batch, n_q, max_pages, heads, kv heads, window, sinks)."""
    rows = ll.run(f"""
result = []
for b, n, p, h, k, w, s in {cases!r}:
    need = lib.prichs_kv_cache_attention_workspace(b, n, h, k, p)
    L.check(lib.prichs_kv_cache_attention(P, 128 * h, P, 1000, P, p, P, P, 128 * h, None, b, n, h,
                                          k, 128, w, s, 1, P, need, None))
    result.append([need, launches()])
""")
    return [(need, ll.as_launches(x)) for need, x in rows]


def test_window_attention_variants():
    # 4 heads that share tiles, 32 rows: 4 * 3 * 64 workgroups of 32 rows; few of
    # them take 16 rows a wave, and heads 2 or 1 at a time where the group is odd.
    (_, big), (_, small), (_, two), (_, one) = window(
        [(4, 2048, 12, 3, 512, 4), (1, 777, 12, 3, 256, 4), (2, 300, 6, 3, 0, 0),
         (1, 300, 5, 5, 0, 0)])
    assert big[0].kernel == "attn_fwd_kernel<4, 2, true, false>" and big[0].grid == [3, 4, 64]
    assert big[1].kernel == "window_dq_kernel<4, 2, false>" and big[1].grid == [3, 4, 64]
    assert small[0].kernel == "attn_fwd_kernel<4, 1, true, false>" and small[0].grid == [3, 1, 49]
    assert small[1].kernel == "window_dq_kernel<4, 1, false>"
    assert two[0].kernel == "attn_fwd_kernel<2, 1, true, false>"
    assert one[0].kernel == "attn_fwd_kernel<1, 1, true, false>"
    for launches in (big, small, two, one):
        assert launches[2].kernel == "window_dkv_kernel<false>" and launches[2].lds <= 160 * 1024


def test_key_blocks_are_cut_where_few_or_seen_by_many_rows():
    # Blocks of 128 keys: whole where there are enough, the block of the sinks in
    # parts, every block in parts for one short sequence.
    shapes = [(4, 2048, 12, 3, 512, 0), (4, 2048, 12, 3, 512, 4), (1, 777, 12, 3, 256, 0),
              (8, 4096, 12, 3, 512, 0)]
    (need0, plain), (need1, sinks), (need2, short), (_, many) = window(shapes)
    assert plain[2].grid == [16, 3, 4] and len(plain) == 3
    assert sinks[2].grid[0] > 16 and sinks[3].kernel == "window_dkv_join_kernel"
    assert sinks[3].grid == [8 * 16, 3, 4]
    assert short[2].grid[0] > 7 and len(short) == 4
    assert many[2].grid == [32, 3, 8] and len(many) == 3
    # The partial sums of an item are 128 keys of d_k and of d_v in f32.
    stats = 4 * 12 * 64 * 64 * 4
    assert need0 == stats and need1 == stats + sinks[2].grid[0] * 12 * 2 * 128 * 128 * 4


def test_long_sequences_are_dealt_to_the_dies():
    # With a window from 8192 rows on: runs of 8 row blocks (8 key blocks) in a grid of one
    # dimension.
    (_, long), (_, ragged), (_, whole), (_, few) = window(
        [(3, 8192, 12, 3, 512, 0), (1, 8200, 6, 3, 64, 0), (3, 8192, 12, 3, 0, 0),
         (1, 8200, 4, 1, 64, 0)])
    assert long[0].kernel == "attn_fwd_kernel<4, 2, true, true>" and long[0].grid == [256 * 9, 1, 1]
    assert long[1].kernel == "window_dq_kernel<4, 2, true>" and long[1].grid == [256 * 9, 1, 1]
    assert long[2].kernel == "window_dkv_kernel<true>" and long[2].grid == [64 * 9, 1, 1]
    # 129 blocks of 64 rows: 17 runs for each of 3 pairs, in 7 rounds of the 8 dies.
    assert ragged[0].grid == [7 * 64, 1, 1] and ragged[1].grid == [7 * 64, 1, 1]
    assert whole[0].grid == [3, 3, 256] and whole[1].grid == [3, 3, 256]
    assert whole[2].kernel == "window_dkv_kernel<false>"
    assert few[0].grid == [1, 1, 513] and few[1].kernel == "window_dq_kernel<4, 1, false>"
    assert few[2].kernel == "window_dkv_kernel<true>"


@pytest.mark.parametrize("case,kernel,splits", [
    ((1, 1, 2, 12, 3, 0, 0), 4, 1), ((1, 1, 5, 12, 3, 0, 0), 8, 1), ((1, 1, 16, 12, 3, 0, 0), 8, 1),
    ((1, 1, 17, 12, 3, 0, 0), 4, 5), ((1, 1, 128, 12, 3, 0, 0), 4, 32),
    ((1, 1, 128, 12, 3, 700, 4), 8, 1), ((32, 1, 94, 12, 3, 0, 0), 4, 8),
    ((86, 1, 16, 12, 3, 0, 0), 4, 2), ((2, 256, 68, 12, 3, 0, 0), 4, 2),
    ((400, 1, 64, 8, 2, 0, 0), 4, 1)])
def test_cache_attention_splits(case, kernel, splits):
    (need, got), = attend([case])
    b, n, _, h, k = case[:5]
    tiles = -(-n * (h // k) // 16)
    assert got[0].kernel == f"kv_attend_kernel<{kernel}>" and got[0].grid == [k * tiles, splits, b]
    assert len(got) == (1 if splits == 1 else 2)
    if splits > 1:
        wide = splits > 8
        assert got[1].kernel == f"kv_join_kernel<{8 if wide else 1}>"
        assert got[1].grid[0] == (n * (h // k) if wide else -(-n * (h // k) // 8))
        assert need >= b * k * tiles * splits * 16 * 130 * 4


def test_the_gpu_tests_reach_every_variant():
    from tests.test_gpu_kv_cache import ATTEND, PAGE
    from tests.test_gpu_window_attention import CASES, LONG

    cases = [c[:6] for c in CASES] + [(*c[:5], 0) for c in LONG]
    names = {x.kernel for _, ls in window(cases) for x in ls}
    kinds = [(h, n, d) for h in (1, 2, 4) for n, d in ((1, "false"), (2, "false"), (2, "true"))]
    want = {f"attn_fwd_kernel<{h}, {n}, true, {d}>" for h, n, d in kinds}
    want |= {f"window_dq_kernel<{h}, {n}, {d}>" for h, n, d in kinds}
    assert names == want | {"window_dkv_kernel<false>", "window_dkv_kernel<true>",
                            "window_dkv_join_kernel"}
    cases = [(b, n, -(-max(max(lens), 1) // PAGE), h, k, w, s) for b, n, lens, h, k, w, s in ATTEND]
    names = {x.kernel for _, ls in attend(cases) for x in ls}
    assert names == {"kv_attend_kernel<4>", "kv_attend_kernel<8>", "kv_join_kernel<1>",
                     "kv_join_kernel<8>"}
