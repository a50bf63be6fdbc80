"""Limits of the window attention and KV cache entry points as documented, on the
CPU (tests/launch_log.py): the largest calls launch, the next ones are refused."""
import os
import subprocess

import pytest

from prichs_amd import _lib as L
from tests import launch_log as ll

ITEMS = (1 << 28) - 16  # of one cache call: batch * n * n_kv_heads


def cache_call(name, batch, n, kv):
    """(status, launches) of a cache write or read."""
    return ll.run(f"""
rc = lib.prichs_kv_cache_{name}(P, 4, P, 2, P, None, P, 128 * {kv}, P, 128 * {kv}, {batch}, {n}, {kv},
                                128, 1, None)
result = [rc, launches()]
""")


@pytest.mark.parametrize("name", ["write", "read"])
def test_items_of_a_cache_call(name):
    rc, got = cache_call(name, 1, ITEMS, 1)
    assert rc == L.PRICHS_OK and len(got) == 1
    (_, _, grid, block, _, _), = got
    assert grid[0] * block < 1 << 32 and grid[0] * block // 16 == ITEMS
    for batch, n, kv in ((1, ITEMS + 1, 1), (1, (1 << 28) - 1, 1), (3, ((1 << 28) - 1) // 3, 1),
                         (5, ((1 << 28) - 1) // 15, 3)):
        assert ITEMS < batch * n * kv < 1 << 28
        assert cache_call(name, batch, n, kv) == [L.PRICHS_ERR_INVALID_ARGUMENT, []], (batch, n, kv)


# Answers to hipFuncSetAttribute and to the count of compute units that a test
# chooses, before launch_log's.
STANDINS = r"""
#define __HIP_PLATFORM_AMD__
#include <hip/hip_runtime_api.h>
#include <cstdlib>
extern "C" hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int) {
  return std::getenv("REFUSE_LDS") ? hipErrorInvalidValue : hipSuccess;
}
extern "C" hipError_t hipDeviceGetAttribute(int *v, hipDeviceAttribute_t, int) {
  const char *cus = std::getenv("CUS");
  *v = cus ? std::atoi(cus) : 256;
  return hipSuccess;
}
"""


@pytest.fixture(scope="module")
def standins(tmp_path_factory):
    """A library to load first (LD_PRELOAD) that reads REFUSE_LDS and CUS."""
    at = tmp_path_factory.mktemp("standins")
    (at / "standins.cpp").write_text(STANDINS)
    so = at / "standins.so"
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-fPIC", "-shared", "-w", "-I",
                    os.path.join(ll.ROCM, "include"), str(at / "standins.cpp"), "-o", str(so)],
                   check=True)
    return str(so)


def window_calls(cases, **env):
    """For each (batch, seq_len, heads, kv heads, window, sinks): status and launches of
    a forward, the workspace's size, status and launches of a backward."""
    rows = ll.run(f"""
result = []
for b, S, h, k, w, s in {cases!r}:
    H, K = 128 * h, 128 * k
    f = lib.prichs_window_attention_forward(P, H, P, K, P, K, P, H, P, None, b, S, h, k, 128, w, s, 1,
                                            None)
    f = [f, launches()]
    need = lib.prichs_window_attention_backward_workspace(b, S, h, k, w, s)
    g = lib.prichs_window_attention_backward(P, H, P, H, P, K, P, K, P, H, P, None, P, H, P, K, P, K,
                                             b, S, h, k, 128, w, s, 1, P, need, None)
    result.append([*f, need, g, launches()])
""", **env)
    return [(f, ll.as_launches(x), need, g, ll.as_launches(y)) for f, x, need, g, y in rows]


def test_no_launch_before_a_refused_lds_limit(standins):
    for case in ((1, 100, 4, 1, 0, 0), (1, 9000, 48, 12, 64, 0)):
        (f, fwd, _, g, bwd), = window_calls([case], LD_PRELOAD=standins, REFUSE_LDS="1")
        assert (f, g) == (L.PRICHS_ERR_HIP, L.PRICHS_ERR_HIP)
        assert fwd == [] and bwd == []


@pytest.mark.parametrize("heads,kv", [(4, 1), (12, 3), (2, 1), (1, 1), (3, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 0), (4096, 4)])
def test_the_longest_sequence(heads, kv, window, sinks):
    """2^21 rows in both directions, whatever the heads, in grids of at most 65535 row
    blocks; one row more is refused by all three entry points."""
    longest, past = window_calls([(1, 1 << 21, heads, kv, window, sinks),
                                  (1, (1 << 21) + 1, heads, kv, window, sinks)])
    f, fwd, need, g, bwd = longest
    assert (f, g) == (L.PRICHS_OK, L.PRICHS_OK) and need > 0
    for x in (*fwd, *bwd):
        assert x.grid[0] * x.block < 1 << 32 and max(x.grid[1:]) <= 65535, x
    # 128 rows a workgroup, or 64 of each of two heads: all of them.
    share = 1 if (heads // kv) % 2 else 2
    for x in (fwd[0], bwd[0]):
        n = (1 << 21) // (128 // share) * (heads // share)
        assert f"<{share}, 2," in x.kernel
        assert x.grid[0] * x.grid[1] * x.grid[2] == n, x
    f, fwd, need, g, bwd = past
    assert (f, need, g) == (L.PRICHS_ERR_INVALID_ARGUMENT, 0, L.PRICHS_ERR_INVALID_ARGUMENT)
    assert fwd == [] and bwd == []


def rows_a_wave(launch):
    """16-row blocks of a wave of a forward or d_q kernel."""
    return launch.kernel.split(",")[1].strip()


@pytest.mark.parametrize("cus,rows", [(256, "1111"), (64, "1122"), (32, "1222"), (512, "1111")])
def test_both_directions_take_16_rows_a_wave_by_one_rule(standins, cus, rows):
    """Where the workgroups of 32 rows a wave are at most one and a half a CU of the
    device: 75, 192 and 384 of 777, 2048 and 4096 rows, and 3 of one row."""
    cases = [(1, S, 12, 3, 0, 0) for S in (1, 777, 2048, 4096)]
    calls = window_calls(cases, LD_PRELOAD=standins, CUS=str(cus))
    assert "".join(rows_a_wave(c[1][0]) for c in calls) == rows
    assert "".join(rows_a_wave(c[4][0]) for c in calls) == rows


@pytest.mark.parametrize("B,S,H,K,W", [(64, 2048, 12, 3, 512), (6, 1500, 4, 4, 60),
                                       (10, 1100, 4, 4, 60)])
def test_workspace_holds_partial_sums_of_cut_blocks_only(B, S, H, K, W):
    """With a few sinks the first block of 128 keys is cut into items and the others are
    not; 128 KiB of f32 sums an item."""
    (_, _, need, _, bwd), = window_calls([(B, S, H, K, W, 4)])
    assert bwd[-1].kernel == "window_dkv_join_kernel"
    items, blocks = bwd[1].grid[0], -(-S // 128)
    stats = -(-S // 32) * 256 * B * H
    assert 1 < items - (blocks - 1) < items
    assert need == -(-stats // 256) * 256 + (items - (blocks - 1)) * B * K * (128 << 10)


def test_workspace_of_a_large_batch_with_sinks():
    (_, _, none, _, _), (_, _, few, _, _) = window_calls([(16, 8192, 32, 8, 512, s)
                                                          for s in (0, 4)])
    assert none == 32 << 20 and few <= 256 << 20


def test_window_attention_without_lse_has_kernels_of_its_own():
    """One for each that forms it, in the same grids."""
    from tests.test_gpu_attention_edges import WITHOUT_LSE

    rows = ll.run(f"""
result = []
for b, S, h, k, w, s in {WITHOUT_LSE!r}:
    for lse in (P, None):
        H, K = 128 * h, 128 * k
        L.check(lib.prichs_window_attention_forward(P, H, P, K, P, K, P, H, lse, None, b, S, h, k, 128,
                                                    w, s, 1, None))
    result.append(launches())
""")
    seen = set()
    for one, two in (ll.as_launches(x) for x in rows):
        kind = one.kernel[len("attn_fwd_kernel<"):].replace("true, ", "", 1)
        assert two.kernel == "window_fwd_kernel<" + kind and one[2:] == two[2:]
        seen.add(kind)
    assert len(seen) == 9


def test_cache_attention_with_lse_has_kernels_of_its_own():
    """One for each without, in the same grids, from workspaces of one size."""
    rows = ll.run("""
result = []
for b, n, p in ((1, 1, 5), (1, 1, 16), (1, 1, 2), (1, 1, 128), (2, 256, 68)):
    need = lib.prichs_kv_cache_attention_workspace(b, n, 12, 3, p)
    for lse in (None, P):
        L.check(lib.prichs_kv_cache_attention(P, 1536, P, 1000, P, p, P, P, 1536, lse, b, n, 12, 3, 128,
                                              0, 0, 1, P, need, None))
        result.append(launches())
""")
    seen = set()
    for one, two in zip(*(map(ll.as_launches, rows[i::2]) for i in (0, 1))):
        assert len(one) == len(two)
        for x, y in zip(one, two):
            assert y.kernel == x.kernel.replace("_kernel", "_lse_kernel") and x[2:4] == y[2:4]
            seen.add(y.kernel)
    assert seen == {"kv_attend_lse_kernel<4>", "kv_attend_lse_kernel<8>", "kv_join_lse_kernel<1>",
                    "kv_join_lse_kernel<8>"}


def test_gpu_tests_deal_rows_and_key_blocks_and_join_cut_blocks_in_one_call():
    from tests.test_gpu_attention_edges import DEALT

    share = set()
    for _, fwd, _, _, bwd in window_calls([c[:6] for c in DEALT]):
        assert fwd[0].kernel.endswith("true, true>") and bwd[0].kernel.endswith("2, true>")
        assert [x.kernel for x in bwd[1:]] == ["window_dkv_kernel<true>", "window_dkv_join_kernel"]
        share.add(fwd[0].kernel)
    assert len(share) == 3
