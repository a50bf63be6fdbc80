"""Norms of queries and keys with rotation: the rows without a position in outputs that the
call allocates, and backwards whose workgroups take several blocks of rows."""
import numpy as np
import pytest
import torch

import norm_rope_ref as R
from prichs_amd import ops
from tests.test_gpu_qk_norm_rope import BF, EPS, F32, case, close, i32, tensors, wide

pytestmark = pytest.mark.gpu


def poison(rows, heads, hd, dtype):
    """Memory of the outputs' sizes, full of NaN and free again: what the next allocations
    of those sizes are given."""
    held = [torch.full((rows, h * hd), float("nan"), dtype=dtype, device="cuda")
            for h in heads if h]
    assert all(t.isnan().all() for t in held)


# (rows, query heads, key heads, head_dim): every number of lanes a head can have, heads that
# leave lanes idle, groups of lanes that hold fewer than three heads, one operand alone.
PADDED = [(1, 12, 3, 128), (60, 3, 2, 128), (33, 4, 1, 8), (21, 7, 2, 40), (50, 6, 2, 80),
          (13, 2, 2, 192), (64, 0, 3, 128), (64, 2, 0, 64), (700, 12, 3, 128)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,Hq,Hk,hd", PADDED)
def test_rows_without_a_position_are_zeros_where_the_call_allocates(cuda, rows, Hq, Hk, hd, dtype):
    print("case:", rows, Hq, Hk, hd, dtype, flush=True)
    rng = np.random.default_rng(rows + hd)
    pos = rng.integers(0, 20, rows)
    pad = rng.random(rows) < 0.4
    pad[rows // 2] = True
    given = np.where(pad, rng.choice([-1, -(1 << 31), 20, (1 << 31) - 1], rows), pos)
    c = case(rows, Hq, Hk, hd, dtype, 5, pos, 20)
    for a in c["x"]:
        a[pad] = np.nan
    args, at = tensors(c, positions=i32(given.tolist()))
    poison(rows, c["heads"], hd, dtype)
    outs = ops.qk_norm_rope(*args, **at)
    into = [None if o is None else torch.full_like(o, 7.0) for o in outs]
    ops.qk_norm_rope(*args, **at, q_out=into[0], k_out=into[1])
    keep = torch.from_numpy(~pad).cuda()
    for i in range(2):
        if c["heads"][i] == 0:
            assert outs[i] is None
            continue
        assert (outs[i][~keep] == 0).all()
        if not pad.all():
            r = R.norm_rope(c["x"][i][~pad], c["w"][i], c["cos"][pos[~pad]], c["sin"][pos[~pad]],
                            EPS, dtype)
            close(outs[i][keep], r["out"], r["e_out"], "out")
        # Outputs that the caller gave: the same rows, and the others as they were.
        assert torch.equal(into[i][keep], outs[i][keep]) and (into[i][~keep] == 7).all()


def test_one_output_given_and_one_allocated(cuda):
    """The given one keeps its rows without a position, the allocated one has zeros there."""
    c = case(40, 3, 2, 128, BF, 6, None, 9)
    pos = [i % 9 if i % 3 else -1 for i in range(40)]
    args, at = tensors(c, positions=i32(pos))
    live = torch.tensor([p >= 0 for p in pos], device="cuda")
    want = ops.qk_norm_rope(*args, **at)
    for given in range(2):
        out = torch.full_like(want[given], 7.0)
        poison(40, c["heads"], 128, BF)
        got = ops.qk_norm_rope(*args, **at, **{("q_out", "k_out")[given]: out})
        assert got[given] is out and (out[~live] == 7).all()
        assert torch.equal(out[live], want[given][live])
        assert torch.equal(got[1 - given], want[1 - given]) and not want[given][~live].any()


def test_rows_that_lose_their_position_between_replays(cuda):
    """Outputs that a captured call allocated: rows with a position at one replay and
    without one at the next."""
    c = case(48, 4, 2, 64, BF, 7, None, 30)
    args, _ = tensors(c)
    pos = i32([0] * 48)
    ops.qk_norm_rope(*args, positions=pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.qk_norm_rope(*args, positions=pos)
    rng = np.random.default_rng(2)
    for _ in range(4):
        now = rng.integers(-12, 40, 48)
        pos.copy_(i32(now.tolist()))
        graph.replay()
        got = [t.clone() for t in held]
        live = torch.from_numpy((now >= 0) & (now < 30)).cuda()
        want = [torch.zeros_like(t) for t in held]
        ops.qk_norm_rope(*args, positions=pos, q_out=want[0], k_out=want[1])
        assert live.any() and not live.all()
        for a, b in zip(got, want):
            assert torch.equal(a, b) and not a[~live].any()


# Backwards of more than the 1024 workgroups that there are at most, and of one more: some
# take one block of rows more than others.  Every number of lanes a head can have.
LONG = [(3277, 12, 3, 128), (8195, 12, 3, 128), (9001, 3, 1, 256), (12001, 7, 2, 64),
        (20001, 12, 3, 32)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,Hq,Hk,hd", LONG)
def test_backward_of_more_blocks_than_workgroups(cuda, rows, Hq, Hk, hd, dtype):
    """Rows without a position among them, in the later blocks too."""
    print("case:", rows, Hq, Hk, hd, dtype, flush=True)
    rng = np.random.default_rng(rows + hd)
    pos = rng.integers(0, 50, rows)
    pad = rng.random(rows) < 0.1
    pad[rows - 40:rows - 20] = True
    c = case(rows, Hq, Hk, hd, dtype, rows + hd, pos, 50)
    for a in c["x"] + c["d"]:
        a[pad] = np.nan
    args, at = tensors(c, positions=i32(np.where(pad, -1, pos).tolist()))
    d = [wide(a, dtype) for a in c["d"]]
    got = ops.qk_norm_rope_backward(*d, *args, **at)
    keep = torch.from_numpy(~pad).cuda()
    for i in range(2):
        r = R.norm_rope(c["x"][i][~pad], c["w"][i], c["cos"][pos[~pad]], c["sin"][pos[~pad]], EPS,
                        dtype, c["d"][i][~pad])
        close(got[i][keep], r["dx"], r["e_dx"], "dx")
        close(got[2 + i], r["dw"], r["e_dw"], "dw")
        assert (got[i][~keep] == 0).all()
    # The same bits again, in place, and added to what there is.
    dw = [torch.full((hd,), 2.0, device="cuda") for _ in range(2)]
    again = ops.qk_norm_rope_backward(*d, *args, **at, d_q=d[0], d_k=d[1], d_wq=dw[0], d_wk=dw[1],
                                      accumulate=True)
    for i in range(2):
        assert torch.equal(again[i], got[i]) and torch.equal(dw[i], got[2 + i] + 2.0)
