"""Norms of queries and keys with their rotation, and the gradients, through the C ABI
against norm_rope_ref in 64 bits and its bounds."""
import numpy as np
import pytest
import torch

import norm_rope_ref as R
from prichs_amd import _lib as L
from prichs_amd import ops

pytestmark = pytest.mark.gpu
EPS = 1e-5
BF, F32 = torch.bfloat16, torch.float32


def dev(a, dtype=F32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to("cuda").to(dtype)


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def values(rng, shape, dtype, std=1.0):
    """f32 values that `dtype` holds exactly, as float64."""
    t = torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32))
    return t.to(dtype).double().numpy()


def case(rows, Hq, Hk, hd, dtype, seed, positions, cache_rows):
    rng = np.random.default_rng(seed)
    c = dict(rows=rows, heads=(Hq, Hk), hd=hd, dtype=dtype, positions=positions)
    c["x"] = [values(rng, (rows, h * hd), dtype, 3.0) for h in (Hq, Hk)]
    c["d"] = [values(rng, (rows, h * hd), dtype) for h in (Hq, Hk)]
    c["w"] = [values(rng, (hd,), F32, 0.3) + 1 for _ in range(2)]
    c["w"] = [w.astype(np.float32).astype(np.float64) for w in c["w"]]
    angle = np.arange(cache_rows)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)
    c["cos"], c["sin"] = (f(angle).astype(np.float32).astype(np.float64) for f in (np.cos, np.sin))
    return c


def wide(a, dtype, pad=8):
    """A row view of a wider buffer."""
    t = torch.full((len(a) + 1, a.shape[1] + 2 * pad), float("nan"), dtype=dtype, device="cuda")
    t[:len(a), pad:pad + a.shape[1]] = dev(a, dtype)
    return t[:len(a), pad:pad + a.shape[1]]


def tensors(c, **at):
    dt = c["dtype"]
    q, k = (wide(a, dt) if h else None for a, h in zip(c["x"], c["heads"]))
    w = [dev(x) for x in c["w"]]
    return (q, k, *w, dev(c["cos"]), dev(c["sin"]), *c["heads"], c["hd"], EPS), at


def close(got, want, bound, what):
    err = np.abs(host(got) - want)
    assert (err <= bound).all(), (what, err.max(), err.flat[np.argmax(err - bound)],
                                  bound.flat[np.argmax(err - bound)])


# (rows, query heads, key heads, head_dim): one token, a few, odd numbers of heads and rows,
# every number of lanes a head can have, heads that leave lanes idle.
SHAPES = [(1, 12, 3, 128), (33, 12, 3, 128), (700, 5, 1, 128), (40, 4, 4, 64), (17, 3, 3, 8),
          (9, 2, 1, 32), (21, 7, 2, 40), (50, 6, 2, 80), (13, 2, 2, 192), (30, 3, 1, 256),
          (64, 0, 3, 128), (64, 3, 0, 128), (3000, 12, 3, 128)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,Hq,Hk,hd", SHAPES)
def test_forward_and_backward(cuda, rows, Hq, Hk, hd, dtype):
    print("case:", rows, Hq, Hk, hd, dtype, flush=True)
    rng = np.random.default_rng(rows + hd)
    pos = rng.integers(0, 50, rows)
    c = case(rows, Hq, Hk, hd, dtype, rows + Hq + hd, pos, 50)
    args, at = tensors(c, positions=i32(pos))
    outs = ops.qk_norm_rope(*args, **at)
    d = [wide(a, dtype) if h else None for a, h in zip(c["d"], c["heads"])]
    got = ops.qk_norm_rope_backward(*d, *args, **at)
    for i in range(2):
        if c["heads"][i] == 0:
            assert outs[i] is None and got[i] is None and got[2 + i] is None
            continue
        r = R.norm_rope(c["x"][i], c["w"][i], c["cos"][pos], c["sin"][pos], EPS, dtype, c["d"][i])
        close(outs[i], r["out"], r["e_out"], "out")
        close(got[i], r["dx"], r["e_dx"], "dx")
        close(got[2 + i], r["dw"], r["e_dw"], "dw")
    # The same bits again, and in place (outputs over inputs, gradients over gradients).
    for a, b in zip(got, ops.qk_norm_rope_backward(*d, *args, **at)):
        assert a is None or torch.equal(a, b)
    into = dict(zip(("d_q", "d_k"), d))
    for a, b in zip(got, ops.qk_norm_rope_backward(*d, *args, **at, **into)):
        assert a is None or torch.equal(a, b)
    ops.qk_norm_rope(*args, **at, q_out=args[0], k_out=args[1])
    for a, b in zip(outs, args[:2]):
        assert a is None or torch.equal(a, b)


def test_positions_from_the_rows_and_weights_added(cuda):
    """Three sequences of 11 rows from position 5 on; weights' gradients added to what is
    there."""
    c = case(33, 4, 2, 128, F32, 3, None, 16)
    args, at = tensors(c, seq_len=11, pos_offset=5)
    pos = np.tile(np.arange(5, 16), 3)
    outs = ops.qk_norm_rope(*args, **at)
    d = [dev(a) for a in c["d"]]
    dw = [torch.full((128,), 2.0, device="cuda") for _ in range(2)]
    got = ops.qk_norm_rope_backward(*d, *args, **at, d_wq=dw[0], d_wk=dw[1], accumulate=True)
    assert got[2] is dw[0] and got[3] is dw[1]
    for i in range(2):
        r = R.norm_rope(c["x"][i], c["w"][i], c["cos"][pos], c["sin"][pos], EPS, F32, c["d"][i])
        close(outs[i], r["out"], r["e_out"], "out")
        close(got[i], r["dx"], r["e_dx"], "dx")
        close(dw[i], r["dw"] + 2, r["e_dw"] + 2.0 ** -24 * (np.abs(r["dw"]) + 2), "dw")
    # One sequence where no length is given.
    first = (args[0][:11], args[1][:11], *args[2:])
    assert torch.equal(ops.qk_norm_rope(*first, pos_offset=5)[0], outs[0][:11])


def test_padding_rows_stay_and_add_nothing(cuda):
    rng = np.random.default_rng(4)
    pos = rng.integers(0, 20, 60)
    pad = rng.random(60) < 0.4
    given = np.where(pad, rng.choice([-1, -(1 << 31), 20, (1 << 31) - 1], 60), pos)
    c = case(60, 3, 2, 128, BF, 5, pos, 20)
    for a in c["x"] + c["d"]:
        a[pad] = np.nan
    args, at = tensors(c, positions=i32(given.tolist()))
    out = [torch.full((60, h * 128), 7.0, dtype=BF, device="cuda") for h in (3, 2)]
    ops.qk_norm_rope(*args, **at, q_out=out[0], k_out=out[1])
    got = ops.qk_norm_rope_backward(*[dev(a, BF) for a in c["d"]], *args, **at)
    for i in range(2):
        r = R.norm_rope(c["x"][i][~pad], c["w"][i], c["cos"][pos[~pad]], c["sin"][pos[~pad]], EPS,
                        BF, c["d"][i][~pad])
        keep = torch.from_numpy(~pad).cuda()
        close(out[i][keep], r["out"], r["e_out"], "out")
        close(got[i][keep], r["dx"], r["e_dx"], "dx")
        close(got[2 + i], r["dw"], r["e_dw"], "dw")
        assert (out[i][~keep] == 7).all() and (got[i][~keep] == 0).all()


def test_zeros_infinities_and_nan_stay_in_their_head(cuda):
    c = case(8, 4, 1, 128, F32, 6, None, 8)
    c["x"][0][1, :128] = 0
    c["x"][0][2, 130] = np.inf
    c["x"][0][3, 260] = np.nan
    args, at = tensors(c)
    q, _ = ops.qk_norm_rope(*args, **at)
    pos = np.arange(8)
    h = host(q).reshape(8, 4, 128)
    bad = np.zeros((8, 4), bool)
    bad[2, 1] = bad[3, 2] = True
    with np.errstate(all="ignore"):
        r = R.norm_rope(c["x"][0], c["w"][0], c["cos"][pos], c["sin"][pos], EPS, F32)
    err = np.abs(h - r["out"].reshape(h.shape)) <= r["e_out"].reshape(h.shape)
    assert err[~bad].all() and not h[1, 0].any()
    assert np.isnan(h[2, 1]).any() and np.isnan(h[3, 2]).all()


def test_no_rows(cuda):
    c = case(0, 2, 1, 128, BF, 7, None, 4)
    q, k = (torch.empty((0, h * 128), dtype=BF, device="cuda") for h in (2, 1))
    args, at = tensors(c)
    args = (q, k, *args[2:])
    assert ops.qk_norm_rope(*args, **at)[0].shape == (0, 256)
    got = ops.qk_norm_rope_backward(q, k, *args, **at)
    assert (got[2] == 0).all() and (got[3] == 0).all()
    dw = [torch.full((128,), 3.0, device="cuda") for _ in range(2)]
    ops.qk_norm_rope_backward(q, k, *args, **at, d_wq=dw[0], d_wk=dw[1], accumulate=True)
    assert (dw[0] == 3).all() and (dw[1] == 3).all()


def test_offsets_past_32_bits(cuda):
    """Rows 2^20 elements apart: the last ones lie past 2^32 elements."""
    rows, ld = 4200, 1 << 20
    buf = torch.empty((rows * ld,), dtype=BF, device="cuda")
    q = buf.as_strided((rows, 128), (ld, 1), 0)
    k = buf.as_strided((rows, 128), (ld, 1), 128)
    c = case(rows, 1, 1, 128, BF, 8, np.arange(rows) % 7, 7)
    q.copy_(dev(c["x"][0], BF)), k.copy_(dev(c["x"][1], BF))
    args, at = tensors(c, seq_len=7)
    narrow = ops.qk_norm_rope(*args, **at)
    d = [dev(a, BF) for a in c["d"]]
    want = ops.qk_norm_rope_backward(*d, *args, **at)
    far = (q, k, *args[2:])
    got = ops.qk_norm_rope_backward(*d, *far, **at)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    ops.qk_norm_rope(*far, **at, q_out=q, k_out=k)
    assert torch.equal(q.contiguous(), narrow[0]) and torch.equal(k.contiguous(), narrow[1])


def test_graph_and_streams(cuda):
    """A captured forward and backward, replayed on other inputs and positions between eager
    calls; a call on a stream of its own."""
    c = case(64, 4, 2, 128, BF, 9, None, 100)
    args, _ = tensors(c)
    pos = i32([0] * 64)
    d = [dev(a, BF) for a in c["d"]]

    def step():
        return [*ops.qk_norm_rope(*args, positions=pos),
                *ops.qk_norm_rope_backward(*d, *args, positions=pos)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    rng = np.random.default_rng(1)
    for i in range(4):
        pos.copy_(i32(rng.integers(-1, 100, 64).tolist()))
        args[0].copy_(dev(values(rng, (64, 512), BF), BF))
        for t in held:
            t.zero_()
        graph.replay()
        got = [t.clone() for t in held]
        want = [torch.zeros_like(t) for t in held[:2]]
        ops.qk_norm_rope(*args, positions=pos, q_out=want[0], k_out=want[1])
        want += ops.qk_norm_rope_backward(*d, *args, positions=pos)
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    pos.fill_(3)
    a = ops.qk_norm_rope(*args, positions=pos)
    side.wait_stream(torch.cuda.current_stream())
    b = ops.qk_norm_rope(*args, positions=pos, stream=side)
    side.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_against_differences(cuda):
    """Gradients of sum(out * d) in f32 against central differences of the 64-bit formula."""
    c = case(3, 1, 1, 16, F32, 11, None, 3)
    args, at = tensors(c)
    got = ops.qk_norm_rope_backward(*[dev(a) for a in c["d"]], *args, **at)
    pos = np.arange(3)

    def loss(x, w):
        return (R.norm_rope(x, w, c["cos"][pos], c["sin"][pos], EPS, F32)["out"] * c["d"][0]).sum()

    step = 1e-5
    for name, base, grad in (("x", c["x"][0], got[0]), ("w", c["w"][0], got[2])):
        num = np.zeros_like(base)
        for i in np.ndindex(base.shape):
            e = np.zeros_like(base)
            e[i] = step
            args2 = ((c["x"][0] + e, c["w"][0]), (c["x"][0] - e, c["w"][0])) if name == "x" else \
                ((c["x"][0], c["w"][0] + e), (c["x"][0], c["w"][0] - e))
            num[i] = (loss(*args2[0]) - loss(*args2[1])) / (2 * step)
        # Differences are off by step^2 and 2^-52 / step; f32 by some 2^-20 of the sums.
        assert np.abs(host(grad) - num).max() < 1e-5 * (1 + np.abs(num).max()), name


def test_wrapper_refusals(cuda):
    c = case(4, 2, 1, 128, BF, 12, None, 4)
    args, _ = tensors(c)
    q, k, wq, wk, cos, sin = args[:6]
    f = ops.qk_norm_rope
    with pytest.raises(TypeError):
        f(q.half(), k.half(), wq, wk, cos, sin, 2, 1)
    with pytest.raises(TypeError):
        f(q, k.float(), wq, wk, cos, sin, 2, 1)
    with pytest.raises(ValueError):
        f(q, k[:3], wq, wk, cos, sin, 2, 1)
    with pytest.raises(ValueError):
        f(q, k, wq[:64], wk, cos, sin, 2, 1)
    with pytest.raises(ValueError):
        f(q, k, wq, wk, cos[:, :32], sin[:, :32], 2, 1)
    with pytest.raises(ValueError):
        f(q, k, wq, wk, cos, sin[:3], 2, 1)
    with pytest.raises(ValueError):
        f(q, k, wq, wk, cos, sin, 2, 1, positions=i32([0, 1]))
    with pytest.raises(ValueError):
        f(q, None, wq, wk, cos, sin, 2, 1)
    with pytest.raises(ValueError):
        f(None, None, wq, wk, cos, sin, 0, 0)
    with pytest.raises(ValueError):
        f(q, k, wq, wk, cos.cpu(), sin, 2, 1)
    with pytest.raises(L.PrichsError):  # position 4 is past the tables
        f(q, k, wq, wk, cos, sin, 2, 1, pos_offset=1)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_backward(q, k, q, k, wq, wk, cos, sin, 2, 1, accumulate=True)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_backward(q[:3], k[:3], q, k, wq, wk, cos, sin, 2, 1)
