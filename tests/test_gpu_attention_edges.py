"""Window attention of the longest sequence."""
import numpy as np
import pytest
import torch

import attention_ref as R
from prichs_amd import ops

pytestmark = pytest.mark.gpu
HD = 128


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def say(*a):
    print(*a, flush=True)


def near(got, want, bound, name):
    err = np.abs(host(got) - want)
    worst = np.argmax(err - bound)
    assert (err <= bound).all(), (name, err.flat[worst], bound.flat[worst])


def piece(q, k, v, d_out, a, z, W, sinks):
    """R.attention of the rows a .. z - 1 of one head (window W > 0) and the keys that
    they see, and those keys.  The sinks before the window take the places right before
    it, which leaves the mask as it is."""
    lo = max(0, a - W + 1)
    s = min(sinks, lo)
    keys = np.concatenate([np.arange(s), np.arange(lo, z)])
    return R.attention(q[a:z], k[keys], v[keys], W, s if lo > s else sinks, first=a - lo + s,
                       d_out=d_out[a:z]), keys


@pytest.mark.parametrize("spans", [[(0, 200), ((1 << 20) - 100, (1 << 20) + 100),
                                    ((1 << 21) - 300, 1 << 21)]])
def test_the_longest_sequence(cuda, spans):
    """2^21 rows: the first, some in the middle and the last, in both directions."""
    S, H, K, W = 1 << 21, 4, 1, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv, d_o = (torch.randn((S, n * HD), generator=g, device="cuda", dtype=torch.bfloat16)
                for n in (H + 2 * K, H))
    q, k, v = qkv[:, :H * HD], qkv[:, H * HD:(H + K) * HD], qkv[:, (H + K) * HD:]
    out, lse = ops.window_attention(q, k, v, 1, S, H, K, W, want_lse=True)
    dq, dk, dv = ops.window_attention_backward(d_o, q, k, v, out, lse, 1, S, H, K, W)
    for a, z in spans:
        say("rows:", a, z)
        lo, end = max(0, a - W), min(S, z + W)  # and what sees their keys
        rows = slice(lo, end)
        x = [host(t[rows]) for t in (q, k, v, d_o)]
        for h in range(H):
            c = slice(h * HD, (h + 1) * HD)
            # Rows from max(lo, a) on see nothing before lo.
            one, keys = piece(x[0][:, c], x[1], x[2], x[3][:, c], a - lo, end - lo, W, 0)
            for name, t in (("out", out), ("dq", dq)):
                near(t[a:z, c], one[name][:z - a], one["e_" + name][:z - a], name)
            if h == 0:
                sums = {e + n: 0 for n in ("dk", "dv") for e in ("", "e_")}
            for name in sums:
                sums[name] = sums[name] + one[name][keys >= a - lo][:z - a]
        for name, t in (("dk", dk), ("dv", dv)):
            near(t[a:z], sums[name], sums["e_" + name], name)
