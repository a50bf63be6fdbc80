"""Float64 reference of heads normed and rotated, with its gradients and the bounds that
f32 arithmetic with one rounding of the result is held to."""
import numpy as np
import torch

F = 2.0 ** -24


def norm_rope(x, w, cos, sin, eps, dtype, d=None):
    """x, d [rows, heads * hd], w [hd], cos / sin [rows, hd / 2], float64.  Returns out and
    (with d) dx, dw, and each one's bound under e_out, e_dx, e_dw for results of `dtype`."""
    rows, hd = len(x), len(w)
    u = torch.finfo(dtype).eps / 2
    x = x.reshape(rows, -1, hd)
    c, s = cos[:, None], sin[:, None]

    def turn(y, s):
        o = np.empty_like(y)
        o[..., 0::2] = y[..., 0::2] * c - y[..., 1::2] * s
        o[..., 1::2] = y[..., 0::2] * s + y[..., 1::2] * c
        return o

    def size(y):  # of the two terms of a rotated value
        o = np.empty_like(y)
        o[..., 0::2] = np.abs(y[..., 0::2] * c) + np.abs(y[..., 1::2] * s)
        o[..., 1::2] = np.abs(y[..., 0::2] * s) + np.abs(y[..., 1::2] * c)
        return o

    inv = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh = x * inv
    out = turn(xh * w, s)
    # The sum of squares is off by at most 14 roundings (8 values a lane, 32 lanes, the
    # mean, eps), inv by half of that and 3 more; then two products and the rotation's three
    # operations.
    e_out = 16 * F * size(xh * w) + u * np.abs(out)
    flat = lambda a: a.reshape(rows, -1)  # noqa: E731
    r = dict(out=flat(out), e_out=flat(e_out * (1 + u)))
    if d is None:
        return r
    d = d.reshape(rows, -1, hd)
    g, mag = turn(d, -s), size(d)
    t = g * w
    m = (t * xh).mean(-1, keepdims=True)
    mag_m = (mag * np.abs(w * xh)).mean(-1, keepdims=True)
    dx = inv * (t - xh * m)
    # t is off by 4 roundings of its terms, the mean by 14 more and inv's 10 twice; the
    # difference and the product with inv by 3 and inv's 10.
    e_dx = inv * F * (20 * mag * np.abs(w) + 64 * np.abs(xh) * mag_m) + u * np.abs(dx)
    # A lane adds up what its rows and heads (at most 4 of a row) give, at most 1024
    # workgroups of 8 groups or more share the rows; then 8 to 64 groups, and the workgroups'
    # sums by way of a thread's 8, 3 exchanges and 16 waves.
    chain = 4 * -(-rows * x.shape[1] // (4 * 1024 * 8)) + 64 + 64 + 20
    dw, mag_w = (g * xh).sum((0, 1)), (mag * np.abs(xh)).sum((0, 1))
    r.update(dx=flat(dx), e_dx=flat(e_dx * (1 + u)), dw=dw, e_dw=chain * F * mag_w)
    return r
