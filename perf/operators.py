"""Window attention, its gradient, the 4-bit KV cache and the attention over it:
their performance cases and plain forms.

Kinds of case:

* ``window``  a causal GQA attention forward with a sliding window and sinks
              over whole sequences (``ops.window_attention``).
* ``train``   the same with its backward: outputs and the gradients of q, k, v
              (``ops.window_attention_backward``).
* ``cache``   new tokens quantised into a paged 4-bit cache and read back
              (``ops.kv_cache_write``, ``ops.kv_cache_read``).
* ``attend``  the attention of a few new tokens over a filled 4-bit cache
              (``ops.kv_cache_attention``).

A query at position i sees the keys j <= i with i - j < window (window 0: all
of them) or j < sinks.  Sequences of a padded batch end at their own length;
rows past it give zeros.  The cache holds groups of 32 values along the head as
e2m1 codes with one power-of-two scale: the least, from 2^-126 to 2^125, whose
sevenfold reaches the group's largest magnitude.
"""
import math

import torch

own = False

HD = 128
GROUP = 32
PAGE = 64
SCALE = 1.0 / math.sqrt(HD)
CHUNK = 512  # query rows whose scores the plain forms hold at once


def _attn(kind, name, batch, S, window, sinks, heads=12, kv=3, ragged=False):
    return dict(name=name, kind=kind, batch=batch, S=S, window=window, sinks=sinks, heads=heads,
                kv=kv, ragged=ragged)


def _cache(name, batch, n, past, kv=3, dtype="bf16"):
    return dict(name=name, kind="cache", batch=batch, n=n, past=past, kv=kv, dtype=dtype)


def _attend(name, batch, n_q, length, window, sinks, heads=12, kv=3, ragged=False):
    return dict(name=name, kind="attend", batch=batch, n_q=n_q, length=length, window=window,
                sinks=sinks, heads=heads, kv=kv, ragged=ragged)


def listed():
    return [
        # One prompt of odd length, its window shorter than the prompt.
        _attn("window", "window_1x777", 1, 777, 256, 4),
        # A batch of whole sequences at the block's training length.
        _attn("window", "window_4x2048", 4, 2048, 512, 4),
        # One long document.
        _attn("window", "window_1x16384", 1, 16384, 4096, 16),
        # A training step over a padded batch of short sequences.
        _attn("train", "train_3x500_ragged", 3, 500, 128, 4, ragged=True),
        # A training step at the block's training length.
        _attn("train", "train_4x2048", 4, 2048, 512, 4),
        # A training step on longer sequences, every earlier token visible.
        _attn("train", "train_1x4096_full", 1, 4096, 0, 0),
        # One decode step's keys and values of 32 sequences.
        _cache("cache_32x1", 32, 1, 1000),
        # The keys and values of four prompts.
        _cache("cache_4x2048", 4, 2048, 0),
        # A decode step of one sequence over a long cache.
        _attend("attend_1x1_8192", 1, 1, 8192, 0, 0),
        # A decode step of 32 sequences of different lengths, windowed.
        _attend("attend_32x1_ragged", 32, 1, 6000, 4096, 4, ragged=True),
        # Eight sequences with five drafted tokens each, to be verified.
        _attend("attend_8x5_4096", 8, 5, 4096, 0, 0),
        # A chunk of two prompts behind what the cache already holds.
        _attend("attend_2x256_4352", 2, 256, 4352, 2048, 4),
    ]


def _loguniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _pairs(S, window, sinks, first=0):
    """Visible (query, key) pairs of queries first .. S - 1."""
    total = 0
    for i in range(first, S):
        lo = 0 if window == 0 else max(0, i - window + 1)
        total += i + 1 - lo + min(lo, sinks)
    return total


def draw(rng):
    kind = rng.choice(["window", "window", "train", "train", "cache", "attend", "attend", "attend"])
    heads, kv = rng.choice([(12, 3), (12, 3), (8, 2), (4, 4), (6, 3), (8, 1), (10, 2)])
    if kind == "cache":
        n = _loguniform(rng, 1, 2048)
        return _cache("cache", rng.randint(1, 4 if n > 256 else 32), n,
                      rng.choice([0, rng.randint(0, 2000)]), kv=min(kv, 3),
                      dtype=rng.choice(["bf16", "bf16", "f32"]))
    window = rng.choice([0, _loguniform(rng, 1, 4096), _loguniform(rng, 64, 2048)])
    sinks = 0 if window == 0 else rng.choice([0, 4, rng.randint(1, 100)])
    if kind == "attend":
        length = _loguniform(rng, 1, 8192)
        n_q = min(length, rng.choice([1, 1, 1, rng.randint(2, 8), _loguniform(rng, 9, 256)]))
        top = 2 if n_q > 64 else 8 if n_q > 8 else 32
        return _attend("attend", rng.randint(1, top), n_q, length, window, sinks, heads, kv,
                       ragged=rng.random() < 0.5)
    S = _loguniform(rng, 1, 8192 if kind == "window" else 2048)
    batch = rng.randint(1, 4 if S <= 2048 else 1)
    return _attn(kind, kind, batch, S, window, sinks, heads, kv, ragged=rng.random() < 0.5)


# ------------------------------------------------------------------- inputs --
def _lengths(case, top, low, g):
    if not case["ragged"]:
        return [top] * case["batch"]
    r = torch.rand((case["batch"],), generator=g, device="cuda").cpu()
    return [min(top, low + int(x * (top - low + 1))) for x in r.tolist()]


def _inputs(case, seed):
    """The case's tensors, from the seed alone (k and v of what a cache holds)."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    def i32(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    st = dict(case=case)
    if case["kind"] in ("window", "train"):
        rows = case["batch"] * case["S"]
        # q, k and v as a block has them: column slices of one projection.
        H, K = case["heads"] * HD, case["kv"] * HD
        qkv = randn(rows, H + 2 * K)
        st.update(q=qkv[:, :H], k=qkv[:, H:H + K], v=qkv[:, H + K:])
        st["lens"] = _lengths(case, case["S"], 1, g)
        st["seq_lens"] = i32(st["lens"]) if case["ragged"] else None
        if case["kind"] == "train":
            st["d_out"] = randn(rows, H, std=0.1)
        return st
    kv, batch = case["kv"], case["batch"]
    if case["kind"] == "cache":
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        top = case["past"] + case["n"]
        st["k"] = randn(batch * case["n"], kv * HD, dtype=dt)
        st["v"] = randn(batch * case["n"], kv * HD, dtype=dt)
        st["starts"] = [case["past"]] * batch
    else:
        top = case["length"]
        st["lens"] = _lengths(case, top, case["n_q"], g)
        st["q"] = randn(batch * case["n_q"], case["heads"] * HD)
        st["k"], st["v"] = (randn(batch * top, kv * HD) for _ in range(2))
        st["starts"] = [0] * batch
    # Every sequence's pages, in the order in which they came free.
    per = -(-top // PAGE)
    table = torch.randperm(batch * per, generator=g, device="cuda").int().view(batch, per)
    st["table"], st["start"] = table, i32(st["starts"])
    if case["kind"] == "attend":
        st["len32"] = i32(st["lens"])
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if case["kind"] in ("window", "train"):
        return st
    n_pages, kv = st["table"].numel(), case["kv"]
    if own:
        from prichs_amd import ops

        st["cache"] = ops.kv_cache_pages(n_pages, kv)
    else:
        # Plain pages: codes and scale bytes of [page][slot][kv head].
        for name in ("k", "v"):
            for part, width in (("codes_", HD // 2), ("scale_", HD // GROUP)):
                st[part + name] = torch.zeros((n_pages, PAGE, kv, width), dtype=torch.uint8,
                                              device="cuda")
    if case["kind"] == "attend":
        # The cache as earlier steps filled it.
        k, v = st.pop("k"), st.pop("v")
        if own:
            ops.kv_cache_write(st["cache"], st["table"], st["start"], k, v, case["batch"],
                               case["length"], kv)
        else:
            _plain_write(st, k, v, case["batch"], case["length"], kv)
    return st


# -------------------------------------------------------------- plain forms --
def _levels(device):
    pos = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)
    return torch.cat([pos, -pos])


def _quantise(x):
    """x [..., kv, 128] f32 -> packed codes [..., kv, 64], scale bytes [..., kv, 4]."""
    x = x.reshape(*x.shape[:-1], HD // GROUP, GROUP)
    amax = x.abs().amax(-1)
    # amax = m 2^e with m in [0.5, 1): the least s with amax <= 7 2^s is e - 3,
    # one more where m passes 7/8.
    m, e = torch.frexp(amax)
    s = e - 3 + (m > 0.875).int()
    s = torch.where(amax == 0, torch.full_like(s, -126), s).clamp(-126, 125)
    a = torch.ldexp(x.abs(), -s.unsqueeze(-1))
    # Nearest level; a value midway goes to the level of even code.
    c = torch.zeros_like(a, dtype=torch.int32)
    for mid, even in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)):
        c += ((a >= mid) if even else (a > mid)).int()
    c += 8 * (x < 0).int()
    c = c.reshape(*c.shape[:-2], HD)
    return (c[..., 0::2] + 16 * c[..., 1::2]).to(torch.uint8), (s + 127).to(torch.uint8)


def _dequantise(codes, scale):
    c = codes.to(torch.int64)
    x = _levels(codes.device)[torch.stack([c & 15, c >> 4], -1).flatten(-2)]
    x = x.reshape(*x.shape[:-1], HD // GROUP, GROUP)
    return torch.ldexp(x, scale.int().unsqueeze(-1) - 127).flatten(-2)


def _slots(st, batch, n):
    """(page, slot) of positions start .. start + n - 1 of every sequence."""
    pos = st["start"].long()[:, None] + torch.arange(n, device="cuda")
    page = torch.gather(st["table"].long(), 1, pos // PAGE)
    return page.flatten(), (pos % PAGE).flatten()


def _plain_write(st, k, v, batch, n, kv):
    page, slot = _slots(st, batch, n)
    for name, x in (("k", k), ("v", v)):
        codes, scale = _quantise(x.float().view(batch * n, kv, HD))
        st["codes_" + name][page, slot] = codes
        st["scale_" + name][page, slot] = scale


def _plain_read(st, batch, n):
    page, slot = _slots(st, batch, n)
    return [_dequantise(st["codes_" + name][page, slot], st["scale_" + name][page, slot])
            for name in ("k", "v")]


def _visible(i, j, window, sinks):
    ok = j <= i
    if window:
        ok = ok & ((i - j < window) | (j < sinks))
    return ok


def _plain_attention(q, k, v, first, window, sinks, d_out=None):
    """q [n, Hq, 128] at positions first.., k / v [L, Hkv, 128], all f32: the
    outputs, and with d_out the gradients of q, k, v."""
    n, H, _ = q.shape
    L, K, _ = k.shape
    G = H // K
    kt, vt = k.permute(1, 0, 2), v.permute(1, 0, 2)  # [K, L, 128]
    out = torch.zeros_like(q)
    if d_out is not None:
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(kt), torch.zeros_like(vt)
    for a in range(0, n, CHUNK):
        b = min(n, a + CHUNK)
        hi = first + b

        def heads(x):  # [rows, Hq, 128] -> [K, G * rows, 128]
            return x[a:b].reshape(b - a, K, G, HD).permute(1, 2, 0, 3).reshape(K, -1, HD)

        def rows(x):
            return x.reshape(K, G, b - a, HD).permute(2, 0, 1, 3).reshape(b - a, H, HD)

        i = torch.arange(first + a, hi, device=q.device)[:, None]
        j = torch.arange(hi, device=q.device)[None, :]
        hidden = ~_visible(i, j, window, sinks)
        s = (heads(q) @ kt[:, :hi].transpose(1, 2)) * SCALE
        s = s.view(K, G, b - a, hi).masked_fill(hidden, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).view(K, -1, hi)
        out[a:b] = rows(p @ vt[:, :hi])
        if d_out is not None:
            do = heads(d_out)
            dv[:, :hi] += p.transpose(1, 2) @ do
            dp = do @ vt[:, :hi].transpose(1, 2)
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * SCALE
            dq[a:b] = rows(ds @ kt[:, :hi])
            dk[:, :hi] += ds.transpose(1, 2) @ heads(q)
    if d_out is None:
        return out
    return out, dq, dk.permute(1, 0, 2), dv.permute(1, 0, 2)


def _run_plain(st):
    c = st["case"]
    batch, kv = c["batch"], c["kv"]
    if c["kind"] == "cache":
        _plain_write(st, st["k"], st["v"], batch, c["n"], kv)
        return [x.to(st["k"].dtype).view(batch * c["n"], kv * HD)
                for x in _plain_read(st, batch, c["n"])]
    H = c["heads"]
    if c["kind"] == "attend":
        n_q, top = c["n_q"], c["length"]
        k, v = (x.view(batch, top, kv, HD) for x in _plain_read(st, batch, top))
        q = st["q"].float().view(batch, n_q, H, HD)
        out = [_plain_attention(q[b], k[b, :L], v[b, :L], L - n_q, c["window"], c["sinks"])
               for b, L in enumerate(st["lens"])]
        return torch.stack(out).to(st["q"].dtype).view(batch * n_q, H * HD)
    S = c["S"]
    names = ["q", "k", "v"] + (["d_out"] if c["kind"] == "train" else [])
    x = {n: st[n].float().view(batch, S, -1, HD) for n in names}
    got = [torch.zeros((batch, S, h, HD), device="cuda")
           for h in ([H] if c["kind"] == "window" else [H, H, kv, kv])]
    for b, L in enumerate(st["lens"]):
        if L:
            r = _plain_attention(*(x[n][b, :L] for n in ("q", "k", "v")), 0, c["window"],
                                 c["sinks"], x["d_out"][b, :L] if "d_out" in x else None)
            for dst, src in zip(got, [r] if c["kind"] == "window" else r):
                dst[b, :L] = src
    return [t.to(torch.bfloat16).flatten(2).flatten(0, 1) for t in got]


def run(st):
    if not own:
        return _run_plain(st)
    from prichs_amd import ops

    c = st["case"]
    batch, kv = c["batch"], c["kv"]
    if c["kind"] == "cache":
        ops.kv_cache_write(st["cache"], st["table"], st["start"], st["k"], st["v"], batch, c["n"],
                           kv)
        return list(ops.kv_cache_read(st["cache"], st["table"], st["start"], batch, c["n"], kv,
                                      out_dtype=st["k"].dtype))
    if c["kind"] == "attend":
        return ops.kv_cache_attention(st["q"], st["cache"], st["table"], st["len32"], batch,
                                      c["n_q"], c["heads"], kv, window=c["window"],
                                      sinks=c["sinks"])[0]
    train = c["kind"] == "train"
    args = (batch, c["S"], c["heads"], kv, c["window"], c["sinks"], st["seq_lens"])
    out, lse = ops.window_attention(st["q"], st["k"], st["v"], *args, want_lse=train)
    if not train:
        return [out]
    return [out, *ops.window_attention_backward(st["d_out"], st["q"], st["k"], st["v"], out, lse,
                                                *args)]


# --------------------------------------------------------------------- work --
def work(case):
    kv, batch = case["kv"], case["batch"]
    if case["kind"] == "cache":
        # Each value read once and written once in its own type, its 4.25 bits
        # written once and read once.
        size = 2 if case["dtype"] == "bf16" else 4
        vals = 2 * batch * case["n"] * kv * HD
        return {"bytes": vals * (2 * size + 2 * 4.25 / 8), "flops": 4 * vals}
    H, W, sinks = case["heads"], case["window"], case["sinks"]
    # Ragged lengths are uniform up to the longest: priced at the middle.
    if case["kind"] == "attend":
        n_q = case["n_q"]
        L = (case["length"] + n_q) // 2 if case["ragged"] else case["length"]
        lo = 0 if W == 0 else max(0, L - n_q - W + 1)
        keys = L - lo + min(lo, sinks)
        return {"bytes": batch * (keys * kv * 2 * HD * 4.25 / 8 + n_q * H * HD * 4),
                "flops": 4 * HD * H * batch * _pairs(L, W, sinks, L - n_q)}
    S = (case["S"] + 1) // 2 if case["ragged"] else case["S"]
    pairs = batch * _pairs(S, W, sinks)
    rows = batch * S
    if case["kind"] == "window":
        return {"bytes": rows * 2 * HD * (2 * H + 2 * kv), "flops": 4 * HD * H * pairs}
    # Forward and backward: q, k, v, d_out read, the output and three gradients
    # written; two products a pair forward, five backward.
    return {"bytes": rows * 2 * HD * (4 * H + 4 * kv), "flops": 14 * HD * H * pairs}


# -------------------------------------------------------------------- exact --
def _exact_values(x):
    """The values that the cache stands for, in 64 bits."""
    x = x.double().unflatten(-1, (-1, GROUP))
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, 2.0 ** -126)
    for e in range(-125, 126):
        scale = torch.where(top > 7.0 * 2.0 ** (e - 1), torch.full_like(top, 2.0 ** e), scale)
    y = (x / scale).abs()
    # The step is 1/2 below 2, 1 below 4 and 2 above; torch.round is half to even.
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    y = (torch.round(y / step) * step).clamp(max=6.0)
    return (torch.sign(x) * y * scale).flatten(-2)


def _exact_rows(q, k, v, at, window, sinks, do=None):
    """One kv head: q / do [G, n, 128] at positions at [n], k / v [L, 128]."""
    j = torch.arange(k.shape[0], device=q.device)
    off = j[None] > at[:, None]
    if window:
        off |= (j[None] <= at[:, None] - window) & (j[None] >= sinks)
    logit = torch.einsum("gnd,ld->gnl", q, k) / math.sqrt(HD)
    prob = torch.softmax(logit.masked_fill(off, -math.inf), dim=-1)
    o = torch.einsum("gnl,ld->gnd", prob, v)
    if do is None:
        return (o,)
    dv = torch.einsum("gnl,gnd->ld", prob, do)
    g = torch.einsum("gnd,ld->gnl", do, v) - (do * o).sum(-1, keepdim=True)
    g = g * prob / math.sqrt(HD)
    return o, torch.einsum("gnl,ld->gnd", g, k), torch.einsum("gnl,gnd->ld", g, q), dv


def exact(case, seed):
    st = _inputs(case, seed)
    kv, batch = case["kv"], case["batch"]
    if case["kind"] == "cache":
        return [_exact_values(st[n].view(-1, kv, HD)).flatten(1) for n in ("k", "v")]
    H = case["heads"]
    G = H // kv
    if case["kind"] == "attend":
        n, top = case["n_q"], case["length"]
        keys, vals = (_exact_values(st[x].view(batch, top, kv, HD)) for x in ("k", "v"))
        first = [L - n for L in st["lens"]]
    else:
        n = case["S"]
        keys, vals = (st[x].double().view(batch, n, kv, HD) for x in ("k", "v"))
        first = [0] * batch
    qs = st["q"].double().view(batch, n, kv, G, HD)
    res = [torch.zeros_like(qs)]
    if case["kind"] == "train":
        dos = st["d_out"].double().view(batch, n, kv, G, HD)
        res += [torch.zeros_like(qs), torch.zeros_like(keys), torch.zeros_like(vals)]
    for b in range(batch):
        L = st["lens"][b]
        count = n if case["kind"] == "attend" else L
        for h in range(kv):
            for a in range(0, count, 1024):
                z = min(count, a + 1024)
                at = torch.arange(first[b] + a, first[b] + z, device="cuda")
                do = dos[b, a:z, h].transpose(0, 1) if len(res) > 1 else None
                r = _exact_rows(qs[b, a:z, h].transpose(0, 1), keys[b, :L, h], vals[b, :L, h], at,
                                case["window"], case["sinks"], do)
                for t, x in zip(res[:2], r[:2]):
                    t[b, a:z, h] = x.transpose(0, 1)
                for t, x in zip(res[2:], r[2:]):
                    t[b, :L, h] += x
    flat = [res[0].reshape(batch * n, H * HD)]
    if case["kind"] == "attend":
        return flat[0]
    if case["kind"] == "train":
        flat += [res[1].reshape(batch * n, H * HD)] + [t.reshape(batch * n, kv * HD)
                                                       for t in res[2:]]
    return flat
