"""Stage-level wrappers over the C ABI, on torch device tensors.

torch provides device memory and the current stream only; every computation
runs in libprichs_hip.so.  Each wrapper names the C entry point it calls.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import numpy as np
import torch

from . import _lib as L

_TORCH_DTYPES = {torch.float32: L.DTYPE_F32, torch.bfloat16: L.DTYPE_BF16}
_DTYPE_TORCH = {L.DTYPE_F32: torch.float32, L.DTYPE_BF16: torch.bfloat16}


def dtype_code(t_or_dtype) -> int:
    dt = t_or_dtype.dtype if isinstance(t_or_dtype, torch.Tensor) else t_or_dtype
    if isinstance(dt, str):
        return {"f32": L.DTYPE_F32, "bf16": L.DTYPE_BF16}[dt]
    if isinstance(dt, int):
        return dt
    try:
        return _TORCH_DTYPES[dt]
    except KeyError:
        raise TypeError(f"unsupported dtype {dt}") from None


def torch_dtype(code: int) -> torch.dtype:
    return _DTYPE_TORCH[code]


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def _dev(t: torch.Tensor) -> torch.Tensor:
    if not t.is_cuda or not t.is_contiguous():
        raise ValueError("expected a contiguous device tensor")
    return t


# ------------------------------------------------------------------ router --
def router_num_blocks(T: int, E: int) -> int:
    return L.load().prichs_router_num_blocks(T, E)


def router_topk(x, w_router, router_bias, k, concept_bias=None, stream=None):
    """prichs_router_topk -> (logits f32 [T,E], idx i32 [T,k], w f32 [T,k], block_counts)."""
    lib = L.load()
    x = _dev(x)
    T, d = x.shape
    E = w_router.shape[1]
    dev = x.device
    nb = lib.prichs_router_num_blocks(T, E)
    logits = torch.empty((T, E), dtype=torch.float32, device=dev)
    idx = torch.empty((T, k), dtype=torch.int32, device=dev)
    w = torch.empty((T, k), dtype=torch.float32, device=dev)
    bc = torch.empty((max(nb * E, 1),), dtype=torch.int32, device=dev)
    nc = 0 if concept_bias is None else concept_bias.numel()
    L.check(lib.prichs_router_topk(_p(x), dtype_code(x), _p(_dev(w_router)), _p(_dev(router_bias)),
                                   _p(concept_bias), nc, T, d, E, k, _p(logits), _p(idx), _p(w),
                                   _p(bc), _stream(stream)))
    return logits, idx, w, bc


def permute(idx, w, block_counts, E, stream=None):
    """prichs_permute -> (offsets [E+2], row_token [T*k+T], row_weight [T*k], token_row [T*k])."""
    lib = L.load()
    T, k = idx.shape
    dev = idx.device
    offsets = torch.empty((E + 2,), dtype=torch.int32, device=dev)
    row_token = torch.empty((T * k + T,), dtype=torch.int32, device=dev)
    row_weight = torch.empty((T * k,), dtype=torch.float32, device=dev)
    token_row = torch.empty((T * k,), dtype=torch.int32, device=dev)
    L.check(lib.prichs_permute(_p(idx), _p(w), _p(block_counts), T, E, k, _p(offsets),
                               _p(row_token), _p(row_weight), _p(token_row), _stream(stream)))
    return offsets, row_token, row_weight, token_row


# ----------------------------------------------------------------- packing --
def _np_dtype(code):
    return np.uint16 if code == L.DTYPE_BF16 else np.float32


def pack_gate_up(gate: np.ndarray, up: np.ndarray, dtype) -> np.ndarray:
    """prichs_pack_gate_up (host): packed [Np, d] (bf16 bits as uint16, or f32;
    bf16 is fragment-tiled, see packed_rows)."""
    lib = L.load()
    code = dtype_code(dtype)
    d, f = gate.shape
    n = lib.prichs_packed_gate_up_elems(d, f, code)
    out = np.empty(n, dtype=_np_dtype(code))
    g = np.ascontiguousarray(gate, dtype=np.float32)
    u = np.ascontiguousarray(up, dtype=np.float32)
    L.check(lib.prichs_pack_gate_up(g.ctypes.data, u.ctypes.data, d, f, code, out.ctypes.data))
    return out.reshape(-1, d)


def pack_down(down: np.ndarray, dtype) -> np.ndarray:
    """prichs_pack_down (host): packed [roundup(d, 256), f] (bf16 fragment-tiled,
    see packed_rows)."""
    lib = L.load()
    code = dtype_code(dtype)
    f, d = down.shape
    n = lib.prichs_packed_down_elems(d, f, code)
    out = np.empty(n, dtype=_np_dtype(code))
    w = np.ascontiguousarray(down, dtype=np.float32)
    L.check(lib.prichs_pack_down(w.ctypes.data, d, f, code, out.ctypes.data))
    return out.reshape(-1, f)


def packed_rows(packed: np.ndarray, dtype) -> np.ndarray:
    """Logical [Np, K] rows of a packed weight.  f32 packing is row-major; bf16
    packing is fragment-major: fragment (n // 16, k // 32) is 512 contiguous
    elements, lane n % 16 + 16 * ((k % 32) // 8) holding k % 8 in 8 of them."""
    np_, K = packed.shape
    if dtype_code(dtype) != L.DTYPE_BF16:
        return packed
    t = packed.reshape(np_ // 16, K // 32, 4, 16, 8)      # [nb][ks][kq][nr][e]
    return t.transpose(0, 3, 1, 2, 4).reshape(np_, K)      # [nb][nr][ks][kq][e]


def to_device_packed(packed: list, dtype, device="cuda") -> torch.Tensor:
    """Concatenates per-expert packed arrays into one device tensor of the GEMM dtype."""
    code = dtype_code(dtype)
    host = np.concatenate([p.reshape(-1) for p in packed])
    t = torch.from_numpy(host.view(np.int16) if code == L.DTYPE_BF16 else host)
    t = t.to(device)
    return t.view(torch.bfloat16) if code == L.DTYPE_BF16 else t


# ------------------------------------------------------------------- GEMMs --
def grouped_gate_up_swiglu(x, row_token, offsets, G, rows, w_packed, d, f, stream=None,
                           out=None):
    """prichs_grouped_gate_up_swiglu -> act [rows, f] (rows = offsets[G]); out: a
    contiguous [rows, f] tensor to write (any element alignment)."""
    lib = L.load()
    act = torch.empty((rows, f), dtype=x.dtype, device=x.device) if out is None else _dev(out)
    L.check(lib.prichs_grouped_gate_up_swiglu(_p(_dev(x)), _p(row_token), _p(offsets), G, rows,
                                              _p(w_packed), d, f, dtype_code(x), _p(act),
                                              _stream(stream)))
    return act


def grouped_down(act, offsets, G, rows, w_packed, d, f, stream=None):
    """prichs_grouped_down -> y [rows, d]."""
    lib = L.load()
    y = torch.empty((rows, d), dtype=act.dtype, device=act.device)
    L.check(lib.prichs_grouped_down(_p(_dev(act)), _p(offsets), G, rows, _p(w_packed), d, f,
                                    dtype_code(act), _p(y), _stream(stream)))
    return y


def moe_combine(y, idx, w, token_row, has_shared=True, out_dtype=torch.float32, stream=None):
    """prichs_moe_combine -> out [T, d]."""
    lib = L.load()
    T, k = idx.shape
    d = y.shape[1]
    out = torch.empty((T, d), dtype=out_dtype, device=y.device)
    L.check(lib.prichs_moe_combine(_p(_dev(y)), dtype_code(y), _p(idx), _p(w), _p(token_row), T,
                                   d, k, 1 if has_shared else 0, _p(out), dtype_code(out),
                                   _stream(stream)))
    return out


# ------------------------------------------------------- memory-bound ops --
def rmsnorm(x, w, eps=1e-5, out_dtype=None, want_rstd=True, stream=None, out=None):
    """prichs_rmsnorm_forward -> (out, rstd)."""
    lib = L.load()
    x = _dev(x)
    d = x.shape[-1]
    T = x.numel() // d
    if out is None:
        out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    rstd = torch.empty((T,), dtype=torch.float32, device=x.device) if want_rstd else None
    L.check(lib.prichs_rmsnorm_forward(_p(x), dtype_code(x), _p(_dev(w)), _p(out), dtype_code(out),
                                       _p(rstd), T, d, eps, _stream(stream)))
    return out, rstd


def rope_(qk, cos, sin, cache_rows, batch, seq_len, pos_offset=0, sign=1, stream=None):
    """prichs_rope_forward, in place on qk [batch, seq_len, heads, head_dim]."""
    lib = L.load()
    qk = _dev(qk)
    hd = qk.shape[-1]
    H = qk.shape[-2]
    L.check(lib.prichs_rope_forward(_p(qk), dtype_code(qk), _p(_dev(cos)), _p(_dev(sin)),
                                    cache_rows, batch, seq_len, H, hd, pos_offset, sign,
                                    _stream(stream)))
    return qk


def hbm_copy(src, dst, stream=None):
    """prichs_hbm_copy: dst = src (device tensors of equal byte size, a multiple
    of 16), the library's streaming copy kernel."""
    nbytes = src.numel() * src.element_size()
    if dst.numel() * dst.element_size() != nbytes:
        raise ValueError("hbm_copy: src and dst sizes differ")
    L.check(L.load().prichs_hbm_copy(_p(src), _p(dst), nbytes, _stream(stream)))
    return dst


# ------------------------------------------------------- block sub-layers --
def pack_weight(w: np.ndarray, dtype) -> np.ndarray:
    """prichs_pack_weight (host): W [K, N] -> packed [roundup(N, 256), K]."""
    lib = L.load()
    code = dtype_code(dtype)
    K, N = w.shape
    n = lib.prichs_packed_weight_elems(K, N, code)
    out = np.empty(n, dtype=_np_dtype(code))
    wc = np.ascontiguousarray(w, dtype=np.float32)
    L.check(lib.prichs_pack_weight(wc.ctypes.data, K, N, code, out.ctypes.data))
    return out.reshape(-1, K)


def gemm(a, w_packed, N, out=None, stream=None):
    """prichs_gemm: C[M, N] = A[M, K] @ W (W packed by pack_weight / to_device_packed)."""
    lib = L.load()
    a = _dev(a)
    M, K = a.shape
    if out is None:
        out = torch.empty((M, N), dtype=a.dtype, device=a.device)
    L.check(lib.prichs_gemm(_p(a), K, M, K, _p(w_packed), N, _p(out), out.stride(0),
                            dtype_code(a), _stream(stream)))
    return out


def matmul_f32(op, a, b, out=None, stream=None):
    """prichs_matmul_f32 on f32 device tensors, in the reference's (m, k, n)
    naming: op MATMUL_AB: a [m, k] @ b [k, n]; MATMUL_ATB: a [m, k]^T @ b [m, n];
    MATMUL_ABT: a [m, k] @ b [n, k]^T.  Any sizes."""
    lib = L.load()
    a, b = _dev(a), _dev(b)
    if a.dtype != torch.float32 or b.dtype != torch.float32:
        raise TypeError("matmul_f32 takes float32 tensors")
    m, k = a.shape
    if op == L.MATMUL_AB:
        assert b.shape[0] == k
        n, shape = b.shape[1], (m, b.shape[1])
    elif op == L.MATMUL_ATB:
        assert b.shape[0] == m
        n, shape = b.shape[1], (k, b.shape[1])
    else:
        assert b.shape[1] == k
        n, shape = b.shape[0], (m, b.shape[0])
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=a.device)
    L.check(lib.prichs_matmul_f32(op, _p(a), _p(b), _p(_dev(out)), m, k, n, _stream(stream)))
    return out


def add(a, b, out_dtype=None, stream=None):
    """prichs_add: a + b in f32 arithmetic."""
    lib = L.load()
    a, b = _dev(a), _dev(b)
    out = torch.empty(a.shape, dtype=out_dtype or a.dtype, device=a.device)
    L.check(lib.prichs_add(_p(a), dtype_code(a), _p(b), dtype_code(b), _p(out), dtype_code(out),
                           a.numel(), _stream(stream)))
    return out


def attention(q, k, v, batch, seq_len, n_heads, n_kv_heads, head_dim=128, out=None,
              stream=None, rope_q=None):
    """prichs_attention_forward on 2-D row views (rows = batch * seq_len; q/k/v may
    be column slices of one fused buffer: their row strides are passed).

    rope_q = (cos, sin, pos_offset): prichs_attention_forward_rope_q instead --
    q is rotated by RoPE as the kernel loads it (cos / sin: device f32 tables
    [cache_rows, head_dim / 2]); k must be rotated already."""
    lib = L.load()
    if out is None:
        out = torch.empty((batch * seq_len, n_heads * head_dim), dtype=q.dtype, device=q.device)
    for t in (q, k, v, out):
        if t.stride(1) != 1:
            raise ValueError("attention operands need unit column stride")
    args = (_p(q), q.stride(0), _p(k), k.stride(0), _p(v), v.stride(0), _p(out), out.stride(0),
            batch, seq_len, n_heads, n_kv_heads, head_dim, dtype_code(q))
    if rope_q is None:
        L.check(lib.prichs_attention_forward(*args, _stream(stream)))
    else:
        cos, sin, pos_offset = rope_q
        for t in (cos, sin):
            if t.dtype != torch.float32 or not t.is_contiguous() or not t.is_cuda:
                raise ValueError("rope tables must be contiguous f32 device tensors")
        cache_rows = cos.numel() // (head_dim // 2)
        L.check(lib.prichs_attention_forward_rope_q(*args, _p(cos), _p(sin), cache_rows,
                                                    pos_offset, _stream(stream)))
    return out


# ---------------------------------------- window attention and KV cache ----
_BF16 = (torch.bfloat16,)
_FLOATS = (torch.bfloat16, torch.float32)


def _rows(t, name, rows, cols, dtypes=_BF16):
    """Checks an operand of at least `rows` rows whose columns are contiguous and
    returns its row stride (of a single row its width, whatever torch keeps)."""
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: unsupported dtype {t.dtype}")
    shape = t.shape
    if len(shape) != 2 or shape[0] < rows or shape[1] != cols:
        raise ValueError(f"{name}: expected [{rows}, {cols}], got {list(shape)}")
    ld, unit = t.stride()
    if unit != 1:
        raise ValueError(f"{name}: operands need unit column stride")
    return ld if shape[0] > 1 else cols


def _a(t):
    return None if t is None else t.data_ptr()


def _i32(t, name, n, dim=1):
    if t.dtype != torch.int32 or not t.is_contiguous() or t.dim() != dim or t.shape[0] != n:
        raise ValueError(f"{name}: expected contiguous int32 of {n} rows, got {t.dtype} "
                         f"{list(t.shape)}")


_HERE = contextlib.nullcontext()


def _launch_on(stream, first, *others):
    """(context, raw stream) of a launch on the operands' device, which must be one
    for all: the given stream, or torch's current one there.  Outputs and
    workspaces allocated in the context belong to that stream."""
    dev = first.get_device()
    for t in (first, *others):
        if t is not None and t.get_device() != dev or dev < 0:
            raise ValueError("expected device tensors, all on one device")
    if stream is not None:
        if stream.device_index != dev:
            raise ValueError(f"a stream of {stream.device} with operands on cuda:{dev}")
        return torch.cuda.stream(stream), stream.cuda_stream
    raw = torch._C._cuda_getCurrentRawStream(dev)
    return (_HERE if torch.cuda.current_device() == dev else torch.cuda.device(dev)), raw


def window_attention(q, k, v, batch, seq_len, n_heads, n_kv_heads, window, sinks=0,
                     seq_lens=None, head_dim=128, out=None, want_lse=False, stream=None):
    """prichs_window_attention_forward on 2-D row views, as ``attention``: each query
    sees its last `window` keys, itself included (0: all earlier ones), and the
    first `sinks` keys.  seq_lens: int32 device [batch], the rows of each sequence
    of a padded batch.  -> (out, lse f32 [batch, n_heads, seq_len], or None)."""
    rows, H, K = batch * seq_len, n_heads * head_dim, n_kv_heads * head_dim
    ldq, ldk, ldv = _rows(q, "q", rows, H), _rows(k, "k", rows, K), _rows(v, "v", rows, K)
    if seq_lens is not None:
        _i32(seq_lens, "seq_lens", batch)
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    ctx, s = _launch_on(stream, q, k, v, seq_lens, out)
    with ctx:
        if out is None:
            out = q.new_empty((rows, H))
        ldo = _rows(out, "out", rows, H)
        lse = None
        if want_lse:
            lse = torch.empty((batch, n_heads, seq_len), dtype=torch.float32, device=q.device)
        L.check(L.load().prichs_window_attention_forward(
            q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, out.data_ptr(), ldo, _a(lse),
            _a(seq_lens), batch, seq_len, n_heads, n_kv_heads, head_dim, window, sinks,
            L.DTYPE_BF16, s))
    return out, lse


def window_attention_backward(d_out, q, k, v, out, lse, batch, seq_len, n_heads, n_kv_heads,
                              window, sinks=0, seq_lens=None, head_dim=128, d_q=None, d_k=None,
                              d_v=None, stream=None):
    """prichs_window_attention_backward -> (d_q, d_k, d_v) bf16, from the operands,
    the output and the lse of window_attention (want_lse=True).  d_q, d_k, d_v:
    row views to write, e.g. column slices of one fused gradient; they must not
    overlap the operands."""
    lib = L.load()
    rows, H, K = batch * seq_len, n_heads * head_dim, n_kv_heads * head_dim
    args = []
    for t, name, cols in ((d_out, "d_out", H), (q, "q", H), (k, "k", K), (v, "v", K),
                          (out, "out", H)):
        ld = _rows(t, name, rows, cols)
        args += (t.data_ptr(), ld)
    if lse is None or lse.dtype != torch.float32 or not lse.is_contiguous() or \
            lse.shape != (batch, n_heads, seq_len):
        raise ValueError("lse: expected the contiguous f32 [batch, n_heads, seq_len] of "
                         "window_attention(want_lse=True)")
    if seq_lens is not None:
        _i32(seq_lens, "seq_lens", batch)
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    ctx, s = _launch_on(stream, d_out, q, k, v, out, lse, seq_lens, d_q, d_k, d_v)
    with ctx:
        grads, to = [], []
        for t, name, cols in ((d_q, "d_q", H), (d_k, "d_k", K), (d_v, "d_v", K)):
            if t is None:
                t = torch.empty((rows, cols), dtype=q.dtype, device=q.device)
            ld = _rows(t, name, rows, cols)
            grads.append(t)
            to += (t.data_ptr(), ld)
        need = lib.prichs_window_attention_backward_workspace(batch, seq_len, n_heads, n_kv_heads,
                                                              window, sinks)
        ws = torch.empty((need,), dtype=torch.uint8, device=q.device)
        L.check(lib.prichs_window_attention_backward(
            *args, lse.data_ptr(), _a(seq_lens), *to, batch, seq_len, n_heads, n_kv_heads,
            head_dim, window, sinks, L.DTYPE_BF16, ws.data_ptr(), need, s))
    return tuple(grads)


def kv_cache_pages(n_pages, n_kv_heads, device="cuda"):
    """A 4-bit KV cache of n_pages pages, each of L.KV_PAGE positions of every kv
    head: uint8 [n_pages, n_kv_heads, L.KV_PAGE_BYTES], not initialised."""
    return torch.empty((n_pages, n_kv_heads, L.KV_PAGE_BYTES), dtype=torch.uint8, device=device)


def _kv_cache(cache, page_table, batch, n_kv_heads):
    if cache.dtype != torch.uint8 or not cache.is_contiguous() or \
            cache.shape != (cache.shape[0], n_kv_heads, L.KV_PAGE_BYTES):
        raise ValueError("cache: expected the pages of kv_cache_pages for these kv heads")
    _i32(page_table, "page_table", batch, dim=2)


def kv_cache_write(cache, page_table, start, k, v, batch, n, n_kv_heads, counts=None,
                   stream=None):
    """prichs_kv_cache_write: rows b * n + i of k and v (bf16 or f32, 2-D row views)
    quantised into position start[b] + i of sequence b, whose pages page_table
    (int32 device [batch, max_pages]) names; i < counts[b] where counts is given.
    start, counts: int32 device [batch]."""
    _kv_cache(cache, page_table, batch, n_kv_heads)
    cols = n_kv_heads * 128
    ldk, ldv = _rows(k, "k", batch * n, cols, _FLOATS), _rows(v, "v", batch * n, cols, _FLOATS)
    if k.dtype != v.dtype:
        raise TypeError("k and v have different dtypes")
    _i32(start, "start", batch)
    if counts is not None:
        _i32(counts, "counts", batch)
    ctx, s = _launch_on(stream, cache, page_table, start, counts, k, v)
    with ctx:
        L.check(L.load().prichs_kv_cache_write(
            cache.data_ptr(), cache.shape[0], page_table.data_ptr(), page_table.shape[1],
            start.data_ptr(), _a(counts), k.data_ptr(), ldk, v.data_ptr(), ldv, batch, n,
            n_kv_heads, 128, _TORCH_DTYPES[k.dtype], s))


def kv_cache_read(cache, page_table, start, batch, n, n_kv_heads, counts=None,
                  out_dtype=torch.bfloat16, k=None, v=None, stream=None):
    """prichs_kv_cache_read: positions start[b] .. start[b] + n - 1 of every sequence
    -> (k, v) [batch * n, n_kv_heads * 128].  Rows past counts[b] keep what k and v
    held (zeros where this call allocates them)."""
    _kv_cache(cache, page_table, batch, n_kv_heads)
    _i32(start, "start", batch)
    if counts is not None:
        _i32(counts, "counts", batch)
    rows, cols = batch * n, n_kv_heads * 128
    ctx, s = _launch_on(stream, cache, page_table, start, counts, k, v)
    with ctx:
        make = torch.empty if counts is None else torch.zeros
        if k is None:
            k = make((rows, cols), dtype=out_dtype, device=cache.device)
            if v is None and counts is None:
                v = torch.empty_like(k)
        if v is None:
            v = make((rows, cols), dtype=out_dtype, device=cache.device)
        ldk, ldv = _rows(k, "k", rows, cols, _FLOATS), _rows(v, "v", rows, cols, _FLOATS)
        if k.dtype != v.dtype:
            raise TypeError("k and v have different dtypes")
        L.check(L.load().prichs_kv_cache_read(
            cache.data_ptr(), cache.shape[0], page_table.data_ptr(), page_table.shape[1],
            start.data_ptr(), _a(counts), k.data_ptr(), ldk, v.data_ptr(), ldv, batch, n,
            n_kv_heads, 128, _TORCH_DTYPES[k.dtype], s))
    return k, v


def kv_cache_attention(q, cache, page_table, lens, batch, n_q, n_heads, n_kv_heads, window=0,
                       sinks=0, head_dim=128, out=None, want_lse=False, stream=None):
    """prichs_kv_cache_attention: row b * n_q + i of q is the query at position
    lens[b] - n_q + i of sequence b, over the cached keys and values (its own
    among them); lens: int32 device [batch].  -> (out, lse f32 [batch, n_heads,
    n_q], or None)."""
    lib = L.load()
    _kv_cache(cache, page_table, batch, n_kv_heads)
    rows, H = batch * n_q, n_heads * head_dim
    ldq = _rows(q, "q", rows, H)
    _i32(lens, "lens", batch)
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    ctx, s = _launch_on(stream, q, cache, page_table, lens, out)
    with ctx:
        if out is None:
            out = q.new_empty((rows, H))
        ldo = _rows(out, "out", rows, H)
        lse = None
        if want_lse:
            lse = torch.empty((batch, n_heads, n_q), dtype=torch.float32, device=q.device)
        max_pages = page_table.shape[1]
        need = lib.prichs_kv_cache_attention_workspace(batch, n_q, n_heads, n_kv_heads, max_pages)
        ws = q.new_empty((need + 1) // 2) if need else None  # of two bytes each: a faster call
        L.check(lib.prichs_kv_cache_attention(
            q.data_ptr(), ldq, cache.data_ptr(), cache.shape[0], page_table.data_ptr(), max_pages,
            lens.data_ptr(), out.data_ptr(), ldo, _a(lse), batch, n_q, n_heads, n_kv_heads,
            head_dim, window, sinks, L.DTYPE_BF16, _a(ws), need, s))
    return out, lse


def kv_cache_shared_attention(q, cache, page_table, lens, group_start, shared, batch, n_q, n_heads,
                              n_kv_heads, window=0, sinks=0, head_dim=128, out=None,
                              want_lse=False, stream=None):
    """prichs_kv_cache_shared_attention: kv_cache_attention of a batch whose sequences
    group_start[g] .. group_start[g + 1] - 1 hold their first shared[g] positions in the
    same pages (group_start int32 device [n_groups + 1], shared [n_groups]), which are
    read once for the group.  -> (out, lse f32 [batch, n_heads, n_q], or None).  Behind
    short prompts, or with long text of each sequence's own, kv_cache_attention is faster."""
    lib = L.load()
    _kv_cache(cache, page_table, batch, n_kv_heads)
    rows, H = batch * n_q, n_heads * head_dim
    ldq = _rows(q, "q", rows, H)
    _i32(lens, "lens", batch)
    n_groups = shared.shape[0] if shared.dim() == 1 else -1
    _i32(shared, "shared", n_groups)
    _i32(group_start, "group_start", n_groups + 1)
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    ctx, s = _launch_on(stream, q, cache, page_table, lens, group_start, shared, out)
    with ctx:
        ldo = H
        if out is None:
            out = q.new_empty((rows, H))
        else:
            ldo = _rows(out, "out", rows, H)
        lse = None
        if want_lse:
            lse = torch.empty((batch, n_heads, n_q), dtype=torch.float32, device=q.device)
        max_pages = page_table.shape[1]
        need = lib.prichs_kv_cache_shared_attention_workspace(batch, n_q, n_heads, n_kv_heads,
                                                              max_pages, n_groups)
        ws = q.new_empty((need + 1) // 2) if need else None  # of two bytes each: a faster call
        L.check(lib.prichs_kv_cache_shared_attention(
            q.data_ptr(), ldq, cache.data_ptr(), cache.shape[0], page_table.data_ptr(), max_pages,
            lens.data_ptr(), group_start.data_ptr(), shared.data_ptr(), n_groups, out.data_ptr(),
            ldo, _a(lse), batch, n_q, n_heads, n_kv_heads, head_dim, window, sinks, L.DTYPE_BF16,
            _a(ws), need, s))
    return out, lse


# --------------------------------------------------- pages of the KV cache ----
def kv_pages_refs(n_pages, device="cuda"):
    """Counts for a cache whose pages are all free: int32 [n_pages], zeros."""
    return torch.zeros((n_pages,), dtype=torch.int32, device=device)


def _pages(refs, page_table):
    _i32(refs, "refs", refs.shape[0] if refs.dim() == 1 else -1)
    _i32(page_table, "page_table", page_table.shape[0] if page_table.dim() == 2 else -1, dim=2)
    return refs.shape[0], page_table.shape[0], page_table.shape[1]


def _pages_cache(cache, n_pages, n_kv_heads):
    if cache.dtype != torch.uint8 or not cache.is_contiguous() or \
            cache.shape != (n_pages, n_kv_heads, L.KV_PAGE_BYTES):
        raise ValueError("cache: expected the pages of kv_cache_pages for these refs and kv heads")


def _pages_work(lib, refs, n_pages, batch, n):
    need = lib.prichs_kv_pages_workspace(n_pages, batch, n)
    return refs.new_empty((need + 3) // 4), need


def kv_pages_reserve(refs, page_table, lens, counts, shortfall=None, stream=None):
    """prichs_kv_pages_reserve: pages for positions lens[b] .. lens[b] + counts[b] - 1 of
    every sequence (int32 device [batch]) where page_table (int32 device [batch,
    max_pages]) names none; refs: int32 device [n_pages], the count of each page's
    holders.  shortfall: int32 device [1], gets the number of pages that were not to be
    had."""
    n_pages, batch, max_pages = _pages(refs, page_table)
    _i32(lens, "lens", batch)
    _i32(counts, "counts", batch)
    if shortfall is not None:
        _i32(shortfall, "shortfall", 1)
    ctx, s = _launch_on(stream, refs, page_table, lens, counts, shortfall)
    with ctx:
        lib = L.load()
        ws, need = _pages_work(lib, refs, n_pages, batch, 0)
        L.check(lib.prichs_kv_pages_reserve(
            refs.data_ptr(), n_pages, page_table.data_ptr(), max_pages, lens.data_ptr(),
            counts.data_ptr(), batch, _a(shortfall), ws.data_ptr(), need, s))


def kv_pages_fork(cache, refs, page_table, lens, parents, children, n_kv_heads, shortfall=None,
                  stream=None):
    """prichs_kv_pages_fork: row children[i] of the table and of lens becomes a copy of
    row parents[i] (int32 device [n]); whole pages are shared, a partly filled last page
    is copied into a new one.  The children's rows must hold no pages (release them
    first).  shortfall as for kv_pages_reserve."""
    n_pages, batch, max_pages = _pages(refs, page_table)
    _pages_cache(cache, n_pages, n_kv_heads)
    _i32(lens, "lens", batch)
    n = parents.shape[0] if parents.dim() == 1 else -1
    _i32(parents, "parents", n)
    _i32(children, "children", n)
    if shortfall is not None:
        _i32(shortfall, "shortfall", 1)
    ctx, s = _launch_on(stream, cache, refs, page_table, lens, parents, children, shortfall)
    with ctx:
        lib = L.load()
        ws, need = _pages_work(lib, refs, n_pages, batch, n)
        L.check(lib.prichs_kv_pages_fork(
            cache.data_ptr(), refs.data_ptr(), n_pages, page_table.data_ptr(), max_pages,
            lens.data_ptr(), batch, parents.data_ptr(), children.data_ptr(), n, n_kv_heads,
            _a(shortfall), ws.data_ptr(), need, s))


def kv_pages_release(refs, page_table, rows, keep=None, stream=None):
    """prichs_kv_pages_release: rows rows[i] of the table (int32 device [n]) keep the
    pages of their first keep[i] positions (int32 device [n]; None: no positions) and
    give the others back."""
    n_pages, batch, max_pages = _pages(refs, page_table)
    n = rows.shape[0] if rows.dim() == 1 else -1
    _i32(rows, "rows", n)
    if keep is not None:
        _i32(keep, "keep", n)
    ctx, s = _launch_on(stream, refs, page_table, rows, keep)
    with ctx:
        L.check(L.load().prichs_kv_pages_release(
            refs.data_ptr(), n_pages, page_table.data_ptr(), max_pages, batch, rows.data_ptr(),
            _a(keep), n, s))


def kv_pages_compact(cache, refs, page_table, n_kv_heads, stream=None):
    """prichs_kv_pages_compact: the pages in use moved to the front of the cache.  ->
    (number of pages in use int32 [1], each old page's new number int32 [n_pages], -1 for
    a free one)."""
    n_pages, batch, max_pages = _pages(refs, page_table)
    _pages_cache(cache, n_pages, n_kv_heads)
    ctx, s = _launch_on(stream, cache, refs, page_table)
    with ctx:
        lib = L.load()
        ws, need = _pages_work(lib, refs, n_pages, 0, 0)
        n_live, new_page = refs.new_empty(1), refs.new_empty(n_pages)
        L.check(lib.prichs_kv_pages_compact(
            cache.data_ptr(), refs.data_ptr(), n_pages, page_table.data_ptr(), max_pages, batch,
            n_kv_heads, new_page.data_ptr(), n_live.data_ptr(), ws.data_ptr(), need, s))
    return n_live, new_page


def kv_cache_copy(dst, src, to, from_, n_kv_heads, stream=None):
    """prichs_kv_cache_copy: page from_[i] of the cache src becomes page to[i] of dst
    (int32 device [n]); dst may be src where no page is both."""
    _pages_cache(dst, dst.shape[0], n_kv_heads)
    _pages_cache(src, src.shape[0], n_kv_heads)
    n = to.shape[0] if to.dim() == 1 else -1
    _i32(to, "to", n)
    _i32(from_, "from_", n)
    ctx, s = _launch_on(stream, dst, src, to, from_)
    with ctx:
        L.check(L.load().prichs_kv_cache_copy(dst.data_ptr(), dst.shape[0], src.data_ptr(),
                                              src.shape[0], to.data_ptr(), from_.data_ptr(), n,
                                              n_kv_heads, s))
    return dst


# ------------------------------------- norms of queries and keys, rotated ----
def _qk(q, k, n_heads, n_kv_heads, head_dim, names):
    """(rows, row strides of q and k, dtype) of a pair of operands, either of which is None
    where it has no heads."""
    first = q if n_heads else k
    if first is None or n_heads and q is None or n_kv_heads and k is None:
        raise ValueError(f"{names[0]}, {names[1]}: missing, or no heads at all")
    rows, dtype = first.shape[0], first.dtype
    ldq = _rows(q, names[0], rows, n_heads * head_dim, _FLOATS) if n_heads else 0
    if not n_kv_heads:
        return rows, ldq, 0, dtype
    ldk = _rows(k, names[1], rows, n_kv_heads * head_dim, _FLOATS)
    if k.dtype != dtype:
        raise TypeError(f"{names[0]} and {names[1]} have different dtypes")
    if k.shape[0] != rows:
        raise ValueError(f"{names[0]} and {names[1]} have different numbers of rows")
    return rows, ldq, ldk, dtype


def _f32(t, name, n):
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name}: expected contiguous f32 of {n} elements")


def _norm_rope_args(w_q, w_k, cos, sin, n_heads, n_kv_heads, head_dim, positions, seq_len,
                    pos_offset, rows):
    """Checks them and returns (positions of the tables, seq_len)."""
    if n_heads:
        _f32(w_q, "w_q", head_dim)
    if n_kv_heads:
        _f32(w_k, "w_k", head_dim)
    shape = cos.shape
    if len(shape) != 2 or shape[1] * 2 != head_dim:
        raise ValueError("cos, sin: expected f32 [positions, head_dim / 2]")
    n = shape[0] * shape[1]
    _f32(cos, "cos", n)
    _f32(sin, "sin", n)
    if positions is not None:
        _i32(positions, "positions", rows)
    if seq_len is None:
        seq_len = rows
    if pos_offset < 0 or seq_len < 0:
        raise ValueError("seq_len and pos_offset must not be negative")
    return shape[0], seq_len if rows else 1


def qk_norm_rope(q, k, w_q, w_k, cos, sin, n_heads, n_kv_heads, head_dim=128, eps=1e-5,
                 positions=None, seq_len=None, pos_offset=0, q_out=None, k_out=None, stream=None):
    """prichs_qk_norm_rope_forward (_zeros): each head of q and k (2-D row views, bf16 or
    f32) normed with w_q / w_k (f32 [head_dim]) and rotated to its row's position:
    positions[r] (int32 device [rows]), or r % seq_len + pos_offset (seq_len None: the rows
    are one sequence).  cos, sin: f32 [positions, head_dim / 2].  q_out / k_out may be q / k.
    With n_heads or n_kv_heads 0 that operand is None.  -> (q_out, k_out).  Rows at positions
    outside the tables keep what q_out and k_out held (zeros where this call allocates
    them)."""
    rows, ldq, ldk, dtype = _qk(q, k, n_heads, n_kv_heads, head_dim, ("q", "k"))
    n_pos, seq_len = _norm_rope_args(w_q, w_k, cos, sin, n_heads, n_kv_heads, head_dim, positions,
                                     seq_len, pos_offset, rows)
    if not n_heads:
        q = w_q = q_out = None
    if not n_kv_heads:
        k = w_k = k_out = None
    ctx, s = _launch_on(stream, cos, q, k, w_q, w_k, sin, positions, q_out, k_out)
    with ctx:
        ldqo, ldko = n_heads * head_dim, n_kv_heads * head_dim
        lib = L.load()
        forward = lib.prichs_qk_norm_rope_forward
        if q_out is None and k_out is None:  # of q's and k's rows and dtype, without gaps
            q_out = q.new_empty((rows, ldqo)) if n_heads else None
            k_out = k.new_empty((rows, ldko)) if n_kv_heads else None
            forward = lib.prichs_qk_norm_rope_forward_zeros
        else:
            make = torch.empty if positions is None else torch.zeros  # all rows have one, or not
            if q_out is None and n_heads:
                q_out = make((rows, ldqo), dtype=dtype, device=q.device)
            if k_out is None and n_kv_heads:
                k_out = make((rows, ldko), dtype=dtype, device=k.device)
            r2, ldqo, ldko, d2 = _qk(q_out, k_out, n_heads, n_kv_heads, head_dim,
                                     ("q_out", "k_out"))
            if r2 != rows or d2 != dtype:
                raise ValueError("q_out, k_out: expected the rows and the dtype of q and k")
        L.check(forward(
            _a(q), ldq, _a(k), ldk, _a(w_q), _a(w_k), cos.data_ptr(), sin.data_ptr(), n_pos,
            _a(positions), seq_len, pos_offset, _a(q_out), ldqo, _a(k_out), ldko, rows, n_heads,
            n_kv_heads, head_dim, eps, _TORCH_DTYPES[dtype], s))
    return q_out, k_out


def qk_norm_rope_backward(d_q_out, d_k_out, q, k, w_q, w_k, cos, sin, n_heads, n_kv_heads,
                          head_dim=128, eps=1e-5, positions=None, seq_len=None, pos_offset=0,
                          d_q=None, d_k=None, d_wq=None, d_wk=None, accumulate=False, stream=None):
    """prichs_qk_norm_rope_backward -> (d_q, d_k, d_wq, d_wk): gradients of q and k (d_q /
    d_k may be d_q_out / d_k_out) and, in f32, of the weights (added to d_wq and d_wk with
    accumulate)."""
    lib = L.load()
    rows, ldq, ldk, dtype = _qk(q, k, n_heads, n_kv_heads, head_dim, ("q", "k"))
    r2, lddqo, lddko, d2 = _qk(d_q_out, d_k_out, n_heads, n_kv_heads, head_dim,
                               ("d_q_out", "d_k_out"))
    if r2 != rows or d2 != dtype:
        raise ValueError("d_q_out, d_k_out: expected the rows and the dtype of q and k")
    n_pos, seq_len = _norm_rope_args(w_q, w_k, cos, sin, n_heads, n_kv_heads, head_dim, positions,
                                     seq_len, pos_offset, rows)
    if not n_heads:
        q = w_q = d_q_out = d_q = d_wq = None
    if not n_kv_heads:
        k = w_k = d_k_out = d_k = d_wk = None
    if accumulate and (n_heads and d_wq is None or n_kv_heads and d_wk is None):
        raise ValueError("accumulate needs the d_wq and d_wk to add to")
    ctx, s = _launch_on(stream, cos, d_q_out, d_k_out, q, k, w_q, w_k, sin, positions, d_q, d_k,
                        d_wq, d_wk)
    with ctx:
        lddq, lddk = n_heads * head_dim, n_kv_heads * head_dim
        given = d_q is not None or d_k is not None
        if n_heads:
            d_q = q.new_empty((rows, lddq)) if d_q is None else d_q
            if d_wq is None:
                d_wq = w_q.new_empty(head_dim)
            else:
                _f32(d_wq, "d_wq", head_dim)
        if n_kv_heads:
            d_k = k.new_empty((rows, lddk)) if d_k is None else d_k
            if d_wk is None:
                d_wk = w_k.new_empty(head_dim)
            else:
                _f32(d_wk, "d_wk", head_dim)
        if given:
            r2, lddq, lddk, d2 = _qk(d_q, d_k, n_heads, n_kv_heads, head_dim, ("d_q", "d_k"))
            if r2 != rows or d2 != dtype:
                raise ValueError("d_q, d_k: expected the rows and the dtype of q and k")
        need = lib.prichs_qk_norm_rope_backward_workspace(rows, n_heads, n_kv_heads, head_dim)
        ws = cos.new_empty((need + 3) // 4)
        L.check(lib.prichs_qk_norm_rope_backward(
            _a(d_q_out), lddqo, _a(d_k_out), lddko, _a(q), ldq, _a(k), ldk, _a(w_q), _a(w_k),
            cos.data_ptr(), sin.data_ptr(), n_pos, _a(positions), seq_len, pos_offset, _a(d_q),
            lddq, _a(d_k), lddk, _a(d_wq), _a(d_wk), int(accumulate), rows, n_heads, n_kv_heads,
            head_dim, eps, _TORCH_DTYPES[dtype], ws.data_ptr(), need, s))
    return d_q, d_k, d_wq, d_wk
