"""Refusals of the window attention and KV cache entry points (no GPU needed:
arguments are checked before any HIP call)."""
import pytest

from prichs_amd import _lib as L

P, Q = 1 << 20, (1 << 20) + 8  # an aligned address and one that is not; never dereferenced
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    return L.load()


FWD = dict(q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, o=P, ldo=512, lse=None, seq_lens=None, batch=1,
           seq_len=8, n_heads=4, n_kv_heads=2, head_dim=128, window=4, sinks=0, dtype=1, stream=None)
BWD = dict(d_o=P, ldd=512, q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, o=P, ldo=512, lse=P,
           seq_lens=None, d_q=P, lddq=512, d_k=P, lddk=256, d_v=P, lddv=256, batch=1, seq_len=8,
           n_heads=4, n_kv_heads=2, head_dim=128, window=4, sinks=0, dtype=1, workspace=P,
           workspace_bytes=BIG, stream=None)
WRITE = dict(cache=P, n_pages=4, page_table=P, max_pages=2, start=P, counts=None, k=P, ldk=256, v=P,
             ldv=256, batch=1, n=8, n_kv_heads=2, head_dim=128, dtype=1, stream=None)
ATTEND = dict(q=P, ldq=512, cache=P, n_pages=4, page_table=P, max_pages=2, lens=P, o=P, ldo=512,
              lse=None, batch=1, n_q=1, n_heads=4, n_kv_heads=2, head_dim=128, window=0, sinks=0,
              dtype=1, workspace=P, workspace_bytes=BIG, stream=None)
INV, UNS, CAP = L.PRICHS_ERR_INVALID_ARGUMENT, L.PRICHS_ERR_UNSUPPORTED, L.PRICHS_ERR_CAPACITY

ROWS = [dict(ldq=504), dict(ldq=516), dict(o=Q), dict(ldo=500), dict(q=None), dict(o=None),
        dict(n_heads=3), dict(n_kv_heads=0), dict(n_heads=0), dict(dtype=0), dict(dtype=7),
        dict(batch=70000)]
BAD = (
    [("prichs_window_attention_forward", FWD, d, INV) for d in ROWS + [
        dict(k=Q), dict(ldv=248), dict(ldk=1 << 25), dict(v=None), dict(seq_len=1 << 40),
        dict(batch=65535, seq_len=1 << 21)]]
    + [("prichs_window_attention_backward", BWD, d, INV) for d in ROWS + [
        dict(d_q=None), dict(d_k=Q), dict(lddv=250), dict(lse=None), dict(workspace=None),
        dict(workspace=Q), dict(d_o=None), dict(ldd=8)]]
    + [("prichs_window_attention_backward", BWD, dict(workspace_bytes=0), CAP)]
    + [(f"prichs_kv_cache_{w}", WRITE, d, INV) for w in ("write", "read") for d in [
        dict(cache=None), dict(cache=Q), dict(page_table=None), dict(start=None), dict(k=Q),
        dict(v=None), dict(ldk=200), dict(ldv=260), dict(dtype=2), dict(n_kv_heads=0),
        dict(n_kv_heads=70000, ldk=1 << 30, ldv=1 << 30), dict(batch=1 << 20, n=1 << 20),
        dict(n=1 << 33), dict(n_pages=1 << 33), dict(max_pages=1 << 31)]]
    + [("prichs_kv_cache_attention", ATTEND, d, INV) for d in ROWS + [
        dict(cache=Q), dict(cache=None), dict(page_table=None), dict(lens=None),
        dict(n_q=1 << 31), dict(n_pages=1 << 33), dict(max_pages=1 << 31)]]
    + [(f, base, dict(head_dim=64), UNS) for f, base in (
        ("prichs_window_attention_forward", FWD), ("prichs_window_attention_backward", BWD),
        ("prichs_kv_cache_write", WRITE), ("prichs_kv_cache_read", WRITE),
        ("prichs_kv_cache_attention", ATTEND))]
)


def call(lib, name, args):
    return getattr(lib, name)(*args.values())


@pytest.mark.parametrize("name,base,change,status", BAD,
                         ids=[f"{n[7:]}-{'-'.join(map(str, c))}-{i}" for i, (n, _, c, _) in
                              enumerate(BAD)])
def test_refused(lib, name, base, change, status):
    assert set(change) <= set(base)
    lib.prichs_clear_error()
    args = {**base, **change}
    if name == "prichs_kv_cache_read":  # cache, table, start, counts, k, v as for a write
        assert list(args) == list(WRITE)
    assert call(lib, name, args) == status
    assert L.last_error()


@pytest.mark.parametrize("name,base", [
    ("prichs_window_attention_forward", FWD), ("prichs_window_attention_backward", BWD),
    ("prichs_kv_cache_write", WRITE), ("prichs_kv_cache_read", WRITE),
    ("prichs_kv_cache_attention", ATTEND)])
def test_an_empty_batch_is_nothing_to_do(lib, name, base):
    assert call(lib, name, {**base, "batch": 0}) == L.PRICHS_OK
    rows = next(n for n in ("seq_len", "n", "n_q") if n in base)
    assert call(lib, name, {**base, rows: 0}) == L.PRICHS_OK


def test_workspaces(lib):
    need = lib.prichs_window_attention_backward_workspace(4, 2048, 12, 3, 4, 0)
    assert need >= 4 * 2048 * 12 * 4
    assert call(lib, "prichs_window_attention_backward",
                {**BWD, "batch": 4, "seq_len": 2048, "n_heads": 12, "n_kv_heads": 3, "ldq": 1536,
                 "ldd": 1536, "ldo": 1536, "ldk": 384, "ldv": 384, "lddq": 1536, "lddk": 384,
                 "lddv": 384, "workspace_bytes": need - 1}) == CAP
    need = lib.prichs_kv_cache_attention_workspace(1, 1, 12, 3, 128)
    if need:
        assert call(lib, "prichs_kv_cache_attention",
                    {**ATTEND, "max_pages": 128, "n_heads": 12, "n_kv_heads": 3, "ldq": 1536,
                     "ldo": 1536, "workspace_bytes": need - 1}) == CAP
