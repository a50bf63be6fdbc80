"""Refusals of the norms with rotation, the page calls and the attention over shared
pages (no GPU needed: arguments are checked before any HIP call)."""
import pytest

from prichs_amd import _lib as L

P, Q = 1 << 20, (1 << 20) + 8  # an aligned address and one that is not; never dereferenced
BIG = 1 << 40
INV, UNS, CAP = L.PRICHS_ERR_INVALID_ARGUMENT, L.PRICHS_ERR_UNSUPPORTED, L.PRICHS_ERR_CAPACITY

NORM = dict(q=P, ldq=512, k=P, ldk=256, w_q=P, w_k=P, cos=P, sin=P, cache_rows=16, positions=P,
            seq_len=0, pos_offset=0, q_out=P, ldqo=512, k_out=P, ldko=256, rows=8, n_heads=4,
            n_kv_heads=2, head_dim=128, eps=1e-5, dtype=1, stream=None)
BWD = dict(d_qo=P, lddqo=512, d_ko=P, lddko=256, q=P, ldq=512, k=P, ldk=256, w_q=P, w_k=P, cos=P,
           sin=P, cache_rows=16, positions=P, seq_len=0, pos_offset=0, d_q=P, lddq=512, d_k=P,
           lddk=256, d_wq=P, d_wk=P, beta=0, rows=8, n_heads=4, n_kv_heads=2, head_dim=128,
           eps=1e-5, dtype=1, workspace=P, workspace_bytes=BIG, stream=None)
RESERVE = dict(refs=P, n_pages=9, page_table=P, max_pages=4, lens=P, counts=P, batch=3,
               shortfall=None, workspace=P, workspace_bytes=BIG, stream=None)
FORK = dict(cache=P, refs=P, n_pages=9, page_table=P, max_pages=4, lens=P, batch=3, parents=P,
            children=P, n=2, n_kv_heads=2, shortfall=None, workspace=P, workspace_bytes=BIG,
            stream=None)
RELEASE = dict(refs=P, n_pages=9, page_table=P, max_pages=4, batch=3, rows=P, keep=None, n=2,
               stream=None)
COMPACT = dict(cache=P, refs=P, n_pages=9, page_table=P, max_pages=4, batch=3, n_kv_heads=2,
               new_page=P, n_live=P, workspace=P, workspace_bytes=BIG, stream=None)
COPY = dict(dst=P, dst_pages=9, src=P, src_pages=9, to=P, frm=P, n=2, n_kv_heads=2, stream=None)
SHARED = dict(q=P, ldq=512, cache=P, n_pages=4, page_table=P, max_pages=40, lens=P, group_start=P,
              shared=P, n_groups=1, o=P, ldo=512, lse=None, batch=2, n_q=1, n_heads=4,
              n_kv_heads=2, head_dim=128, window=0, sinks=0, dtype=1, workspace=P,
              workspace_bytes=BIG, stream=None)

ROTATE = [dict(ldq=504), dict(ldq=516), dict(ldk=128), dict(q=Q), dict(k=None), dict(w_q=None),
          dict(w_k=Q), dict(cos=None), dict(sin=Q), dict(n_heads=0, n_kv_heads=0),
          dict(n_heads=70000, ldq=1 << 24), dict(rows=1 << 31), dict(cache_rows=1 << 31),
          dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=2), dict(positions=None),
          dict(positions=None, seq_len=17), dict(positions=None, seq_len=16, pos_offset=1),
          dict(positions=None, seq_len=4, pos_offset=1 << 63)]
TABLE = [dict(refs=None), dict(page_table=None), dict(n_pages=1 << 25), dict(batch=1 << 21),
         dict(max_pages=1 << 28), dict(batch=1 << 20, max_pages=1 << 12)]
WORK = [dict(workspace=None), dict(workspace=Q)]
HEADS = [dict(n_kv_heads=0), dict(n_kv_heads=70000), dict(cache=None), dict(cache=Q)]
BAD = (
    [("prichs_qk_norm_rope_forward", NORM, d, INV) for d in ROTATE + [
        dict(q_out=None), dict(k_out=Q), dict(ldqo=8), dict(ldko=260)]]
    + [("prichs_qk_norm_rope_backward", BWD, d, INV) for d in ROTATE + WORK + [
        dict(d_q=None), dict(d_k=Q), dict(lddq=8), dict(d_qo=None), dict(d_ko=Q), dict(lddko=12),
        dict(d_wq=None), dict(d_wk=None), dict(beta=2), dict(rows=0, d_wq=None)]]
    + [(f"prichs_qk_norm_rope_{w}", b, dict(head_dim=h), UNS)
       for w, b in (("forward", NORM), ("backward", BWD)) for h in (0, 4, 100, 264, 1 << 40)]
    + [("prichs_kv_pages_reserve", RESERVE, d, INV) for d in TABLE + WORK + [
        dict(lens=None), dict(counts=None)]]
    + [("prichs_kv_pages_fork", FORK, d, INV) for d in TABLE + WORK + HEADS + [
        dict(lens=None), dict(parents=None), dict(children=None), dict(n=1 << 21)]]
    + [("prichs_kv_pages_release", RELEASE, d, INV) for d in TABLE + [dict(rows=None),
                                                                     dict(n=1 << 21)]]
    + [("prichs_kv_pages_compact", COMPACT, d, INV) for d in TABLE + WORK + HEADS + [
        dict(new_page=None), dict(n_live=None)]]
    + [(n, b, dict(workspace_bytes=w), CAP) for n, b, w in (
        ("prichs_qk_norm_rope_backward", BWD, 0), ("prichs_kv_pages_reserve", RESERVE, 8),
        ("prichs_kv_pages_fork", FORK, 0), ("prichs_kv_pages_compact", COMPACT, 100),
        ("prichs_kv_cache_shared_attention", SHARED, 0))]
    + [("prichs_kv_cache_copy", COPY, d, INV) for d in [
        dict(dst=None), dict(src=Q), dict(to=None), dict(frm=None), dict(n=1 << 31),
        dict(n_kv_heads=0), dict(dst_pages=1 << 31), dict(src_pages=1 << 31)]]
    + [("prichs_kv_cache_shared_attention", SHARED, d, INV) for d in WORK + [
        dict(ldq=504), dict(ldq=516), dict(ldo=500), dict(q=None), dict(o=Q), dict(cache=Q),
        dict(cache=None), dict(page_table=None), dict(lens=None), dict(group_start=None),
        dict(shared=None), dict(n_groups=70000), dict(n_heads=3), dict(n_kv_heads=0),
        dict(dtype=0), dict(batch=70000), dict(n_q=1 << 31), dict(n_pages=1 << 33),
        dict(max_pages=1 << 31), dict(batch=60000, n_q=1000)]]
    + [("prichs_kv_cache_shared_attention", SHARED, dict(head_dim=64), UNS)]
)


def call(lib, name, args):
    return getattr(lib, name)(*args.values())


@pytest.fixture(scope="module")
def lib():
    return L.load()


@pytest.mark.parametrize("name,base,change,status", BAD,
                         ids=[f"{n[7:]}-{'-'.join(map(str, c))}-{i}" for i, (n, _, c, _) in
                              enumerate(BAD)])
def test_refused(lib, name, base, change, status):
    assert set(change) <= set(base)
    lib.prichs_clear_error()
    assert call(lib, name, {**base, **change}) == status
    assert L.last_error()


@pytest.mark.parametrize("name,args", [
    ("prichs_qk_norm_rope_forward", {**NORM, "rows": 0}),
    ("prichs_kv_pages_reserve", {**RESERVE, "batch": 0}),
    ("prichs_kv_pages_fork", {**FORK, "n": 0}),
    ("prichs_kv_pages_release", {**RELEASE, "n": 0}),
    ("prichs_kv_pages_release", {**RELEASE, "max_pages": 0}),
    ("prichs_kv_cache_copy", {**COPY, "n": 0}),
    ("prichs_kv_cache_copy", {**COPY, "src_pages": 0}),
    ("prichs_kv_cache_shared_attention", {**SHARED, "batch": 0}),
    ("prichs_kv_cache_shared_attention", {**SHARED, "n_q": 0})])
def test_nothing_to_do(lib, name, args):
    assert call(lib, name, args) == L.PRICHS_OK


def test_workspaces(lib):
    need = lib.prichs_qk_norm_rope_backward_workspace(8, 4, 2, 128)
    assert need >= 2 * 128 * 4
    assert call(lib, "prichs_qk_norm_rope_backward", {**BWD, "workspace_bytes": need - 1}) == CAP
    assert lib.prichs_qk_norm_rope_backward_workspace(0, 4, 2, 128) == 0
    assert lib.prichs_qk_norm_rope_backward_workspace(1 << 30, 12, 3, 128) <= 1 << 21
    need = lib.prichs_kv_pages_workspace(9, 3, 2)
    assert call(lib, "prichs_kv_pages_fork", {**FORK, "workspace_bytes": need - 1}) == CAP
    assert lib.prichs_kv_pages_workspace(1 << 25, 1, 1) == 0
    need = lib.prichs_kv_cache_shared_attention_workspace(2, 1, 4, 2, 40, 1)
    assert need >= 2 * 4 * 2 * 130 * 4
    assert call(lib, "prichs_kv_cache_shared_attention",
                {**SHARED, "workspace_bytes": need - 1}) == CAP
