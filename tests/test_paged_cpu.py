"""CPU tests of the paged operators: what the host side refuses before it
launches anything, the workspace's size, and the references that the GPU
tests compare with."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged_ref

PTR = 1 << 20   # an aligned address that nothing reads: every call here is refused first


def _cache(pkg, **kw):
    d = dict(k=PTR, v=PTR, dtype=pkg.T3B_F16, n_pages=10, n_kv_head=4, page_size=16, head_dim=64)
    return pkg.PagedKv(**{**d, **kw})


def _attn(pkg, cache=None, **kw):
    d = dict(q=PTR, out=PTR, q_stride=512, out_stride=512, len=PTR, table=PTR, row_start=PTR, prefix_start=PTR,
             prefix_len=PTR, prefix_table=PTR, workspace=PTR, workspace_bytes=1 << 30, dtype=pkg.T3B_F32, n_head=8, n=4,
             rows=4, max_blocks=3, n_prefix=1, prefix_max_blocks=2)
    return pkg.SharedAttn(cache=_cache(pkg, **(cache or {})), **{**d, **kw})


BAD_CACHE = [dict(dtype=0), dict(dtype=8), dict(page_size=0), dict(page_size=24), dict(page_size=4), dict(page_size=512),
             dict(head_dim=80), dict(head_dim=256), dict(n_pages=0), dict(n_pages=1 << 28, page_size=256),
             dict(n_kv_head=0), dict(n_kv_head=5000), dict(k=None), dict(v=None), dict(k=PTR + 8), dict(v=PTR + 2),
             dict(page_stride=4095), dict(page_stride=4097), dict(page_stride=-8)]


@pytest.mark.parametrize("cache", BAD_CACHE, ids=str)
def test_bad_caches_are_refused(pkg, cache):
    L = pkg.lib()
    for f in (L.t3b_op_attention_shared, L.t3b_op_attention_shared_prompt):
        assert f(C.byref(_attn(pkg, cache)), None) == -1, cache
        assert "t3b_op_attention_shared" in pkg.last_error()
    a = pkg.KvAppend(cache=_cache(pkg, **cache), k=PTR, v=PTR, stride=512, slots=PTR, dtype=pkg.T3B_F32, rows=3)
    assert L.t3b_op_kv_append(C.byref(a), None) == -1
    assert "t3b_op_kv_append" in pkg.last_error()


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(len=None), dict(table=None), dict(prefix_start=None),
                                 dict(prefix_len=None), dict(prefix_table=None), dict(q=PTR + 4), dict(out=PTR + 8),
                                 dict(dtype=30), dict(dtype=8), dict(n_head=6), dict(n_head=0), dict(n_head=68),
                                 dict(n=0, rows=0), dict(n=-1), dict(n=70000, rows=70000), dict(n_prefix=-1),
                                 dict(n_prefix=70000), dict(max_blocks=0), dict(max_blocks=1 << 27),
                                 dict(prefix_max_blocks=0), dict(prefix_max_blocks=1 << 27), dict(q_stride=511),
                                 dict(q_stride=508), dict(out_stride=514), dict(out_stride=0), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(rows=-1), dict(rows=(1 << 26) + 1), dict(q_stride=516)], ids=str)
def test_bad_attention_calls_are_refused(pkg, bad):
    L = pkg.lib()
    for f in (L.t3b_op_attention_shared, L.t3b_op_attention_shared_prompt):
        assert f(C.byref(_attn(pkg, **bad)), None) == -1, bad
        assert pkg.last_error()
        assert f(None, None) == -1


def test_each_form_refuses_what_only_it_needs(pkg):
    L = pkg.lib()
    assert L.t3b_op_attention_shared(C.byref(_attn(pkg, rows=5)), None) == -1            # one row per request
    assert L.t3b_op_attention_shared_prompt(C.byref(_attn(pkg, row_start=None)), None) == -1
    assert L.t3b_op_attention_shared_prompt(C.byref(_attn(pkg, rows=0)), None) == 0      # nothing to do


def test_a_short_workspace_is_refused(pkg):
    L = pkg.lib()
    a = _attn(pkg)
    need = L.t3b_op_attention_shared_workspace(C.byref(a))
    if need:
        for kw in (dict(workspace=None), dict(workspace=PTR + 4), dict(workspace_bytes=need - 1)):
            assert L.t3b_op_attention_shared(C.byref(_attn(pkg, **kw)), None) == -1, kw
            assert "workspace" in pkg.last_error()
    assert L.t3b_op_attention_shared_workspace(C.byref(_attn(pkg, n=0))) == 0
    # pointers are not looked at, and more of anything never needs less
    sizes = [L.t3b_op_attention_shared_workspace(C.byref(_attn(pkg, q=None, workspace=None, n=n, rows=n))) for n in (1, 8, 64, 500)]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("heads,kv,dim,dtype", [(8, 4, 64, 0), (16, 1, 128, 1), (6, 2, 128, 0)])
def test_a_batch_that_shares_a_long_prefix_needs_its_workspace(pkg, heads, kv, dim, dtype):
    """Where a prefix is computed once for the batch (re-reading it would
    cost over 48 MB) the workspace holds an own part of head_dim + 4 floats a
    row and head, and a call without it is refused before anything runs."""
    L = pkg.lib()
    kw = dict(n_head=heads, q_stride=heads * dim, out_stride=heads * dim, dtype=dtype, prefix_max_blocks=2000)

    def attn(n, **more):
        return _attn(pkg, dict(n_kv_head=kv, head_dim=dim), **{**kw, "n": n, "rows": n, **more})

    n = 64
    need = L.t3b_op_attention_shared_workspace(C.byref(attn(n)))
    assert (n - 1) * 2000 * 16 * 4 * kv * dim > 48e6
    assert need == n * heads * (dim + 4) * 4
    for bad in (dict(workspace=None), dict(workspace=PTR + 4), dict(workspace_bytes=need - 1), dict(workspace_bytes=0)):
        assert L.t3b_op_attention_shared(C.byref(attn(n, **bad)), None) == -1, bad
        assert "workspace" in pkg.last_error() and str(need) in pkg.last_error()
    # pointers are not looked at, and more requests never need less, on both sides of the 48 MB
    sizes = [L.t3b_op_attention_shared_workspace(C.byref(attn(m, q=None, workspace=None, prefix_max_blocks=200))) for m in (1, 2, 8, 64, 500, 65535)]
    assert sizes == sorted(sizes) and sizes[0] == 0 and sizes[-1] == 65535 * heads * (dim + 4) * 4
    # a prompt needs none
    assert L.t3b_op_attention_shared_workspace(C.byref(attn(n, rows=n + 1))) == 0


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(slots=None), dict(rows=-1), dict(dtype=30), dict(dtype=8),
                                 dict(stride=255), dict(stride=258), dict(k=PTR + 8), dict(v=PTR + 4)], ids=str)
def test_bad_appends_are_refused(pkg, bad):
    L = pkg.lib()
    d = dict(k=PTR, v=PTR, stride=256, slots=PTR, dtype=pkg.T3B_F32, rows=3)
    assert L.t3b_op_kv_append(C.byref(pkg.KvAppend(cache=_cache(pkg), **{**d, **bad})), None) == -1
    assert L.t3b_op_kv_append(None, None) == -1
    assert L.t3b_op_kv_append(C.byref(pkg.KvAppend(cache=_cache(pkg), **{**d, "rows": 0})), None) == 0


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=8193), dict(page_size=12), dict(page_size=512), dict(max_blocks=0),
                                 dict(max_blocks=1 << 27), dict(rows_cap=-1), dict(free_cap=-1), dict(len=None),
                                 dict(add=None), dict(free_pages=None), dict(n_free=None), dict(n_free_out=None),
                                 dict(table=None), dict(row_start=None), dict(n=8000, max_blocks=1 << 18)], ids=str)
def test_bad_plans_are_refused(pkg, bad):
    d = dict(n=4, page_size=16, max_blocks=8, rows_cap=10, len=PTR, add=PTR, release=PTR, free_pages=PTR, free_cap=9,
             n_free=PTR, n_free_out=PTR, table=PTR, row_start=PTR, row_req=PTR, row_pos=PTR, slots=PTR, len_out=PTR)
    L = pkg.lib()
    assert L.t3b_op_kv_plan(C.byref(pkg.KvPlan(**{**d, **bad})), None) == -1, bad
    assert "t3b_op_kv_plan" in pkg.last_error()
    assert L.t3b_op_kv_plan(None, None) == -1


def test_plan_reference_keeps_pages_apart():
    """Over many random steps no page is held twice and none is lost."""
    rng = np.random.default_rng(0)
    n, width, page = 7, 6, 8
    total = n * width - 5
    free, n_free = np.arange(total), total
    table, ln = np.full((n, width), -1), np.zeros(n, np.int64)
    for _ in range(200):
        rel = np.where(rng.random(n) < 0.2, ln, 0)
        ln = np.where(rel > 0, 0, ln)
        add = np.minimum(rng.integers(0, 20, n), width * page - ln)
        r = paged_ref.plan(ln, add, rel, page, table, free, n_free, 1000)
        if r is None:
            add[:] = 0
            r = paged_ref.plan(ln, add, rel, page, table, free, n_free, 1000)
        table, free, n_free, ln = r["table"], r["free"], r["n_free"], r["len_out"]
        held = [p for i in range(n) for p in table[i, :paged_ref.blocks(ln[i], page)]]
        assert sorted(held + list(free[:n_free])) == list(range(total))
        live = r["slots"][r["slots"] >= 0]
        assert len(set(live)) == add.sum() == r["row_start"][-1]


def test_attention_reference_is_a_softmax():
    """The reference of a batch with a prefix equals a dense softmax over the joined keys."""
    b = paged_ref.Batch("f32", [5, 0, 9], 4, 2, 64, 8, prefix_lens=[3], prefix_start=[0, 2], adds=[2, 0, 9], device="cpu")
    out, tol = b.reference()
    k, v = b.keys(0)
    assert k.shape == (8, 2, 64) and (tol > 0).all() and tol.max() < 1e-3
    q = b.q.double().reshape(11, 4, 64)
    w = torch.softmax(q[0, 3] @ k[:7, 1].T / 8, -1)              # row 0 of request 0: the prefix and 4 of its 5 keys
    assert torch.allclose(out[0, 3 * 64:], w @ v[:7, 1])
    w = torch.softmax(q[10, 0] @ b.own[2][0, :, 0].double().T / 8, -1)
    assert torch.allclose(out[10, :64], w @ b.own[2][1, :, 0].double())
