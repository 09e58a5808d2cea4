"""GPU tests of the paged operators (t3b_op_kv_plan, t3b_op_kv_append,
t3b_op_attention_shared, t3b_op_attention_shared_prompt) against plain
references in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import paged_ref
from paged_ref import Batch, blocks

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()


@pytest.fixture(autouse=True)
def _clean(pkg):
    """No error is left over from another test, and none is left behind."""
    pkg.lib().t3b_op_check(_stream())
    yield
    assert pkg.lib().t3b_op_check(_stream()) == 0, pkg.last_error()


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# --------------------------------------------------------------------------
# plan
# --------------------------------------------------------------------------

class Plan:
    """The device arrays of a t3b_kv_plan, with a guard value behind each."""

    def __init__(self, pkg, ln, add, release, page, table, free, n_free, rows_cap, in_place=False, want=True):
        self.n, self.width = table.shape
        self.in_ = dict(len=_i32(ln), add=_i32(add), table=_i32(np.r_[table.ravel(), 77]), free=_i32(np.r_[free, 77]), n_free=_i32([n_free]))
        self.release = None if release is None else _i32(release)
        self.out = {k: torch.full((m + 1,), 77, dtype=torch.int32, device="cuda")
                    for k, m in (("row_start", self.n + 1), ("row_req", rows_cap), ("row_pos", rows_cap), ("slots", rows_cap),
                                 ("len_out", self.n), ("n_free_out", 1))}
        self.in_place = in_place
        if in_place:
            self.out["len_out"], self.out["n_free_out"] = self.in_["len"], self.in_["n_free"]
        p = lambda t: t.data_ptr()  # noqa: E731
        self.d = pkg.KvPlan(n=self.n, page_size=page, max_blocks=self.width, rows_cap=rows_cap, len=p(self.in_["len"]),
                            add=p(self.in_["add"]), release=None if release is None else p(self.release),
                            free_pages=p(self.in_["free"]), free_cap=len(free), n_free=p(self.in_["n_free"]),
                            n_free_out=p(self.out["n_free_out"]), table=p(self.in_["table"]), row_start=p(self.out["row_start"]))
        if want:
            self.d.row_req, self.d.row_pos = p(self.out["row_req"]), p(self.out["row_pos"])
            self.d.slots, self.d.len_out = p(self.out["slots"]), p(self.out["len_out"])

    def got(self):
        o = {k: v.cpu().numpy().astype(np.int64) for k, v in self.out.items()}
        whole = ("len_out", "n_free_out") if self.in_place else ()
        for k in o:
            assert k in whole or o[k][-1] == 77, k                 # nothing is written past an array
        r = {k: o[k] if k in whole else o[k][:-1] for k in o}
        t, f = (self.in_[k].cpu().numpy().astype(np.int64) for k in ("table", "free"))
        assert t[-1] == 77 and f[-1] == 77
        return dict(r, table=t[:-1].reshape(self.n, self.width), free=f[:-1], n_free=int(r["n_free_out"][0]))


def _same(got, ref):
    for k, v in ref.items():
        assert np.array_equal(np.asarray(got[k]), np.asarray(v)), k


def _random_step(rng, n, page, width, readmit):
    total = n * width
    ids = rng.permutation(total)
    used = rng.integers(0, width * page // 2, n)
    kind = rng.integers(0, 4, n)                                   # decode, prompt, idle, finished
    ln = np.where(kind == 1, 0, used)
    release = np.where(kind == 3, used, 0)
    ln = np.where(release > 0, 0, ln)
    add = np.select([kind == 0, kind == 1], [np.ones(n, int), rng.integers(0, width * page + 1, n)], 0)
    if readmit:
        add = np.where(release > 0, rng.integers(0, width * page + 1, n), add)
    add = np.minimum(add, width * page - ln)
    table, at = np.full((n, width), -1), 0
    for i in range(n):
        b = blocks(ln[i] if release[i] == 0 else release[i], page)
        table[i, :b] = ids[at:at + b]
        at += b
    free = np.r_[ids[at:], np.full(at, -5)]
    return ln, add, release, table, free, total - at


@pytest.mark.parametrize("n,page,width", [(1, 8, 1), (1, 256, 3), (2, 16, 4), (31, 8, 5), (64, 16, 40), (1000, 32, 6),
                                          (1024, 8, 3), (1025, 64, 4), (8192, 16, 3)])
@pytest.mark.parametrize("readmit", [False, True])
def test_plan_matches_its_definition(pkg, n, page, width, readmit):
    rng = np.random.default_rng(n + page)
    for trial in range(3):
        ln, add, release, table, free, n_free = _random_step(rng, n, page, width, readmit)
        cap = int(add.sum()) + [0, 1, 700][trial]
        p = Plan(pkg, ln, add, release, page, table, free, n_free, cap, in_place=trial == 1)
        pkg.check(pkg.lib().t3b_op_kv_plan(C.byref(p.d), _stream()))
        ref = paged_ref.plan(ln, add, release, page, table, free, n_free, cap)
        assert ref is not None
        _same(p.got(), ref)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,page,width,rows_cap", [(700, 16, 9, None), (3000, 8, 8, None), (300, 32, 20, 100003), (5, 256, 40, 40000)])
def test_plan_of_many_rows(pkg, n, page, width, rows_cap, in_place):
    """Steps of tens of thousands of rows, with in-place lengths and room to spare."""
    rng = np.random.default_rng(n)
    ln, add, release, table, free, n_free = _random_step(rng, n, page, width, True)
    cap = rows_cap or int(add.sum())
    assert 16384 < cap and add.sum() <= cap
    p = Plan(pkg, ln, add, release, page, table, free, n_free, cap, in_place=in_place)
    pkg.check(pkg.lib().t3b_op_kv_plan(C.byref(p.d), _stream()))
    _same(p.got(), paged_ref.plan(ln, add, release, page, table, free, n_free, cap))
    # one page too few: nothing changes, all of the large row maps are -1
    q = Plan(pkg, ln, add, release, page, table, free, 0, cap, in_place=in_place)
    if paged_ref.plan(ln, add, release, page, table, free, 0, cap) is None:
        pkg.check(pkg.lib().t3b_op_kv_plan(C.byref(q.d), _stream()))
        assert pkg.lib().t3b_op_check(_stream()) == -5
        got = q.got()
        assert all((got[k] == -1).all() for k in ("row_req", "row_pos", "slots")) and np.array_equal(got["table"], table)


def test_plan_without_the_optional_arrays(pkg):
    rng = np.random.default_rng(5)
    ln, add, _, table, free, n_free = _random_step(rng, 40, 16, 6, False)
    p = Plan(pkg, ln, add, None, 16, table, free, n_free, int(add.sum()), want=False)
    pkg.check(pkg.lib().t3b_op_kv_plan(C.byref(p.d), _stream()))
    ref = paged_ref.plan(ln, add, None, 16, table, free, n_free, int(add.sum()))
    got = p.got()
    _same({k: got[k] for k in ("table", "free", "n_free", "row_start")},
          {k: ref[k] for k in ("table", "free", "n_free", "row_start")})
    assert (got["row_req"] == 77).all() and (got["len_out"] == 77).all()


def test_plan_without_row_maps_does_not_look_for_rows(pkg):
    """Without row_req, row_pos and slots no row is mapped: ids of pages that
    are held already, which only the maps need, are not looked at."""
    rng = np.random.default_rng(6)
    ln, add, _, table, free, n_free = _random_step(rng, 40, 16, 6, False)
    ln[0], add[0], table[0, 0] = 5, 1, -9
    p = Plan(pkg, ln, add, None, 16, table, free, n_free, int(add.sum()), want=False)
    pkg.check(pkg.lib().t3b_op_kv_plan(C.byref(p.d), _stream()))
    pkg.check(pkg.lib().t3b_op_check(_stream()))
    ref = paged_ref.plan(ln, add, None, 16, table, free, n_free, int(add.sum()))
    got = p.got()
    _same({k: got[k] for k in ("table", "free", "n_free", "row_start")},
          {k: ref[k] for k in ("table", "free", "n_free", "row_start")})


BAD_STEPS = {
    "negative length": dict(len={3: -1}), "negative new": dict(add={0: -2}), "negative release": dict(release={2: -7}),
    "past the table": dict(add={1: 97}), "far past the table": dict(add={1: 2 ** 31 - 1}), "release past the table": dict(release={2: 97}, len={2: 0}),
    "release of a live slot": dict(release={3: 5}), "too few pages": dict(n_free=2), "too few rows": dict(rows=19),
    "stack below zero": dict(n_free=-1), "stack past its end": dict(n_free=1000),
    "no room for returned pages": dict(free_cap=29, release={2: 90}, len={2: 0}, add={2: 0}),
}


@pytest.mark.parametrize("bad", list(BAD_STEPS), ids=str)
@pytest.mark.parametrize("in_place", [False, True])
def test_a_step_that_does_not_fit_changes_nothing(pkg, bad, in_place):
    n, page, width = 5, 16, 6
    ln, add, release = np.array([0, 16, 0, 5, 33]), np.array([17, 1, 0, 1, 1]), np.zeros(5, int)
    what = BAD_STEPS[bad]
    for name, arr in (("len", ln), ("add", add), ("release", release)):
        for i, v in what.get(name, {}).items():
            arr[i] = v
    table = np.full((n, width), -1)
    table[1, :1], table[2], table[3, :1], table[4, :3] = 40, np.arange(50, 56), 41, [42, 43, 44]
    free = np.arange(30)
    p = Plan(pkg, ln, add, release, page, table, free[:what.get("free_cap", 30)], what.get("n_free", 28), what.get("rows", 40), in_place)
    assert paged_ref.plan(ln, add, release, page, table, free[:what.get("free_cap", 30)], what.get("n_free", 28), what.get("rows", 40)) is None
    pkg.check(pkg.lib().t3b_op_kv_plan(C.byref(p.d), _stream()))
    assert pkg.lib().t3b_op_check(_stream()) == -5
    assert "range" in pkg.last_error() or "out-of-pages" in pkg.last_error()
    got = p.got()
    _same({k: got[k] for k in ("table", "free", "n_free")}, dict(table=table, free=free[:what.get("free_cap", 30)], n_free=what.get("n_free", 28)))
    assert (got["row_start"] == 0).all() and np.array_equal(got["len_out"], ln)
    assert all((got[k] == -1).all() for k in ("row_req", "row_pos", "slots"))


def test_captured_plan_evolves_its_state(pkg):
    """A captured step with in-place lengths and stack, replayed: each replay
    is the next step; pages run out at the right one."""
    n, page, width = 33, 8, 4
    ln, add = np.arange(n) % 5, np.ones(n, int)
    table, free = np.full((n, width), -1), np.arange(70)[::-1].copy()
    table[ln > 0, 0] = 100 + np.arange(n)[ln > 0]
    p = Plan(pkg, ln, add, None, page, table, free, 70, 64, in_place=True)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        pkg.check(pkg.lib().t3b_op_kv_plan(C.byref(p.d), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    state = dict(len_out=ln, table=table, free=free, n_free=70)
    for step in range(25):
        ref = paged_ref.plan(state["len_out"], add, None, page, state["table"], state["free"], state["n_free"], 64)
        g.replay()
        torch.cuda.synchronize()
        if ref is None:
            assert pkg.lib().t3b_op_check(_stream()) == -5
            break
        _same(p.got(), ref)
        state = ref
    assert step > 10 and ref is None


# --------------------------------------------------------------------------
# append
# --------------------------------------------------------------------------

@pytest.mark.parametrize("src,cache", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("rows,kv,dim,page,pad,gap", [(1, 1, 64, 8, 0, 0), (5, 16, 64, 16, 0, 0), (333, 3, 128, 32, 24, 8),
                                                      (2049, 8, 128, 64, 0, 8 * 64 * 128), (64, 2, 64, 256, 8, 0), (9001, 8, 64, 16, 16, 0)])
def test_append_matches_its_definition(pkg, src, cache, rows, kv, dim, page, pad, gap):
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    ids = {"f32": 0, "f16": 1, "bf16": 30}
    g = torch.Generator().manual_seed(rows)
    n_pages = blocks(rows, page) + 3
    stride = kv * page * dim + gap
    pool = torch.randn(2, n_pages * stride, generator=g).to(t[cache]).cuda()
    before = pool.clone()
    new = (torch.randn(2, rows, kv * dim + pad, generator=g) * 50).to(t[src]).cuda()
    if src == "f32":
        new[0, 0, :4] = torch.tensor([7e4, -1e30, float("inf"), float("nan")])   # past f16, and not finite
    slots = torch.randperm(n_pages * page, generator=g)[:rows].to(torch.int32)
    if rows > 4:
        slots[1::5] = -1
    sd = slots.cuda()
    c = pkg.PagedKv(k=pool[0].data_ptr(), v=pool[1].data_ptr(), page_stride=stride, dtype=ids[cache], n_pages=n_pages,
                    n_kv_head=kv, page_size=page, head_dim=dim)
    a = pkg.KvAppend(cache=c, k=new[0].data_ptr(), v=new[1].data_ptr(), stride=kv * dim + pad, slots=sd.data_ptr(),
                     dtype=ids[src], rows=rows)
    pkg.check(pkg.lib().t3b_op_kv_append(C.byref(a), _stream()))
    for x in range(2):
        want = before[x].cpu().clone()
        view = want.view(n_pages, stride)[:, :kv * page * dim].view(n_pages, kv, page, dim)
        for r in range(rows):
            s = int(slots[r])
            if s >= 0:
                view[s // page, :, s % page] = new[x, r, :kv * dim].cpu().to(t[cache]).view(kv, dim)
        assert torch.equal(pool[x].cpu().view(torch.int16), want.view(torch.int16)) or \
            torch.allclose(pool[x].cpu(), want, rtol=0, atol=0, equal_nan=True)


def test_append_reports_a_slot_past_the_pool(pkg):
    pool = torch.zeros(2, 4 * 16 * 64, dtype=torch.float16, device="cuda")
    new = torch.ones(2, 3, 64, device="cuda")
    slots = _i32([3, 64, 2 ** 31 - 1])
    c = pkg.PagedKv(k=pool[0].data_ptr(), v=pool[1].data_ptr(), dtype=1, n_pages=4, n_kv_head=1, page_size=16, head_dim=64)
    a = pkg.KvAppend(cache=c, k=new[0].data_ptr(), v=new[1].data_ptr(), stride=64, slots=slots.data_ptr(), dtype=0, rows=3)
    pkg.check(pkg.lib().t3b_op_kv_append(C.byref(a), _stream()))
    assert pkg.lib().t3b_op_check(_stream()) == -5
    assert "page-out-of-range" in pkg.last_error()
    assert float(pool.sum()) == 2 * 64


# --------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------

def _attend(pkg, b, **kw):
    d = b.desc(pkg, **kw)
    f = pkg.lib().t3b_op_attention_shared if b.adds is None else pkg.lib().t3b_op_attention_shared_prompt
    pkg.check(f(C.byref(d), _stream()))
    torch.cuda.synchronize()
    return d


def _close(b, out=None, scale=None, skip=()):
    ref, tol = b.reference(scale)
    w = b.heads * b.dim
    got = (b.out_all if out is None else out)[:b.rows, :w].cpu().double()
    keep = torch.ones(b.rows, dtype=torch.bool)
    for i in skip:
        keep[b.starts[i]:b.starts[i + 1]] = False
    got, ref, tol = got[keep], ref[keep], tol[keep]
    assert torch.isfinite(got).all()
    over = (got - ref).abs() / tol
    assert over.max() <= 1, (float(over.max()), int(over.argmax()))
    if b.kind == "f32" and ref.numel() and ref.norm() > 0:
        # errors of 22-bit factors and 32-bit sums do not add up in one direction
        assert (got - ref).norm() / ref.norm() < 3e-6
    # rows behind the last one and the padding of each row stay as they were
    if out is None:
        assert (b.out_all[b.rows:] == -7).all() and (b.out_all[:b.rows, w:] == -7).all()


LAYOUTS = [(1, 1, 64, 16), (4, 4, 64, 8), (16, 16, 64, 16), (8, 2, 128, 32), (6, 2, 64, 64), (16, 1, 128, 128),
           (7, 1, 64, 256), (5, 5, 128, 16), (10, 2, 128, 64), (24, 2, 64, 32)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("heads,kv,dim,page", LAYOUTS)
def test_decode_attention_matches_fp64(pkg, kind, heads, kv, dim, page, share):
    lens = [1, 0, page - 1, page, page + 1, 2 * page + 3, 63, 64, 65, 300, 129]
    for prefix, start in (([], None), ([1], [0, 11]), ([page + 3, 0, 200], [1, 4, 6, 10]), ([64, 128], [0, 1, 11])):
        b = Batch(kind, lens, heads, kv, dim, page, prefix, start, seed=heads * 7 + len(prefix), gap=8 * len(prefix), q_pad=8 * len(prefix), share=share)
        d = _attend(pkg, b)
        assert (d.workspace_bytes > 0) == (share and len(prefix) > 0)
        _close(b)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,heads,kv,dim,page,prefix,lo,hi", [
    (1, 16, 16, 64, 16, 376, 1, 1), (2, 16, 16, 64, 16, 376, 88, 1088), (3, 4, 4, 64, 16, 1, 1500, 1501), (1, 8, 8, 128, 64, 0, 5000, 5001),
    (130, 4, 2, 64, 16, 77, 1, 40), (65, 32, 8, 128, 32, 1000, 1, 90), (300, 2, 1, 64, 8, 513, 0, 30), (1, 1, 1, 128, 16, 4000, 0, 1)])
def test_decode_attention_sizes(pkg, kind, n, heads, kv, dim, page, prefix, lo, hi):
    rng = np.random.default_rng(n + heads)
    for share in (False, True):
        b = Batch(kind, rng.integers(lo, hi + 1, n).tolist(), heads, kv, dim, page, [prefix], [0, n], seed=n, share=share)
        _attend(pkg, b)
        _close(b)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim,page", LAYOUTS)
def test_prompt_attention_matches_fp64_ragged(pkg, kind, heads, kv, dim, page):
    adds = [1, 0, page, 33, 5, 0, 130, 64]
    lens = [1, 0, page, 50, 5 + page, 7, 130, 300]
    for prefix, start in (([], None), ([page + 3, 0, 200], [0, 2, 3, 7]), ([65], [0, 8])):
        b = Batch(kind, lens, heads, kv, dim, page, prefix, start, adds=adds, seed=heads * 3 + len(prefix), gap=8, q_pad=16)
        _attend(pkg, b)
        _close(b)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("adds,past,heads,kv,dim,page,prefix", [
    ([88, 120, 20], [0, 0, 0], 16, 16, 64, 16, 376), ([700, 1], [333, 2000], 4, 2, 128, 64, 129), ([1000], [0], 2, 1, 64, 32, 0),
    ([3], [4000], 8, 8, 64, 16, 500), ([1] * 150, [7] * 150, 4, 1, 128, 16, 40), ([257, 256, 255], [1, 0, 127], 3, 3, 128, 128, 1)])
def test_prompt_attention_sizes(pkg, kind, adds, past, heads, kv, dim, page, prefix):
    b = Batch(kind, [a + p for a, p in zip(adds, past)], heads, kv, dim, page, [prefix], [0, len(adds)], adds=adds, seed=adds[0])
    _attend(pkg, b)
    _close(b)


@pytest.mark.parametrize("prompt,share", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("kind,q_scale", [("f32", 3e4), ("f32", 1e-6), ("f16", 100.0), ("bf16", 300.0), ("f32", 0.0)])
def test_large_and_small_queries(pkg, kind, q_scale, prompt, share):
    """Scores of thousands (the softmax picks one key) and of nothing (it averages)."""
    lens = [40, 200, 1]
    b = Batch(kind, lens, 4, 2, 64, 16, [100], [0, 3], adds=[40, 30, 1] if prompt else None, seed=3, q_scale=q_scale,
              share=share)
    _attend(pkg, b)
    ref, tol = b.reference()
    got = b.out_all[:b.rows].cpu().double()
    assert torch.isfinite(got).all()
    assert ((got - ref).abs() <= tol).all()


@pytest.mark.parametrize("prompt,share", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("scale", [0.3, -0.125])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_scale_argument(pkg, prompt, share, scale, kind):
    b = Batch(kind, [40, 100], 4, 2, 64, 16, [50], [0, 2], adds=[40, 30] if prompt else None, seed=4, share=share)
    d = b.desc(pkg)
    d.scale = scale
    f = pkg.lib().t3b_op_attention_shared_prompt if prompt else pkg.lib().t3b_op_attention_shared
    pkg.check(f(C.byref(d), _stream()))
    torch.cuda.synchronize()
    _close(b, scale=scale)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind,prefix", [("f32", 70), ("f16", 70), ("bf16", 70), ("f32", 2000), ("bf16", 2000)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_values_of_later_tokens_stay_there(pkg, kind, prefix, value, in_place):
    """A NaN or infinity in the K or V of a token reaches the rows that see
    it, and no row before it; also where out is q, and where the keys are
    split over CTAs (the long prefix)."""
    b = Batch(kind, [100, 30], 6, 2, 64, 16, [prefix], [0, 2], adds=[60, 30], seed=31)
    q = b.q_all.clone()
    ref, tol = b.reference()
    key = 85                                                      # own key 85 of request 0: rows from 45 on see it
    slot = int(b.table[0, key // 16]), key % 16
    for pool, dims in ((b.v, slice(3, 5)), (b.k, slice(9, 10))):
        view = pool.view(b.n_pages, b.kv, 16, 64)
        old = view[slot[0], 1, slot[1]].clone()
        view[slot[0], 1, slot[1], dims] = value                   # kv head 1: query heads 3, 4 and 5
        b.out_all.fill_(-7)
        _attend(pkg, b, out=b.q_all if in_place else None)
        view[slot[0], 1, slot[1]] = old
        got = (b.q_all if in_place else b.out_all)[:90].cpu().double()
        b.q_all.copy_(q)
        clean = torch.ones_like(ref, dtype=torch.bool)
        clean[45:60, 3 * 64:] = False
        assert ((got - ref).abs() <= tol)[clean].all()
        if pool is b.v:
            hit = got[45:60].view(15, 6, 64)[:, 3:, dims]
            assert (~torch.isfinite(hit)).all()
            if value != value:
                assert torch.isnan(hit).all()


@pytest.mark.parametrize("prompt,share", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_output_in_place_of_q(pkg, prompt, share, kind):
    b = Batch(kind, [40, 3, 700], 8, 4, 64, 16, [300], [0, 2], adds=[40, 2, 300] if prompt else None, seed=5, share=share)
    out = b.q_all.clone()
    b.q_all, b.q = out, out[:, :8 * 64]
    ref, tol = b.reference()
    _attend(pkg, b, out=out)
    assert ((out.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("prompt,shared", [(False, False), (False, True), (True, False)])
def test_bad_lengths_and_pages_are_reported(pkg, prompt, shared):
    """A request with a bad length leaves its rows unwritten, a bad page's
    keys count as absent, and the other requests are right; also where the
    prefix is computed once for the batch (long enough for that)."""
    lens, adds = [40, 30, 20, 50], [3, 30, 2, 1]
    for what in ("long", "negative", "page", "prefix"):
        b = Batch("f32", lens, 4, 2, 64, 16, [20, 20], [0, 2, 4], adds=adds if prompt else None, seed=6, share=shared)
        skip = [1]
        assert (b.desc(pkg).workspace_bytes > 0) == shared
        if what == "long":
            b.len[1] = b.table.shape[1] * 16 + 1
        elif what == "negative":
            b.len[1] = -3
        elif what == "prefix":
            b.plen[0], skip = 16 * b.ptable.shape[1] + 1, [0, 1]
        else:
            b.table[1, 0] = [b.n_pages, -1][prompt]
        _attend(pkg, b)
        assert pkg.lib().t3b_op_check(_stream()) == -5
        assert ("page-out-of-range" if what == "page" else "length-out-of-range") in pkg.last_error()
        _close(b, skip=skip)
        rows = b.out_all[b.starts[1]:b.starts[2]]
        if what == "page":                                        # the other 14 own keys and the prefix are left
            b.own[1] = b.own[1][:, 16:]
            if not prompt:
                _close(b)
        else:
            assert (rows == -7).all()


def test_more_rows_than_keys_are_reported(pkg):
    b = Batch("f32", [4, 9], 4, 2, 64, 16, [20], [0, 2], adds=[4, 9], seed=6)
    b.len[0] = 3
    _attend(pkg, b)
    assert pkg.lib().t3b_op_check(_stream()) == -5
    _close(b, skip=[0])
    assert (b.out_all[:4] == -7).all()


def test_a_workspace_of_another_call_leaves_no_trace(pkg):
    """Two batches through one workspace, one after the other and back."""
    x = Batch("f32", [40] * 20, 4, 4, 64, 16, [300], [0, 20], seed=7, share=True)
    y = Batch("f32", [3, 500, 60], 4, 4, 64, 16, [20, 700], [0, 1, 3], seed=8, share=True)
    dx, dy = x.desc(pkg), y.desc(pkg)
    assert dx.workspace_bytes > 0 and dy.workspace_bytes > 0
    big = torch.empty(max(dx.workspace_bytes, dy.workspace_bytes, 16), dtype=torch.uint8, device="cuda").fill_(0xFF)
    for b, d in ((x, dx), (y, dy), (x, dx)):
        d.workspace, d.workspace_bytes = big.data_ptr(), big.numel()
        b.out_all.fill_(-7)
        pkg.check(pkg.lib().t3b_op_attention_shared(C.byref(d), _stream()))
        torch.cuda.synchronize()
        _close(b)


@pytest.mark.parametrize("prompt,share", [(False, False), (False, True), (True, False)])
def test_repeated_calls_give_the_same_bits(pkg, prompt, share):
    b = Batch("f32", [40, 900, 7, 333], 8, 8, 64, 16, [377], [0, 4], adds=[40, 60, 7, 100] if prompt else None, seed=9, share=share)
    _attend(pkg, b)
    first = b.out_all.clone()
    for _ in range(5):
        _attend(pkg, b)
        assert torch.equal(b.out_all, first)


@pytest.mark.parametrize("kind", ["prompt", "decode", "shared"])
def test_two_calls_at_once_on_two_streams(pkg, kind):
    bs = [Batch("f32", [200, 30, 77] * 8, 8, 8, 64, 16, [377], [0, 24], adds=[150, 30, 1] * 8 if kind == "prompt" else None,
                seed=10 + i, share=kind == "shared") for i in range(2)]
    ds = [b.desc(pkg) for b in bs]
    f = pkg.lib().t3b_op_attention_shared_prompt if kind == "prompt" else pkg.lib().t3b_op_attention_shared
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for d, s in zip(ds, streams):
            pkg.check(f(C.byref(d), C.c_void_p(s.cuda_stream)))
    torch.cuda.synchronize()
    for b in bs:
        _close(b)


@pytest.mark.parametrize("dim,prompt,share", [(64, False, False), (128, False, True), (128, True, False)])
def test_pages_past_2_to_the_31_elements(pkg, dim, prompt, share):
    """Page offsets that do not fit 32 bits: K and V of 4.4 GB each."""
    page, kv = 64, 8
    at = (1 << 31) // (page * kv * dim) + 3
    b = Batch("f16", [70, 200], 8, kv, dim, page, [300], [0, 2], adds=[70, 10] if prompt else None, seed=11, pages_at=at, share=share)
    assert b.k.numel() > 1 << 31
    _attend(pkg, b)
    _close(b)


@pytest.mark.parametrize("mode", ["decode", "shared", "prompt"])
def test_more_than_32_prefixes(pkg, mode):
    rng = np.random.default_rng(13)
    start = np.cumsum(np.r_[1, rng.integers(0, 4, 41)]).tolist()   # some prefixes have no request, some requests no prefix
    n = start[-1] + 2
    adds = rng.integers(0, 9, n).tolist() if mode == "prompt" else None
    lens = [int(x) + (a if adds else 0) for x, a in zip(rng.integers(0, 60, n), adds or [0] * n)]
    b = Batch("f32", lens, 4, 2, 64, 16, rng.integers(0, 150, 41).tolist(), start, adds=adds, seed=14, share=mode == "shared")
    _attend(pkg, b)
    _close(b)


@pytest.mark.parametrize("mode", ["decode", "prompt"])
def test_as_many_requests_as_allowed(pkg, mode):
    """65535 requests of one key each: every row is that key's V."""
    n, page = 65535, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.randn(n, 1, page, 64, generator=g, device="cuda").half()
    v = torch.randn(n, 1, page, 64, generator=g, device="cuda").half()
    q = torch.randn(n, 64, generator=g, device="cuda")
    out = torch.full((n, 64), -7.0, device="cuda")
    table, ln = torch.randperm(n, generator=g, device="cuda").to(torch.int32), torch.ones(n, dtype=torch.int32, device="cuda")
    starts = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    d = pkg.SharedAttn(cache=pkg.PagedKv(k=k.data_ptr(), v=v.data_ptr(), dtype=1, n_pages=n, n_kv_head=1, page_size=page, head_dim=64),
                       q=q.data_ptr(), out=out.data_ptr(), q_stride=64, out_stride=64, len=ln.data_ptr(), table=table.data_ptr(),
                       row_start=starts.data_ptr(), dtype=0, n_head=1, n=n, rows=n, max_blocks=1)
    f = pkg.lib().t3b_op_attention_shared if mode == "decode" else pkg.lib().t3b_op_attention_shared_prompt
    pkg.check(f(C.byref(d), _stream()))
    want = v[table.long(), 0, 0].float()
    assert ((out - want).abs() <= want.abs() * 2.0 ** -20).all()      # one key: its weight is 1 to a few roundings


def test_rows_without_a_request_stay_as_they_were(pkg):
    """A prompt call whose requests bring no rows, with room for some."""
    b = Batch("f32", [5, 0, 3], 4, 2, 64, 16, [20], [0, 3], adds=[0, 0, 0], seed=15)
    b.q_all = torch.zeros(7, 256, device="cuda")
    b.q = b.q_all
    out = torch.full((7, 256), -7.0, device="cuda")
    _attend(pkg, b, out=out, rows=7)
    assert (out == -7).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_calls_one_after_the_other_without_waiting(pkg, kind):
    """Two batches take turns on one stream through one workspace, nothing
    waited for in between; what each left is copied right behind it."""
    bs = [Batch(kind, lens, 8, 4, 64, 16, [p], [0, len(lens)], seed=16 + p, share=True)
          for lens, p in (([40, 3, 200, 77] * 9, 700), ([5, 600], 90))]
    ds = [b.desc(pkg) for b in bs]
    big = torch.empty(max(d.workspace_bytes for d in ds), dtype=torch.uint8, device="cuda").fill_(0xFF)
    left = []
    for d in ds:
        d.workspace, d.workspace_bytes = big.data_ptr(), big.numel()
    for _ in range(25):
        for b, d in zip(bs, ds):
            b.out_all.fill_(-7)
            pkg.check(pkg.lib().t3b_op_attention_shared(C.byref(d), _stream()))
            left.append(b.out_all.clone())
    torch.cuda.synchronize()
    for b in bs:
        _close(b)
    assert all(torch.equal(x, left[i % 2]) for i, x in enumerate(left))


def test_append_right_behind_a_large_plan(pkg):
    """The row maps of a large step are there when the append that follows reads them."""
    rng = np.random.default_rng(17)
    n, page, width = 900, 16, 12
    ln, add, release, table, free, n_free = _random_step(rng, n, page, width, True)
    cap = int(add.sum()) + 100
    ref = paged_ref.plan(ln, add, release, page, table, free, n_free, cap)
    p = Plan(pkg, ln, add, release, page, table, free, n_free, cap, in_place=True)
    assert cap > 16384
    rows = torch.randn(2, cap, 64, device="cuda")
    pool = torch.zeros(2, n * width, 1, page, 64, dtype=torch.float16, device="cuda")
    a = pkg.KvAppend(cache=pkg.PagedKv(k=pool[0].data_ptr(), v=pool[1].data_ptr(), dtype=1, n_pages=n * width, n_kv_head=1, page_size=page,
                                       head_dim=64),
                     k=rows[0].data_ptr(), v=rows[1].data_ptr(), stride=64, slots=p.out["slots"].data_ptr(), dtype=0, rows=cap)
    pkg.check(pkg.lib().t3b_op_kv_plan(C.byref(p.d), _stream()))
    pkg.check(pkg.lib().t3b_op_kv_append(C.byref(a), _stream()))
    torch.cuda.synchronize()
    want = torch.zeros(2, n * width * page, 64, dtype=torch.float16)
    live = torch.from_numpy(ref["slots"] >= 0)
    want[:, torch.from_numpy(ref["slots"][ref["slots"] >= 0])] = rows.cpu()[:, live].half()
    assert torch.equal(pool.cpu().view(2, -1, 64), want)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("what", ["no request has a prefix", "every prefix is refused"])
def test_what_follows_a_shared_call_finds_its_output(pkg, what, graph):
    """The two-kernel way of a decode call where no row tile has work (all
    prefix ranges empty, or all prefix lengths refused): a projection queued
    right behind it, whose kernel may start early, reads what the call wrote."""
    H, n = 16, 3
    b = Batch("f32", [3000, 2000, 6000], H, H, 64, 16, [20, 20], [0, 0, 0] if "no" in what else [0, 1, 2], seed=41, share=True)
    d = b.desc(pkg)
    assert d.workspace_bytes > 0
    refused = [] if "no" in what else [0, 1]
    if refused:
        b.plen.fill_(16 * b.ptable.shape[1] + 1)
    L, N = pkg.lib(), 256
    w = (torch.randn(N, H * 64, generator=torch.Generator().manual_seed(2)) * 0.05).half().numpy()
    wd = torch.empty(N * L.t3b_op_row_bytes(1, H * 64), dtype=torch.uint8, device="cuda")
    pkg.check(L.t3b_op_repack(1, w.ctypes.data, N, H * 64, C.c_void_p(wd.data_ptr())))
    y = torch.zeros(n, N, device="cuda")

    def project():
        pkg.check(L.t3b_op_gemv(1, C.c_void_p(wd.data_ptr()), N, H * 64, C.c_void_p(b.out_all.data_ptr()), n, None, None, 0.0, None, None, 0,
                                C.c_void_p(y.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream)))

    def both():
        pkg.check(L.t3b_op_attention_shared(C.byref(d), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        project()

    pkg.check(L.t3b_op_attention_shared(C.byref(d), _stream()))
    torch.cuda.synchronize()
    project()
    want = y.clone()
    torch.cuda.synchronize()
    run = both
    if graph:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            both()
        run = g.replay
    for _ in range(20):
        b.out_all.fill_(-7)
        y.zero_()
        run()
        left = b.out_all.clone()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert torch.equal(left, b.out_all)
    if refused:
        assert L.t3b_op_check(_stream()) == -5
        assert (b.out_all[:2] == -7).all()
    _close(b, skip=refused)


@pytest.mark.parametrize("prompt,share", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("kind,prefix", [("f32", 70), ("bf16", 70), ("f32", 2000), ("f16", 2000)])
@pytest.mark.parametrize("where", ["q", "first prefix key", "first own key", "a prefix value"])
def test_nan_reaches_every_row_that_sees_it(pkg, kind, prefix, prompt, share, where):
    """A NaN in a query or in the K of the first key makes the whole output of
    the rows and heads that meet it NaN, whatever the order of the keys, and
    one in a V its element; the other rows and heads stay right."""
    b = Batch(kind, [100, 30, 40], 6, 2, 64, 16, [prefix], [0, 2], adds=[60, 30, 7] if prompt else None, seed=37, share=share)
    ref, tol = b.reference()
    hit = torch.zeros(b.rows, 6, 64, dtype=torch.bool)
    k, v = (x.view(b.n_pages, b.kv, 16, 64) for x in (b.k, b.v))
    nan = float("nan")
    if where == "q":
        b.q[b.starts[1], 4 * 64 + 9] = nan                        # one row, one head
        hit[b.starts[1], 4] = True
    elif where == "first prefix key":
        k[int(b.ptable[0, 0]), 1, 0, 5] = nan                     # kv head 1: query heads 3, 4 and 5
        hit[:b.starts[2], 3:] = True
    elif where == "first own key":
        k[int(b.table[1, 0]), 1, 0, 5] = nan
        hit[b.starts[1]:b.starts[2], 3:] = True
    else:
        v[int(b.ptable[0, 0]), 1, 3, 5] = nan
        hit[:b.starts[2], 3:, 5] = True
    _attend(pkg, b)
    got = b.out_all[:b.rows].cpu().double()
    hit = hit.view(b.rows, -1)
    assert torch.isnan(got[hit]).all()
    assert ((got - ref).abs() <= tol)[~hit].all()


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("what", ["past the rows", "all past the rows", "backwards", "below zero"])
def test_row_ranges_out_of_bounds_are_reported_wherever_they_are(pkg, heads, kv, dim, what):
    """A bad row range is reported, and the other requests are right, also
    behind the first requests and behind the last row tile."""
    n, at = 100, 70
    adds = [1 + i % 3 for i in range(n)]
    b = Batch("f16", [5 + a for a in adds], heads, kv, dim, 16, [20], [0, n], adds=adds, seed=38)
    rows = b.rows
    if what == "past the rows":                                   # rows that the call does not have: the last 30 requests'
        rows, skip = b.starts[at], range(at, n)
    elif what == "all past the rows":
        rows, skip = 1, range(1, n)
    elif what == "backwards":                                     # request 70 ends before it begins, 71 has a row of 69's too
        b.row_start[at + 1] = b.starts[at] - 1
        skip = [at - 1, at, at + 1]
    else:
        b.row_start[0], skip = -2, [0]
    _attend(pkg, b, rows=rows)
    assert pkg.lib().t3b_op_check(_stream()) == -5
    assert "length-out-of-range" in pkg.last_error()
    _close(b, skip=skip)
    if what in ("past the rows", "all past the rows", "below zero"):
        assert all((b.out_all[b.starts[i]:b.starts[i + 1]] == -7).all() for i in skip)


def test_prefix_ranges_out_of_bounds_are_reported_wherever_they_are(pkg):
    """The same for the prefixes of a decode batch: the last of 70 has
    requests that the call does not have."""
    G = 70
    start = list(range(0, 2 * G + 1, 2))
    b = Batch("f32", [9] * (2 * G), 4, 4, 64, 16, [20] * G, start, seed=39, share=True)
    b.pstart[G] = 2 * G + 1
    _attend(pkg, b)
    assert pkg.lib().t3b_op_check(_stream()) == -5
    assert "length-out-of-range" in pkg.last_error()
    _close(b, skip=[2 * G - 2, 2 * G - 1])


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("room", [-1, -(1 << 31), 1 << 27, (1 << 31) - 1])
def test_prefix_room_counts_for_nothing_without_prefixes(pkg, prompt, room):
    b = Batch("f32", [40, 3, 70], 4, 2, 64, 16, adds=[4, 3, 70] if prompt else None, seed=40)
    d = b.desc(pkg)
    d.prefix_max_blocks = room
    f = pkg.lib().t3b_op_attention_shared_prompt if prompt else pkg.lib().t3b_op_attention_shared
    pkg.check(f(C.byref(d), _stream()))
    torch.cuda.synchronize()
    _close(b)


@pytest.mark.parametrize("mode", ["prompt", "shared", "own"])
@pytest.mark.parametrize("dim", [64, 128])
def test_f32_over_8000_keys_of_one_cta(pkg, mode, dim):
    """F32 outputs stay within 1e-6 of 64 bits (2-norm) where one CTA takes
    all of 8000 keys: 5 row tiles of 16 heads are more than half of 148 SMs
    and 40 requests of 16 heads more than four times as many, so nothing is
    split.  What is off in 32 bits: weights of 22 bits, 2^-22 / sqrt(3) =
    1.4e-7; exponents of up to 2^3 held to 2^-22, 2e-7; scores, whose sum of
    dim / 16 steps loses up to 2^-24 of itself at each, 5e-7 at 128 dimensions
    times a weighted spread of about 1 between the scores; at most 500
    roundings of O, sqrt(500) 2^-25 = 7e-7 where they all met its final size
    and half of that as it grows.  Squares added: 7e-7.  One running sum of
    the tensor cores, which is cut off at each step, comes to 2.5e-6 and more."""
    G, H = 5, 16
    adds = [3] * G if mode == "prompt" else None
    per = 1 if mode == "prompt" else 2
    if mode == "own":
        b = Batch("f32", [8000] * 40, H, H, dim, 64, seed=42)
    else:
        b = Batch("f32", [3] * (G * per), H, H, dim, 64, [8000] * G, [per * i for i in range(G + 1)], adds=adds, seed=42, share=mode == "shared")
    d = _attend(pkg, b)
    assert (d.workspace_bytes > 0) == (mode == "shared")
    _close(b)
    ref, _ = b.reference()
    got = b.out_all[:b.rows].cpu().double()
    assert (got - ref).norm() / ref.norm() < 1e-6
    for i in range(len(b.lens)):                                  # each request by itself too
        rows = slice(b.starts[i], b.starts[i + 1])
        assert (got - ref)[rows].norm() / ref[rows].norm() < 1e-6


@pytest.mark.parametrize("prompt,share", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("kind,heads,kv,dim", [("f16", 8, 2, 128), ("bf16", 8, 2, 128), ("bf16", 16, 1, 64), ("f16", 32, 2, 128)])
def test_repeated_16_bit_calls_give_the_same_bits(pkg, kind, heads, kv, dim, prompt, share):
    b = Batch(kind, [40, 900, 7, 333] * 6, heads, kv, dim, 16, [4001], [0, 24], adds=[40, 260, 7, 100] * 6 if prompt else None, seed=43, share=share)
    _attend(pkg, b)
    first = b.out_all.clone()
    _close(b)
    for _ in range(5):
        b.out_all.fill_(-7)
        _attend(pkg, b)
        assert torch.equal(b.out_all, first)


@pytest.mark.parametrize("prompt,share", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("kind,heads,kv,dim", [("f32", 4, 4, 64), ("bf16", 8, 2, 128)])
def test_k_and_v_of_two_layers_in_one_page(pkg, kind, heads, kv, dim, prompt, share):
    """K and V (and another layer's) side by side in each page, by page_stride;
    the append writes there too, and nowhere else."""
    page = 16
    lens = [40, 3, 17, 200]
    b = Batch(kind, lens, heads, kv, dim, page, [150], [0, 3], adds=[40, 2, 1, 60] if prompt else None, seed=44, share=share)
    dense = kv * page * dim
    pool = torch.full((b.n_pages, 2, 2, dense), float("nan"), dtype=b.k.dtype, device="cuda")    # [page][layer][K, V]
    pool[:, 1, 0], pool[:, 1, 1] = b.k.view(b.n_pages, dense), b.v.view(b.n_pages, dense)
    b.stride, b.k, b.v = 4 * dense, pool[0, 1, 0], pool[0, 1, 1]
    _attend(pkg, b)
    _close(b)
    if not prompt and not share:
        before = pool.clone()
        new = torch.randn(2, 4, kv * dim, device="cuda")
        slots = _i32([int(b.table[i, (n - 1) // page]) * page + (n - 1) % page for i, n in enumerate(lens)])
        c = b.desc(pkg).cache
        a = pkg.KvAppend(cache=c, k=new[0].data_ptr(), v=new[1].data_ptr(), stride=kv * dim, slots=slots.data_ptr(), dtype=0, rows=4)
        pkg.check(pkg.lib().t3b_op_kv_append(C.byref(a), _stream()))
        view = before.view(b.n_pages, 2, 2, kv, page, dim)
        for r, s in enumerate(slots.tolist()):
            for x in range(2):
                view[s // page, 1, x, :, s % page] = new[x, r].to(pool.dtype).view(kv, dim)
        assert torch.equal(pool.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("mode", ["decode", "shared", "prompt"])
@pytest.mark.parametrize("kind,heads,kv,dim,page", [("f32", 4, 4, 64, 8), ("f16", 8, 2, 128, 32), ("bf16", 32, 2, 128, 16), ("f32", 3, 1, 128, 64)])
def test_tables_much_wider_than_the_lengths(pkg, mode, kind, heads, kv, dim, page):
    """Tables with room for thousands of keys and few in them: clusters of
    which most CTAs have no key."""
    lens = [1, 0, page, 130, 5]
    b = Batch(kind, lens, heads, kv, dim, page, [40, 3], [0, 2, 4], adds=[1, 0, page - 1, 130, 2] if mode == "prompt" else None, seed=45)
    wide = torch.full((len(lens), 6000 // page), 1 << 28, dtype=torch.int32, device="cuda")
    b.table = torch.cat([b.table, wide], 1).contiguous()
    room = 50_000_000 // (4 * kv * dim * page * 3) + 1 if mode == "shared" else 3000 // page if mode == "prompt" else 1000 // page
    b.ptable = torch.cat([b.ptable, torch.full((2, room), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
    d = _attend(pkg, b)
    assert (d.workspace_bytes > 0) == (mode == "shared")
    _close(b)


@pytest.mark.parametrize("which", [("row_req", "row_pos", "slots"), ("slots",), ("row_pos",), ("row_req", "slots")])
@pytest.mark.parametrize("n,page,width", [(50, 16, 12), (900, 16, 12)])
def test_plan_with_some_row_maps_that_are_not_16_byte_aligned(pkg, which, n, page, width):
    rng = np.random.default_rng(n)
    ln, add, release, table, free, n_free = _random_step(rng, n, page, width, True)
    cap = int(add.sum()) + 3
    ref = paged_ref.plan(ln, add, release, page, table, free, n_free, cap)
    p = Plan(pkg, ln, add, release, page, table, free, n_free, cap)
    for k in ("row_req", "row_pos", "slots"):
        p.out[k] = torch.full((cap + 4,), 77, dtype=torch.int32, device="cuda")
        setattr(p.d, k, p.out[k].data_ptr() + 4 if k in which else None)
    pkg.check(pkg.lib().t3b_op_kv_plan(C.byref(p.d), _stream()))
    for k in ("row_req", "row_pos", "slots"):
        got = p.out[k].cpu().numpy()
        assert got[0] == 77 and (got[cap + 1:] == 77).all()
        assert np.array_equal(got[1:cap + 1], ref[k]) if k in which else (got == 77).all(), k


# --------------------------------------------------------------------------
# the operators together
# --------------------------------------------------------------------------

@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("graph", [False, True])
def test_a_serving_loop_matches_dense_attention(pkg, graph, share):
    """Plan, append and attention as a server runs them: prompts of a common
    prefix are admitted, decode, finish, and their slots are taken over by
    others; every step's output equals t3b_op_attention on dense caches that
    hold prefix and own keys of each request.  With `graph` each kind of step
    is captured once and replayed."""
    L = pkg.lib()
    H, D, page, n, width, cap, P = 16, 64, 16, 6, 7, 64, 37
    rng = np.random.default_rng(12)
    g = torch.Generator(device="cuda").manual_seed(1)
    n_pages = 40
    pool = torch.full((2, n_pages, H, page, D), float("nan"), dtype=torch.float16, device="cuda")
    pre_pages = blocks(P, page)
    dense = torch.zeros(2, n, H, 256, D, dtype=torch.float16, device="cuda")
    kvp = torch.randn(2, P, H, D, generator=g, device="cuda").half()
    room = 200 if share else pre_pages                   # 3200 keys of room: the prefix is computed once for the batch
    ptable = torch.full((room,), -1, dtype=torch.int32, device="cuda")
    ptable[:pre_pages] = torch.arange(pre_pages)
    for t in range(P):
        pool[:, t // page, :, t % page] = kvp[:, t]
    dense[:, :, :, :P] = kvp.permute(0, 2, 1, 3)[:, None]
    st = torch.cuda.Stream()
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    ln, add, rel, table = z(n), z(n), z(n), z(n, width)
    free, n_free = torch.arange(pre_pages, n_pages, dtype=torch.int32, device="cuda"), _i32([n_pages - pre_pages])
    row_start, req, pos, slots = z(n + 1), z(cap), z(cap), z(cap)
    plen, pstart = _i32([P]), _i32([0, n])
    q, k, v, out = (torch.zeros(cap, H * D, device="cuda") for _ in range(4))
    p = lambda t: t.data_ptr()  # noqa: E731
    dplan = pkg.KvPlan(n=n, page_size=page, max_blocks=width, rows_cap=cap, len=p(ln), add=p(add), release=p(rel), free_pages=p(free),
                       free_cap=free.numel(), n_free=p(n_free), n_free_out=p(n_free), table=p(table), row_start=p(row_start),
                       row_req=p(req), row_pos=p(pos), slots=p(slots), len_out=p(ln))
    cache = pkg.PagedKv(k=p(pool[0]), v=p(pool[1]), dtype=1, n_pages=n_pages, n_kv_head=H, page_size=page, head_dim=D)
    dapp = pkg.KvAppend(cache=cache, k=p(k), v=p(v), stride=H * D, slots=p(slots), dtype=0, rows=cap)
    da = pkg.SharedAttn(cache=cache, q=p(q), out=p(out), q_stride=H * D, out_stride=H * D, len=p(ln), table=p(table),
                        row_start=p(row_start), prefix_start=p(pstart), prefix_len=p(plen), prefix_table=p(ptable), dtype=0,
                        n_head=H, n=n, rows=cap, max_blocks=width, n_prefix=1, prefix_max_blocks=room)
    dd = pkg.SharedAttn.from_buffer_copy(da)
    dd.rows, dd.row_start = n, None
    assert (L.t3b_op_attention_shared_workspace(C.byref(dd)) > 0) == share
    size = max(L.t3b_op_attention_shared_workspace(C.byref(da)), L.t3b_op_attention_shared_workspace(C.byref(dd)))
    ws = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    for d in (da, dd):
        d.workspace, d.workspace_bytes = p(ws), ws.numel()

    def step(decode):
        s = C.c_void_p(torch.cuda.current_stream().cuda_stream)
        pkg.check(L.t3b_op_kv_plan(C.byref(dplan), s))
        pkg.check(L.t3b_op_kv_append(C.byref(dapp), s))
        if decode:
            pkg.check(L.t3b_op_attention_shared(C.byref(dd), s))
        else:
            pkg.check(L.t3b_op_attention_shared_prompt(C.byref(da), s))

    graphs = {}
    if graph:
        for decode in (False, True):
            graphs[decode] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graphs[decode], stream=st):
                step(decode)
    lens, live = np.zeros(n, int), np.zeros(n, bool)
    for it in range(24):
        decode = it % 3 != 0
        a, r = np.zeros(n, int), np.zeros(n, int)
        if decode:
            a[:] = 1                                   # one row per request: every slot gets a token
        else:
            gone = live & (rng.random(n) < 0.5)
            r[gone], lens[gone] = lens[gone], 0
            a = np.where(lens == 0, rng.integers(1, 10, n), 1)
        a = np.minimum(a, width * page - lens)
        live[:] = True
        add.copy_(_i32(a)); rel.copy_(_i32(r))
        if r.any():
            ln.copy_(_i32(lens))
        x = torch.randn(3, cap, H * D, generator=g, device="cuda")
        q.copy_(x[0]); k.copy_(x[1]); v.copy_(x[2]); out.fill_(-7.0)
        torch.cuda.synchronize()
        if graph:
            graphs[decode].replay()
        else:
            step(decode)
        torch.cuda.synchronize()
        pkg.check(L.t3b_op_check(_stream()))
        starts = np.cumsum(np.r_[0, a])
        total = int(starts[-1])
        assert row_start.tolist() == starts.tolist() and ln.tolist() == (lens + a).tolist()
        rows, rlen = [], []
        for i in range(n):
            for t in range(a[i]):
                dense[0, i, :, P + lens[i] + t] = k[starts[i] + t].half().view(H, D)
                dense[1, i, :, P + lens[i] + t] = v[starts[i] + t].half().view(H, D)
                rows.append(i)
                rlen.append(P + lens[i] + t + 1)
        kd, vd = dense[0][rows].contiguous(), dense[1][rows].contiguous()
        want = torch.zeros(total, H * D, device="cuda")
        pkg.check(L.t3b_op_attention(p(q), p(kd), p(vd), total, H, 256, p(_i32(rlen)), p(want), _stream()))
        torch.cuda.synchronize()
        assert (out[:total] - want).abs().max() <= 1e-5 * want.abs().max()     # the bound of each against 64 bits
        assert (out[total:] == -7).all()
        lens = lens + a


@pytest.mark.parametrize("form", ["decode", "prompt"])
def test_a_serving_loop_with_idle_slots(pkg, form):
    """Steps in which some slots get no token: the plan's rows are compact
    (row r belongs to slot row_req[r]), the decode form's are by slot.  The
    decode form takes q by slot, and its K/V rows are gathered through row_req
    for the append; the prompt form takes all of them in the plan's order,
    prompts of admitted requests among them.  Every row against 64 bits."""
    L = pkg.lib()
    H, D, page, n, width, cap, P = 4, 64, 8, 7, 6, 64, 21
    rng = np.random.default_rng(19)
    g = torch.Generator(device="cuda").manual_seed(5)
    n_pages, pre = 50, blocks(P, page)
    pool = torch.full((2, n_pages, H, page, D), float("nan"), dtype=torch.float16, device="cuda")
    prefix = torch.randn(2, P, H, D, generator=g, device="cuda").half()
    for t in range(P):
        pool[:, t // page, :, t % page] = prefix[:, t]
    held = [prefix.new_zeros(2, 0, H, D) for _ in range(n)]       # the own K and V of each slot
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    ln, add, rel, table, row_start = z(n), z(n), z(n), z(n, width), z(n + 1)
    req, pos, slots = z(cap), z(cap), z(cap)
    free, n_free = torch.arange(pre, n_pages, dtype=torch.int32, device="cuda"), _i32([n_pages - pre])
    ptable, plen, pstart = torch.arange(pre, dtype=torch.int32, device="cuda"), _i32([P]), _i32([0, n])
    q, k, v, out = (torch.zeros(cap, H * D, device="cuda") for _ in range(4))
    p = lambda t: t.data_ptr()  # noqa: E731
    dplan = pkg.KvPlan(n=n, page_size=page, max_blocks=width, rows_cap=cap, len=p(ln), add=p(add), release=p(rel), free_pages=p(free),
                       free_cap=free.numel(), n_free=p(n_free), n_free_out=p(n_free), table=p(table), row_start=p(row_start),
                       row_req=p(req), row_pos=p(pos), slots=p(slots), len_out=p(ln))
    cache = pkg.PagedKv(k=p(pool[0]), v=p(pool[1]), dtype=1, n_pages=n_pages, n_kv_head=H, page_size=page, head_dim=D)
    app = pkg.KvAppend(cache=cache, k=p(k), v=p(v), stride=H * D, slots=p(slots), dtype=0, rows=cap)
    at = pkg.SharedAttn(cache=cache, q=p(q), out=p(out), q_stride=H * D, out_stride=H * D, len=p(ln), table=p(table), prefix_start=p(pstart),
                        prefix_len=p(plen), prefix_table=p(ptable), dtype=0, n_head=H, n=n, rows=n, max_blocks=width, n_prefix=1,
                        prefix_max_blocks=pre)
    if form == "prompt":
        at.row_start, at.rows = p(row_start), cap
    lens = np.zeros(n, int)
    for it in range(30):
        a, r = (rng.random(n) < 0.6).astype(int), np.zeros(n, int)    # some slots idle in every step
        gone = (lens > 0) & (rng.random(n) < 0.15)
        r[gone], lens[gone] = lens[gone], 0
        if form == "prompt":
            a = np.where((lens == 0) & (a > 0), rng.integers(1, 9, n), a)
        a[gone & (rng.random(n) < 0.5)] = 0
        a = np.minimum(a, width * page - lens)
        for i in np.nonzero(gone)[0]:
            held[i] = held[i][:, :0]
        ln.copy_(_i32(lens)); add.copy_(_i32(a)); rel.copy_(_i32(r))
        starts, total = np.cumsum(np.r_[0, a]), int(a.sum())
        x = torch.randn(3, n if form == "decode" else cap, H * D, generator=g, device="cuda")   # what the model's QKV step gives
        out.fill_(-7.0)
        pkg.check(L.t3b_op_kv_plan(C.byref(dplan), _stream()))
        q[:x.shape[1]] = x[0]
        if form == "decode":
            rows = req.clamp(min=0).long()
            k.copy_(x[1][rows]); v.copy_(x[2][rows])
        else:
            k.copy_(x[1]); v.copy_(x[2])
        pkg.check(L.t3b_op_kv_append(C.byref(app), _stream()))
        pkg.check((L.t3b_op_attention_shared if form == "decode" else L.t3b_op_attention_shared_prompt)(C.byref(at), _stream()))
        pkg.check(L.t3b_op_check(_stream()))
        assert row_start.tolist() == starts.tolist() and (req[total:] == -1).all()
        for i in range(n):
            own = slice(i, i + a[i]) if form == "decode" else slice(starts[i], starts[i] + a[i])
            new = x[1:, own].half().view(2, -1, H, D)
            held[i] = torch.cat([held[i], new], 1)
            for t in range(a[i]):
                kk, vv = torch.cat([prefix, held[i][:, :lens[i] + t + 1]], 1).double()
                qq = x[0, own.start + t].double().view(H, D)
                w = torch.softmax(torch.einsum("hd,khd->hk", qq, kk) / 8, -1)
                want = torch.einsum("hk,khd->hd", w, vv).reshape(-1)
                # 32-bit results: 2^-18 of the largest value, which is above 64 roundings
                assert (out[own.start + t].double() - want).abs().max() <= 2.0 ** -18 * vv.abs().max(), (it, i, t)
        lens = lens + a
        if form == "prompt":
            assert (out[total:] == -7).all()
    assert lens.max() > page                                      # requests grew over several pages
