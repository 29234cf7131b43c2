"""Calls of the paged cache's operators that are refused, recorded or have to
leave something as it was, on the CPU (KILN_HIP_INTERPRET=1: the library's CPU
meaning)."""

import ctypes

import pytest
import torch

import kiln
import paged_reference as ref
from kiln.hip import lib as kl


@pytest.fixture(autouse=True)
def interpreting(monkeypatch):
    monkeypatch.setenv("KILN_HIP_INTERPRET", "1")


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


# -- the C entries -----------------------------------------------------------------------------


@pytest.mark.parametrize("stride", ["kp_t", "vp_t", "k_n", "v_n"])
def test_negative_token_strides_are_refused(stride):
    """The kernels count rows inside a tile with unsigned 32-bit offsets."""
    op = kl.Paged(kl.PAGED_ATTENTION, 1, 2, 1, 1, 64, 16, 4, 2, 0, kl.TYPE_F32, kl.TYPE_F32, 0, 1.0)
    size = ctypes.c_size_t()
    assert kl.load().kh_paged_workspace_bytes(op, size) == kl.OK
    setattr(op, stride, -64)
    assert kl.load().kh_paged_workspace_bytes(op, size) == kl.ERR_INVALID
    assert kl.load().kh_paged_host(op) == kl.ERR_INVALID
    assert b"negative" in kl.load().kh_last_error()
    launch = kl.LaunchDesc()
    launch.family, launch.variant, launch.n_refs, launch.rank = kl.FAM_PAGED, kl.PAGED_ATTENTION, 8, 6
    for i, x in enumerate((1, 2, 1, 1, 64, 16)):
        launch.shape[i] = x
    launch.gemm[0], launch.gemm[1] = 4, 2
    at = {"k_n": (1, 1), "v_n": (2, 1), "kp_t": (3, 2), "vp_t": (4, 2)}[stride]
    launch.refs[at[0]].strides[at[1]] = -64
    handle = ctypes.c_void_p()
    assert kl.load().kh_plan_create(ctypes.byref(launch), 1, ctypes.byref(handle)) == kl.ERR_INVALID


# -- tracers and dispatch modes ------------------------------------------------------------------


def attention_calls():
    p = ref.problem(gen(), lengths=(70, 17))
    means = p["k_pages"].mean(2)
    names = list(p)

    def tree(*args):
        return kiln.tree_attention(**dict(zip(names, args)))

    def picked(*args):
        p = dict(zip(names, args))
        sel = kiln.select_pages(p["q"], args[-1], p["table"], p["lengths"], page_size=16, pages=2)
        return kiln.selected_attention(**p, selected=sel)

    return [(tree, tuple(p.values())), (picked, (*p.values(), means))]


def append_call():
    k_pages, v_pages = (torch.randn(9, 3, 16, 8, generator=gen(s)) for s in (1, 2))
    table, lengths = torch.tensor([[4, 2], [0, 7]], dtype=torch.int32), torch.tensor([14, 3], dtype=torch.int32)
    rows = torch.tensor([[0, 2, 4, 6], [9, 1, -1, 3]], dtype=torch.int32)
    k, v = (torch.randn(2, 11, 3, 8, generator=gen(s)) for s in (3, 4))

    def append(k, v, k_pages, v_pages, means):
        kiln.cache_append(k, v, k_pages, v_pages, table, lengths, rows=rows, k_means=means)
        kiln.copy_pages([k_pages, v_pages], [4, 0], [1, 3])
        return k_pages + v_pages

    return append, (k, v, k_pages, v_pages, k_pages.mean(2))


@pytest.mark.parametrize("how", ["jit", "make_fx"])
@pytest.mark.parametrize("which", [0, 1], ids=["tree", "picked"])
def test_traces_hold_the_operators(how, which):
    from torch.fx.experimental.proxy_tensor import make_fx

    fn, args = attention_calls()[which]
    traced = torch.jit.trace(fn, args) if how == "jit" else make_fx(fn)(*args)
    assert "paged_attention" in str(traced.graph)
    other = [t.clone() for t in args]
    other[0].mul_(-0.7)
    other[6].sub_(9)
    assert torch.equal(traced(*other), fn(*other))


def test_traces_hold_what_changes_the_cache():
    from torch.fx.experimental.proxy_tensor import make_fx

    fn, args = append_call()
    traced = make_fx(fn)(*[t.clone() for t in args])
    assert "cache_append" in str(traced.graph) and "copy_pages" in str(traced.graph)
    mine, want = [t.clone() for t in args], [t.clone() for t in args]
    for x in (mine, want):
        x[0].mul_(-2)
    out = traced(*mine)
    assert torch.equal(out, fn(*want))
    assert all(torch.equal(a, b) for a, b in zip(mine, want)) and not torch.equal(mine[2], args[2])


def test_a_trace_that_would_drop_them_is_refused():
    fn, args = append_call()
    for call in (fn, lambda pool: kiln.copy_pages([pool], [0], [1]) or pool):
        before = [t.clone() for t in args]
        with pytest.raises(NotImplementedError, match="trace"):
            torch.jit.trace(call, args if call is fn else args[2:3])
        assert all(torch.equal(a, b) for a, b in zip(args, before))


def test_dispatch_modes_see_the_operators():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Names(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    for fn, args in attention_calls():
        want = fn(*args)
        with Names() as mode:
            got = fn(*args)
        assert torch.equal(got, want) and "kiln.paged_attention.default" in mode.seen
    fn, args = append_call()
    mine = [t.clone() for t in args]
    want = fn(*args)
    with Names() as mode:
        got = fn(*mine)
    assert torch.equal(got, want) and {"kiln.cache_append.default", "kiln.copy_pages.default"} <= set(mode.seen)
    assert all(torch.equal(a, b) for a, b in zip(mine, args))


def test_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode() as mode:
        for fn, args in attention_calls():
            out = fn(*[mode.from_tensor(t) for t in args] if not isinstance(args[0], torch._subclasses.FakeTensor) else args)
            assert out.shape == args[0].shape and isinstance(out, torch._subclasses.FakeTensor)
        fn, args = append_call()
        fn(*args)


# -- autograd -------------------------------------------------------------------------------------


@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_is_refused(no_grad):
    """A dual tensor's tangent would be lost; tensors without one go through."""
    import torch.autograd.forward_ad as fw

    p = ref.problem(gen(), lengths=(70, 17))
    means = p["k_pages"].mean(2)

    def attend(p):
        return kiln.tree_attention(**p)

    def pick(q, means):
        return kiln.select_pages(q, means, p["table"], p["lengths"], page_size=16, pages=2)

    def append(k, v, k_pages, v_pages, m):
        return kiln.cache_append(k, v, k_pages, v_pages, p["table"], p["lengths"], k_means=m)

    def copy(pool):
        return kiln.copy_pages([pool], [0], [1])

    want, picked = attend(p), pick(p["q"], means)
    with fw.dual_level(), torch.set_grad_enabled(not no_grad):
        def dual(t):
            return fw.make_dual(t.clone(), torch.ones_like(t))

        for name in ("q", "k", "v", "k_pages", "v_pages"):
            with pytest.raises(NotImplementedError, match="forward"):
                attend(dict(p, **{name: dual(p[name])}))
        for args in ((dual(p["q"]), means), (p["q"], dual(means))):
            with pytest.raises(NotImplementedError, match="forward"):
                pick(*args)
        args = [p["k"], p["v"], p["k_pages"], p["v_pages"], means]
        for i in range(5):
            mine = [t.clone() for t in args]
            mine[i] = dual(args[i])
            with pytest.raises(NotImplementedError, match="forward"):
                append(*mine)
        with pytest.raises(NotImplementedError, match="forward"):
            copy(dual(means))
        assert torch.equal(attend(p), want) and torch.equal(pick(p["q"], means), picked)


@pytest.mark.parametrize("seen", [False, True], ids=["alone", "dispatch mode"])
def test_what_changed_counts_as_changed(seen):
    """Values saved for a backward pass and changed before it: torch's error, no gradient of other values."""
    from torch.utils.flop_counter import FlopCounterMode

    fn, (k, v, k_pages, v_pages, means) = append_call()
    table, lengths = torch.tensor([[4, 2], [0, 7]], dtype=torch.int32), torch.tensor([14, 3], dtype=torch.int32)

    def run(call):
        if not seen:
            return call()
        with FlopCounterMode(display=False):
            return call()

    for call, changed in ((lambda: kiln.cache_append(k, v, k_pages, v_pages, table, lengths, k_means=means), (k_pages, v_pages, means)),
                          (lambda: kiln.copy_pages([k_pages, v_pages], [4], [1]), (k_pages, v_pages))):
        for t in changed:
            x = torch.ones((), requires_grad=True)
            y = (x * t.view(-1)[5:]).sum()      # saves a view
            before = [t._version for t in changed]
            run(call)
            assert all(t._version > n for t, n in zip(changed, before))
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
    before = k_pages._version, v_pages._version
    for refused in (lambda: kiln.copy_pages([k_pages, v_pages], [4], [4]), lambda: kiln.copy_pages([k_pages, v_pages], [], [])):
        try:
            refused()
        except ValueError:
            pass
    assert (k_pages._version, v_pages._version) == before
    with torch.inference_mode():                # (such tensors count no versions)
        kiln.copy_pages([k_pages.clone()], [4], [1])
        kiln.cache_append(k, v, k_pages.clone(), v_pages.clone(), table, lengths)


# -- kiln.PagedCache ------------------------------------------------------------------------------


@pytest.mark.parametrize("upload", [0, 1, 2])
@pytest.mark.parametrize("error", [RuntimeError, MemoryError, KeyboardInterrupt])
def test_an_append_that_fails_on_its_way_gives_its_pages_back(monkeypatch, upload, error):
    """The accepted rows, the table or the lengths do not reach the device."""
    cache = kiln.PagedCache(1, 6, 16, 2, 8, dtype=torch.float32)
    a = cache.open()
    k = torch.randn(1, 1, 20, 2, 8, generator=gen())
    cache.append([a], k, k)
    b, = cache.fork(a)
    before = cache.k.clone(), list(cache._refs), sorted(cache._free), cache.pages_of(b)
    done = []

    def fails(t):
        done.append(t)
        if len(done) > upload:
            raise error("no more")
        return t

    with monkeypatch.context() as m:
        m.setattr(cache, "_upload", fails)
        with pytest.raises(error):
            cache.append([b], k, k, rows=[list(range(20))])
    assert sorted(cache._free) == before[2] and cache._refs == before[1] and cache.pages_of(b) == before[3]
    assert cache.length(b) == 20 and torch.equal(cache.k[:, list(before[3])], before[0][:, list(before[3])])
    cache.append([b], k, k)
    assert cache.length(b) == 40 and cache.free_pages == 2


# -- calls whose forms are kept ---------------------------------------------------------------------


def test_forms_of_different_operators():
    """Tensors of the same shapes, strides and types in another operator's places."""
    k, pages, means = torch.randn(9, 5, 9, 8, generator=gen()), torch.zeros(9, 9, 16, 8), torch.zeros(9, 9, 8)
    table, lengths = torch.arange(9, dtype=torch.int32).view(9, 1), torch.zeros(9, dtype=torch.int32)
    rows = torch.zeros(9, 4, dtype=torch.int32)
    args = (k, k.clone(), pages, pages.clone(), table, lengths)
    kiln.cache_append(*args, rows=rows, k_means=means)
    assert means.abs().sum() > 0
    with pytest.raises(TypeError, match="pool"):      # lengths are no pool: as without the append before
        kiln.copy_pages([*args, rows, means], [0], [1])
    pools = [*args[:5], rows, means]
    kiln.copy_pages(pools, [0], [1])
    assert all(torch.equal(t[1], t[0]) for t in pools)


def test_the_cache_refuses_to_be_captured(monkeypatch):
    cache = kiln.PagedCache(1, 6, 16, 2, 8, dtype=torch.float32)
    a = cache.open()
    k = torch.randn(1, 1, 20, 2, 8, generator=gen())
    cache.append([a], k, k)
    b = cache.open()
    cache.append([b], k, k)
    cache.free(a)
    before = cache.k.clone(), cache.pages_of(b), cache.free_pages
    with monkeypatch.context() as m:
        m.setattr(cache, "device", torch.device("cuda"))
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        for call in (lambda: cache.append([b], k, k), lambda: cache.batch([b]), cache.compact):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    assert torch.equal(cache.k, before[0]) and cache.pages_of(b) == before[1] and cache.free_pages == before[2]
    assert cache.compact() == 2


@pytest.mark.parametrize("variant", [kl.PAGED_ATTENTION, kl.PAGED_SELECT])
def test_tables_whose_last_tile_passes_32_bits_are_refused(variant):
    """Tiles of a sequence are counted as (length + keys of a tile - 1) / keys of a tile, in 32 bits."""
    size = ctypes.c_size_t()
    for page, width, rc in ((16, 2 ** 27 - 1, kl.ERR_UNSUPPORTED), (16, 2 ** 27 - 4, kl.ERR_UNSUPPORTED), (16, 2 ** 27 - 8, kl.OK),
                            (1024, 2 ** 21 - 1, kl.OK), (1024, 2 ** 21, kl.ERR_UNSUPPORTED)):
        op = kl.Paged(variant, 1, 1, 1, 1, 64, page, 4, width, variant, kl.TYPE_F32, kl.TYPE_F32, 0, 1.0)
        assert kl.load().kh_paged_workspace_bytes(op, size) == rc, (page, width)


def test_more_items_than_a_launch_holds_are_refused():
    """A workgroup of eight waves per (sequence, head, token): 2^32 work items are one too many."""
    size = ctypes.c_size_t()
    for draft, batch, rc in ((15, 4096, kl.OK), (16, 4096, kl.ERR_UNSUPPORTED), (16, 4095, kl.OK)):
        op = kl.Paged(kl.PAGED_ATTENTION, batch, draft, 128, 128, 8, 16, 4, 2, 2, kl.TYPE_BF16, kl.TYPE_BF16, 0, 1.0)
        assert kl.load().kh_paged_workspace_bytes(op, size) == rc
    for draft, rc in ((31, kl.OK), (32, kl.ERR_UNSUPPORTED)):     # (heads of 256: four waves)
        op = kl.Paged(kl.PAGED_ATTENTION, 4096, draft, 128, 128, 256, 16, 4, 2, 2, kl.TYPE_BF16, kl.TYPE_BF16, 0, 1.0)
        assert kl.load().kh_paged_workspace_bytes(op, size) == rc
    p = ref.problem(gen(), batch=4096, draft=16, heads=128, kv=128, dim=8, lengths=[0] * 4096, spare=4, columns=2, tree=False,
                    cache=torch.bfloat16, act=torch.bfloat16)
    p["q"], p["k"], p["v"] = (t[:, :, :1, :].expand(4096, 16, 128, 8) for t in (p["q"], p["k"], p["v"]))
    with pytest.raises(NotImplementedError, match="launch"):
        kiln.selected_attention(**p, selected=torch.zeros(1, 1, 1, 2, dtype=torch.int32).expand(4096, 16, 128, 2))


# -- models ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("change", [lambda y: y.sum(-1, dtype=torch.float16), lambda y: y.mean(-1, dtype=torch.bfloat16),
                                    lambda y: y.half(), lambda y: y.sum(-1, dtype=torch.int32)])
def test_models_that_change_the_type_are_refused(change):
    """Beside a cache too: everything but the cache's own operands is float32."""
    from kiln.frontend.fx_import import Unsupported, import_exported

    p = ref.problem(gen(), lengths=(40, 17), dim=16)

    class Model(torch.nn.Module):
        def forward(self, q, k_pages, table, lengths):
            return change(kiln.tree_attention(q, q[:, :, :2], q[:, :, :2], k_pages, k_pages, table, lengths))

    class Plain(torch.nn.Module):
        def forward(self, q):
            return change(q)

    for model, args in ((Model(), (p["q"], p["k_pages"], p["table"], p["lengths"])), (Plain(), (p["q"],))):
        with pytest.raises(Unsupported):
            import_exported(torch.export.export(model.eval(), args).run_decompositions())
