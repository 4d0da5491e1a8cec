"""Calls of the paged cache's operators that must not reach a kernel, on the
CPU: what the native module would be told is recorded instead."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from crowdllama_amd.ops import kv


class Recorder:
    """Stands in for the native module."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            if name.endswith("_workspace"):
                return 64
            self.calls.append((name, args))
        return call


@pytest.fixture
def core(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(kv, "_get", lambda dev: rec)
    monkeypatch.setattr(kv, "_stream", lambda dev: 0)
    return rec


def tensors(device="cpu"):
    kw = dict(device=device)
    half = dict(dtype=torch.bfloat16, **kw)
    ints = dict(dtype=torch.int32, **kw)
    return dict(pool=torch.zeros(8, 2, 2, 16, 64, **half),
                all=torch.zeros(8, 3, 2, 2, 16, 64, **half),
                q=torch.zeros(2, 4, 64, **half), k=torch.zeros(2, 2, 64, **half),
                v=torch.zeros(2, 2, 64, **half),
                table=torch.zeros(2, 4, **ints), lens=torch.ones(2, **ints),
                now=torch.ones(2, **ints), mass=torch.zeros(2, 2, 64, **kw),
                pos=torch.zeros(2, 2, 64, **ints),
                masses=torch.zeros(3, 2, 2, 64, **kw),
                places=torch.zeros(3, 2, 2, 64, **ints),
                inv=torch.ones(32, **kw))


def append(t, **kw):
    kw = {"q": t["q"], "inv_freq": t["inv"], "mass": t["mass"],
          "pos": t["pos"], **kw}
    return kv.append(t["k"], t["v"], t["pool"], t["table"], t["lens"],
                     t["now"], **kw)


def attend(t, **kw):
    kw = {"mass": t["mass"], **kw}
    return kv.attend(t["q"], t["pool"], t["table"], t["lens"], **kw)


def observe(t, **kw):
    return kv.observe(t["q"], t["pool"], t["table"], t["lens"], t["mass"],
                      **kw)


def evict(t, **kw):
    kw = {"keep": 5, **kw}
    return kv.evict(t["all"], t["table"], t["lens"], t["now"], t["masses"],
                    t["places"], **kw)


OPERATORS = [append, attend, observe, evict]
operators = pytest.mark.parametrize("op", OPERATORS,
                                    ids=[x.__name__ for x in OPERATORS])


@operators
def test_a_plain_call_reaches_the_kernel(core, op):
    op(tensors())
    assert [name for name, _ in core.calls] == ["kv_" + op.__name__]


@operators
def test_fake_tensors_are_refused(core, op):
    with FakeTensorMode():
        t = tensors("cuda")
        with pytest.raises(ValueError, match="traced"):
            op(t)
    with pytest.raises(ValueError, match="no memory"):
        op(t)                        # outside of the mode too
    real = tensors()
    with FakeTensorMode(allow_non_fake_inputs=True):
        with pytest.raises(ValueError, match="traced"):
            op(real)                 # its outputs would be fake
    assert not core.calls


@operators
@pytest.mark.parametrize("only", sorted(tensors()))
def test_one_tensor_without_memory_is_refused(core, op, only):
    """Each of the tensors that the operator takes."""
    t = tensors()
    t[only] = torch._to_functional_tensor(t[only])
    before = len(core.calls)
    if only in {"append": ("all", "masses", "places"),
                "attend": ("all", "k", "v", "now", "pos", "masses", "places",
                           "inv"),
                "observe": ("all", "k", "v", "now", "pos", "masses", "places",
                            "inv"),
                "evict": ("pool", "q", "k", "v", "mass", "pos", "inv")}[
                    op.__name__]:
        op(t)
        assert len(core.calls) == before + 1
    else:
        with pytest.raises(ValueError, match="no memory"):
            op(t)
        assert not core.calls


@operators
def test_tracing_is_refused(core, op):
    t = tensors()

    def go(q, pool):
        op({**t, "q": q, "pool": pool})
        return q + 1
    with pytest.raises(ValueError, match="traced"):
        make_fx(go)(t["q"], t["pool"])
    with pytest.raises((ValueError, RuntimeError)):
        make_fx(go, tracing_mode="fake")(t["q"], t["pool"])
    assert not core.calls


@pytest.mark.parametrize("op,only", [
    (append, "k"), (append, "v"), (append, "q"), (append, "pool"),
    (append, "mass"), (append, "inv"), (attend, "q"), (attend, "pool"),
    (attend, "mass"), (observe, "q"), (observe, "pool"), (observe, "mass"),
    (evict, "all"), (evict, "masses")])
def test_tangents_are_refused(core, op, only):
    t = tensors()
    with forward_ad.dual_level():
        op(t)                        # a level alone says nothing
        t[only] = forward_ad.make_dual(t[only], torch.ones_like(t[only]))
        with pytest.raises(ValueError, match="gradient"):
            op(t)
    with torch.enable_grad():
        t = tensors()
        t[only].requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            op(t)
    assert len(core.calls) == 1


@pytest.mark.parametrize("transform", [
    lambda f, x: torch.func.vmap(f)(x.expand(3, *x.shape)),
    lambda f, x: torch.func.jvp(f, (x,), (x,)),
    lambda f, x: torch.func.functionalize(f)(x)],
    ids=["vmap", "jvp", "functionalize"])
def test_transforms_are_refused(core, transform):
    t = tensors()
    with pytest.raises((ValueError, RuntimeError)):
        transform(lambda q: attend({**t, "q": q}), t["q"])
    assert not core.calls


def test_outputs_of_a_written_tensor_are_checked_too(core):
    t = tensors()
    fake = torch._to_functional_tensor
    for call in (lambda: append(t, q_out=fake(t["q"] + 0)),
                 lambda: attend(t, out=fake(t["q"] + 0)),
                 lambda: append(t, starts=fake(t["lens"].new_zeros(3))),
                 lambda: observe(t, starts=fake(t["lens"].new_zeros(3))),
                 lambda: evict(t, out=(fake(t["masses"] + 0), t["places"],
                                       t["lens"])),
                 lambda: evict(t, out=(t["masses"], fake(t["places"] + 0),
                                       t["lens"])),
                 lambda: evict(t, out=(t["masses"], t["places"],
                                       fake(t["lens"] + 0)))):
        with pytest.raises(ValueError, match="no memory"):
            call()
    assert not core.calls


def rows_of(base, at, n, heads=4, stride=None):
    """[n, heads, 64] from element `at` of a flat tensor on."""
    return base.as_strided((n, heads, 64), (stride or heads * 64, 64, 1), at)


def test_outputs_over_inputs_are_refused(core):
    """All but exactly the queries: other workgroups still read what one
    writes."""
    t = tensors()
    base = torch.zeros(4096, dtype=torch.bfloat16)
    t["q"] = rows_of(base, 256, 2)
    for at, stride in ((0, None), (256 + 64, None), (256 + 256, None),
                       (256, 512), (256 + 448, 64 * 5), (256 - 192, None)):
        for call in (append, attend):
            name = "q_out" if call is append else "out"
            with pytest.raises(ValueError, match=name + " overlaps q"):
                call(t, **{name: rows_of(base, at, 2, stride=stride)})
    swapped = t["q"].as_strided((2, 4, 64), (64, 128, 1))
    with pytest.raises(ValueError, match="out overlaps q"):
        attend(t, out=swapped)
    for name in ("k", "v"):
        both = tensors()
        both[name] = rows_of(base, 0, 2, heads=2)
        for at in (0, 64, 192):
            with pytest.raises(ValueError, match=f"q_out overlaps {name}"):
                append(both, q_out=rows_of(base, at, 2))
    assert not core.calls
    for out in (t["q"], rows_of(base, 256, 2), rows_of(base, 768, 2),
                rows_of(base, 1024, 2, stride=1024)):
        assert append(t, q_out=out) is out and attend(t, out=out) is out
    assert len(core.calls) == 8


def test_outputs_over_the_cache_are_refused(core):
    t = tensors()
    pool = t["pool"].reshape(-1)
    out = rows_of(pool, pool.numel() - 600, 2)
    for call, name in ((append, "q_out"), (attend, "out")):
        with pytest.raises(ValueError, match=name + " overlaps pool"):
            call(t, **{name: out})
        whole = torch.zeros(4096, dtype=torch.bfloat16)
        for part, dtype in (("mass", torch.float32), ("table", torch.int32),
                            ("lens", torch.int32)):
            u = dict(t)
            n = t[part].numel() * 2
            u[part] = whole[64:64 + n].view(dtype).view(t[part].shape)
            with pytest.raises(ValueError, match=f"{name} overlaps {part}"):
                call(u, **{name: rows_of(whole, 0, 2)})
    assert not core.calls


def test_outputs_between_inputs_are_taken(core):
    """Rows of one fused product, and other strides that meet nowhere."""
    wide = torch.zeros(2, 8 * 64 + 64, dtype=torch.bfloat16)
    t = tensors()
    t["q"] = wide[:, :256].view(2, 4, 64)
    t["k"] = wide[:, 256:384].view(2, 2, 64)
    t["v"] = wide[:, 384:512].view(2, 2, 64)
    append(t, q_out=t["q"])
    base = torch.zeros(4096, dtype=torch.bfloat16)
    t["q"] = base.as_strided((2, 4, 64), (1024, 128, 1))
    between = base.as_strided((2, 4, 64), (1024, 128, 1), 64)
    append(t, q_out=between)
    attend(t, out=between)
    attend(t, out=base.as_strided((2, 4, 64), (1024, 64, 1), 512))
    assert len(core.calls) == 4
    with pytest.raises(ValueError, match="out overlaps q"):
        attend(t, out=base.as_strided((2, 4, 64), (1024, 64, 1), 440))


def test_more_than_one_sequence_may_read_one_row(core):
    """Inputs may overlap themselves and each other."""
    t = tensors()
    t["q"] = t["q"][:1].expand(2, 4, 64)
    t["k"] = t["v"] = t["k"][:1].expand(2, 2, 64)
    append(t)
    attend(t, out=torch.zeros(2, 4, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="overlap itself"):
        append(t, q_out=t["q"])


def test_one_row_has_no_stride(core):
    t = tensors()
    t["q"] = torch.zeros(1, 512, dtype=torch.bfloat16)[:, :256].view(1, 4, 64)
    for x in ("table", "lens", "mass"):
        t[x] = t[x][:1]
    out = t["q"].as_strided((1, 4, 64), (256, 64, 1))
    assert attend(t, out=out) is out


@pytest.mark.parametrize("op", [attend, observe])
def test_scales_that_float32_does_not_hold(core, op):
    """As it is, and times log2(e)."""
    t = tensors()
    for scale in (1e-40, 1e-320, 2.4e38, 2.9e38, 1e300):
        with pytest.raises(ValueError, match="scale must be positive"):
            op(t, scale=scale)
    assert not core.calls
    for scale in (2.0 ** -126, 1, 2.0 ** 127):
        op(t, scale=scale)
        assert core.calls[-1][1][-3] == scale


def test_outputs_with_a_gradient_are_refused(core):
    """They would be written behind autograd's back."""
    t = tensors()
    grad = lambda x: (x + 0).requires_grad_()  # noqa: E731
    for call in (lambda: append(t, q_out=grad(t["q"])),
                 lambda: attend(t, out=grad(t["q"])),
                 lambda: evict(t, out=(grad(t["masses"]), t["places"],
                                       t["lens"]))):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    assert len(core.calls) == 3
