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
