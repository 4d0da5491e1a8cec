"""What the paged cache's operators refuse, and what they decide from values
on the device, on the CPU."""
import math

import pytest
import torch

from crowdllama_amd.ops import get_core, kv


def pool(pages=8, heads=2, page=16, dim=64, dtype=torch.bfloat16, layers=None):
    lead = (pages,) if layers is None else (pages, layers)
    return torch.zeros(*lead, heads, 2, page, dim, dtype=dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def attend_args(**kw):
    a = dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16), pool=pool(),
             table=torch.zeros(2, 4, dtype=torch.int32), lens=ints(1, 2))
    a.update(kw)
    return a


def refused(call, args, match):
    with pytest.raises(ValueError, match=match):
        call(**args)


def test_all_is_checked_before_the_device():
    refused(kv.attend, attend_args(), "must be on a GPU")
    refused(kv.attend, attend_args(mass=torch.zeros(2, 2, 64)),
            "must be on a GPU")


@pytest.mark.parametrize("kw,match", [
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.float16)), "does not go with"),
    (dict(q=torch.zeros(2, 4, 64), pool=pool(dtype=torch.float16)),
     "does not go with"),
    (dict(pool=pool(dtype=torch.float32)), "bfloat16 or float16"),
    (dict(q=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), "kv heads"),
    (dict(q=torch.zeros(2, 34, 64, dtype=torch.bfloat16)), "kv heads"),
    (dict(q=torch.zeros(2, 0, 64, dtype=torch.bfloat16)), "kv heads"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(2, 4, 96, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(2, 4, 128, dtype=torch.bfloat16)[..., ::2]),
     "contiguous"),
    (dict(q=torch.zeros(2, 4, 68, dtype=torch.bfloat16)[..., 4:]),
     "16-byte aligned"),
    (dict(lens=ints(1)), "lens must have 2"),
    (dict(lens=torch.tensor([1, 2])), "lens must be torch.int32"),
    (dict(lens=[1, 2]), "lens must be a tensor"),
    (dict(table=torch.zeros(2, 4)), "table must be torch.int32"),
    (dict(table=torch.zeros(2, 8, dtype=torch.int32)[:, ::2]), "contiguous"),
    (dict(table=torch.zeros(2, 0, dtype=torch.int32)), "empty"),
    (dict(pool=torch.zeros(8, 2, 64, 64, dtype=torch.bfloat16)),
     "pool must be"),
    (dict(pool=pool().transpose(2, 3)), "pool must be"),
    (dict(pool=pool(pages=1).expand(8, -1, -1, -1, -1)), "overlap"),
    (dict(pool=pool()[..., :32]), "contiguous"),
    (dict(mass=torch.zeros(2, 2, 65)), "1 to 64 places"),
    (dict(mass=torch.zeros(2, 4, 64)), "mass must be"),
    (dict(mass=torch.zeros(2, 2, 64, dtype=torch.float64)), "mass must be"),
    (dict(mass=torch.zeros(2, 1, 64).expand(2, 2, 64)), "overlap"),
    (dict(out=torch.zeros(2, 4, 64)), "out must be torch.bfloat16"),
    (dict(out=torch.zeros(1, 4, 64, dtype=torch.bfloat16).expand(2, 4, 64)),
     "overlap"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16, requires_grad=True)),
     "gradient"),
    (dict(scale=0.), "positive"), (dict(scale=-1.), "positive"),
    (dict(scale=math.nan), "positive"), (dict(scale=math.inf), "positive"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="meta")),
     "q is on meta"),
])
def test_attend_refuses(kw, match):
    refused(kv.attend, attend_args(**kw), match)


@pytest.mark.parametrize("kw,match", [
    (dict(), "must be on a GPU"),
    (dict(v=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), "v must be"),
    (dict(k=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), "k must be"),
    (dict(q=torch.zeros(2, 4, 64)), "q must be torch.bfloat16"),
    (dict(q_out=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), "without q"),
    (dict(inv_freq=torch.zeros(64)), "32 values"),
    (dict(inv_freq=torch.zeros(32).double()), "inv_freq must be"),
    (dict(starts=ints(0, 1)), "starts must have 3"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.bfloat16),
          v=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), "without starts"),
    (dict(pos=torch.zeros(2, 2, 64)), "pos must be torch.int32"),
    (dict(next_pos=ints(1)), "next_pos must have 2"),
])
def test_append_refuses(kw, match):
    a = dict(k=torch.zeros(2, 2, 64, dtype=torch.bfloat16),
             v=torch.zeros(2, 2, 64, dtype=torch.bfloat16), pool=pool(),
             table=torch.zeros(2, 4, dtype=torch.int32), lens=ints(0, 0),
             next_pos=ints(0, 0))
    a.update(kw)
    refused(kv.append, a, match)


@pytest.mark.parametrize("kw,match", [
    (dict(), "must be on a GPU"),
    (dict(mass=None), "mass must be a tensor"),
    (dict(starts=None), "without starts"),
    (dict(starts=ints(0, 1, 2, 3)), "starts must have 3"),
    (dict(q=torch.zeros(5, 64, dtype=torch.bfloat16)), "3 dimensions"),
])
def test_observe_refuses(kw, match):
    a = dict(q=torch.zeros(5, 4, 64, dtype=torch.bfloat16), pool=pool(),
             table=torch.zeros(2, 4, dtype=torch.int32), lens=ints(3, 2),
             mass=torch.zeros(2, 2, 64), starts=ints(0, 3, 5))
    a.update(kw)
    refused(kv.observe, a, match)


def evict_args(**kw):
    a = dict(pool=pool(layers=3), table=torch.zeros(2, 4, dtype=torch.int32),
             lens=ints(3, 2), next_pos=ints(3, 2),
             mass=torch.zeros(3, 2, 2, 64),
             pos=torch.zeros(3, 2, 2, 64, dtype=torch.int32), keep=5)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(), "must be on a GPU"),
    (dict(keep=0), "keep must be"),
    (dict(recent=-1), "keep must be"),
    (dict(limit=4), "keep must be"),
    (dict(limit=1 << 31), "below 2"),
    (dict(pool=pool()), "pool must be"),
    (dict(pos=torch.zeros(3, 2, 2, 63, dtype=torch.int32)), "equally many"),
    (dict(mass=torch.zeros(2, 2, 2, 64)), "mass must be"),
    (dict(pool=pool(layers=1).expand(8, 3, -1, -1, -1, -1)), "overlap"),
    (dict(out=(torch.zeros(3, 2, 2, 60),
               torch.zeros(3, 2, 2, 64, dtype=torch.int32), ints(0, 0))),
     "as many places"),
    (dict(mass=torch.zeros(1).expand(3, 2, 2, 64)), "contiguous"),
    (dict(mass=torch.zeros(3, 2, 1, 64).expand(3, 2, 2, 64)), "overlap"),
    (dict(mass=torch.zeros(3, 2, 2, 64, requires_grad=True)), "gradient"),
])
def test_evict_refuses(kw, match):
    refused(kv.evict, evict_args(**kw), match)


def test_evict_refuses_a_mixed_out():
    a = evict_args()
    b = torch.zeros(3, 2, 2, 65)
    a["mass"] = b[..., :64]
    refused(kv.evict, {**a, "out": (b[..., 1:], a["pos"], a["lens"])}, "apart")
    refused(kv.evict, {**a, "out": (a["mass"], a["pos"], a["next_pos"])},
            "apart")
    refused(kv.evict, {**a, "out": (a["mass"], a["pos"], a["lens"])},
            "must be on a GPU")
    refused(kv.evict, {**a, "out": (torch.zeros(3, 2, 2, 64), a["pos"],
                                    ints(0, 0))}, "must be on a GPU")


def test_evict_refuses_what_overlaps():
    a = evict_args()
    refused(kv.evict, {**a, "next_pos": a["lens"]}, "apart")
    refused(kv.evict, {**a, "pos": a["mass"].view(torch.int32)}, "apart")
    both = ints(1, 2, 3)
    refused(kv.evict, {**a, "lens": both[:2], "next_pos": both[1:]}, "apart")
    both = ints(1, 2, 3, 4)
    refused(kv.evict, {**a, "lens": both[2:], "next_pos": both[:2]},
            "must be on a GPU")


def test_evict_refuses_an_out_that_overlaps():
    a, t = evict_args(), torch.zeros(3, 2, 2, 64)
    refused(kv.evict, {**a, "out": (t, t.view(torch.int32), ints(0, 0))},
            "apart")
    refused(kv.evict, {**a, "out": (a["pos"].view(torch.float32), a["pos"],
                                    a["lens"])}, "apart")
    refused(kv.evict, {**a, "next_pos": a["lens"],
                       "out": (t, a["pos"], a["lens"])}, "apart")
    refused(kv.evict, {**a, "next_pos": a["lens"],
                       "out": (t, a["pos"], ints(0, 0))}, "must be on a GPU")


def pages_arg(page=16, dim=64, slots=1, heads=1, kind=2, max_pages=4):
    return (0, 0, 1, 0, 0, max_pages, page, slots, heads, dim, kind, 0)


@pytest.mark.parametrize("kw,reach,match", [
    (dict(page=8), 32, "page size"), (dict(page=40), 32, "page size"),
    (dict(page=2048), 32, "page size"), (dict(dim=80), 32, "head_dim"),
    (dict(dim=256), 32, "head_dim"), (dict(kind=0), 32, "bfloat16"),
    (dict(), 65, "2\\^30"), (dict(), -1, "2\\^30"),
    (dict(max_pages=1 << 27), (1 << 30) + 1, "2\\^30"),
    (dict(max_pages=1 << 26, slots=4096), 1 << 30, "too many places"),
])
def test_sizes_that_the_kernels_do_not_take(kw, reach, match):
    core = get_core()
    with pytest.raises(RuntimeError, match=match):
        core.kv_attend_workspace(pages_arg(**kw), 1, reach, True)


def test_a_chunk_needs_no_more_than_the_most():
    """The workspace of fewer rows may be larger (they are cut finer): the
    engine takes the most over all chunks."""
    core = get_core()
    page = pages_arg(max_pages=8192, heads=8, dim=128)
    need = [core.kv_observe_workspace(page, 32, m, 131072, 0)
            for m in range(1, 1025)]
    assert all(n > 0 for n in need) and max(need) < 64 << 20
    with pytest.raises(RuntimeError, match="too many rows"):
        core.kv_observe_workspace(page, 32, 1 << 27, 131072, 0)


@pytest.mark.parametrize("first,then", [
    ("import torch", "from crowdllama_amd.ops import get_core; get_core()"),
    ("from crowdllama_amd.ops import get_core; get_core()", "import torch")])
def test_one_hip_runtime(first, then):
    """torch's runtime serves both if it is loaded first; otherwise the
    operators would be handed streams of another runtime, and refuse."""
    import subprocess
    import sys
    code = (f"{first}\n{then}\nfrom crowdllama_amd.ops import kv\n"
            "try:\n    kv._one_runtime()\n    print('one')\n"
            "except RuntimeError as e:\n    print(str(e)[:16])\n"
            "print(sum('libamdhip64' in x and x.split()[2] == '00000000'\n"
            "          for x in open('/proc/self/maps')))")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True,
                         text=True, timeout=120, check=True).stdout.split("\n")
    # where the system's and torch's libraries are one file, both orders work
    assert out[0] == ("one" if out[1] == "1" else "two HIP runtimes")
    if first == "import torch":
        assert out[0] == "one"


def test_pages_outside_the_pool_are_not_followed():
    find = get_core().test_kv_page_of
    row = [3, -1, 5, 4, 2 ** 31 - 1, -2 ** 31]
    assert [find(row, i, 5) for i in range(-1, 8)] == [
        -1, 3, -1, -1, 4, -1, -1, -1, -1]
    assert find(row, 2 ** 40, 5) == -1 and find(row, -2 ** 40, 5) == -1


def test_lengths_are_cut():
    cut = get_core().test_kv_clamp_len
    assert [cut(x, 64) for x in (-2 ** 31, -1, 0, 1, 64, 65, 2 ** 31 - 1)] \
        == [0, 0, 0, 1, 64, 64, 64]


def test_order_of_eviction():
    key = get_core().test_kv_rank_key
    masses = [math.nan, -math.inf, -3e38, -1., -1e-45, 0., 1e-45, 1e-3, 1.,
              3e38, math.inf]
    keys = [key(m, False) for m in masses]
    assert keys == sorted(keys) and len(set(keys)) == len(keys)
    assert key(-0., False) == key(0., False)
    assert key(math.copysign(math.nan, -1), False) == keys[0]
    assert all(key(m, True) == 2 ** 32 - 1 > max(keys) for m in masses)


def test_token_budget():
    from crowdllama_amd.engine.api import token_budget
    assert token_budget(100, 20, 64, 64) == 43
    assert token_budget(10, 20, 64, 64) == 10
    assert token_budget(100, 63, 64, 64) == 0
    assert token_budget(100, 20, 64, 1024, kv_keep=40) == 100
    assert token_budget(5000, 20, 64, 1024, kv_keep=40) == 1024
    assert token_budget(100, 63, 64, 1024, kv_keep=40) < 1


def test_reference_evicts(tmp_path):
    """The numpy reference past max_seq: every head keeps the newest tokens,
    and its places' masses add up to what the tokens gave."""
    from crowdllama_amd.engine.ref_numpy import RefLlama
    from crowdllama_amd.models import write_synthetic_gguf
    path = write_synthetic_gguf(str(tmp_path / "t.gguf"), "testllama",
                                scheme="f32", mode="exact", seed=1)
    full = RefLlama(path)
    ref = RefLlama(path, max_seq=12, kv_keep=7, kv_recent=3)
    for i in range(12):
        a, b = full.step(i + 3), ref.step(i + 3)
        assert abs(a - b).max() < 1e-5 * abs(a).max()
    ref.step(50)
    for layer in ref.places:
        for row in layer:
            pos = [e[3] for e in row]
            assert len(row) == 8 and len(set(pos)) == 8 and pos[-1] == 12
            assert {9, 10, 11} <= set(pos)
    ref.reset()
    assert ref.n_past == 0 and ref.places[0][0] == []
