"""Decoding past the end of the KV cache: the engine with kv_keep against the
numpy reference. The engine's products round to bfloat16 on some paths, so its
masses are near the reference's but may order two places otherwise: which
places stay is checked against the engine's own masses, and the reference goes
on with the same ones."""
import numpy as np
import pytest

import kv_oracle as oracle

pytestmark = pytest.mark.gpu

MAX_SEQ, KEEP, RECENT = 48, 30, 6

# Prefill and batched products round both operands to bfloat16: an output is
# off by 2^-9 sqrt(2 / 3) = 1.6e-3 of its size (rms), after a path of some
# eight products by sqrt(8) times that, 4.5e-3. Of 512 logits the one that is
# furthest off is at 3.5 of that and the largest logit at 3.4 of theirs, so
# 4.6e-3 of the largest is ordinary, and three times that is not.
LOGITS = 1.5e-2


@pytest.fixture(scope="module")
def core():
    from crowdllama_amd.ops import get_core
    c = get_core()
    if c.device_count() == 0:
        pytest.skip("no GPU")
    return c


@pytest.fixture(scope="module")
def gguf(tmp_path_factory):
    from crowdllama_amd.models import write_synthetic_gguf
    path = str(tmp_path_factory.mktemp("m") / "tiny.gguf")
    return write_synthetic_gguf(path, "testllama", scheme="f32",
                                mode="exact", seed=11)


def engine(core, gguf, batch=1, keep=KEEP, max_seq=MAX_SEQ, **kw):
    cfg = core.EngineConfig()
    cfg.batch, cfg.max_seq = batch, max_seq
    cfg.act_q8 = False
    cfg.kv_keep, cfg.kv_recent = keep, RECENT if keep else 0
    for k, v in kw.items():
        setattr(cfg, k, v)
    return core.Engine(gguf, cfg)


def prompt(n, seed=3):
    return np.random.default_rng(seed).integers(3, 512, n).tolist()


def reference(gguf):
    from crowdllama_amd.engine.ref_numpy import RefLlama
    # it never evicts by itself
    return RefLlama(gguf, max_seq=1 << 30, kv_keep=1)


def follow(eng, refs):
    """Before a step: evict in the references whose slots are full what the
    engine's masses say."""
    for slot, (ref, n) in enumerate(zip(refs, eng.kv_lens())):
        if n < MAX_SEQ:
            continue
        late = eng.n_past()[slot] - RECENT
        for layer, rows in enumerate(ref.places):
            pos, mass = eng.kv_places(layer, slot)
            for h, row in enumerate(rows):
                stay = oracle.survivors(mass[h], pos[h], late, KEEP)
                come = iter([row[p] for p in sorted(stay) if p >= KEEP])
                rows[h] = [row[p] if p in stay else next(come)
                           for p in range(KEEP)]


def check_places(eng, ref, slot):
    n = eng.kv_lens()[slot]
    for layer, rows in enumerate(ref.places):
        pos, mass = eng.kv_places(layer, slot)
        assert pos.shape == (len(rows), n)
        for h, row in enumerate(rows):
            assert len(row) == n
            assert pos[h].tolist() == [e[3] for e in row]
            np.testing.assert_allclose(mass[h], [e[2] for e in row],
                                       rtol=2e-2, atol=1e-4)


@pytest.mark.parametrize("use_graph", [True, False])
@pytest.mark.parametrize("chunk", [1024, 16])
def test_engine_goes_on_past_max_seq(core, gguf, use_graph, chunk):
    """Two evictions; after each token the logits are the reference's, which
    is fed the engine's tokens."""
    eng = engine(core, gguf, use_graph=use_graph, prefill_chunk=chunk)
    ref = reference(gguf)
    ids = prompt(41)
    eng.prefill(np.array([ids], dtype=np.int32))
    for t in ids:
        want = ref.step(t)
    check_places(eng, ref, 0)
    for _ in range(45):
        got = np.asarray(eng.logits(0))
        assert np.abs(got - want).max() < LOGITS * np.abs(want).max()
        follow(eng, [ref])
        want = ref.step(eng.cur_token(0))
        eng.decode(1)
        check_places(eng, ref, 0)
    # full at 48 and, 18 tokens later, at 66 and 84
    assert eng.n_past() == [86] and eng.kv_lens() == [KEEP + 86 - 84]


def test_without_a_full_cache_nothing_changes(core, gguf):
    a, b = engine(core, gguf), engine(core, gguf, keep=0)
    ids = np.array([prompt(20)], dtype=np.int32)
    for e in (a, b):
        e.prefill(ids)
    for _ in range(10):
        x, y = np.asarray(a.logits(0)), np.asarray(b.logits(0))
        assert np.abs(x - y).max() < LOGITS * np.abs(y).max()
        b.set_cur_token(0, a.cur_token(0))
        a.decode(1)
        b.decode(1)
    assert a.kv_lens() == b.kv_lens() == [30]


def test_a_cache_longer_than_one_workgroup_takes(core, gguf):
    """The attention's form for long rows: the logits of the engine without
    eviction, and weights that sum to one for each query head of each token."""
    a = engine(core, gguf, keep=1000, max_seq=1100)
    b = engine(core, gguf, keep=0, max_seq=1100)
    ids = np.array([prompt(700)], dtype=np.int32)
    for e in (a, b):
        e.prefill(ids)
    for _ in range(10):
        x, y = np.asarray(a.logits(0)), np.asarray(b.logits(0))
        assert np.abs(x - y).max() < LOGITS * np.abs(y).max()
        b.set_cur_token(0, a.cur_token(0))
        a.decode(1)
        b.decode(1)
    sums = [a.kv_places(layer, 0)[1].sum(-1) for layer in (0, 1)]
    # the last token's own weights count too; 710 sums of up to 710 weights
    ref = reference(gguf)
    group = ref.heads // ref.kv_heads
    np.testing.assert_allclose(sums, 710 * group, rtol=1e-3)


@pytest.mark.parametrize("batch", [2, 5])
def test_slots_evict_on_their_own(core, gguf, batch):
    """Slots of other lengths, one parked on the way: each is as it would be
    alone, in the same strides."""
    eng = engine(core, gguf, batch=batch)
    refs, wants = [], []
    for b in range(batch):
        ref = reference(gguf)
        ids = prompt(5 + 9 * b, seed=b)
        eng.prefill_slot(b, ids)
        for t in ids:
            want = ref.step(t)
        refs.append(ref)
        wants.append(want)
    parked = batch - 1
    for i in range(50):
        if i == 10:
            eng.set_slot_active(parked, False)
        if i == 15:
            eng.set_slot_active(parked, True)
        follow(eng, refs)
        for b in range(batch):
            if b == parked and 10 <= i < 15:
                continue
            if b == parked and i == 15:
                # its logits were written while it was parked
                wants[b] = refs[b].step(eng.cur_token(b))
                continue
            got = np.asarray(eng.logits(b))
            assert np.abs(got - wants[b]).max() < \
                LOGITS * np.abs(wants[b]).max(), (i, b)
            wants[b] = refs[b].step(eng.cur_token(b))
        eng.decode(1)
        if 10 <= i < 15:
            check_places(eng, refs[parked], parked)
    for b in range(batch):
        check_places(eng, refs[b], b)
    assert eng.kv_lens()[0] < MAX_SEQ


def test_a_slot_starts_anew(core, gguf):
    """After an eviction too, a prompt finds an empty slot."""
    eng = engine(core, gguf)
    ids = np.array([prompt(30)], dtype=np.int32)
    eng.prefill(ids)
    first = np.asarray(eng.logits(0))
    for again in (eng.reset, lambda: eng.reset_slot(0), lambda: None):
        eng.decode(60)
        assert eng.n_past() == [90] and KEEP < eng.kv_lens()[0] < MAX_SEQ
        again()
        eng.prefill(ids)
        assert eng.kv_lens() == [30] and eng.n_past() == [30]
        for layer in range(2):
            pos, mass = eng.kv_places(layer, 0)
            assert (pos == np.arange(30)).all()
            # two query heads' weights of 30 tokens
            assert np.allclose(mass.sum(1), 60, atol=1e-3)
        got = np.asarray(eng.logits(0))
        assert np.abs(got - first).max() < LOGITS * np.abs(first).max()


def test_quantized_and_many_slots(core, tmp_path_factory):
    """The int8 GEMM path, whose output projection has its own quantizer
    where attention does not quantize."""
    from crowdllama_amd.models import write_synthetic_gguf
    path = str(tmp_path_factory.mktemp("m") / "q.gguf")
    write_synthetic_gguf(path, "testllama", scheme="q4_k_m", mode="exact",
                         seed=7)
    a = engine(core, path, batch=4, act_q8=True)
    b = engine(core, path, batch=4, keep=0, act_q8=True)
    for e in (a, b):
        for s in range(4):
            e.prefill_slot(s, prompt(12 + s, seed=s))
        e.decode(3)
    for s in range(4):
        x, y = np.asarray(a.logits(s)), np.asarray(b.logits(s))
        assert np.abs(x - y).max() < 5e-2 * np.abs(y).max()
    a.decode(100)
    assert all(KEEP <= n <= MAX_SEQ for n in a.kv_lens())
    assert a.n_past() == [115, 116, 117, 118]


@pytest.mark.parametrize("kw,match", [
    (dict(kv_keep=MAX_SEQ), "kv_keep"), (dict(kv_keep=-1), "kv_keep"),
    (dict(kv_recent=KEEP + 1), "kv_recent"),
    (dict(kv_recent=-1), "kv_recent"), (dict(page_size=24), "page_size")])
def test_refusals(core, gguf, kw, match):
    with pytest.raises(RuntimeError, match=match):
        engine(core, gguf, **kw)
    with pytest.raises(RuntimeError, match="no kv_keep"):
        engine(core, gguf, keep=0).kv_places(0, 0)
    with pytest.raises(RuntimeError, match="no such layer"):
        engine(core, gguf).kv_places(2, 0)


def test_served_past_max_seq(core, gguf):
    """Both engines give a request more tokens than the cache has places."""
    import asyncio
    from crowdllama_amd.engine.batching import BatchingHipEngine
    from crowdllama_amd.engine.hip_engine import HipEngine
    for cls, kw in ((HipEngine, {}), (BatchingHipEngine, {"batch": 3})):
        eng = cls("testllama", gguf, max_seq=64, kv_keep=40, kv_recent=8,
                  **kw)
        r = asyncio.run(eng.generate("hello", 150))
        assert r.tokens_generated == 150 or r.done_reason == "stop"
        asyncio.run(eng.close())
