"""The engines' loops around the native engine, on the CPU: what they ask of it
and what they make of its tokens."""
import threading
import time

import pytest

from crowdllama_amd.engine.api import RollingRate, TextStream
from crowdllama_amd.engine.batching import BatchingHipEngine, _Req, _Slot
from crowdllama_amd.engine.hip_engine import HipEngine
from crowdllama_amd.tokenizer import NativeTokenizer, Tokenizer

BYTES = ["<unk>", "<s>", "</s>"] + [f"<0x{b:02X}>" for b in range(256)]
EOS = 2
TEXT = "na\u00efve \u20ac5 \U0001f600 \ufffd ok"


class Native:
    """A native engine that generates the given tokens, then others."""

    def __init__(self, texts):
        self.texts, self.made = texts, [0] * len(texts)
        self.active = [True] * len(texts)
        self.steps, self.handed = 0, 0

    def reset(self):
        self.made = [0] * len(self.texts)

    def reset_slot(self, slot):
        self.made[slot] = 0

    def set_slot_active(self, slot, on):
        self.active[slot] = on

    def prefill(self, ids):
        self.made = [1] * len(self.texts)

    def prefill_slot(self, slot, ids):
        self.made[slot], self.active[slot] = 1, True

    def decode(self, n):
        self.steps += n
        self.made = [m + n * a for m, a in zip(self.made, self.active)]

    def gen_tokens(self, slot, first=0):
        t = self.texts[slot]
        out = [t[i] if i < len(t) else 3 + 65
               for i in range(first, self.made[slot])]
        self.handed += len(out)
        return out


def tokens(text, eos=True):
    return [3 + b for b in text.encode()] + [EOS] * eos


def hip(texts, max_seq=4096):
    e = HipEngine.__new__(HipEngine)
    e.eng, e.tok = Native(texts), NativeTokenizer(BYTES)
    e._lock, e._rate = threading.Lock(), RollingRate()
    e.max_seq, e.gen_cap, e.kv_keep = max_seq, 16 * max_seq, max_seq // 2
    return e


def batching(texts):
    e = BatchingHipEngine.__new__(BatchingHipEngine)
    e.eng, e.tok = Native(texts), NativeTokenizer(BYTES)
    e._rate, e._active = RollingRate(), len(texts)
    e._slots = [_Slot() for _ in texts]
    return e


@pytest.mark.parametrize("kind", [Tokenizer, NativeTokenizer])
def test_text_as_it_comes(kind):
    """In pieces of any size it is the whole text, and no piece ends within a
    character."""
    tok = kind(BYTES)
    ids = tokens(TEXT) + [3 + 0xE2, 3 + 0x82]      # and a part of one
    whole = tok.decode(ids)
    assert whole == TEXT + "\ufffd"
    assert tok.decode_bytes(ids) == TEXT.encode() + b"\xe2\x82"
    for size in range(1, len(ids) + 1):
        text = TextStream(tok)
        parts = [text.add(ids[i:i + size], i + size >= len(ids))
                 for i in range(0, len(ids), size)]
        assert "".join(parts) == whole
        assert whole.startswith("".join(parts[:-1]))


@pytest.mark.parametrize("limit", [5000, 20, 7, 1])
def test_stream(limit):
    e, got = hip([tokens(TEXT * 30)]), []
    e._stream_sync("hello", limit, 0.0, got.append)
    want = tokens(TEXT * 30, eos=False)[:limit]
    assert "".join(r.text for r in got) == e.tok.decode(want)
    assert [bool(r.done_reason) for r in got] == [False] * (len(got) - 1) + [
        True]
    assert got[-1].tokens_generated == len(want)
    assert got[-1].done_reason == ("stop" if len(want) < limit else "length")
    # each token is handed out once
    assert e.eng.handed <= len(want) + e.STREAM_STRIDE


def run(e, reqs):
    class Loop:
        def call_soon_threadsafe(self, f, x):
            f(x)

    class Chunks(list):
        put_nowait = list.append

    for slot, (i, (limit, stream)) in zip(e._slots, enumerate(reqs)):
        req = _Req(ids=[1], max_new=limit, t0=time.monotonic_ns())
        if stream:
            req.chunks, req.loop = Chunks(), Loop()
        e.eng.prefill_slot(i, req.ids)
        slot.req, slot.collected = req, 0
        slot.text, slot.parts = TextStream(e.tok), []
    all_ = [s.req for s in e._slots]
    for _ in range(10000):
        if not e._active:
            return all_
        e.eng.decode(8)
        e._harvest()
    raise AssertionError("does not end")


def test_harvest():
    texts = [TEXT * 30, TEXT, "x" * 50, ""]
    limits = [(5000, True), (9, True), (50, False), (10, True)]
    e = batching([tokens(t) for t in texts])
    for (limit, stream), text, req in zip(limits, texts, run(e, limits)):
        want = tokens(text, eos=False)[:limit]
        r = req.future.result(timeout=0)
        assert r.text == e.tok.decode(want)
        assert r.tokens_generated == len(want)
        assert r.done_reason == ("stop" if len(want) < limit else "length")
        if stream:
            assert "".join(c.text for c in req.chunks) == r.text
            assert req.chunks[-1].done_reason == r.done_reason
            assert not any(c.done_reason for c in req.chunks[:-1])
    assert not any(e.eng.active)
    assert e.eng.handed <= sum(len(tokens(t)) + 8 for t in texts)


@pytest.mark.parametrize("limit", [5000, 70, 33, 32, 2, 1])
@pytest.mark.parametrize("text", [TEXT * 30, TEXT, "x" * 31, ""])
def test_greedy(limit, text):
    """A request that ends early does not hold the engine to its limit."""
    e = hip([tokens(text)])
    r = e._generate_sync("hello", limit)
    want = tokens(text)[:limit]
    ended = EOS in want
    assert r.text == e.tok.decode(want)
    assert r.tokens_generated == len(want) - ended
    assert r.done_reason == ("stop" if ended else "length")
    assert len(want) - 1 <= e.eng.steps < len(want) + e.STRIDE
    assert e.eng.steps <= limit - 1


@pytest.mark.parametrize("gone", [False, True])
def test_a_failed_step_parks_the_slots(gone):
    """Every request hears of it, and no slot goes on without one."""
    e = batching([tokens(TEXT), tokens(TEXT)])
    e._stop, e._admit = False, lambda: None

    def decode(n):
        e._stop = True
        raise RuntimeError("step")
    e.eng.decode = decode
    if gone:
        def park(slot, on):
            raise RuntimeError("gone")
        e.eng.set_slot_active = park
    reqs = [_Req(ids=[1], max_new=9) for _ in e._slots]
    for i, (slot, req) in enumerate(zip(e._slots, reqs)):
        e.eng.prefill_slot(i, req.ids)
        slot.req = req
    e._loop()
    for req in reqs:
        with pytest.raises(RuntimeError, match="step"):
            req.future.result(timeout=0)
    assert e._active == 0 and e.eng.active == [gone, gone]


@pytest.mark.gpu
def test_idle_slots_stay_empty(tmp_path):
    """One request of four slots' engine, twice its cache: the others neither
    fill theirs nor evict, before and after."""
    import asyncio
    from crowdllama_amd.models import write_synthetic_gguf
    path = write_synthetic_gguf(str(tmp_path / "t.gguf"), "testllama",
                                scheme="f32", mode="exact", seed=11)
    eng = BatchingHipEngine("m", path, batch=4, max_seq=64, kv_keep=40,
                            kv_recent=8)

    def empty():
        # a slot is parked right after its request is told
        for _ in range(100):
            if eng.eng.kv_lens() == eng.eng.n_past() == [0] * 4:
                return True
            time.sleep(0.01)
        return False
    try:
        asyncio.run(eng.generate("hello", 150))
        assert empty()
        async def go():
            await asyncio.gather(eng.generate("hello", 150),
                                 eng.generate("there", 30))
        asyncio.run(go())
        assert empty()
    finally:
        asyncio.run(eng.close())
