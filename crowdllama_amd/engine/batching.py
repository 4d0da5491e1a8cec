"""Continuous-batching engine: concurrent requests share the decode slots
of one HIP engine instance.

The reference serves one request per worker at a time (its per-request
Ollama POST); this is the MI355X-native upgrade: the decode step is
weight-bandwidth-bound, so B concurrent sequences cost barely more than
one (measured: B=32 decodes ~5000 tok/s aggregate vs ~300 at B=1 on
llama3-8b Q4_K_M). A background thread admits queued prompts into free
slots (per-slot chunked-GEMM prefill), steps all slots together in decode
strides, and completes futures as sequences hit EOS or their token budget.
"""

from __future__ import annotations

import asyncio
import queue
import threading
import time
from concurrent.futures import Future
from dataclasses import dataclass, field


from ..quant.gguf import GGUFReader
from ..tokenizer import NativeTokenizer, Tokenizer
from .api import EngineBase, GenerateResult, RollingRate, TextStream
from .api import EVICTING_GEN, token_budget

DECODE_STRIDE = 8  # graph replays between slot bookkeeping passes


@dataclass
class _Req:
    ids: list[int]
    max_new: int
    future: Future = field(default_factory=Future)
    t0: int = 0
    # streaming: deltas are pushed onto `chunks` (an asyncio.Queue) via
    # `loop.call_soon_threadsafe` from the batcher thread
    chunks: object = None
    loop: object = None

    def push(self, item) -> None:
        if self.chunks is not None and self.loop is not None:
            self.loop.call_soon_threadsafe(self.chunks.put_nowait, item)


class _Slot:
    def __init__(self):
        self.req: _Req | None = None
        self.collected = 0                    # tokens that are in `parts`
        self.text: TextStream | None = None
        self.parts: list[str] = []


class BatchingHipEngine(EngineBase):
    def __init__(self, model_name: str, gguf_path: str, device: int = 0,
                 batch: int = 8, max_seq: int = 4096, max_new: int = 256,
                 kv_keep: int = 0, kv_recent: int = 0):
        from ..ops import get_core
        core = self._core = get_core()
        if core.device_count() == 0:
            raise RuntimeError("BatchingHipEngine requires a GPU")
        self.model_name = model_name
        cfg = core.EngineConfig()
        cfg.batch = batch
        cfg.max_seq = max_seq
        # size the generated-token ring from max_seq so a request's max_new
        # can never exceed it (with max_new > gen_cap it would saturate the
        # ring and decode forever)
        cfg.gen_cap = max_seq * EVICTING_GEN if kv_keep else max_seq
        # past max_seq by eviction, as HipEngine
        cfg.kv_keep, cfg.kv_recent = kv_keep, kv_recent
        self.kv_keep = kv_keep
        cfg.device = device
        self.eng = core.Engine(gguf_path, cfg)
        self.gen_cap = cfg.gen_cap
        with GGUFReader(gguf_path) as r:
            try:
                self.tok = NativeTokenizer.from_gguf(r)
            except Exception:
                import logging
                logging.getLogger("crowdllama_amd.engine").warning(
                    "native tokenizer unavailable for %s; falling back to "
                    "the Python tokenizer", gguf_path, exc_info=True)
                self.tok = Tokenizer.from_gguf(r)
        self._props = core.device_props(device)
        self.batch = batch
        self.max_seq = max_seq
        self.default_max_new = max_new
        self._rate = RollingRate()
        # bounded admission queue: reject instead of piling unbounded work
        # behind a saturated engine (gateway failover retries elsewhere)
        self._queue: "queue.Queue[_Req]" = queue.Queue(maxsize=8 * batch)
        self._slots = [_Slot() for _ in range(batch)]
        # a slot without a request is parked: with kv_keep it would fill its
        # cache, attend to all of it and evict, for nothing
        for i in range(batch):
            self.eng.set_slot_active(i, False)
        self._wake = threading.Event()
        self._stop = False
        self._active = 0
        self._thread = threading.Thread(target=self._loop, daemon=True,
                                        name="cla-batcher")
        self._thread.start()

    # -------------------------------------------------------------- loop

    def _admit(self) -> None:
        for i, slot in enumerate(self._slots):
            if slot.req is not None:
                continue
            try:
                req = self._queue.get_nowait()
            except queue.Empty:
                return
            self.eng.reset_slot(i)
            self.eng.prefill_slot(i, req.ids)
            slot.req = req
            slot.collected = 0
            slot.text, slot.parts = TextStream(self.tok), []
            self._active += 1

    def _park(self, i: int) -> None:
        self.eng.set_slot_active(i, False)
        self.eng.reset_slot(i)

    def _harvest(self) -> None:
        for i, slot in enumerate(self._slots):
            req = slot.req
            if req is None:
                # idle slots are parked (set_slot_active False) when their
                # request completes: the decode step no longer advances them,
                # so no per-stride reset is needed
                continue
            # the new ones only: a long request must not cost more a stride
            toks = list(self.eng.gen_tokens(i, slot.collected))
            done = False
            if self.tok.eos_id in toks:
                toks = toks[: toks.index(self.tok.eos_id)]
                done = True
            if slot.collected + len(toks) >= req.max_new:
                toks = toks[: req.max_new - slot.collected]
                done = True
            slot.collected += len(toks)
            delta = slot.text.add(toks, done)
            slot.parts.append(delta)
            count = slot.collected
            if done:
                self._rate.add(count)
                reason = "stop" if count < req.max_new else "length"
                req.push(GenerateResult(
                    text=delta, tokens_generated=count,
                    duration_ns=time.monotonic_ns() - req.t0,
                    done_reason=reason))
                req.future.set_result(GenerateResult(
                    text="".join(slot.parts), tokens_generated=count,
                    duration_ns=time.monotonic_ns() - req.t0,
                    done_reason=reason))
                slot.req = None
                self._active -= 1
                self._park(i)
            elif delta:
                req.push(GenerateResult(text=delta, tokens_generated=count,
                                        done_reason=""))

    def _loop(self) -> None:
        while not self._stop:
            try:
                self._admit()
                if self._active == 0:
                    self._wake.wait(timeout=0.05)
                    self._wake.clear()
                    continue
                self.eng.decode(DECODE_STRIDE)
                self._harvest()
            except Exception as e:  # noqa: BLE001
                # fatal engine error: fail every waiting request instead of
                # leaving their futures hanging, then keep serving new ones
                for i, slot in enumerate(self._slots):
                    req, slot.req = slot.req, None
                    if req is None:
                        continue
                    self._active -= 1
                    req.push(GenerateResult(text="", done_reason="error"))
                    if not req.future.done():
                        req.future.set_exception(RuntimeError(
                            f"batch engine error: {e}"))
                    try:
                        self._park(i)
                    except Exception:  # noqa: BLE001  the engine is gone
                        pass

    # --------------------------------------------------------------- api

    def _make_req(self, prompt: str, max_new_tokens: int, **kw) -> _Req:
        ids = self.tok.encode(prompt)
        # clamp to both the sequence budget and the engine's generated-token
        # ring (gen_cap): tokens past gen_cap are never recorded, so a
        # max_new above it would otherwise decode forever
        max_new = token_budget(max_new_tokens or self.default_max_new,
                               len(ids), self.max_seq, self.gen_cap,
                               self.kv_keep)
        if max_new < 1:
            raise ValueError("prompt exceeds max_seq")
        return _Req(ids=ids or [self.tok.bos_id], max_new=max_new,
                    t0=time.monotonic_ns(), **kw)

    def _enqueue(self, req: _Req) -> None:
        try:
            self._queue.put_nowait(req)
        except queue.Full:
            raise RuntimeError("engine request queue full") from None
        self._wake.set()

    async def generate(self, prompt: str, max_new_tokens: int = 256,
                       temperature: float = 0.0) -> GenerateResult:
        # batched mode is greedy (per-slot host sampling would serialize)
        req = self._make_req(prompt, max_new_tokens)
        self._enqueue(req)
        return await asyncio.wrap_future(req.future)

    async def generate_stream(self, prompt: str, max_new_tokens: int = 256,
                              temperature: float = 0.0):
        """Streaming under continuous batching: deltas are emitted as the
        shared decode strides advance this request's slot."""
        req = self._make_req(prompt, max_new_tokens,
                             chunks=asyncio.Queue(),
                             loop=asyncio.get_running_loop())
        self._enqueue(req)
        while True:
            chunk = await req.chunks.get()
            yield chunk
            if chunk.done_reason:
                break
        await asyncio.wrap_future(req.future)

    def throughput(self) -> float:
        r = self._rate.rate()
        return r if r > 0 else 100.0

    def load(self) -> float:
        return min(1.0, self._active / max(1, self.batch))

    def vram_gb(self) -> float:
        return float(self._props["total_mem_gb"])

    def gpu_model(self) -> str:
        return str(self._props["name"])

    async def close(self) -> None:
        self._stop = True
        self._wake.set()
        self._thread.join(timeout=5)
