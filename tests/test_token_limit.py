"""How many tokens a worker generates for a request, from its configuration to
the engine."""
import asyncio

import pytest

from crowdllama_amd import cli
from crowdllama_amd.config import Config
from crowdllama_amd.engine.api import EngineBase, GenerateResult
from crowdllama_amd.mesh import pb
from crowdllama_amd.mesh.peer import Peer


class Wire:
    """A stream that holds one request and takes the answers."""

    def __init__(self, message):
        self.message, self.answers = message, []

    async def read_frame(self, timeout=None):
        return self.message.encode()

    async def write_frame(self, data):
        self.answers.append(pb.BaseMessage.decode(data).generate_response)


class Counting(EngineBase):
    def __init__(self):
        self.asked = []

    async def generate(self, prompt, max_new_tokens=256, temperature=0.0):
        self.asked.append(max_new_tokens)
        return GenerateResult("x " * max_new_tokens, max_new_tokens)


def ask(engine, cfg, stream):
    peer = Peer(cfg, worker_mode=True, engines={"m": engine})
    wire = Wire(pb.request_message("m", "hello", stream))
    asyncio.run(peer._handle_inference(wire))
    return wire.answers


@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("limit", [None, 1, 5000])
def test_a_worker_asks_its_engine_for_as_many(tmp_path, stream, limit):
    kw = {} if limit is None else {"max_new_tokens": limit}
    engine = Counting()
    answers = ask(engine, Config(key_path=str(tmp_path / "k"), **kw), stream)
    assert engine.asked == [limit or 256]
    assert len(answers[-1].response.split()) == (limit or 256)


def test_the_command_line_says_it(monkeypatch, capsys):
    seen = []

    async def start(args):
        seen.append((args.max_new_tokens, args.kv_keep, args.kv_recent))
    monkeypatch.setattr(cli, "_run_start", start)
    cli.main(["start", "--worker-mode"])
    cli.main(["start", "--worker-mode", "--max-new-tokens", "9000",
              "--kv-keep", "2048", "--kv-recent", "512"])
    assert seen == [(256, 0, 0), (9000, 2048, 512)]
    for wrong in (["--max-new-tokens", "0"], ["--kv-recent", "5"]):
        with pytest.raises(SystemExit):
            cli.main(["start", *wrong])
        assert wrong[0] in capsys.readouterr().err


@pytest.mark.gpu
@pytest.mark.parametrize("stream", [False, True])
@pytest.mark.parametrize("batch", [1, 2])
def test_served_past_max_seq(tmp_path, stream, batch):
    """More tokens than the cache has places, through the worker."""
    from crowdllama_amd.engine.batching import BatchingHipEngine
    from crowdllama_amd.engine.hip_engine import HipEngine
    from crowdllama_amd.models import write_synthetic_gguf
    path = write_synthetic_gguf(str(tmp_path / "t.gguf"), "testllama",
                                scheme="f32", mode="exact", seed=11)
    kw = dict(max_seq=64, kv_keep=40, kv_recent=8)
    engine = (HipEngine("m", path, **kw) if batch == 1 else
              BatchingHipEngine("m", path, batch=batch, **kw))
    try:
        last = ask(engine, Config(key_path=str(tmp_path / "k"),
                                  max_new_tokens=300), stream)[-1]
    finally:
        asyncio.run(engine.close())
    # (another order of sums may lead to an end-of-text token)
    assert last.eval_count == 300 or last.done_reason == "stop"
    assert last.done
