#!/usr/bin/env python3
"""Flagship bench: llama3-8b Q4_K_M decode on N MI355X GPUs as N DP workers.

Driver contract: `python bench.py --gpus N --steps K --warmup W`; for N>1
launched via torch.distributed.run with one rank per GPU. One "step" = one
decode iteration of the engine's whole batch (B tokens per step per GPU).
Rank 0 prints ONE JSON line with the aggregate whole-job tokens/sec
(the metric: aggregate tokens/sec + p50 latency, llama3:8b Q4_K across
1/2/4/8 workers); weights are random-init GGUF (no network for real
checkpoints), prompts synthetic.
"""

from __future__ import annotations

import argparse
import json
import os
import sys
import time

import numpy as np


def log(msg: str) -> None:
    print(f"[bench] {msg}", file=sys.stderr, flush=True)


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=256)
    ap.add_argument("--warmup", type=int, default=32)
    ap.add_argument("--model", default="llama3-8b")
    ap.add_argument("--scheme", default="q4_k_m")
    ap.add_argument("--mode", default="dp", choices=["dp", "tp", "serve"],
                    help="dp: one replica worker per GPU (default). tp: ONE worker spanning "
                         "all ranks via RCCL tensor parallelism "
                         "(e.g. --mode tp --model "
                         "llama3-70b --scheme bf16). serve: the FULL "
                         "serving path — DHT + worker (continuous "
                         "batching) + gateway /api/chat, concurrent HTTP "
                         "clients, true request p50/p95")
    ap.add_argument("--concurrency", type=int, default=32,
                    help="serve mode: concurrent in-flight HTTP requests")
    ap.add_argument("--models", default="",
                    help="serve mode: comma-separated models for a mixed "
                         "fleet (one worker per model on this GPU; "
                         "requests round-robin across models: model-aware "
                         "routing)")
    ap.add_argument("--max-new", type=int, default=64,
                    help="serve mode: max_new_tokens per request")
    ap.add_argument("--batch", type=int, default=16,
                    help="decode slots per GPU (the serving stack batches "
                         "concurrent requests into these slots — "
                         "crowdllama_amd/engine/batching.py; use 1 for the "
                         "single-stream latency point)")
    ap.add_argument("--prompt-len", type=int, default=128)
    ap.add_argument("--max-seq", type=int, default=4096)
    ap.add_argument("--act-q8", dest="act_q8", action="store_true",
                    default=True,
                    help="int8-quantized activations for quantized-weight "
                         "GEMMs (default on; the i8 MFMA batched path)")
    ap.add_argument("--no-act-q8", dest="act_q8", action="store_false",
                    help="force the f32-activation bf16-staging GEMM path")
    args = ap.parse_args()

    if args.mode == "serve":
        serve_bench(args)
        return

    rank = int(os.environ.get("RANK", "0"))
    world = int(os.environ.get("WORLD_SIZE", "1"))
    local_rank = int(os.environ.get("LOCAL_RANK", str(rank)))
    n_gpus = max(args.gpus, world)

    import torch
    import torch.distributed as dist
    distributed = world > 1
    if distributed:
        # DP replicas share no tensors; gloo carries the control barriers.
        # (The TP=8 worker path is where RCCL over xGMI runs — see
        # crowdllama_amd/parallel/.)
        dist.init_process_group(backend="gloo")

    def barrier():
        if distributed:
            dist.barrier()

    from crowdllama_amd.models import get_preset, synth_path

    cfg = get_preset(args.model)
    # rank 0 generates the shared checkpoint; same /tmp on a 1-node job
    if rank == 0:
        t0 = time.time()
        path = synth_path(args.model, scheme=args.scheme, mode="fast")
        log(f"checkpoint ready in {time.time() - t0:.1f}s: {path}")
    barrier()
    path = synth_path(args.model, scheme=args.scheme, mode="fast")

    from crowdllama_amd.ops import get_core
    core = get_core()
    if core.device_count() == 0:
        log("no GPU visible — printing a null result")
        if rank == 0:  # contract: exactly one JSON line, from rank 0
            print(json.dumps({"metric": "aggregate_tokens_per_sec",
                              "value": None, "error": "no GPU"}),
                  flush=True)
        if distributed:
            dist.destroy_process_group()
        return

    ecfg = core.EngineConfig()
    ecfg.batch = args.batch
    ecfg.max_seq = args.max_seq
    ecfg.act_q8 = args.act_q8
    ecfg.device = local_rank if core.device_count() > local_rank else 0
    if args.mode == "tp":
        # one worker spanning all ranks: RCCL over xGMI
        ecfg.tp_rank = rank
        ecfg.tp_size = world
        if world > 1:
            if rank == 0:
                nid = core.nccl_unique_id()
                obj = [nid]
            else:
                obj = [None]
            dist.broadcast_object_list(obj, src=0)
            ecfg.nccl_id = obj[0]
    t0 = time.time()
    eng = core.Engine(path, ecfg)
    log(f"rank {rank}: engine loaded in {time.time() - t0:.1f}s "
        f"({eng.vram_bytes() / 1e9:.2f} GB VRAM)")

    # synthetic prompt prefill (untimed in the decode metric; measured for
    # the p50-latency story)
    rng = np.random.default_rng(1234 + rank)
    prompts = rng.integers(3, cfg.vocab_size - 1,
                           size=(args.batch, args.prompt_len)).astype(np.int32)
    t_pf = time.perf_counter()
    eng.prefill(prompts)
    prefill_ms = (time.perf_counter() - t_pf) * 1e3

    # warmup
    if args.warmup > 0:
        eng.decode(args.warmup)
    barrier()
    torch.cuda.synchronize() if torch.cuda.is_available() else None

    t_start = time.perf_counter()
    eng.decode(args.steps)  # one hipDeviceSynchronize inside after K replays
    torch.cuda.synchronize() if torch.cuda.is_available() else None
    elapsed = time.perf_counter() - t_start
    barrier()

    # MAX over ranks of elapsed
    if distributed:
        t = torch.tensor([elapsed], dtype=torch.float64)
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        elapsed = float(t.item())

    if args.mode == "tp":
        tokens_total = args.batch * args.steps  # one worker, whole job
    else:
        tokens_total = n_gpus * args.batch * args.steps
    value = tokens_total / elapsed
    ms_per_step = elapsed / args.steps * 1e3

    if rank == 0:
        result = {
            "metric": "aggregate_tokens_per_sec",
            "value": value,
            "unit": "tokens/s",
            "n_gpus": n_gpus,
            "steps": args.steps,
            "warmup": args.warmup,
            "ms_per_step": ms_per_step,
            "p50_latency_ms": ms_per_step,  # per-token latency at this batch
            "higher_is_better": True,
            "scaling": "weak",
            "vs_baseline": None,  # reference publishes no numbers
            # act_q8: per-32-block int8 activations for quantized-weight
            # GEMMs — the same activation-quantization scheme llama.cpp's
            # MMQ path (the reference's compute backend) uses for these
            # weight formats; --no-act-q8 forces f32 activations
            "dtype": args.scheme + ("+int8-activations" if args.act_q8
                                    else "+f32-activations"),
            "data": "synthetic",
            "config": {
                "model": args.model,
                "quant": args.scheme,
                "global_batch": n_gpus * args.batch,
                "seq_len": args.prompt_len,
                "parallelism": (f"tp{world}" if args.mode == "tp" else f"dp{n_gpus}"),
                "engine_ms_per_step": eng.last_decode_ms() / args.steps,
                "prefill_ms": prefill_ms,
            },
        }
        print(json.dumps(result), flush=True)

    if distributed:
        dist.destroy_process_group()


def serve_bench(args) -> None:
    """The serving path: N concurrent /api/chat
    requests through DHT + worker + gateway on loopback; reports aggregate
    generated tokens/sec AND true request-level p50/p95."""
    import asyncio
    import statistics

    from crowdllama_amd.models import get_preset, synth_path

    models = [m for m in args.models.split(",") if m] or [args.model]
    paths = {}
    for m in models:
        get_preset(m)  # validate
        paths[m] = synth_path(m, scheme=args.scheme, mode="fast")
        log(f"checkpoint ready: {paths[m]}")

    from crowdllama_amd.ops import get_core
    if get_core().device_count() == 0:
        print(json.dumps({"metric": "serving_tokens_per_sec", "value": None,
                          "error": "no GPU"}), flush=True)
        return

    async def go():
        import aiohttp

        from crowdllama_amd.config import Config
        from crowdllama_amd.engine.batching import BatchingHipEngine
        from crowdllama_amd.mesh.dhtnode import DHTServer
        from crowdllama_amd.mesh.gateway import Gateway
        from crowdllama_amd.mesh.peer import Peer

        import tempfile
        kd = tempfile.mkdtemp(prefix="clabench-keys-")

        def mk(c):
            return Config(test_mode=True, listen_host="127.0.0.1",
                          key_path=os.path.join(kd, f"{c}.key"))

        dht = DHTServer(mk("dht"))
        dht_port = await dht.start("127.0.0.1", 0)
        boot = [f"127.0.0.1:{dht_port}"]
        # one worker per model, all on this GPU (288 GB HBM holds a mixed
        # fleet, e.g. 2 models with model-aware routing).
        # Per-request token budget rides the engine default max_new (the
        # PB GenerateRequest is reference-schema: model/prompt/stream).
        workers = []
        for i, m in enumerate(models):
            engine = BatchingHipEngine(m, paths[m], batch=args.batch,
                                       max_seq=args.max_seq,
                                       max_new=args.max_new)
            wcfg = mk(f"worker{i}")
            wcfg.bootstrap_peers = boot
            w = Peer(wcfg, worker_mode=True, engines={m: engine})
            await w.start()
            workers.append(w)
        ccfg = mk("consumer")
        ccfg.bootstrap_peers = boot
        consumer = Peer(ccfg, worker_mode=False)
        await consumer.start()
        gw = Gateway(consumer, ccfg)
        gw_port = await gw.start(port=0)
        url = f"http://127.0.0.1:{gw_port}/api/chat"

        # wait for discovery of every model
        deadline = time.time() + 120
        while any(gw.find_best_worker(m) is None for m in models):
            if time.time() > deadline:
                raise RuntimeError("worker never discovered")
            await asyncio.sleep(0.2)
        log("workers discovered; running serve bench")

        rng = np.random.default_rng(7)
        words = ["alpha", "beta", "gamma", "delta", "omega", "sigma",
                 "theta", "lambda"]

        def mk_prompt():
            n = max(4, args.prompt_len // 4)  # ~4 BPE tokens/word is plenty
            return " ".join(rng.choice(words) for _ in range(n))

        lat: list[float] = []
        toks = [0]

        rr = [0]

        async def one_request(session):
            model = models[rr[0] % len(models)]
            rr[0] += 1
            t0 = time.perf_counter()
            async with session.post(url, json={
                    "model": model,
                    "messages": [{"role": "user", "content": mk_prompt()}],
                    "options": {"num_predict": args.max_new}}) as r:
                body = await r.json()
                if r.status != 200:
                    raise RuntimeError(f"chat failed: {body}")
            lat.append(time.perf_counter() - t0)
            toks[0] += int(body.get("eval_count", 0))

        async def run_n(session, n):
            sem = asyncio.Semaphore(args.concurrency)

            async def guarded():
                async with sem:
                    await one_request(session)
            await asyncio.gather(*[guarded() for _ in range(n)])

        warm = max(args.concurrency, args.warmup)
        total = max(args.steps, 2 * args.concurrency)
        async with aiohttp.ClientSession() as session:
            await run_n(session, warm)          # warmup (untimed)
            lat.clear()
            toks[0] = 0
            t0 = time.perf_counter()
            await run_n(session, total)
            elapsed = time.perf_counter() - t0

        await gw.stop()
        await consumer.stop()
        for w in workers:
            await w.stop()
        await dht.stop()

        lat_ms = sorted(x * 1e3 for x in lat)
        result = {
            "metric": "serving_tokens_per_sec",
            "value": toks[0] / elapsed,
            "unit": "tokens/s",
            "n_gpus": 1,
            "steps": total,                    # requests completed (timed)
            "warmup": warm,
            "requests_per_sec": total / elapsed,
            "p50_latency_ms": statistics.median(lat_ms),
            "p95_latency_ms": lat_ms[int(0.95 * (len(lat_ms) - 1))],
            "higher_is_better": True,
            "scaling": "weak",
            "vs_baseline": None,
            "dtype": args.scheme + "+int8-activations",
            "data": "synthetic",
            "config": {
                "model": ",".join(models),
                "quant": args.scheme,
                "path": "dht+worker+gateway /api/chat (loopback, "
                        "encrypted mesh streams)",
                "concurrency": args.concurrency,
                "batch_slots": args.batch,
                "max_new_tokens": args.max_new,
                "prompt_len": args.prompt_len,
                "parallelism": "dp1",
            },
        }
        print(json.dumps(result), flush=True)

    asyncio.run(go())


if __name__ == "__main__":
    main()
