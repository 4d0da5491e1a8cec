"""What the paged cache's operators compute and which calls of them are timed.

Four operators share one cache: `append` (rotary positions and the new keys and values), `attend` (one new
token over the paged cache, adding each place's weight to the cache's mass), `observe` (the weight that a
prompt's rows gave to the places) and `evict` (which places stay once a sequence is too long).

A pool holds pages `[page][layer][kv head][K, V][place][head_dim]`; a sequence's place p lies in row
`p % page` of page `page_table[b, p // page]`.  `mass` (float32) and `pos` (int32) have a value for each layer,
sequence, kv head and place."""
import math
import random

import torch

own = False

# head counts and sizes of the model presets, and page sizes around the engine's 64
_HEADS = ((32, 8, 128), (32, 4, 64), (32, 32, 128), (64, 8, 128), (4, 2, 64), (40, 40, 128), (24, 8, 96), (6, 2, 64))
_TYPES = (("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float16", "float16"))
_PAGES = (16, 32, 64, 128)


def _case(op, heads, types, **more):
    return {"op": op, "heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "q": types[0], "cache": types[1], **more}


def listed():
    f32, bf16, f16 = _TYPES
    return [
        # one user's next token in one layer: the engine's float32 projections, one slot
        _case("append", _HEADS[0], f32, name="append one token", batch=1, rows=1, held=600, page=64),
        # all slots of a full continuous batch, each one token on
        _case("append", _HEADS[1], bf16, name="append a step of 64 slots", batch=64, rows=1, held=1900, page=64),
        # ragged prompts of several users, together
        _case("append", _HEADS[0], bf16, name="append ragged prompts", batch=8, rows=2047, held=70, page=64),
        # a short chat: latency counts
        _case("attend", _HEADS[0], f32, name="attend one short", batch=1, n=601, page=64),
        # a full batch of sequences of all lengths
        _case("attend", _HEADS[1], bf16, name="attend 64 ragged", batch=64, n=4096, page=64),
        # one very long document
        _case("attend", _HEADS[0], f32, name="attend one long", batch=1, n=131071, page=64),
        # every head has keys of its own: the most bytes a token
        _case("attend", _HEADS[2], f16, name="attend 16 without shared heads", batch=16, n=8191, page=128),
        # a short prompt
        _case("observe", _HEADS[0], f32, name="observe a short prompt", batch=1, rows=300, n=300, page=64),
        # a prompt as long as the presets allow
        _case("observe", _HEADS[0], bf16, name="observe a long prompt", batch=1, rows=8192, n=8192, page=64),
        # the last chunks of long prompts of several users
        _case("observe", _HEADS[0], f32, name="observe chunks", batch=3, rows=500, n=16001, page=64),
        # one layer of one slot
        _case("evict", _HEADS[0], f32, name="evict one short", batch=1, layers=1, n=512, keep=385, recent=128, page=64),
        # all layers of a model whose slot has filled its cache
        _case("evict", _HEADS[0], bf16, name="evict all layers", batch=1, layers=32, n=8192, keep=6144, recent=2048, page=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "observe", "evict"))
    heads, types, page = rng.choice(_HEADS), rng.choice(_TYPES), rng.choice(_PAGES)
    a_place = heads[1] * heads[2] * 4
    if op == "append":
        batch, rows = _log(rng, 1, 64), _log(rng, 1, 2048)
        while batch * rows * (heads[0] + heads[1]) > 8 * 2047 * 40:
            batch, rows = -(-batch // 2), -(-rows // 2)
        return _case(op, heads, types, batch=batch, rows=rows, held=rng.randrange(0, 300), page=page)
    if op == "attend":
        batch, n = _log(rng, 1, 64), _log(rng, 1, 131072)
        while batch * n * a_place > 1 << 31:
            batch, n = -(-batch // 2), -(-n // 2)
        return _case(op, heads, types, batch=batch, n=n, page=page)
    if op == "observe":
        batch, n = _log(rng, 1, 8), _log(rng, 1, 16384)
        rows = _log(rng, 1, min(n, 8192))
        while batch * rows * n * heads[0] * heads[2] > 8192 * 8192 * 2048:
            batch, rows = -(-batch // 2), -(-rows // 2)
        return _case(op, heads, types, batch=batch, rows=rows, n=n, page=page)
    batch, layers, n = _log(rng, 1, 16), _log(rng, 1, 32), _log(rng, 64, 16384)
    while batch * layers * n * a_place > 1 << 30:
        batch, layers = -(-batch // 2), -(-layers // 2)
        if batch == layers == 1:
            break
    keep = rng.randrange(n // 4 + 1, n)
    return _case(op, heads, types, batch=batch, layers=layers, n=n, keep=keep, recent=rng.randrange(0, keep + 1), page=page)


def _lens(case, most, least=0):
    """Lengths of a batch: the first has the most, one of more than two has the least, the others are spread."""
    rng = random.Random("%d %d %d" % (case["batch"], most, least))
    got = [most] + [rng.randint(least, most) for _ in range(case["batch"] - 1)]
    if len(got) > 2:
        got[1] = least
    return got


def _rows(case):
    """How many new rows each sequence of a case has."""
    if case["rows"] == 1:
        return [1] * case["batch"]
    return _lens(case, case["rows"], 0)


def _held(case):
    """How many places of each sequence are in use, the new rows of `observe` among them."""
    if case["op"] == "append":
        return _lens(case, case["held"], 0)
    if case["op"] == "observe":
        return [max(r, x) for r, x in zip(_rows(case), _lens(case, case["n"], 1))]
    if case["op"] == "evict":
        return _lens(case, case["n"], case["keep"] // 2)
    return _lens(case, case["n"], 0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    op, B, NH, NKV, D, page = (case[k] for k in ("op", "batch", "heads", "kv_heads", "dim", "page"))
    qt, ct = getattr(torch, case["q"]), getattr(torch, case["cache"])
    L = case.get("layers", 1)
    held = _held(case)
    rows = _rows(case) if op in ("append", "observe") else [1] * B
    cap = -(-(max(held) + (max(rows) if op == "append" else 0)) // page) * page
    pages = cap // page
    P = B * pages + 3
    s = {"case": case, "cap": cap, "n": max(held), "lens": ints(held)}
    # pages in no order; what no sequence uses is in the pool too
    s["table"] = torch.randperm(P, generator=g, device="cuda")[: B * pages].to(torch.int32).view(B, pages)
    pool = torch.empty(P, L, NKV, 2, page, D, dtype=ct, device="cuda")
    for i in range(0, P, 256):  # in pieces, to keep the float32 values few
        pool[i:i + 256] = normal(min(256, P - i), L, NKV, 2, page, D)
    s["pool"] = pool
    if op in ("append", "observe"):
        s["starts"] = ints([sum(rows[:b]) for b in range(B + 1)])
        s["rows"] = max(rows)
    T = sum(rows)
    if op == "append":
        # the projections of one layer, side by side as the engine's fused product leaves them
        qkv = normal(T, (NH + 2 * NKV) * D).to(qt)
        s["q"] = qkv[:, : NH * D].view(T, NH, D)
        s["k"] = qkv[:, NH * D:(NH + NKV) * D].view(T, NKV, D)
        s["v"] = qkv[:, (NH + NKV) * D:].view(T, NKV, D)
        s["inv_freq"] = (500000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)).float()
        # tokens that the cache has seen: some sequences have lost places before, so positions run ahead
        s["next_pos"] = s["lens"] + torch.randint(0, 100000, (B,), generator=g, device="cuda", dtype=torch.int32)
        s["mass"] = normal(B, NKV, cap).abs()
        s["pos"] = torch.randint(0, 1000, (B, NKV, cap), generator=g, device="cuda", dtype=torch.int32)
    elif op in ("attend", "observe"):
        s["q"] = (1.5 * normal(B if op == "attend" else T, NH, D)).to(qt)
        # what a few rows before these have left
        s["mass"] = normal(B, NKV, cap).abs() * (NH / NKV / s["n"])
    else:
        # a few places hold most of the weight; equal weights (places that nothing looked at) are common
        s["mass"] = torch.exp(2.5 * normal(L, B, NKV, cap) - 3)
        s["mass"][s["mass"] < 0.005] = 0
        # the first `keep` places are what an earlier call left, in no order; the others came after it, in order
        order = torch.arange(cap, dtype=torch.int32, device="cuda")
        old = torch.rand(L, B, NKV, case["keep"], generator=g, device="cuda").argsort(-1).to(torch.int32)
        s["pos"] = torch.cat([old, order[case["keep"]:].expand(L, B, NKV, -1)], -1) + 1000
        s["next_pos"] = s["lens"] + 1000
        s["out"] = (torch.zeros_like(s["mass"]), torch.zeros_like(s["pos"]), torch.zeros_like(s["lens"]))
    return s


def _places(s, pool):
    """One layer's keys and values in float32, sequence after sequence: [B][kv head][K, V][place][dim]."""
    x = pool[s["table"].long()].permute(0, 2, 3, 1, 4, 5)
    return x.reshape(*x.shape[:3], -1, x.shape[-1])[..., : s["n"], :].float()


def _padded(s):
    """For each sequence and row of the longest: the packed row's number, and whether there is one."""
    i = torch.arange(s["rows"], device="cuda")
    first, last = s["starts"][:-1, None].long(), s["starts"][1:, None].long()
    there = first + i < last
    return torch.where(there, first + i, 0), there


def _softmax(x, seen):
    x = x.masked_fill(~seen, -math.inf)
    most = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(most == -math.inf, 0.0, most))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _append(s):
    c, pool = s["case"], s["pool"][:, 0]
    at, there = _padded(s)
    b, i = there.nonzero(as_tuple=True)
    at = at[b, i]
    place = s["lens"].long()[b] + i
    position = s["next_pos"].long()[b] + i
    turn = position[:, None, None].double() * s["inv_freq"].double()
    cos, sin = turn.cos().float(), turn.sin().float()

    def turned(x):
        x = x.float()[at]
        a, z = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - z * sin, a * sin + z * cos), -1).flatten(-2)

    where = s["table"].long()[b, place // c["page"]]
    row = place % c["page"]
    pool[where, :, 0, row] = turned(s["k"]).to(pool.dtype)
    pool[where, :, 1, row] = s["v"][at].float().to(pool.dtype)
    s["mass"][b, :, place] = 0
    s["pos"][b, :, place] = position.to(torch.int32)[:, None]
    q = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    q[at] = turned(s["q"]).to(q.dtype)
    return q, s["pool"], s["mass"], s["pos"]


def _attend(s):
    c, n = s["case"], s["n"]
    B, NKV, D = c["batch"], c["kv_heads"], c["dim"]
    kv = _places(s, s["pool"][:, 0])
    seen = (torch.arange(n, device="cuda") < s["lens"][:, None])[:, None, None]
    q = s["q"].float().view(B, NKV, -1, D)
    w = _softmax(torch.matmul(q, kv[:, :, 0].transpose(-1, -2)) * D ** -0.5, seen)
    out = torch.matmul(w, kv[:, :, 1].masked_fill(~seen.transpose(-1, -2), 0))
    s["mass"][..., :n] += w.sum(2)
    return out.reshape(B, -1, D).to(s["q"].dtype), s["mass"]


def _observe(s):
    c, n = s["case"], s["n"]
    B, NKV, D, M = c["batch"], c["kv_heads"], c["dim"], s["rows"]
    at, there = _padded(s)
    count = s["starts"][1:] - s["starts"][:-1]
    last = (s["lens"] - count)[:, None] + torch.arange(M, device="cuda")
    seen = (torch.arange(n, device="cuda") <= last[..., None]) & there[..., None]
    k = _places(s, s["pool"][:, 0])[:, :, 0]
    q = s["q"].float()[at].view(B, M, NKV, -1, D).permute(0, 2, 3, 1, 4)
    G = q.shape[2]
    x = torch.matmul(q.reshape(B, NKV, G * M, D), k.transpose(-1, -2)).view(B, NKV, G, M, n) * D ** -0.5
    s["mass"][..., :n] += _softmax(x, seen[:, None, None]).sum((2, 3))
    return s["mass"]


def _evict(s):
    c, cap, keep, page = s["case"], s["cap"], s["case"]["keep"], s["case"]["page"]
    place = torch.arange(cap, device="cuda")
    here = (place < s["lens"][:, None])[:, None]
    recent = here & (s["pos"] >= s["next_pos"][:, None, None] - c["recent"])
    # one order of all places: those of late first, then by weight, places that are not in use last
    by = torch.where(recent, math.inf, torch.where(here, s["mass"], -math.inf))
    stays = torch.zeros_like(by, dtype=torch.bool).scatter_(-1, by.sort(dim=-1, descending=True, stable=True)[1][..., :keep], True)
    full = (s["lens"] > keep)[:, None, None]
    free = full & ~stays & (place < keep)
    comes = full & stays & (place >= keep)
    # the k-th free place and the k-th place that moves into it, in the same order
    to, of = free.nonzero(as_tuple=True), comes.nonzero(as_tuple=True)
    mass, pos, lens = s["out"]
    mass.copy_(s["mass"])
    pos.copy_(s["pos"])
    mass[to], pos[to] = s["mass"][of], s["pos"][of]
    torch.minimum(s["lens"], torch.full_like(s["lens"], keep), out=lens)
    l, b, h = to[:3]
    table = s["table"].long()
    dst, src = table[b, to[3] // page], table[b, of[3] // page]
    s["pool"][dst, l, h, :, to[3] % page] = s["pool"][src, l, h, :, of[3] % page]
    return s["pool"], mass, pos, lens


def run(s):
    op = s["case"]["op"]
    if own:
        from crowdllama_amd.ops import kv
        if op == "append":
            q = kv.append(s["k"], s["v"], s["pool"][:, 0], s["table"], s["lens"], s["next_pos"], q=s["q"], inv_freq=s["inv_freq"],
                          starts=s["starts"], mass=s["mass"], pos=s["pos"])
            return q, s["pool"], s["mass"], s["pos"]
        if op == "attend":
            return kv.attend(s["q"], s["pool"][:, 0], s["table"], s["lens"], mass=s["mass"]), s["mass"]
        if op == "observe":
            return kv.observe(s["q"], s["pool"][:, 0], s["table"], s["lens"], s["mass"], starts=s["starts"])
        c = s["case"]
        return s["pool"], *kv.evict(s["pool"], s["table"], s["lens"], s["next_pos"], s["mass"], s["pos"], keep=c["keep"], recent=c["recent"], out=s["out"])
    return {"append": _append, "attend": _attend, "observe": _observe, "evict": _evict}[op](s)


def work(case):
    NH, NKV, D = case["heads"], case["kv_heads"], case["dim"]
    G, q, c = NH // NKV, 4 if case["q"] == "float32" else 2, 2
    held = _held(case)
    if case["op"] == "append":
        T = sum(_rows(case))
        return {"bytes": T * ((2 * NH + 2 * NKV) * D * q + 2 * NKV * D * c + 8 * NKV), "flops": T * (NH + NKV) * D * 3}
    if case["op"] == "attend":
        return {"bytes": sum(held) * NKV * (2 * D * c + 8) + 2 * case["batch"] * NH * D * q, "flops": sum(held) * NH * D * 4}
    if case["op"] == "observe":
        rows = _rows(case)
        pairs = sum(r * (x - r) + r * (r + 1) // 2 for r, x in zip(rows, held))
        return {"bytes": sum(rows) * NH * D * q + sum(x for r, x in zip(rows, held) if r) * NKV * (D * c + 8), "flops": pairs * NH * D * 2}
    # what moves goes by the weights: about as many of the places past `keep` as stay of all, and the late ones among them
    moved = sum(min(x - case["keep"], case["keep"]) * max(case["keep"], case["recent"]) / x for x in held if x > case["keep"])
    return {"bytes": case["layers"] * NKV * (sum(held) * 16 + moved * 4 * D * c), "flops": case["layers"] * NKV * sum(held)}


def exact(case, seed):
    s = prepare(case, seed)
    op, B, NH, NKV, D, page = (case[k] for k in ("op", "batch", "heads", "kv_heads", "dim", "page"))
    held, pool, table = _held(case), s["pool"], s["table"].cpu().tolist()
    if op == "append":
        q, cache, mass, pos = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), pool.double(), s["mass"].double(), s["pos"].clone()
        rows, ahead, t = _rows(case), s["next_pos"].cpu().tolist(), 0
        for b in range(B):
            r = rows[b]
            if not r:
                continue
            where = torch.arange(ahead[b], ahead[b] + r, dtype=torch.float64, device="cuda")
            turns = torch.polar(torch.ones(r, D // 2, dtype=torch.float64, device="cuda"), where[:, None] * s["inv_freq"].double())
            turn = lambda x: torch.view_as_real(torch.view_as_complex(x.double().reshape(r, -1, D // 2, 2)) * turns[:, None]).reshape(r, -1, D)  # noqa: E731
            q[t:t + r], k, v = turn(s["q"][t:t + r]), turn(s["k"][t:t + r]), s["v"][t:t + r].double()
            for p in range(held[b] // page, -(-(held[b] + r) // page)):  # page after page
                lo, hi = max(held[b], p * page), min(held[b] + r, (p + 1) * page)
                if lo < hi:
                    inside, rows_of = slice(lo - p * page, hi - p * page), slice(lo - held[b], hi - held[b])
                    cache[table[b][p], 0, :, 0, inside] = k[rows_of].transpose(0, 1)
                    cache[table[b][p], 0, :, 1, inside] = v[rows_of].transpose(0, 1)
            mass[b, :, held[b]:held[b] + r] = 0
            pos[b, :, held[b]:held[b] + r] = where.to(torch.int32)
            t += r
        return q, cache, mass, pos
    if op in ("attend", "observe"):
        rows = [1] * B if op == "attend" else _rows(case)
        mass, out, t = s["mass"].double(), torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
        for b in range(B):
            n, r = held[b], rows[b]
            if n and r:
                kv = pool[table[b][: -(-n // page)], 0]  # the sequence's pages, in order
                first = torch.arange(n - r + 1, n + 1, device="cuda")[:, None]
                hidden = torch.arange(n, device="cuda") >= first
                for h in range(NH):
                    x = kv[:, h // (NH // NKV)].double()
                    # a thousand rows at a time: the scores in 64 bits are large
                    for i in range(0, r, 1024):
                        j = min(r, i + 1024)
                        score = (s["q"][t + i:t + j, h].double() @ x[:, 0].reshape(-1, D)[:n].T / math.sqrt(D)).masked_fill_(hidden[i:j], -math.inf)
                        w = torch.softmax(score, -1)
                        mass[b, h // (NH // NKV), :n] += w.sum(0)
                        if op == "attend":
                            out[t + i:t + j, h] = w @ x[:, 1].reshape(-1, D)[:n]
            t += r
        return (out, mass) if op == "attend" else mass
    # nothing is rounded here: what stays is looked up row by row
    keep, mass, pos, lens = case["keep"], s["mass"].clone(), s["pos"].clone(), s["lens"].clone()
    late = s["next_pos"].cpu().tolist()
    for b in range(B):
        if held[b] <= keep:
            continue
        lens[b] = keep
        pages = s["table"][b].long()
        for l in range(case["layers"]):
            for h in range(NKV):
                w, p = s["mass"][l, b, h, :held[b]].double(), s["pos"][l, b, h, :held[b]]
                w = torch.where(p >= late[b] - case["recent"], 1e300, w)
                stays = torch.argsort(-w, stable=True)[:keep]
                gone = torch.ones(held[b], dtype=torch.bool, device="cuda")
                gone[stays] = False
                to, of = gone[:keep].nonzero()[:, 0], (~gone[keep:]).nonzero()[:, 0] + keep
                mass[l, b, h, to], pos[l, b, h, to] = s["mass"][l, b, h, of], s["pos"][l, b, h, of]
                pool[pages[to // page], l, h, :, to % page] = pool[pages[of // page], l, h, :, of % page]
    return pool, mass.double(), pos, lens
