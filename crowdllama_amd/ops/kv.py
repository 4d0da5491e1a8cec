"""The paged KV cache's operators on torch tensors.

    append    rotary positions, new keys and values into the pages
    attend    one new token's attention over the cache
    observe   the attention weight that a prompt's rows gave to the places
    evict     keep the places that matter once a sequence is too long

A layer's pool is `[pages, kv_heads, 2, page, head_dim]` (keys, then values;
bfloat16 or float16), all but the first dimension contiguous, so that one pool
of all layers, `[pages, layers, kv_heads, 2, page, head_dim]`, serves as
`pool[:, layer]`. Place p of sequence b is row `p % page` of page
`table[b, p // page]`; `lens[b]` of its places are in use. `mass` (float32) and
`pos` (int32) are `[slots, kv_heads, places]`: the attention weight that each
place has received, summed over tokens and query heads, and the position of
the token in it. A place is not a position: after `evict`, a sequence's tokens
keep their positions (keys are stored rotated) and take other places, which
differ from head to head.

    q = kv.append(k, v, pool[:, l], table, lens, next_pos, q=q,
                  inv_freq=inv_freq, mass=mass[l], pos=pos[l])
    out = kv.attend(q, pool[:, l], table, lens + 1, mass=mass[l])
    ...
    kv.evict(pool, table, lens, next_pos, mass, pos, keep=2048, recent=512)

`table`, `lens`, `next_pos` and `starts` are int32 on the device and are read
there: no call waits for the device, and all may be captured into a graph
(which then goes by the values at replay). Lengths are cut to what the table
and the mass reach; page numbers outside the pool are not followed: such places
have no weight, and no keys and values are stored there. Work goes to the current stream
of the tensors' device. None of the operators has a gradient, and none can be
traced (fake or functional tensors, `make_fx`).
"""

from __future__ import annotations

import numpy
import torch
from torch.autograd import forward_ad

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_NONE = (0, 0, 0)
_core = None


def _one_runtime() -> None:
    """torch brings its own HIP runtime, which the native module takes too if
    it is there first; streams and memory of one are nothing to another."""
    with open("/proc/self/maps") as f:
        found = {line.split(None, 5)[5].strip() for line in f
                 if "libamdhip64" in line}
    if len(found) > 1:
        raise RuntimeError(
            "two HIP runtimes are loaded (%s): import torch before the first "
            "use of crowdllama_amd's native module"
            % ", ".join(sorted(found)))


def _get(dev):
    """The native module, once all arguments are checked."""
    global _core
    if dev.type != "cuda":
        _fail(f"pool must be on a GPU, not on {dev}")
    if _core is None:
        from . import get_core
        core = get_core()
        _one_runtime()
        _core = core
    return _core


def _fail(what: str):
    raise ValueError("kv: " + what)


def _on(t, name: str, dtype, dims: int, device):
    if not isinstance(t, torch.Tensor):
        _fail(f"{name} must be a tensor, not {type(t).__name__}")
    if t.dtype is not dtype:
        _fail(f"{name} must be {dtype}, not {t.dtype}")
    if t.dim() != dims:
        _fail(f"{name} must have {dims} dimensions, not {t.dim()}")
    if t.device != device:
        _fail(f"{name} is on {t.device}, the pool on {device}")


def _dense(t, name: str, n: int):
    """The last n dimensions are contiguous."""
    want = 1
    shape, stride = t.shape, t.stride()
    for i in range(1, n + 1):
        if shape[-i] > 1 and stride[-i] != want:
            _fail(f"{name}'s last {n} dimensions must be contiguous")
        want *= shape[-i]
    return want


_depth = torch._C._len_torch_dispatch_stack
_TRACERS = [getattr(torch._C._TorchDispatchModeKey, x)
            for x in ("FAKE", "PROXY", "FUNCTIONAL")]


def _plain(*tensors):
    """The call is neither differentiated nor traced."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _fail("no operator of the cache has a gradient")
    if forward_ad._current_level >= 0:       # there may be tangents
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _fail("no operator of the cache has a gradient")
    if _depth() and any(torch._C._get_dispatch_mode(x) is not None
                        for x in _TRACERS):
        _fail("the operators work on memory and cannot be traced")


def _memory(t, name: str) -> int:
    """The address of a tensor that has values."""
    at = t.data_ptr()
    if not at and t.numel():
        _fail(f"{name} has no memory (a fake or functional tensor): the "
              "operators work on memory and cannot be traced")
    return at


def _pages(pool, table, layers: bool):
    """What the kernels need of the pool and the table. Most calls pass the
    first test; what does not is looked at piece by piece."""
    try:
        dev = pool.device
        ps, st = pool.shape, pool.stride()
        p, (heads, two, page, dim) = ps[0], ps[-4:]
        per, ts = page * dim, table.shape
        kind, at = _TYPES[pool.dtype], pool.data_ptr()
        if (kind and two == 2 and st[-4:] == (2 * per, per, dim, 1)
                and len(ps) == (6 if layers else 5)
                and not (layers and (st[1] < st[2] * heads or st[1] % 8
                                     or st[0] < st[1] * ps[1]))
                and st[0] >= 2 * per * heads and not (st[0] % 8 or at % 16)
                and p and heads and page and dim and at
                and table.dtype is torch.int32 and len(ts) == 2
                and ts[0] and ts[1] and table.stride()[1] == 1
                and table.device == dev and (pages := table.data_ptr())):
            return dev, ts[1] * page, (
                at, st[0], p, pages, table.stride()[0], ts[1], page, ts[0],
                heads, dim, kind, dev.index)
    except (AttributeError, KeyError, ValueError, IndexError, TypeError,
            RuntimeError):
        pass
    return _pages_slowly(pool, table, layers)


def _pages_slowly(pool, table, layers: bool):
    if not isinstance(pool, torch.Tensor):
        _fail(f"pool must be a tensor, not {type(pool).__name__}")
    if pool.dtype not in (torch.bfloat16, torch.float16):
        _fail(f"pool must be bfloat16 or float16, not {pool.dtype}")
    dims = 6 if layers else 5
    if pool.dim() != dims or pool.shape[-3] != 2:
        _fail("pool must be [pages, %skv_heads, 2, page, head_dim]"
              % ("layers, " if layers else ""))
    dev = pool.device
    size = _dense(pool, "pool", 4)
    shape, stride = pool.shape, pool.stride()
    p, heads, page, dim = shape[0], shape[-4], shape[-2], shape[-1]
    steps = ((stride[0], p),) + (((stride[1], shape[1]),) if layers else ())
    for step, n in steps:
        if n > 1 and (step < size or step % 8):
            _fail("pool's pages must be multiples of 16 bytes apart and must "
                  "not overlap")
    if layers and p > 1 and shape[1] > 1 and not (
            stride[0] >= stride[1] * shape[1]
            or stride[1] >= stride[0] * p):
        _fail("pool's layers and pages must not overlap")
    if pool.numel() == 0 or _memory(pool, "pool") % 16:
        _fail("pool must not be empty and must be 16-byte aligned")
    _on(table, "table", torch.int32, 2, dev)
    _dense(table, "table", 1)
    slots, reach = table.shape[0], table.shape[1] * page
    if not slots or not reach:
        _fail("table must not be empty")
    return dev, reach, (
        pool.data_ptr(), stride[0], p, _memory(table, "table"),
        table.stride(0), table.shape[1], page, slots, heads, dim,
        _TYPES[pool.dtype], dev.index)


def _vector(t, name: str, n: int, dev, dtype=torch.int32):
    try:
        if (t.dtype is dtype and t.shape == (n,) and t.stride() == (1,)
                and t.device == dev):
            at = t.data_ptr()
            if at:
                return at
    except (AttributeError, TypeError):
        pass
    _on(t, name, dtype, 1, dev)
    if t.shape[0] != n:
        _fail(f"{name} must have {n} values, not {t.shape[0]}")
    _dense(t, name, 1)
    return _memory(t, name)


def _heads(t, name: str, rows, heads, dim: int, dtype, dev):
    try:
        n, h, d = t.shape
        s0, s1, s2 = t.stride()
        at = t.data_ptr()
        if (at and d == dim and s2 == 1 and t.dtype is dtype and t.device == dev
                and (rows is None or n == rows)
                and (heads is None or h == heads)
                and not (at % 16 or s0 % 8 or s1 % 8)):
            return at, s0, s1
    except (AttributeError, TypeError, ValueError, RuntimeError):
        pass
    _on(t, name, dtype, 3, dev)
    shape = t.shape
    if ((rows is not None and shape[0] != rows)
            or (heads is not None and shape[1] != heads) or shape[2] != dim):
        _fail(f"{name} must be [{'rows' if rows is None else rows}, "
              f"{'heads' if heads is None else heads}, {dim}], not "
              f"{list(shape)}")
    _dense(t, name, 1)
    s0, s1, _ = t.stride()
    unit = 4 if dtype is torch.float32 else 8
    at = _memory(t, name)
    if at % 16 or (shape[0] > 1 and s0 % unit) or (
            shape[1] > 1 and s1 % unit):
        _fail(f"{name}'s rows must be 16-byte aligned")
    return at, s0, s1


def _apart(t, name: str):
    """A tensor that is written must have a place of its own for each value:
    sorted by stride, each dimension steps over the ones below it."""
    if t.is_contiguous():
        return
    span = 1
    for step, n in sorted((s, n) for n, s in zip(t.shape, t.stride())
                          if n > 1):
        if step < span:
            _fail(f"{name} is written and must not overlap itself")
        span = step * n


def _ends(t):
    """The addresses of a tensor's memory, from its first value to its last."""
    at = t.data_ptr()
    if t.is_contiguous():
        return at, at + t.nbytes
    return at, at + t.element_size() * (
        1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _pieces(t):
    """The first and last address of each contiguous piece of a tensor."""
    size, shape, stride = t.element_size(), list(t.shape), list(t.stride())
    long_ = 1
    while shape and (shape[-1] == 1 or stride[-1] == long_):
        long_ *= shape.pop()
        stride.pop()
    at = numpy.array([t.data_ptr()])
    for n, step in zip(shape, stride):
        if step:
            at = (at[:, None] + numpy.arange(n) * (step * size)).ravel()
    return at, at + (long_ * size - 1)


def _over(t, name: str, inputs):
    """An output that a caller gives must not overlap what the call reads:
    other workgroups read that while one writes."""
    if not t.numel():
        return
    first, last = _ends(t)
    for of, x, at in inputs:
        if not at or at >= last:
            continue
        lo, hi = _ends(x)
        if hi <= first or not x.numel() or (of == "q" and lo == first and all(
                m == n for m, n, size in zip(x.stride(), t.stride(), t.shape)
                if size > 1)):
            continue
        # piece by piece: what lies between an input's rows is free
        a, b = _pieces(t)
        order = numpy.argsort(a)
        a, b = a[order], b[order]
        lo, hi = _pieces(x)
        at = numpy.searchsorted(a, hi, side="right")    # pieces that begin by hi
        if ((at > 0) & (b[at - 1] >= lo)).any():
            _fail(f"{name} overlaps {of}")


def _places(t, name: str, dtype, lead: tuple, reach: int, dev):
    try:
        if (t.shape[:-1] == lead and 0 < t.shape[-1] <= reach
                and t.dtype is dtype and t.is_contiguous()
                and t.device == dev):
            at = t.data_ptr()
            if at:
                return (at, *t.stride()[:-1])
    except (AttributeError, TypeError):
        pass
    _on(t, name, dtype, len(lead) + 1, dev)
    if tuple(t.shape[:-1]) != lead:
        _fail(f"{name} must be {list(lead)} x places, not {list(t.shape)}")
    if not 0 < t.shape[-1] <= reach:
        _fail(f"{name} must have 1 to {reach} places (what the table "
              f"reaches), not {t.shape[-1]}")
    _dense(t, name, 1)
    _apart(t, name)
    return (_memory(t, name), *t.stride()[:-1])


def _queries(q, dtype_of_pool):
    if not isinstance(q, torch.Tensor):
        _fail(f"q must be a tensor, not {type(q).__name__}")
    if q.dtype is not dtype_of_pool and not (
            q.dtype is torch.float32 and dtype_of_pool is torch.bfloat16):
        _fail(f"{q.dtype} does not go with a pool of {dtype_of_pool}: it "
              "must be the pool's type, or float32 over bfloat16")


def _group(heads: int, kv_heads: int):
    if heads % kv_heads or not 1 <= heads // kv_heads <= 16:
        _fail(f"{heads} query heads over {kv_heads} kv heads: 1 to 16 query "
              "heads must share each kv head")


def _scale(scale, dim: int) -> float:
    if scale is None:
        return dim ** -0.5
    scale = float(scale)
    # the kernels multiply by it and log2(e) in float32, without subnormals
    if not 2.0 ** -126 <= scale <= 2.0 ** 127:
        _fail(f"scale must be positive and finite in float32 (2^-126 to "
              f"2^127), not {scale}")
    return scale


def _workspace(n: int, table):
    return table.new_empty(n // 4 + 1) if n else None


def _at(ws) -> int:
    return 0 if ws is None else ws.data_ptr()


# the stream's handle without an object around it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(dev) -> int:
    if _raw_stream is not None:
        return _raw_stream(dev.index)
    return torch.cuda.current_stream(dev).cuda_stream


def append(k, v, pool, table, lens, next_pos, *, q=None, inv_freq=None,
           starts=None, mass=None, pos=None, q_out=None):
    """Store new tokens' keys and values behind each sequence's last place.

    k, v: `[rows, kv_heads, head_dim]`, of the pool's type or float32 over a
    bfloat16 pool (rounded once, when stored). Rows `starts[b]` to
    `starts[b + 1]` are sequence b's next tokens, in order; without `starts`
    row b is sequence b's. Token i of sequence b goes to place `lens[b] + i`,
    and is at position `next_pos[b] + i`.

    inv_freq: float32 `[head_dim / 2]`, the radians per position of each
    adjacent pair; without it nothing is rotated. q `[rows, heads, head_dim]`
    is rotated as k is, and returned (in `q_out`, which may be q itself, but
    must not overlap it, or another input, otherwise).
    mass, pos: the new places' mass becomes 0 and their pos the position.

    `lens` and `next_pos` are only read (all layers share them). Rows past the
    last place that a sequence has are not stored; rows past `starts[-1]`
    belong to no sequence: their queries are returned as they are.
    """
    dev, reach, kv = _pages(pool, table, False)
    slots, heads, dim = kv[7], kv[8], kv[9]
    _queries(k, pool.dtype)
    rows = k.shape[0] if k.dim() else 0
    kh = _heads(k, "k", None, heads, dim, k.dtype, dev)
    vh = _heads(v, "v", rows, heads, dim, k.dtype, dev)
    qh = qo = _NONE
    q_heads, over = 0, None
    if q is not None:
        qh = _heads(q, "q", rows, None, dim, k.dtype, dev)
        q_heads = q.shape[1]
        if q_out is None:
            q_out = q.new_empty((rows, q_heads, dim))
            qo = (q_out.data_ptr(), q_heads * dim, dim)
        else:
            qo = _heads(q_out, "q_out", rows, q_heads, dim, k.dtype, dev)
            over = q_out
            _apart(q_out, "q_out")
    elif q_out is not None:
        _fail("q_out without q")
    if starts is None and rows != slots:
        _fail(f"without starts there must be one row for each of {slots} "
              f"sequences, not {rows}")
    st = 0 if starts is None else _vector(starts, "starts", slots + 1, dev)
    fr = 0 if inv_freq is None else _vector(inv_freq, "inv_freq", dim // 2,
                                            dev, torch.float32)
    ms = ps = _NONE
    if mass is not None:
        ms = _places(mass, "mass", torch.float32, (slots, heads), reach, dev)
        reach = mass.shape[-1]
    if pos is not None:
        ps = _places(pos, "pos", torch.int32, (slots, heads), reach, dev)
        reach = min(reach, pos.shape[-1])
    le = _vector(lens, "lens", slots, dev)
    np = _vector(next_pos, "next_pos", slots, dev)
    if over is not None:
        _over(over, "q_out", (
            ("q", q, qh[0]), ("k", k, kh[0]), ("v", v, vh[0]),
            ("pool", pool, kv[0]), ("mass", mass, ms[0]), ("pos", pos, ps[0]),
            ("table", table, kv[3]), ("lens", lens, le),
            ("next_pos", next_pos, np), ("starts", starts, st),
            ("inv_freq", inv_freq, fr)))
    _plain(k, v, q, pool, mass, inv_freq, over)
    _get(dev).kv_append(kv, kh, vh, qh, qo, q_heads, _TYPES[k.dtype], rows,
                        st, le, np, fr, ms, ps, reach, _stream(dev))
    return q_out


def attend(q, pool, table, lens, *, mass=None, scale=None, out=None):
    """Attention of one new token of each sequence over its first `lens[b]`
    places: `[slots, heads, head_dim]`, of q's type.

    q: `[slots, heads, head_dim]`, of the pool's type or float32 over a
    bfloat16 pool; query heads g * i ... g * i + g - 1 share kv head i.
    mass: each place's weight is added, summed over the query heads that share
    the kv head. scale: of the scores, positive, head_dim ** -0.5 by default.
    out: may be q itself, but must not overlap it, or another input, otherwise.
    A sequence without places gives zeros.
    """
    dev, reach, kv = _pages(pool, table, False)
    slots, heads, dim = kv[7], kv[8], kv[9]
    _queries(q, pool.dtype)
    qh = _heads(q, "q", slots, None, dim, q.dtype, dev)
    q_heads = q.shape[1]
    _group(q_heads, heads)
    ms = _NONE
    if mass is not None:
        ms = _places(mass, "mass", torch.float32, (slots, heads), reach, dev)
        reach = mass.shape[-1]
    given = out
    if given is None:
        out = q.new_empty((slots, q_heads, dim))
        oh = (out.data_ptr(), q_heads * dim, dim)
    else:
        oh = _heads(out, "out", slots, q_heads, dim, q.dtype, dev)
        _apart(out, "out")
    le, scale = _vector(lens, "lens", slots, dev), _scale(scale, dim)
    if given is not None:
        _over(out, "out", (
            ("q", q, qh[0]), ("pool", pool, kv[0]), ("mass", mass, ms[0]),
            ("table", table, kv[3]), ("lens", lens, le)))
    _plain(q, pool, mass, given)
    core = _get(dev)
    ws = _workspace(core.kv_attend_workspace(kv, q_heads, reach,
                                             mass is not None), table)
    core.kv_attend(kv, qh, oh, q_heads, _TYPES[q.dtype], le, ms, reach,
                   scale, _at(ws), _stream(dev))
    return out


def observe(q, pool, table, lens, mass, *, starts=None, scale=None):
    """Add to `mass` the attention weights of each sequence's last tokens.

    q: `[rows, heads, head_dim]`, rotated; rows `starts[b]` to `starts[b + 1]`
    are the queries of sequence b's last tokens (without `starts`, row b is
    that of sequence b's last), whose keys are in the cache: `lens[b]` counts
    them. Each sees the places up to its own; where `lens[b]` goes past the last
    place, the tokens past it have none, and the others see what they would in
    a longer cache. What `attend` adds for one token, this adds for a prompt,
    without making its outputs. Returns mass.
    """
    dev, reach, kv = _pages(pool, table, False)
    slots, heads, dim = kv[7], kv[8], kv[9]
    _queries(q, pool.dtype)
    qh = _heads(q, "q", None, None, dim, q.dtype, dev)
    rows, q_heads = q.shape[0], q.shape[1]
    _group(q_heads, heads)
    ms = _places(mass, "mass", torch.float32, (slots, heads), reach, dev)
    reach = mass.shape[-1]
    if starts is None:
        if rows != slots:
            _fail(f"without starts there must be one row for each of {slots} "
                  f"sequences, not {rows}")
        starts = torch.arange(slots + 1, dtype=torch.int32, device=dev)
    st = _vector(starts, "starts", slots + 1, dev)
    le, scale = _vector(lens, "lens", slots, dev), _scale(scale, dim)
    _plain(q, pool, mass)
    core = _get(dev)
    ws = _workspace(core.kv_observe_workspace(kv, q_heads, rows, reach,
                                              _TYPES[q.dtype]), table)
    core.kv_observe(kv, qh, q_heads, _TYPES[q.dtype], rows, st, le,
                    ms, reach,
                    scale, _at(ws), _stream(dev))
    return mass


def evict(pool, table, lens, next_pos, mass, pos, *, keep, recent=0,
          limit=None, out=None):
    """Keep `keep` places of each sequence with more than `limit` of them
    (default: `keep`), for each layer and kv head its own; returns
    `(mass, pos, lens)`.

    pool: `[pages, layers, kv_heads, 2, page, head_dim]`; mass, pos:
    `[layers, slots, kv_heads, places]`. Places with a pos of at least
    `next_pos[b] - recent` stay before all others, the others by mass; among
    equals the lower place stays, and a NaN counts as less than any number. The
    late ones are equals: of more than `keep` of them those in the lower places
    stay. Survivors below place `keep` stay where they are; the free places
    there take the others, both in order. What lies at and above `keep`
    afterwards is left as it was.

    Keys and values move within the pool, so a page must not serve two places
    of the table, and the pages of a sequence that is to be evicted from must
    be there: mass and pos order and move its places whether they have a page
    or not, keys and values move where both places have one. mass, pos and lens
    are changed in place, or, with `out=(mass, pos, lens)`, written there whole
    while these stay as they were.
    """
    dev, reach, kv = _pages(pool, table, True)
    slots, heads, layers = kv[7], kv[8], pool.shape[1]
    keep, recent = int(keep), int(recent)
    limit = keep if limit is None else int(limit)
    if keep < 1 or recent < 0 or limit < keep:
        _fail(f"keep {keep}, recent {recent}, limit {limit}: keep must be at "
              "least 1, recent not negative and limit not below keep")
    if max(keep, recent, limit) >= 1 << 31:
        _fail("keep, recent and limit must be below 2^31")
    lead = (layers, slots, heads)
    ms = _places(mass, "mass", torch.float32, lead, reach, dev)
    ps = _places(pos, "pos", torch.int32, lead, reach, dev)
    reach = mass.shape[-1]
    if pos.shape[-1] != reach:
        _fail("mass and pos must have equally many places")
    if layers * slots * heads >= 1 << 22:
        _fail("layers x sequences x kv heads must be below 2^22")
    le = _vector(lens, "lens", slots, dev)
    np = _vector(next_pos, "next_pos", slots, dev)
    spans = [_ends(mass), _ends(pos), _ends(lens)]
    if out is None:
        mass_out, pos_out, lens_out = mass, pos, lens
        mo, po, lo = ms, ps, le
    else:
        mass_out, pos_out, lens_out = out
        mo = _places(mass_out, "out's mass", torch.float32, lead, reach, dev)
        po = _places(pos_out, "out's pos", torch.int32, lead, reach, dev)
        lo = _vector(lens_out, "out's lens", slots, dev)
        if mass_out.shape[-1] != reach or pos_out.shape[-1] != reach:
            _fail("out's mass and pos must have as many places as mass")
        if mo != ms:
            spans.append(_ends(mass_out))
        if po != ps:
            spans.append(_ends(pos_out))
        if lo != le:
            spans.append(_ends(lens_out))
    _plain(pool, mass, mass_out)
    if np != le or lo == le:       # both are only read, else
        spans.append(_ends(next_pos))
    spans.sort()
    end = 0
    for first, last in spans:
        if first < end:
            _fail("mass, pos, lens and next_pos must be apart from each "
                  "other, and from each of out that does not replace one")
        end = last
    core = _get(dev)
    ws = _workspace(core.kv_evict_workspace(kv, layers, keep, reach), table)
    core.kv_evict(kv, layers, pool.stride(1), le, lo, np,
                  ms, ps, mo, po, keep, recent, limit, reach, _at(ws),
                  _stream(dev))
    return mass_out, pos_out, lens_out
