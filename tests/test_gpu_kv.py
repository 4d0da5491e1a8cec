"""The paged cache's operators on the GPU against their definitions in 64 bits.

Tolerances, derived: a score is a sum of D products of exact operands in
float32, so it is off by at most (D + 4) 2^-24 of sum |q||k| scale (`size`),
and as much again for the scaling; a weight exp(s - max) / sum by twice that
(score and maximum) plus the sum's own rounding, at most one addition a place
that a lane sees (n / 16) and some 64 for joins and exponentials. An output
adds the weights' 16-bit pieces (2^-16 of sum w|V| with two, nothing with
three) and half a step of its type.
"""
import math

import pytest
import torch

import kv_oracle as oracle

pytestmark = pytest.mark.gpu

STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11,
        torch.bfloat16: 2.0 ** -8}
TYPES = [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float16)]
IDS = ["f32-bf16", "bf16", "f16"]


def weight_error(size, dim, n, scores=1):
    return 2 * 2 * (dim + 4) * 2.0 ** -24 * size + (n / 16 + 64) * 2.0 ** -24


def make(seed, lens, heads, kv_heads, dim, page, types, more=0, layers=None,
         strange=True):
    """q, pool, table on the CPU; unused places and pages hold inf and NaN."""
    g = torch.Generator().manual_seed(seed)
    B, n = len(lens), max(max(lens) + more, 1)
    per = -(-n // page) + 1
    P = B * per + 2
    shape = (P, kv_heads, 2, page, dim)
    if layers:
        shape = (P, layers, *shape[1:])
    pool = torch.randn(shape, generator=g).to(types[1])
    table = torch.randperm(P, generator=g)[:B * per].to(torch.int32)
    table = table.view(B, per)
    if strange:
        used = torch.zeros(P, page, dtype=torch.bool)
        for b, x in enumerate(lens):
            for p in range(x):
                used[table[b, p // page], p % page] = True
        junk = torch.tensor([math.inf, math.nan, -math.inf, 6e4])
        for a, r in (~used).nonzero().tolist():
            pool[a, ..., r, :] = junk[(a + r) % 4]
    q = (1.5 * torch.randn(B, heads, dim, generator=g)).to(types[0])
    return q, pool, table


def ints(v, device="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=device)


def check_attend(q, pool, table, lens, mass=True, scale=None, seed=0, **kw):
    from crowdllama_amd.ops import kv
    B, H, D = q.shape
    cap = table.shape[1] * pool.shape[-2]
    base = torch.rand(B, pool.shape[1], cap,
                      generator=torch.Generator().manual_seed(seed))
    dm = base.cuda() if mass else None
    got = kv.attend(q.cuda(), pool.cuda(), table.cuda(), ints(lens), mass=dm,
                    scale=scale, **kw)
    real = D ** -0.5 if scale is None else scale
    want, add, big, size = oracle.attend(q, pool, table, lens, real)
    err = weight_error(size, D, max(lens))
    piece = 0 if q.dtype is torch.float32 else 2.0 ** -16
    assert got.dtype is q.dtype
    off = (got.double().cpu() - want).abs()
    assert (off <= big * (err + piece) + want.abs() * STEP[q.dtype]
            + 2.0 ** -24).all(), (off.max(), err)
    if mass:
        sum_ = base.double() + add
        off = (dm.double().cpu() - sum_).abs()
        assert (off <= add * err + sum_ * 2.0 ** -24 + 2.0 ** -126).all(), \
            off.max()
    return got, dm


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (16, 1)])
def test_attend(types, dim, heads, kv_heads):
    lens = [70, 0, 1, 16, 17, 33, 128, 129, 300]
    q, pool, table = make(1, lens, heads, kv_heads, dim, 32, types)
    check_attend(q, pool, table, lens)


@pytest.mark.parametrize("page", [16, 48, 64, 128, 1024])
def test_attend_page_sizes(page):
    lens = [page - 1, page, page + 1, 3 * page + 5, 2]
    q, pool, table = make(2, lens, 4, 2, 64, page, TYPES[1])
    check_attend(q, pool, table, lens)
    check_attend(q, pool, table, lens, mass=False, scale=0.3)


@pytest.mark.parametrize("heads,kv_heads", [(7, 1), (10, 2), (24, 8)])
def test_attend_shared_heads(heads, kv_heads):
    lens = [257, 31]
    q, pool, table = make(3, lens, heads, kv_heads, 128, 64, TYPES[0])
    check_attend(q, pool, table, lens)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
def test_attend_long(types):
    """One long sequence over many workgroups beside short ones."""
    lens = [9001, 3, 700]
    q, pool, table = make(4, lens, 8, 2, 64, 64, types, strange=False)
    a, m = check_attend(q, pool, table, lens)
    b, n = check_attend(q, pool, table, lens)
    assert torch.equal(a, b) and torch.equal(m, n)   # and always the same


def test_attend_many_sequences():
    lens = [(7 * i) % 90 for i in range(150)]
    q, pool, table = make(5, lens, 2, 1, 64, 16, TYPES[1])
    check_attend(q, pool, table, lens)


def test_attend_large_scores():
    """One place takes all the weight; the running maximum rises late."""
    lens = [400]
    q, pool, table = make(6, lens, 4, 2, 64, 32, TYPES[0], strange=False)
    for p, f in ((0, 3.), (130, 6.), (399, 20.)):
        pool[table[0, p // 32], :, 0, p % 32] *= f
    check_attend(q, pool, table, lens)


def test_attend_lengths_out_of_range():
    from crowdllama_amd.ops import kv
    lens = [40, 40, 40]
    q, pool, table = make(7, lens, 4, 2, 64, 16, TYPES[1], strange=False)
    cap = table.shape[1] * 16
    mass = torch.zeros(3, 2, cap, device="cuda")
    got = kv.attend(q.cuda(), pool.cuda(), table.cuda(),
                    ints([10 ** 9, -5, 40]), mass=mass)
    want, add, big, _ = oracle.attend(q, pool, table, [cap, 0, 40], 64 ** -.5)
    assert torch.allclose(got.double().cpu(), want, atol=2.0 ** -8 * 4)
    assert (got[1] == 0).all() and (mass[1] == 0).all()
    assert torch.allclose(mass.double().cpu(), add, atol=1e-5)


def test_attend_missing_pages():
    """Pages outside the pool have no weight; one sequence has no other."""
    lens = [100, 60, 50]
    q, pool, table = make(8, lens, 4, 2, 64, 16, TYPES[0])
    table[0, 2], table[0, 5] = -1, pool.shape[0]
    table[1, :] = 2 ** 30
    got, mass = check_attend(q, pool, table, lens)
    assert (got[1] == 0).all()


def test_attend_strides():
    """Queries in a fused product's rows, one layer of a pool, a mass that is
    part of more, the output in another order."""
    from crowdllama_amd.ops import kv
    lens = [90, 33]
    q, pool, table = make(9, lens, 4, 2, 64, 32, TYPES[0], strange=False)
    want, add, big, size = oracle.attend(q, pool, table, lens, 64 ** -.5)
    qkv = torch.zeros(2, 8 * 64, device="cuda")
    qkv[:, :256] = q.reshape(2, 256).cuda()
    three = torch.full((pool.shape[0], 3, *pool.shape[1:]), math.nan,
                       dtype=pool.dtype, device="cuda")
    three[:, 1] = pool.cuda()
    wide = torch.zeros(2, table.shape[1] + 3, dtype=torch.int32,
                       device="cuda")
    wide[:, :table.shape[1]] = table.cuda()
    masses = torch.zeros(2, 2, 5, table.shape[1] * 32 + 7, device="cuda")
    mass = masses[:, :, 2, :table.shape[1] * 32]
    out = torch.zeros(4, 2, 64, device="cuda").transpose(0, 1)
    got = kv.attend(qkv[:, :256].view(2, 4, 64), three[:, 1],
                    wide[:, :table.shape[1]], ints(lens), mass=mass, out=out)
    assert got is out
    err = weight_error(size, 64, 90)
    off = (out.double().cpu() - want).abs()
    assert (off <= big * err + 2.0 ** -24 * want.abs() + 2.0 ** -24).all()
    assert ((mass.double().cpu() - add).abs() <= add * (err + 2.0 ** -24)
            + 2.0 ** -126).all()
    masses[:, :, 2, :table.shape[1] * 32] = 0
    assert (masses == 0).all()


def test_attend_into_its_queries():
    from crowdllama_amd.ops import kv
    lens = [700, 5]
    q, pool, table = make(10, lens, 8, 2, 128, 64, TYPES[1], strange=False)
    dq, pool, table = q.cuda(), pool.cuda(), table.cuda()
    want = kv.attend(dq, pool, table, ints(lens))
    kv.attend(dq, pool, table, ints(lens), out=dq)
    assert torch.equal(dq, want)


def test_attend_nan_and_inf_stay_in_their_head():
    from crowdllama_amd.ops import kv
    lens = [50, 50]
    q, pool, table = make(11, lens, 4, 2, 64, 16, TYPES[1], strange=False)
    want, _, _, _ = oracle.attend(q, pool, table, lens, 64 ** -.5)
    pool[table[0, 1], 1, 0, 3] = math.nan
    pool[table[1, 2], 0, 1, 2, 5] = math.inf
    mass = torch.zeros(2, 2, table.shape[1] * 16, device="cuda")
    got = kv.attend(q.cuda(), pool.cuda(), table.cuda(), ints(lens),
                    mass=mass).double().cpu()
    assert got[0, 2:].isnan().all() and mass[0, 1, :50].isnan().all()
    assert torch.allclose(got[0, :2], want[0, :2], atol=2.0 ** -7)
    assert (got[1, :2, 5] == math.inf).all()
    keep = torch.arange(64) != 5
    assert torch.allclose(got[1, :2][:, keep], want[1, :2][:, keep],
                          atol=2.0 ** -7)
    assert not mass[1].isnan().any() and not mass[0, 0].isnan().any()
    assert (mass[..., 50:] == 0).all()


def test_attend_past_32_bits():
    """Rows whose offset in the pool is past 2^32 bytes and 2^31 elements."""
    from crowdllama_amd.ops import kv
    lens = [100]
    q, pool, table = make(12, lens, 4, 2, 128, 64, TYPES[1], strange=False)
    per = pool[0].numel()
    big = torch.empty((1 << 31) // per + 10, *pool.shape[1:],
                      dtype=pool.dtype, device="cuda")
    at = big.shape[0] - pool.shape[0]
    big[at:] = pool.cuda()
    got = kv.attend(q.cuda(), big, (table + at).cuda(), ints(lens))
    assert torch.equal(got, kv.attend(q.cuda(), pool.cuda(), table.cuda(),
                                      ints(lens)))


def longer(table, page):
    """Room for more places than one workgroup takes: rows go in parts."""
    more = torch.full((table.shape[0], 2048 // page), -1, dtype=torch.int32)
    return torch.cat([table, more], 1)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (16, 1)])
def test_attend_in_parts(types, dim, heads, kv_heads):
    lens = [70, 0, 1, 16, 17, 33, 128, 129, 300]
    q, pool, table = make(1, lens, heads, kv_heads, dim, 32, types)
    check_attend(q, pool, longer(table, 32), lens)


def test_attend_in_parts_odd_pages_and_lengths():
    from crowdllama_amd.ops import kv
    lens = [100, 60, 50, 400]
    q, pool, table = make(8, lens, 4, 2, 64, 16, TYPES[0])
    table[0, 2], table[0, 5] = -1, pool.shape[0]
    table[1, :] = 2 ** 30
    got, _ = check_attend(q, pool, longer(table, 16), lens)
    assert (got[1] == 0).all()
    a = [x.cuda() for x in (q, pool, longer(table, 16))]
    # 10^9 is as many as the table holds, NaN in unused places among them:
    # off - off is NaN where it should be, so not check_attend's comparison
    b = kv.attend(*a, ints([10 ** 9, -5, 50, 0]))
    full, _, _, _ = oracle.attend(q, pool, longer(table, 16),
                                  [10 ** 9, -5, 50, 0], 64 ** -.5)
    assert torch.allclose(b.double().cpu(), full, atol=1e-5, equal_nan=True)
    assert (b[[1, 3]] == 0).all() and torch.equal(b[2], got[2])
    want = kv.attend(*a, ints(lens))
    kv.attend(*a, ints(lens), out=a[0])              # into its queries
    assert torch.equal(a[0], want)


def test_attend_in_parts_nan_and_inf():
    from crowdllama_amd.ops import kv
    lens = [50, 50]
    q, pool, table = make(11, lens, 4, 2, 64, 16, TYPES[1], strange=False)
    want, _, _, _ = oracle.attend(q, pool, table, lens, 64 ** -.5)
    pool[table[0, 1], 1, 0, 3] = math.nan
    pool[table[1, 2], 0, 1, 2, 5] = math.inf
    table = longer(table, 16)
    mass = torch.zeros(2, 2, table.shape[1] * 16, device="cuda")
    got = kv.attend(q.cuda(), pool.cuda(), table.cuda(), ints(lens),
                    mass=mass).double().cpu()
    assert got[0, 2:].isnan().all() and mass[0, 1, :50].isnan().all()
    assert torch.allclose(got[0, :2], want[0, :2], atol=2.0 ** -7)
    assert (got[1, :2, 5] == math.inf).all()
    assert not mass[1].isnan().any() and not mass[0, 0].isnan().any()
    assert (mass[..., 50:] == 0).all()


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("B,kv_heads,cap", [(16, 8, 1024), (2, 2, 768),
                                            (257, 1, 96), (16, 8, 1040),
                                            (1025, 1, 32)])
def test_attend_full_rows(types, B, kv_heads, cap):
    """Full caches at the sizes where one form gives way to the other."""
    lens = [cap - 3 * (b % 7) for b in range(B)]
    q, pool, table = make(13, lens, 2 * kv_heads, kv_heads, 64, 16, types,
                          strange=False)
    table = table[:, :cap // 16].contiguous()
    a, m = check_attend(q, pool, table, lens)
    b, n = check_attend(q, pool, table, lens)
    assert torch.equal(a, b) and torch.equal(m, n)


# ------------------------------------------------------------------- append

@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 2), (96, 3, 1),
                                                (128, 8, 8)])
@pytest.mark.parametrize("ragged", [False, True])
def test_append(types, dim, heads, kv_heads, ragged):
    from crowdllama_amd.ops import kv
    lens = [5, 31, 0, 60]
    rows = [7, 0, 40, 1] if ragged else [1] * 4
    # far positions: 2^24 and past
    ahead = [5, 1 << 24, 2 ** 31 - 100, 77777]
    T, behind = sum(rows), 2 if ragged else 0
    _, pool, table = make(20, lens, heads, kv_heads, dim, 16, types, 40,
                          strange=False)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(T + behind, (heads + 2 * kv_heads) * dim, generator=g)
    qkv = qkv.to(types[0])
    inv = (10000.0 ** (-torch.arange(0, dim, 2).double() / dim)).float()
    cap = table.shape[1] * 16
    mass = torch.rand(4, kv_heads, cap, generator=g)
    pos = torch.randint(0, 99, (4, kv_heads, cap), generator=g,
                        dtype=torch.int32)
    split = lambda x: (x[:, :heads * dim].view(-1, heads, dim),  # noqa: E731
                       x[:, heads * dim:(heads + kv_heads) * dim].view(
                           -1, kv_heads, dim),
                       x[:, (heads + kv_heads) * dim:].view(-1, kv_heads, dim))
    starts = [sum(rows[:b]) for b in range(5)] if ragged else None
    q, k, v = split(qkv)
    owner = sum(([b] * r for b, r in enumerate(rows)), [])
    index = sum((list(range(r)) for r in rows), [])
    positions = torch.tensor([ahead[b] + i for b, i in zip(owner, index)])
    want_q = torch.cat([oracle.turn(q[:T], positions, inv),
                        q[T:].double()])
    want_k = oracle.turn(k[:T], positions, inv)
    # two products and a sum, sines to two units, the angle to half of one
    # of pi: 14 half steps of the larger of the pair, at most 6
    small = 14 * 2.0 ** -24 * 6

    dp, dm, ds = pool.cuda(), mass.cuda(), pos.cuda()
    dq, dk, dv = split(qkv.cuda())
    before = dq.clone()
    got = kv.append(dk, dv, dp, table.cuda(), ints(lens), ints(ahead), q=dq,
                    inv_freq=inv.cuda(),
                    starts=ints(starts) if ragged else None, mass=dm, pos=ds)
    assert torch.equal(dq, before)
    assert ((got.double().cpu() - want_q).abs()
            <= small + want_q.abs() * STEP[types[0]]).all()
    dp2 = pool.cuda()
    same = kv.append(dk, dv, dp2, table.cuda(), ints(lens), ints(ahead),
                     q=dq, q_out=dq, inv_freq=inv.cuda(),
                     starts=ints(starts) if ragged else None)
    assert same is dq and torch.equal(got, dq) and torch.equal(dp, dp2)
    want, told = pool.double(), torch.zeros(pool.shape, dtype=torch.bool)
    for t, (b, i) in enumerate(zip(owner, index)):
        p, r = oracle.place(table, pool.shape[0], 16, b, lens[b] + i)
        want[p, :, 0, r], want[p, :, 1, r] = want_k[t], v[t].double()
        told[p, :, 0, r] = True
        mass[b, :, lens[b] + i] = 0
        pos[b, :, lens[b] + i] = int(positions[t])
    off = (dp.double().cpu() - want).abs()
    assert (off <= told * small + want.abs() * STEP[types[1]]).all()
    untouched = want == pool.double()
    assert torch.equal(dp.cpu()[untouched], pool[untouched])
    assert torch.equal(dm.cpu(), mass) and torch.equal(ds.cpu(), pos)


def test_append_without_rotation_or_queries():
    from crowdllama_amd.ops import kv
    lens = [3, 20]
    _, pool, table = make(21, lens, 4, 2, 64, 16, TYPES[1], 5, strange=False)
    k, v = torch.randn(2, 2, 2, 64).bfloat16().unbind()
    dp = pool.cuda()
    assert kv.append(k.cuda(), v.cuda(), dp, table.cuda(), ints(lens),
                     ints(lens)) is None
    for b in range(2):
        p, r = oracle.place(table, pool.shape[0], 16, b, lens[b])
        pool[p, :, 0, r], pool[p, :, 1, r] = k[b], v[b]
    assert torch.equal(dp.cpu(), pool)


def test_append_past_the_end_and_missing_pages():
    """Rows past a sequence's reach and on pages that are not there."""
    from crowdllama_amd.ops import kv
    lens = [30, 2 ** 31 - 2, -3, 0]
    _, pool, table = make(22, [30, 0, 0, 0], 4, 2, 64, 16, TYPES[1],
                          strange=False)
    table[3, 0] = pool.shape[0]
    cap = table.shape[1] * 16 - 5          # the mass ends before the pages
    k = torch.randn(4 * 20, 2, 64).bfloat16()
    mass = torch.rand(4, 2, cap)
    dp, dm = pool.cuda(), mass.cuda()
    kv.append(k.cuda(), k.cuda(), dp, table.cuda(), ints(lens), ints([0] * 4),
              starts=ints([0, 20, 40, 60, 80]), mass=dm)
    for b, n in enumerate(lens):
        for i in range(20):
            if not 0 <= n + i < cap:
                continue
            mass[b, :, n + i] = 0
            at = oracle.place(table, pool.shape[0], 16, b, n + i)
            if at:
                pool[at[0], :, 0, at[1]] = k[b * 20 + i]
                pool[at[0], :, 1, at[1]] = k[b * 20 + i]
    assert torch.equal(dp.cpu(), pool) and torch.equal(dm.cpu(), mass)


# ------------------------------------------------------------------ observe

def check_observe(q, pool, table, lens, starts, types):
    from crowdllama_amd.ops import kv
    B, heads, D = table.shape[0], pool.shape[1], q.shape[-1]
    cap = table.shape[1] * pool.shape[-2]
    base = torch.rand(B, heads, cap, generator=torch.Generator().manual_seed(1))
    dm = base.cuda()
    assert kv.observe(q.cuda(), pool.cuda(), table.cuda(), ints(lens), dm,
                      starts=None if starts is None else ints(starts)) is dm
    st = starts or list(range(B + 1))
    add, size = oracle.observe(q, pool, table, lens, st, D ** -.5)
    rows = max(b - a for a, b in zip(st, st[1:])) * q.shape[1] // heads
    # a row's sum is taken as its logarithm, which is off by half a step of
    # itself (its size is at most the scores' and log2 of the places);
    # a place's sum has one addition a row
    err = weight_error(size, D, max(lens)) + rows * 2.0 ** -24 + \
        2 * (1.5 * size + math.log2(cap)) * 2.0 ** -24
    want = base.double() + add
    off = (dm.double().cpu() - want).abs()
    assert (off <= add * err + want * 2.0 ** -24 + 2.0 ** -126).all(), \
        (off.max(), err)
    return dm


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 2), (96, 3, 3),
                                                (128, 7, 1)])
def test_observe(types, dim, heads, kv_heads):
    lens = [70, 1, 300, 40, 16]
    rows = [70, 1, 33, 0, 16]
    _, pool, table = make(30, lens, heads, kv_heads, dim, 32, types)
    q = torch.randn(sum(rows) + 3, heads, dim,
                    generator=torch.Generator().manual_seed(2)).to(types[0])
    starts = [sum(rows[:b]) for b in range(6)]
    a = check_observe(q, pool, table, lens, starts, types)
    b = check_observe(q, pool, table, lens, starts, types)
    assert torch.equal(a, b)


def test_observe_as_attend():
    """Of one token it is what attend adds."""
    lens = [70, 200, 3]
    q, pool, table = make(31, lens, 8, 2, 64, 16, TYPES[0])
    check_observe(q, pool, table, lens, None, TYPES[0])


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("long_,n", [(1, 1), (9, 700), (70, 2100)])
def test_observe_few_rows(types, dim, long_, n):
    """Few rows a sequence on average: one may have many more."""
    lens, rows = [n] + [5, 0, 1500, 33, 40, 7, 8], [long_, 1, 0, 3, 2, 2, 1, 8]
    _, pool, table = make(38, lens, 4, 2, dim, 32, types,
                          strange=n < 1000)
    table[4, 0] = -1
    q = torch.randn(sum(rows), 4, dim,
                    generator=torch.Generator().manual_seed(2)).to(types[0])
    q[long_:] *= 8                       # and scores far from 0
    check_observe(q, pool, table, lens,
                  [sum(rows[:b]) for b in range(9)], types)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
def test_observe_longer(types):
    lens = [1500, 777]
    rows = [1030, 777]
    _, pool, table = make(32, lens, 4, 2, 128, 64, types, strange=False)
    q = torch.randn(sum(rows), 4, 128,
                    generator=torch.Generator().manual_seed(2)).to(types[0])
    check_observe(q, pool, table, lens, [0, 1030, 1807], types)


@pytest.mark.parametrize("types", TYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("heads,rows", [(2, 1300), (16, 1300)])
def test_observe_uneven_batch(types, heads, rows):
    """One of 70 sequences has nearly all the rows: several chunks of them,
    which the others' one or none go before and come after."""
    B, long_ = 70, 66
    m = [b % 4 for b in range(B)]
    lens = [x + 5 * (b % 7) for b, x in enumerate(m)]
    m[long_], lens[long_] = rows, rows + 200
    _, pool, table = make(39, lens, heads, 2, 64, 32, types, strange=False)
    q = torch.randn(sum(m) + 2, heads, 64,
                    generator=torch.Generator().manual_seed(2)).to(types[0])
    starts = [sum(m[:b]) for b in range(B + 1)]
    assert torch.equal(check_observe(q, pool, table, lens, starts, types),
                       check_observe(q, pool, table, lens, starts, types))


def test_observe_starts_out_of_order():
    """Nothing is added behind a sequence's places, or to one without rows."""
    from crowdllama_amd.ops import kv
    lens = [900, 40, 700, 0, 64]
    _, pool, table = make(40, lens, 16, 4, 64, 32, TYPES[1], strange=False)
    q = torch.randn(600, 16, 64).bfloat16().cuda()
    cap = table.shape[1] * 32
    for starts in ([0, 600, 0, 600, 0, 600], [2**31 - 1, 0, 600, 5, -7, 900],
                   [0, 600, 600, 600, 600, -2**31]):
        mass = torch.ones(5, 4, cap, device="cuda")
        kv.observe(q, pool.cuda(), table.cuda(), ints(lens), mass,
                   starts=ints(starts))
        mass = mass.cpu()
        for b, n in enumerate(lens):
            assert (mass[b, :, n:] == 1).all()
            if starts[b + 1] <= max(starts[b], 0):
                assert (mass[b] == 1).all()


def test_observe_more_rows_than_places():
    """A row before the first place sees nothing, and adds nothing."""
    from crowdllama_amd.ops import kv
    lens = [10]
    _, pool, table = make(33, lens, 4, 2, 64, 16, TYPES[1], 6)
    q = torch.randn(30, 4, 64).bfloat16()
    cap = table.shape[1] * 16
    a, b = torch.zeros(2, 1, 2, cap, device="cuda").unbind()
    args = pool.cuda(), table.cuda(), ints(lens)
    kv.observe(q.cuda(), *args, a, starts=ints([0, 30]))
    kv.observe(q[20:].cuda().contiguous(), *args, b, starts=ints([0, 10]))
    assert torch.allclose(a, b, atol=1e-5) and (a[..., 10:] == 0).all()
    assert abs(float(a.sum()) - 10 * 4) < 1e-3


def test_observe_missing_pages():
    lens = [100, 40]
    _, pool, table = make(34, lens, 4, 2, 64, 16, TYPES[1])
    table[0, 1], table[1, :] = -7, pool.shape[0]
    q = torch.randn(90, 4, 64).bfloat16()
    check_observe(q, pool, table, lens, [0, 60, 90], TYPES[1])


@pytest.mark.parametrize("types", TYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("factor,shift", [(20., 0.), (1., -30.), (1., 30.),
                                          (6., -12.)])
def test_observe_far_scores(types, factor, shift):
    """Rows whose scores are all far below or above 0, or far apart: their
    exponentials would vanish or overflow."""
    lens, rows = [200, 90], [70, 90]
    _, pool, table = make(35, lens, 4, 2, 64, 16, types, strange=False)
    q = torch.randn(160, 4, 64, generator=torch.Generator().manual_seed(2))
    q, pool = factor * q, pool.float()
    # one dimension of all keys and queries: adds shift * 8 * scale to each
    q[..., 0], pool[:, :, 0, :, 0] = shift, 64.
    check_observe(q.to(types[0]), pool.to(types[1]), table, lens,
                  [0, 70, 160], types)


@pytest.mark.parametrize("types", TYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("shift", [-30., 30.])
def test_observe_far_scores_in_parts(types, shift):
    """The same over several parts of the places, the later of which most rows
    do not see at all."""
    lens, rows = [1700, 600], [1700, 10]
    _, pool, table = make(37, lens, 2, 1, 64, 64, types, strange=False)
    q = torch.randn(1710, 2, 64, generator=torch.Generator().manual_seed(2))
    pool = pool.float()
    q[..., 0], pool[:, :, 0, :, 0] = shift, 64.
    check_observe(q.to(types[0]), pool.to(types[1]), table, lens,
                  [0, 1700, 1710], types)


def test_observe_nan_and_inf():
    """A row with NaN spoils what it sees, in its kv head; a key with NaN
    spoils every row that sees it."""
    from crowdllama_amd.ops import kv
    lens = [120]
    _, pool, table = make(36, lens, 4, 2, 64, 16, TYPES[1], strange=False)
    q = torch.randn(80, 4, 64).bfloat16()
    args = lambda: (pool.cuda(), table.cuda(), ints(lens))  # noqa: E731
    cap = table.shape[1] * 16
    clean = torch.zeros(1, 2, cap, device="cuda")
    kv.observe(q.cuda(), *args(), clean, starts=ints([0, 80]))
    bad = q.clone()
    bad[79, 0, 5] = math.nan                   # the last token
    got = torch.zeros(1, 2, cap, device="cuda")
    kv.observe(bad.cuda(), *args(), got, starts=ints([0, 80]))
    assert got[0, 0, :120].isnan().all() and torch.equal(got[0, 1],
                                                         clean[0, 1])
    bad = q.clone()
    bad[0, 3, 5] = math.inf                    # sees 41 places
    got.zero_()
    kv.observe(bad.cuda(), *args(), got, starts=ints([0, 80]))
    assert got[0, 1, :41].isnan().all() and torch.equal(got[0, 0],
                                                        clean[0, 0])
    # rows beside it are summed relative to their maximum instead of to 0:
    # each way is within weight_error (here below 1e-4) of the exact sum
    assert torch.allclose(got[0, 1, 41:], clean[0, 1, 41:], rtol=2e-4)
    at = oracle.place(table, pool.shape[0], 16, 0, 119)
    pool[at[0], 0, 0, at[1], 3] = math.nan     # seen by the last token only
    got.zero_()
    kv.observe(q.cuda(), *args(), got, starts=ints([0, 80]))
    assert got[0, 0, :120].isnan().all() and torch.equal(got[0, 1],
                                                         clean[0, 1])


def many(types, n, m, seed=41, dim=64, **kw):
    """24 sequences and 8 heads: enough rows for a pass that stages its keys."""
    lens, rows = [n - b for b in range(24)], [m - 2 * b for b in range(24)]
    _, pool, table = make(seed, lens, 8, 8, dim, 16, types, **kw)
    q = torch.randn(sum(rows), 8, dim,
                    generator=torch.Generator().manual_seed(2))
    return q, pool, table, lens, [sum(rows[:b]) for b in range(25)]


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("n,m,dim", [(200, 170, 64), (700, 160, 64),
                                     (700, 160, 96), (700, 160, 128)])
@pytest.mark.parametrize("missing", [False, True])
def test_observe_many_rows(types, n, m, dim, missing):
    q, pool, table, lens, starts = many(types, n, m, dim=dim)
    if missing:
        table[0, 1], table[2, :], table[5, 3], table[7, 0] = -7, 1 << 30, -1, -1
    check_observe(q.to(types[0]), pool, table, lens, starts, types)


@pytest.mark.parametrize("types", TYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("factor,shift", [(20., 0.), (1., -30.), (1., 30.),
                                          (6., -12.)])
@pytest.mark.parametrize("n,m", [(200, 170), (700, 160)])
def test_observe_many_far_rows(types, factor, shift, n, m):
    q, pool, table, lens, starts = many(types, n, m, strange=False)
    q, pool = factor * q, pool.float()
    q[..., 0], pool[:, :, 0, :, 0] = shift, 64.
    check_observe(q.to(types[0]), pool.to(types[1]), table, lens, starts, types)


def test_observe_nan_among_many_rows():
    from crowdllama_amd.ops import kv
    q, pool, table, lens, starts = many(TYPES[1], 200, 170, strange=False)
    q = q.bfloat16()
    cap = table.shape[1] * 16

    def run():
        got = torch.zeros(24, 8, cap, device="cuda")
        return kv.observe(q.cuda(), pool.cuda(), table.cuda(), ints(lens), got,
                          starts=ints(starts)).cpu()
    clean = run()
    q[starts[4] - 1, 2, 5] = math.nan          # sequence 3's last token
    q[starts[9], 6, 5] = math.inf              # 9's first: sees 191 - 152 + 1
    at = oracle.place(table, pool.shape[0], 16, 20, 179)
    pool[at[0], 7, 0, at[1], 3] = math.nan     # 20's last token sees it alone
    got = run()
    assert got[3, 2, :197].isnan().all() and got[9, 6, :40].isnan().all()
    assert got[20, 7, :180].isnan().all()
    # rows of the same workgroup: summed another way, as above
    assert torch.allclose(got[9, 6, 40:], clean[9, 6, 40:], rtol=2e-4)
    got[3, 2], got[9, 6], got[20, 7] = clean[3, 2], clean[9, 6], clean[20, 7]
    assert torch.equal(got, clean)


# -------------------------------------------------------------------- evict

def make_evict(seed, lens, layers, kv_heads, dim, page, dtype, cap=None):
    g = torch.Generator().manual_seed(seed)
    _, pool, table = make(seed, lens, kv_heads, kv_heads, dim, page,
                          (dtype, dtype), layers=layers, strange=False)
    cap = cap or table.shape[1] * page
    shape = (layers, len(lens), kv_heads, cap)
    mass = torch.exp(2 * torch.randn(shape, generator=g))
    mass[torch.rand(shape, generator=g) < 0.3] = 0.
    pos = torch.rand(shape, generator=g).argsort(-1).to(torch.int32)
    return pool, table, mass, pos


def check_evict(pool, table, lens, next_pos, mass, pos, keep, recent, limit):
    from crowdllama_amd.ops import kv
    args = dict(keep=keep, recent=recent, limit=limit)
    d = [x.cuda() for x in (pool, mass, pos)]
    out = [torch.full_like(d[1], 7), torch.full_like(d[2], 7),
           ints([7] * len(lens))]
    dl, dn, dt = ints(lens), ints(next_pos), table.cuda()
    got = kv.evict(d[0], dt, dl, dn, d[1], d[2], out=out, **args)
    assert all(a is b for a, b in zip(got, out))
    assert torch.equal(d[1].cpu().isnan(), mass.isnan())
    assert torch.equal(d[2].cpu(), pos) and dl.tolist() == list(lens)
    d2 = [x.cuda() for x in (pool, mass, pos)]
    l2 = ints(lens)
    kv.evict(d2[0], dt, l2, dn, d2[1], d2[2], **args)
    want = [x.clone() for x in (pool, mass, pos)]
    wl = list(lens)
    oracle.evict(want[0], table, wl, next_pos, want[1], want[2], keep, recent,
                 keep if limit is None else limit)
    for have in ((d[0], *out[:2]), d2):
        for a, b in zip(have, want):
            a = a.cpu()
            assert torch.equal(a, b) or torch.equal(
                a.nan_to_num(nan=-1e9), b.nan_to_num(nan=-1e9))
    assert out[2].tolist() == wl and l2.tolist() == wl


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 48), (128, 64)])
@pytest.mark.parametrize("keep,recent", [(40, 10), (40, 40), (1, 0), (63, 0),
                                         (30, 500)])
def test_evict(dtype, dim, page, keep, recent):
    lens = [100, 41, 40, 0, 64]
    pool, table, mass, pos = make_evict(40, lens, 2, 2, dim, page, dtype)
    check_evict(pool, table, lens, [100, 90, 40, 0, 64], mass, pos, keep,
                recent, None)


@pytest.mark.parametrize("n,keep", [(1024, 1000), (1025, 512), (5000, 2500),
                                    (9000, 100), (40000, 9999)])
def test_evict_long(n, keep):
    lens = [n, n // 2]
    pool, table, mass, pos = make_evict(41, lens, 1, 2, 64, 64,
                                        torch.bfloat16)
    check_evict(pool, table, lens, lens, mass, pos, keep, keep // 3, None)


def test_evict_many_rows():
    """More rows than a grid's second dimension holds."""
    from crowdllama_amd.ops import kv
    g = torch.Generator(device="cuda").manual_seed(0)
    B, heads = 2200, 32
    pool = torch.randn(B, 1, heads, 2, 16, 64, device="cuda").bfloat16()
    table = torch.randperm(B, generator=g, device="cuda").int().view(B, 1)
    mass = torch.rand(1, B, heads, 16, generator=g, device="cuda")
    pos = torch.arange(16, dtype=torch.int32, device="cuda").expand(
        1, B, heads, 16).contiguous()
    lens = torch.full((B,), 16, dtype=torch.int32, device="cuda")
    old, weight = pool.clone(), mass.clone()
    kv.evict(pool, table, lens, lens.clone(), mass, pos, keep=6)
    assert (lens == 6).all()
    stay = weight.topk(6, -1)[1].sort(-1)[0]
    assert torch.equal(pos[..., :6].long().sort(-1)[0], stay)
    assert torch.equal(mass[..., :6], weight.gather(-1, pos[..., :6].long()))
    rows = old[table[:, 0].long(), 0].gather(3, pos[0, :, :, None, :6, None]
                                            .long().expand(-1, -1, 2, -1, 64))
    assert torch.equal(pool[table[:, 0].long(), 0, :, :, :6], rows)


def test_evict_ties_and_strange_masses():
    lens = [64]
    pool, table, mass, pos = make_evict(42, lens, 1, 4, 64, 16,
                                        torch.bfloat16)
    mass[:, :, 0] = 1.                                   # all the same
    mass[:, :, 1] = torch.where(torch.arange(mass.shape[-1]) % 2 == 0, 0., -0.)
    mass[:, :, 2, ::3] = math.nan                        # after all numbers
    mass[:, :, 2, 1::3] = math.inf
    mass[:, :, 3] = -mass[:, :, 3]
    mass[:, :, 3, 5] = -math.inf
    check_evict(pool, table, lens, [0], mass, pos, 30, 0, None)
    check_evict(pool, table, lens, [64], mass, pos, 60, 7, None)


@pytest.mark.parametrize("n", [300, 3000, 33000])
@pytest.mark.parametrize("kind", ["one", "two", "late", "nan", "near"])
def test_evict_rows_of_equals(n, kind):
    """Ties over several waves, and keys that differ in their last bits."""
    lens = [n, n - 65]
    pool, table, mass, pos = make_evict(45, lens, 1, 2, 64, 64,
                                        torch.bfloat16)
    g = torch.Generator().manual_seed(5)
    pick = torch.rand(mass.shape, generator=g)
    late = [0, 0] if kind == "late" else [1 << 30] * 2
    if kind == "nan":
        mass[pick < .8] = math.nan
    elif kind == "near":
        mass = 1 + torch.floor(pick * 300) * 2.0 ** -23
    else:
        mass = torch.full_like(mass, .5) + (pick < .4) * (kind == "two")
    for keep in (n // 3, n - 70):
        check_evict(pool, table, lens, late, mass, pos, keep, 5, None)


def test_evict_limit():
    lens = [50, 51, 30]
    pool, table, mass, pos = make_evict(43, lens, 2, 1, 64, 16,
                                        torch.float16)
    check_evict(pool, table, lens, lens, mass, pos, 20, 4, 50)


def test_evict_missing_pages_and_lengths_out_of_range():
    lens = [60, 2 ** 31 - 1, -1]
    pool, table, mass, pos = make_evict(44, [60, 60, 60], 1, 2, 64, 16,
                                        torch.bfloat16)
    table[0, 1], table[1, 3] = -1, pool.shape[0]
    check_evict(pool, table, lens, [60, 70, 0], mass, pos, 25, 5, None)


def test_evict_keep_past_the_cache():
    lens = [60]
    pool, table, mass, pos = make_evict(45, lens, 1, 2, 64, 16,
                                        torch.bfloat16)
    check_evict(pool, table, lens, [60], mass, pos, 10 ** 6, 5, None)
    check_evict(pool, table, lens, [60], mass, pos, 10, 5, 10 ** 6)


# ---------------------------------------------------------------- together

class Model:
    """A cache of one layer as lists, in 64 bits: entries of a head."""

    def __init__(self, kv_heads):
        self.rows = [[] for _ in range(kv_heads)]   # [k, v, mass, pos]

    def append(self, k, v, position):
        for h, r in enumerate(self.rows):
            r.append([k[h], v[h], 0., position])

    def attend(self, q, scale):
        out, G = [], len(q) // len(self.rows)
        for h, r in enumerate(self.rows):
            k = torch.stack([e[0] for e in r])
            w = torch.softmax(q[h * G:(h + 1) * G] @ k.T * scale, -1)
            out.append(w @ torch.stack([e[1] for e in r]))
            for e, x in zip(r, w.sum(0).tolist()):
                e[2] += x
        return torch.cat(out)

    def evict(self, keep, recent, now):
        for h, r in enumerate(self.rows):
            stay = oracle.survivors([e[2] for e in r], [e[3] for e in r],
                                    now - recent, keep)
            come = iter([r[p] for p in sorted(stay) if p >= keep])
            self.rows[h] = [r[p] if p in stay else next(come)
                            for p in range(keep)]


def test_a_cache_that_goes_on_past_its_end():
    """Prompts, then tokens, through a cache of 64 places that is emptied to
    40 whenever it is full: outputs, masses and positions as a model says."""
    from crowdllama_amd.ops import kv
    L, B, H, heads, D, page, cap, keep, recent = 2, 2, 4, 2, 64, 16, 64, 40, 8
    g = torch.Generator().manual_seed(50)
    pool = torch.zeros(B * 4, L, heads, 2, page, D, dtype=torch.bfloat16,
                       device="cuda")
    table = ints([[3, 1, 6, 0], [7, 2, 5, 4]])
    lens, now = ints([0, 0]), ints([0, 0])
    mass = torch.zeros(L, B, heads, cap, device="cuda")
    pos = torch.full((L, B, heads, cap), -1, dtype=torch.int32, device="cuda")
    inv = (10000.0 ** (-torch.arange(0, D, 2).double() / D)).float()
    models = [[Model(heads) for _ in range(B)] for _ in range(L)]
    seen, scale = [0, 0], D ** -.5
    # sum |q||k| scale stays below 16 for values of this size (64 products
    # of about 0.64, over 8)
    err = weight_error(16., D, cap)
    prompt = [50, 13]
    for step in range(80):
        rows = prompt if step == 0 else [1, 1]
        starts = ints([0, rows[0], sum(rows)])
        held = lens.tolist()
        for l in range(L):
            q, k, v = (torch.randn(sum(rows), n, D, generator=g)
                       for n in (H, heads, heads))
            dq = kv.append(k.cuda(), v.cuda(), pool[:, l], table, lens, now,
                           q=q.cuda(), inv_freq=inv.cuda(), starts=starts,
                           mass=mass[l], pos=pos[l])
            if step == 0:
                kv.observe(dq, pool[:, l], table, lens + ints(rows), mass[l],
                           starts=starts)
            else:
                out = kv.attend(dq, pool[:, l], table, lens + 1,
                                mass=mass[l]).double().cpu()
            stored, dq, t = pool[:, l].double().cpu(), dq.double().cpu(), 0
            for b in range(B):
                for i in range(rows[b]):
                    p = held[b] + i
                    at = stored[int(table[b, p // page]), :, :, p % page]
                    m = models[l][b]
                    m.append(at[:, 0], at[:, 1], seen[b] + i)
                    want = m.attend(dq[t], scale)
                    if step:
                        assert (out[b] - want).abs().max() < 2 * err * 5
                    t += 1
        for b in range(B):
            seen[b] += rows[b]
        lens += ints(rows)
        now += ints(rows)
        kv.evict(pool, table, lens, now, mass, pos, keep=keep, recent=recent,
                 limit=cap - 1)
        for b in range(B):
            if len(models[0][b].rows[0]) == cap:
                for l in range(L):
                    models[l][b].evict(keep, recent, seen[b])
        assert lens.tolist() == [len(models[0][b].rows[0]) for b in range(B)]
        for l in range(L):
            for b in range(B):
                for h in range(heads):
                    r = models[l][b].rows[h]
                    assert pos[l, b, h, :len(r)].tolist() == [e[3] for e in r]
                    have = mass[l, b, h, :len(r)].double().cpu()
                    want = torch.tensor([e[2] for e in r],
                                        dtype=torch.float64)
                    assert ((have - want).abs() <= want * (
                        err + 160 * 2.0 ** -24)).all()
    assert seen == [129, 92] and lens.tolist()[0] < cap


# ------------------------------------------------- streams, graphs, devices

def test_on_another_stream():
    from crowdllama_amd.ops import kv
    lens = [3000, 10]
    q, pool, table = make(60, lens, 8, 2, 64, 64, TYPES[1], strange=False)
    dq, dp, dt, dl = q.cuda(), pool.cuda(), table.cuda(), ints(lens)
    want = kv.attend(dq, dp, dt, dl)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda")
    with torch.cuda.stream(side):
        for _ in range(4):
            big = big @ big.clamp(-1e-3, 1e-3)
        late = dq * 1           # ready only when the products are
        got = kv.attend(late, dp, dt, dl)
    side.synchronize()
    assert torch.equal(got, want)


def test_captured_and_replayed():
    """append, attend and evict in one graph; another graph of attend between
    its replays; lengths change between replays; each checked against eager
    calls."""
    from crowdllama_amd.ops import kv
    B, H, heads, D, cap = 2, 4, 2, 64, 64
    g = torch.Generator().manual_seed(61)
    _, pool, table = make(61, [50, 40], H, heads, D, 16, TYPES[0],
                          layers=1, strange=False)
    table = table[:, :4].contiguous()
    mass = torch.rand(1, B, heads, cap, generator=g)
    pos = torch.arange(cap, dtype=torch.int32).expand(1, B, heads, cap)
    inv = (10000.0 ** (-torch.arange(0, D, 2).double() / D)).float().cuda()

    def fresh():
        return dict(pool=pool.cuda(), mass=mass.cuda(),
                    pos=pos.contiguous().cuda(), lens=ints([50, 40]),
                    now=ints([50, 40]), x=torch.zeros(B, 8, D, device="cuda"),
                    out=torch.zeros(B, H, D, device="cuda"))

    dt = table.cuda()

    def step(s):
        x = s["x"]
        q = kv.append(x[:, 4:6], x[:, 6:], s["pool"][:, 0], dt, s["lens"],
                      s["now"], q=x[:, :4], inv_freq=inv, mass=s["mass"][0],
                      pos=s["pos"][0])
        s["lens"] += 1
        s["now"] += 1
        kv.attend(q, s["pool"][:, 0], dt, s["lens"], mass=s["mass"][0],
                  out=s["out"])
        kv.evict(s["pool"], dt, s["lens"], s["now"], s["mass"], s["pos"],
                 keep=45, recent=6, limit=60)

    step(fresh())                  # loaded before the capture
    a, b = fresh(), fresh()
    other = torch.zeros_like(a["out"])
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    with torch.cuda.graph(second):
        kv.attend(b["x"][:, :4], b["pool"][:, 0], dt, b["lens"], out=other)
    for i in range(40):
        x = torch.randn(B, 8, D, generator=g).cuda()
        a["x"].copy_(x)
        b["x"].copy_(x)
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(other, kv.attend(b["x"][:, :4], b["pool"][:, 0],
                                            dt, b["lens"]))
        step(b)
        for k in a:
            assert torch.equal(a[k], b[k]), (i, k)
    assert int(a["lens"].max()) <= 60 and a["now"].tolist() == [90, 80]


@pytest.mark.parametrize("n,m", [(1500, 700), (700, 30)])
def test_captured_with_workspaces(n, m):
    """attend in parts, observe in parts and chunks, and evict of long rows, in
    two graphs whose replays take turns, with lengths that change between them;
    each replay is what eager calls give, bit for bit."""
    from crowdllama_amd.ops import kv
    B, H, heads, D = 3, 8, 4, 64
    lens = [[n, 20, n // 2], [n // 3, n, 1], [0, n - 1, n]]
    starts = [[0, m, m + 20, 2 * m], [0, 3, m, m + 1], [0, 0, m, 2 * m]]
    _, pool, table = make(62, [n] * B, H, heads, D, 64, TYPES[0], layers=1,
                          strange=False)
    table = longer(table, 64)
    cap = table.shape[1] * 64
    g = torch.Generator().manual_seed(63)
    mass = torch.rand(1, B, heads, cap, generator=g)
    pos = torch.arange(cap, dtype=torch.int32).expand(1, B, heads, cap)
    one = torch.randn(B, H, D, generator=g).cuda()
    q = torch.randn(2 * m, H, D, generator=g).cuda()
    dt = table.cuda()

    def fresh(i):
        return dict(pool=pool.cuda(), mass=mass.cuda(), lens=ints(lens[i]),
                    starts=ints(starts[i]), pos=pos.contiguous().cuda(),
                    out=torch.zeros(B, H, D, device="cuda"))

    def step(s):
        kv.observe(q, s["pool"][:, 0], dt, s["lens"], s["mass"][0],
                   starts=s["starts"])
        kv.attend(one, s["pool"][:, 0], dt, s["lens"], mass=s["mass"][0],
                  out=s["out"])
        kv.evict(s["pool"], dt, s["lens"], s["lens"] + 5, s["mass"], s["pos"],
                 keep=n // 2 - 3, recent=9)

    step(fresh(0))                 # loaded before the capture
    held = [fresh(0), fresh(1)]
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph, s in zip(graphs, held):
        with torch.cuda.graph(graph):
            step(s)
    for i in (0, 1, 2, 0):
        for s, new in zip(held, (fresh(i), fresh((i + 1) % 3))):
            for k in s:
                s[k].copy_(new[k])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s, want in zip(held, (fresh(i), fresh((i + 1) % 3))):
            step(want)
            for k in s:
                assert torch.equal(s[k], want[k]), k
