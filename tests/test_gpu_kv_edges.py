"""The paged cache's operators at the edges of their arithmetic and of what a
call may look like, against the definitions in 64 bits.

Where a query is one 1 among zeros, its scores are one element of each key and
exact but for the scale: a product of three float32 factors, 3 half steps.
"""
import math

import pytest
import torch

import kv_oracle as oracle
from test_gpu_kv import IDS, TYPES, check_attend, ints, longer, make

pytestmark = pytest.mark.gpu


def one_hot(B, heads, dim, dtype):
    """Queries whose scores are element 0 of the keys times the scale."""
    q = torch.zeros(B, heads, dim, dtype=dtype)
    q[..., 0] = 1
    return q


def at(pool, table, b, p):
    """Place p of sequence b in the pool: [kv heads, 2, dim]."""
    page = pool.shape[-2]
    return pool[table[b, p // page], :, :, p % page]


both_forms = pytest.mark.parametrize("parts", [False, True],
                                     ids=["row", "parts"])


@both_forms
def test_attend_bfloat16_is_rounded_once(parts):
    """Each output is the bfloat16 next to a value that is off by float32's
    roundings alone.

    All weights but one lose 0.9 x 2^-15 of themselves if they are cut to two
    pieces of 8 bits; the one has no value. In half steps of
    float32 (2^-24): with scores of at most 1 (their factors 3, their
    difference from the maximum 1 more: 4 ln 2 = 3) and an exponential that is
    off by 2, a weight is off by 5; so is their sum, with 10 additions of its
    own; the products' sum has at most 3 x 32, and the joins and the division
    at most 10. Values of one sign do not cancel.
    """
    from crowdllama_amd.ops import kv
    lens, heads, dim = [32, 31, 17, 9, 30, 25, 5, 28], 16, 128
    _, pool, table = make(70, lens, heads, heads, dim, 16, TYPES[1],
                          strange=False)
    q = one_hot(len(lens), heads, dim, torch.bfloat16)
    pool[:, :, 0, :, 0] = -1.
    pool[:, :, 1] = 1 + pool[:, :, 1].abs() % 1
    for b in range(len(lens)):
        at(pool, table, b, 2)[:, 0, 0] = 0.
        at(pool, table, b, 2)[:, 1] = 0.
    scale = -math.log(.5 * (1 + 2.0 ** -8 + .9 * 2.0 ** -15))
    if parts:
        table = longer(table, 16)
    got = kv.attend(q.cuda(), pool.cuda(), table.cuda(), ints(lens),
                    scale=scale)
    want, _, big, _ = oracle.attend(q, pool, table, lens, scale)
    e = (5 + 5 + 10 + 96 + 10) * 2.0 ** -24 * big
    low, high = (want - e).bfloat16(), (want + e).bfloat16()
    got = got.cpu()
    assert ((low <= got) & (got <= high)).all(), \
        int(((low > got) | (got > high)).sum())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("far", [16, 20, 24, 26, 30])
@both_forms
def test_attend_far_below_one_place(types, far, parts):
    """One place has nearly all the weight and no value (an attention sink);
    the outputs are those of the others, each 2^-far of it."""
    lens = [700, 300, 40]
    q, pool, table = make(71, lens, 4, 2, 64, 16, types, strange=False)
    q = one_hot(3, 4, 64, types[0])
    pool[:, :, 0, :, 0] = 0.
    pool[:, :, 1] = 1 + pool[:, :, 1].abs() % 1
    for b, n in enumerate(lens):
        sink = at(pool, table, b, n // 3)
        sink[:, 0, 0], sink[:, 1] = far, 0.
    if parts:
        table = longer(table, 16)
    check_attend(q, pool, table, lens, scale=math.log(2.))


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@both_forms
def test_attend_infinite_values(types, parts):
    """Infinite wherever a weight meets an infinite value of one sign, also at
    the place with the largest weight, whose 1 is one 16-bit piece."""
    from crowdllama_amd.ops import kv
    lens = [1, 1, 50, 50, 300, 17]
    q, pool, table = make(72, lens, 4, 2, 64, 16, types, strange=False)
    at(pool, table, 0, 0)[:, 1, 3] = math.inf
    at(pool, table, 1, 0)[0, 1, 5] = -math.inf
    for p in range(50):                        # equal weights: all of them 1
        at(pool, table, 2, p)[:, 0] = at(pool, table, 2, 0)[:, 0]
    at(pool, table, 2, 20)[:, 1, 7] = math.inf
    at(pool, table, 3, 11)[1, 1, 9] = -math.inf
    at(pool, table, 4, 250)[:, 1, ::2] = math.inf
    at(pool, table, 4, 3)[:, 1, ::2] = math.inf
    at(pool, table, 5, 2)[:, 1, 1] = math.inf   # both signs: NaN
    at(pool, table, 5, 16)[:, 1, 1] = -math.inf
    if parts:
        table = longer(table, 16)
    mass = torch.zeros(6, 2, table.shape[1] * 16, device="cuda")
    got = kv.attend(q.cuda(), pool.cuda(), table.cuda(), ints(lens),
                    mass=mass).double().cpu()
    want, add, _, _ = oracle.attend(q, pool, table, lens, 64 ** -.5)
    assert want.isinf().sum() == 4 * 1 + 2 * 1 + 4 * 1 + 2 * 1 + 4 * 32
    assert torch.equal(got.isnan(), want.isnan()) and want.isnan().any()
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    fine = want.isfinite()
    # half a step of the coarsest type, of values below 4
    assert torch.allclose(got[fine], want[fine], rtol=0, atol=2.0 ** -6)
    assert torch.allclose(mass.double().cpu(), add, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@both_forms
def test_infinite_keys(types, parts):
    """A score of -inf is a weight of 0, whatever the pieces of the query;
    what attend adds to the mass, observe adds too."""
    from crowdllama_amd.ops import kv
    lens = [40, 300]
    q, pool, table = make(73, lens, 4, 2, 64, 16, types, strange=False)
    q[..., 5] = -1.                  # its second and third pieces are 0
    q[..., 6] = 0.75
    at(pool, table, 0, 7)[:, 0, 5] = math.inf
    at(pool, table, 1, 299)[1, 0, 6] = -math.inf
    at(pool, table, 1, 120)[0, 0, 5:7] = torch.tensor([math.inf, -math.inf])
    # the definition, with the largest negative number for the infinity
    low = pool.double().clamp(-1e9, 1e9)
    if parts:
        table = longer(table, 16)
    args = q.cuda(), pool.cuda(), table.cuda(), ints(lens)
    mass = torch.zeros(2, 2, table.shape[1] * 16, device="cuda")
    got = kv.attend(*args, mass=mass).double().cpu()
    want, add, big, _ = oracle.attend(q, low, table, lens, 64 ** -.5)
    assert (add[0, :, 7] == 0).all() and add[1, 1, 299] == 0
    assert torch.allclose(got, want, rtol=0, atol=2.0 ** -6)
    assert torch.allclose(mass.double().cpu(), add, rtol=1e-4, atol=1e-6)
    for rows in (1, 3):
        many = q.repeat_interleave(rows, 0)
        again = torch.zeros_like(mass)
        kv.observe(many.cuda(), *args[1:], again,
                   starts=ints([0, rows, 2 * rows]))
        add, _ = oracle.observe(many, low, table, lens, [0, rows, 2 * rows],
                                64 ** -.5)
        assert torch.allclose(again.double().cpu(), add, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,n", [(40, 3000), (600, 2000)])
@pytest.mark.parametrize("far", [False, True])
def test_observe_rows_add_up_to_one(types, rows, n, far):
    """The weights that a row gives sum to 1, on average over rows with no
    more than the roundings of their exponentials: the row's own sum must not
    be rounded to fewer bits than they have.

    Scores of at most 8 in base 2 below a sum of n: an exponent of at most 20
    is off by 2^-21 (half a step) one way or the other, and an exponential by
    2^-23; over the row's many places these average to a tenth of that at
    most, as do the additions (a few units of 2^-24 each). A row's logarithm in
    float32 (a sum of 2^11 to 2^19) would be off by up to 2^-20 one way. Far
    scores, of -184 in base 2, are rounded in one pass and not in the other, by
    2^-17 at most: over 160 rows x 1000 places, 2^-17 / 400.
    """
    from crowdllama_amd.ops import kv
    _, pool, table = make(74, [n], 8, 2, 64, 64, types, strange=False)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(rows, 8, 64, generator=g)
    if far:                         # scores far below 0: with a maximum
        q[..., 0], pool[:, :, 0, :, 0] = -64., 16.
    mass = torch.zeros(1, 2, table.shape[1] * 64, device="cuda")
    kv.observe(q.to(types[0]).cuda(), pool.cuda(), table.cuda(), ints([n]),
               mass, starts=ints([0, rows]))
    given = mass.double().sum(-1).cpu() / (rows * 4)
    assert ((given - 1).abs() <= 2.0 ** -23).all(), given - 1


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("past", [0, 1, 5, 29, 30, 31, 1000, 2 ** 31 - 200])
def test_observe_past_the_last_place(types, past):
    """Tokens past the last place were not stored; the rows before them see
    what they would see in a longer cache."""
    from crowdllama_amd.ops import kv
    cap, rows = 128, [30, 30, 4]
    lens = [cap + past, 70, min(cap + 3, cap + past)]
    _, pool, table = make(75, [cap, 70, cap], 4, 2, 64, 16, types,
                          strange=False)
    table = table[:, :cap // 16].contiguous()
    q = torch.randn(64, 4, 64, generator=torch.Generator().manual_seed(2))
    q = q.to(types[0])
    starts = [0, 30, 60, 64]
    mass = torch.zeros(3, 2, cap, device="cuda")
    kv.observe(q.cuda(), pool.cuda(), table.cuda(), ints(lens), mass,
               starts=ints(starts))
    want = torch.zeros(3, 2, cap, dtype=torch.float64)
    for b, n in enumerate(lens):
        k, _, there = oracle.keys_values(pool, table, b, min(n, cap))
        seen = torch.arange(min(n, cap))[None] <= \
            (n - rows[b] + torch.arange(rows[b]))[:, None]
        for h in range(2):
            x = q[starts[b]:starts[b + 1], 2 * h:2 * h + 2].double()
            w, _ = oracle.weights(x.transpose(0, 1), k[h], there, 64 ** -.5,
                                  seen)
            want[b, h, :min(n, cap)] = w.sum((0, 1))
    # 68 x 4 half steps of scores below 16, 30 rows: below 2^-10
    assert torch.allclose(mass.double().cpu(), want, rtol=2.0 ** -10,
                          atol=1e-6)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("in_place", [False, True])
def test_append_leaves_rows_behind_the_last_sequence(types, in_place):
    """As they are, infinities, NaN and signs of zeros among them."""
    from crowdllama_amd.ops import kv
    lens = [3, 8]
    _, pool, table = make(76, lens, 4, 2, 64, 16, types, 4, strange=False)
    x = torch.randn(9, 8, 64, generator=torch.Generator().manual_seed(1))
    x = x.to(types[0])
    x[5, :, ::2], x[5, :, 1::4] = math.inf, -1.
    x[6] = math.nan
    x[7, :, ::3], x[7, :, 1::3] = -0., -2.
    x[8, :, 1::2] = -math.inf
    dx, dp = x.cuda(), pool.cuda()
    inv = torch.rand(32, device="cuda")
    got = kv.append(dx[:, 4:6], dx[:, 6:], dp, table.cuda(), ints(lens),
                    ints([1, 2]), q=dx[:, :4], inv_freq=inv,
                    starts=ints([0, 2, 5]),
                    q_out=dx[:, :4] if in_place else None)
    bits = torch.int32 if types[0] is torch.float32 else torch.int16
    assert torch.equal(got[5:].cpu().contiguous().view(bits),
                       x[5:, :4].contiguous().view(bits))
    assert not got[:5].isnan().any()
