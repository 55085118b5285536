"""GPU: the operators over a paged cache at extremes: lengths next to the largest, scores that are not finite.

What a query sees decides: a NaN or +infinity among its scores makes its row NaN, a score of -infinity has the weight 0, and a row with
nothing but those is NaN (0 / 0)."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import DEV, ci, gen, i32, make_cache, make_table, rnd, rope_tables, starts_of

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def spoil(cache, table, b, j, value):
    """A value of key j of sequence b (4 bits: its first group, which holds no infinity: a NaN)."""
    i = ref.page(cache, table, b, j)
    if cache.bits == 16:
        cache.k[i, :, j % cache.page_size, 0] = value
    else:
        cache.k_scale[i, :, j % cache.page_size, 0] = value


def compare(q, cache, table, kv, new=None, **args):
    """NaN where the definition gives it and nowhere else, the rest within the bound of its roundings."""
    starts = starts_of(new) if new else None
    got = ci().paged_attention(q, cache, table.to(DEV), i32(kv), starts, **args)
    args.pop("max_q_len", None)
    want, bound = ref.attention(q, cache, table, kv, starts, **args)
    got = got.double().view_as(want)
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), (got.isnan() != nan).nonzero()[:8].tolist()
    assert bool(((got - want).abs() <= bound)[~nan].all())
    return nan


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("group", [1, 3])
def test_lengths_next_to_the_largest(group, bits):
    """Lengths just below 2^31, far past the table's row: the tokens see all of the row, the rows of the sequences beside stay theirs."""
    g = gen(group)
    d, page, new = 64, 16, [70, 90]
    cache = make_cache(g, 12, page, 1, d, bits)
    table = i32([[0, 1, 2, 3, 4, 5], [6, 7, 8, 9, 10, 11]])
    T = 200
    q, k, v = (rnd(g, T, h * d).to(torch.bfloat16).to(DEV) for h in (group, 1, 1))
    cos, sin = rope_tables(96, d)

    def all_of(kv, **args):
        out = torch.full((T, group * d), 7.0, dtype=torch.bfloat16, device=DEV)
        ci().paged_attention(q, cache, table, i32(kv), starts_of(new), out=out, **args)
        return out

    pages = [x.clone() for x in (cache.k, cache.v)]
    for first, second in (({}, {}), (dict(max_q_len=90), dict(window=40, sinks=5))):
        want, windowed = all_of([1000, 90], **first), all_of([100000, 90], **second)
        assert bool((want[160:] == 7).all()) and not bool((want[:160] == 7).any())
        for less in [1, 2, 3, 30, 40, 41, 57, 58, 59, 60, 70, 71, 100, 127, 128, 129, 186, 187]:
            assert torch.equal(all_of([2 ** 31 - less, 90], **first), want), less
            assert torch.equal(all_of([2 ** 31 - less, 90], **second), windowed), less
    qr = torch.full((T, group, d), 7.0, dtype=torch.bfloat16, device=DEV)
    ci().rope_paged_append(q, k, v, cos, sin, cache, table, i32([2 ** 31 - 1, 0]), starts_of(new), out=qr)
    assert bool((qr[:160] == 0).all()) and bool((qr[160:] == 7).all())      # past the rotation tables, and below zero
    assert all(torch.equal(x, y) for x, y in zip((cache.k, cache.v), pages))
    gk, gv = ci().paged_gather(cache, table, i32([2 ** 31 - 1, 0]), starts_of(new), 160)
    assert bool((gk == 0).all()) and bool((gv == 0).all())
    one = ci().paged_attention(q[:2], cache, table, i32([2 ** 31 - 1, 96]))
    assert torch.equal(one, ci().paged_attention(q[:2], cache, table, i32([96, 96])))


STEPS = [  # d, group, n_kv, page, tokens of each sequence: alone (parts of them in many blocks), and in a batch that leaves them whole
    (128, 4, 2, 64, [1, 3, 700, 64]),
    (64, 7, 1, 16, [2, 33, 400, 5]),
    (256, 2, 1, 32, [1, 130, 257, 40]),
    (128, 16, 1, 32, [1, 90, 333, 17]),
    (64, 1, 2, 64, [(7 * i) % 60 + 1 for i in range(900)]),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,group,n_kv,page,kv", STEPS)
def test_steps_with_a_nan(d, group, n_kv, page, kv, bits):
    g = gen(d + group)
    pages = sum(-(-n // page) for n in kv) + 1
    cache, table = make_cache(g, pages, page, n_kv, d, bits), make_table(g, kv, page, pages)
    q = rnd(g, len(kv), group * n_kv, d).to(torch.bfloat16).to(DEV)
    q[0, 0, 3] = NAN                                    # all scores of one head
    spoil(cache, table, 1, kv[1] - 1, NAN)              # one key among several
    spoil(cache, table, len(kv) - 1, 0, NAN)
    nan = compare(q, cache, table, kv)
    assert bool(nan[0, 0].all()) and not bool(nan[0, 1:].any()) and bool(nan[1].all()) and not bool(nan[2].any())


@pytest.mark.parametrize("kv", [[1, 1, 40], [1, 700, 40], [1 + i % 50 for i in range(900)]])
def test_steps_with_infinite_scores(kv):
    g = gen(len(kv))
    d, page = 128, 32
    pages = sum(-(-n // page) for n in kv) + 1
    q = rnd(g, len(kv), 4, d).to(torch.bfloat16).to(DEV)
    q[..., 0] = 1.0
    for b, value, where in ((1, -INF, "all"), (1, INF, "all"), (2, INF, "one"), (2, -INF, "one"), (2, -INF, "first 17"), (1, -INF, "but one"), (2, -INF, "last")):
        cache, table = make_cache(gen(3), pages, page, 2, d, 16), make_table(gen(4), kv, page, pages)
        n = kv[b]
        for j in {"all": range(n), "one": [n // 2], "first 17": range(min(n - 1, 17)), "but one": [j for j in range(n) if j != n // 2],
                  "last": [n - 1] if n > 1 else []}[where]:
            spoil(cache, table, b, j, value)
        nan = compare(q, cache, table, kv)
        other = [i for i in range(len(kv)) if i != b]
        assert not bool(nan[other].any())
        if where == "all" or value == INF:
            assert bool(nan[b].all())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [[3, 2], [12, 1]])
def test_few_new_tokens_with_a_nan(new, bits):
    """The tokens in front of a key do not see it."""
    g = gen(7)
    kv, d = [300, 20], 128
    cache, table = make_cache(g, 30, 16, 1, d, bits), make_table(g, kv, 16, 30)
    q = rnd(g, sum(new), 4, d).to(torch.bfloat16).to(DEV)
    spoil(cache, table, 0, kv[0] - 2, NAN)
    nan = compare(q, cache, table, kv, new)
    assert not bool(nan[:new[0] - 2].any()) and bool(nan[new[0] - 2:new[0]].all()) and not bool(nan[new[0]:].any())
    q[new[0] - 3] = NAN
    nan = compare(q, cache, table, kv, new)
    assert bool(nan[new[0] - 3].all())
    compare(q, cache, table, kv, new, window=1)


PROMPTS = [  # d, group, n_kv, page, new, tokens: in one piece, in several
    (128, 2, 1, 32, [300], [600]),
    (64, 3, 2, 64, [200], [500]),
    (256, 2, 1, 16, [140], [400]),
    (128, 4, 1, 64, [40], [5000]),
]


@pytest.mark.parametrize("d,group,n_kv,page,new,kv", PROMPTS)
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_prompts_with_a_key_that_is_not_finite(d, group, n_kv, page, new, kv, value):
    """At each position modulo 8 of a tile that every row sees all of."""
    g = gen(d)
    pages = sum(-(-n // page) for n in kv) + 1
    cache, table = make_cache(g, pages, page, n_kv, d, 16), make_table(g, kv, page, pages)
    q = rnd(g, sum(new), group * n_kv, d).to(torch.bfloat16).to(DEV)
    q[..., 0] = 1.0
    for j in range(136, 144):
        i = ref.page(cache, table, 0, j)
        keep = cache.k[i, :, j % page, 0].clone()
        spoil(cache, table, 0, j, value)
        got = ci().paged_attention(q, cache, table.to(DEV), i32(kv), starts_of(new))
        if value == -INF:
            if j == 137 or j == 142:
                assert not bool(compare(q, cache, table, kv, new).any())
        else:
            assert bool(got.isnan().all()), (j, int(got.isnan().sum()), got.numel())
        cache.k[i, :, j % page, 0] = keep


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,group,n_kv,page,new,kv", PROMPTS)
def test_prompts_with_a_nan(d, group, n_kv, page, new, kv, bits):
    g = gen(d + 1)
    pages = sum(-(-n // page) for n in kv) + 1
    cache, table = make_cache(g, pages, page, n_kv, d, bits), make_table(g, kv, page, pages)
    q = rnd(g, sum(new), group * n_kv, d).to(torch.bfloat16).to(DEV)
    q[5, 1, 7] = NAN                                    # all scores of one row, whatever its tiles
    nan = compare(q, cache, table, kv, new)
    assert bool(nan[5, 1].all()) and int(nan.sum()) == d
    first = kv[0] - new[0]
    spoil(cache, table, 0, first + 20, NAN)             # a key that the first twenty do not see
    nan = compare(q, cache, table, kv, new)
    assert not bool(nan[:5].any()) and not bool(nan[6:20].any()) and bool(nan[20:].all())
    nan = compare(q, cache, table, kv, new, window=1)   # one token sees nothing else, the others not at all
    assert bool(nan[20].all()) and not bool(nan[21:].any()) and not bool(nan[6:20].any())


@pytest.mark.parametrize("d,group,n_kv,page,new,kv", PROMPTS)
def test_prompts_of_nothing_but_infinite_scores(d, group, n_kv, page, new, kv):
    """-infinity as a whole tile, where others follow, and everywhere."""
    g = gen(d + 2)
    pages = sum(-(-n // page) for n in kv) + 1
    cache, table = make_cache(g, pages, page, n_kv, d, 16), make_table(g, kv, page, pages)
    q = rnd(g, sum(new), group * n_kv, d).to(torch.bfloat16).to(DEV)
    q[..., 0] = 1.0
    for j in range(128):
        spoil(cache, table, 0, j, -INF)
    assert not bool(compare(q, cache, table, kv, new).any())
    for j in range(128, kv[0]):
        spoil(cache, table, 0, j, -INF)
    assert bool(compare(q, cache, table, kv, new).all())
    for j in range(3):
        spoil(cache, table, 0, kv[0] - new[0] - j, 0.5)
    assert not bool(compare(q, cache, table, kv, new).any())


@pytest.mark.parametrize("bits", [16, 4])
def test_rows_behind_a_sequence_do_not_change_the_others(bits):
    """NaN in the queries of padding and of the next sequence, which lie in the same tile of query rows."""
    g = gen(23)
    new, kv, d, group = [100, 30], [130, 400], 128, 6
    cache, table = make_cache(g, 60, 16, 1, d, bits), make_table(g, kv, 16, 60)
    q = rnd(g, 180, group, d).to(torch.bfloat16).to(DEV)
    args = (cache, table.to(DEV), i32(kv), starts_of(new))
    want = ci().paged_attention(q, *args)[:100].clone()
    q[100:] = NAN
    junk = rnd(g, 200, group, d).to(torch.bfloat16).to(DEV)
    for _ in range(3):
        ci().paged_attention(junk.fill_(NAN), cache, table.to(DEV), i32([400, 400]), i32([0, 120, 200]))       # NaN left in shared memory
        assert torch.equal(ci().paged_attention(q, *args)[:100], want)


@pytest.mark.parametrize("bits", [16, 4])
def test_a_row_that_sees_nothing_beside_rows_that_see_a_nan(bits):
    """Its page is not there; the tokens behind it have a page, and a NaN among its values."""
    g = gen(29)
    cache = make_cache(g, 12, 32, 1, 64, bits)
    table = torch.tensor([[-1, -1, -1, 0, 1, 2, 3]], dtype=torch.int32)
    if bits == 16:
        cache.v[0, 0, 3, 5] = NAN
    else:
        cache.v_scale[0, 0, 3, 0] = NAN
    for new, kv in (([224], [224]), ([100], [130])):
        q = rnd(g, sum(new), 2, 64).to(torch.bfloat16).to(DEV)
        got = ci().paged_attention(q, cache, table.to(DEV), i32(kv), starts_of(new))
        blind = 96 - (kv[0] - new[0])
        assert bool((got[:blind] == 0).all())
        assert bool(got[blind + 4:, 5].isnan().all())


@pytest.mark.parametrize("d,group,new,kv,window", [(128, 2, 600, 600, 20), (64, 1, 600, 600, 5), (256, 1, 600, 600, 150), (128, 1, 700, 1000, 64)])
def test_values_that_shrink_under_a_window(d, group, new, kv, window):
    """Values of 4 bits that shrink along the sequence by 2^60 (12.8 binary places in a tile of 128 positions), and in the last case tiles
    of 1e20 and of 1 in turn: rows that see the small ones alone, beside rows that see the large ones."""
    g = gen(d + kv)
    table = make_table(g, [kv], 32, kv // 32 + 2)
    pos = torch.arange(kv, dtype=torch.float64)
    grow = 2.0 ** (30.0 - pos / 10.0) if kv == 600 else torch.where(pos % 256 < 128, 1e20, 1.0)
    one, none = torch.ones(kv, d, dtype=torch.bfloat16, device=DEV), torch.zeros(kv, d, dtype=torch.bfloat16, device=DEV)
    cache = ci().PagedKVCache(kv // 32 + 2, 32, 1, d, 4, DEV)
    k, v = rnd(g, kv, d).to(torch.bfloat16).to(DEV), (grow[:, None] * rnd(g, kv, d)).to(torch.bfloat16).to(DEV)
    ci().rope_paged_append(k, k, v, one, none, cache, table.to(DEV), i32([kv]), i32([0, kv]))
    q = rnd(g, new, group, d).to(torch.bfloat16).to(DEV)
    for sinks in (0, 3):
        compare(q, cache, table, [kv], [new], window=window, sinks=sinks)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [None, [3], [80]])
def test_a_nan_among_values_of_the_smallest_weight(new, bits):
    """A weight that is 0 in 32 bits is not 0: a NaN that a token sees makes its channels NaN, wherever in the tiles it lies."""
    g = gen(31)
    d, kv = 128, [300]
    for j in (5, 130, 290 if new != [80] else 219):
        cache, table = make_cache(g, 10, 32, 1, d, bits), make_table(g, kv, 32, 10)
        i = ref.page(cache, table, 0, j)
        if bits == 16:
            cache.k[i, 0, j % 32] = -2.0
            cache.v[i, 0, j % 32, :64] = NAN
        else:
            cache.k_scale[i, 0, j % 32, :, 0] = 0.0
            cache.k_scale[i, 0, j % 32, :, 1] = -2.0
            cache.v_scale[i, 0, j % 32, 0] = NAN
        q = torch.ones(new[0] if new else 1, 4, d, dtype=torch.bfloat16, device=DEV)
        got = ci().paged_attention(q, cache, table.to(DEV), i32(kv), starts_of(new) if new else None, scale=1.0).view(-1, 4, d)
        assert bool(got[..., :64].isnan().all()) and not bool(got[..., 64:].isnan().any())
