"""GPU: the operators over a paged cache and the logit adjustments against plain 64-bit forms."""
import itertools

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


def ci():
    import comp_inference_b200
    return comp_inference_b200


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape):
    return torch.randn(*shape, generator=g)


def make_cache(g, pages, page, n_kv, d, bits, fill=True):
    """A pool as earlier steps left it (keys with channels that stand out)."""
    cache = ci().PagedKVCache(pages, page, n_kv, d, bits, DEV)
    if fill:
        far = 4.0 * (torch.rand(d, generator=g) < 0.05)
        for rows, scale, shift in ((cache.k, cache.k_scale, far), (cache.v, cache.v_scale, 0 * far)):
            x = (rnd(g, pages, n_kv, page, d) + shift).to(torch.bfloat16)
            if bits == 16:
                rows.copy_(x)
            else:
                code, sc = ref.quantise(x)
                packed = torch.zeros(pages, n_kv, page, d // 2, dtype=torch.int64)
                for c, (byte, shift_) in enumerate(ref.nibbles(d)):
                    packed[..., byte] |= code[..., c] << shift_
                rows.copy_(packed.to(torch.uint8))
                scale.copy_(sc)
    return cache


def make_table(g, kv_lens, page, pages, spare=1):
    need = [-(-n // page) for n in kv_lens]
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(kv_lens), max(need + [0]) + spare), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
    return table


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts_of(lens):
    return i32([0] + list(itertools.accumulate(lens)))


def rope_tables(T, d):
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    a = torch.outer(torch.arange(T, dtype=torch.float64), inv)
    a = torch.cat((a, a), 1)
    return a.cos().to(torch.bfloat16).to(DEV), a.sin().to(torch.bfloat16).to(DEV)


def rotate(x, cos, sin):
    """bf16 [.., d] rotated, float32 with one rounding per sum (the products are exact)."""
    h = x.shape[-1] // 2
    x = x.float()
    return (x * cos.float() + torch.cat((-x[..., h:], x[..., :h]), -1) * sin.float()).to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------- append and gather

APPEND = [  # d, n_q, n_kv, page, new tokens, tokens
    (128, 4, 2, 16, None, [1, 17, 16, 40]),
    (64, 3, 3, 32, None, [5]),
    (256, 2, 1, 64, [3, 0, 70, 1], [3, 9, 130, 64]),
    (128, 8, 8, 128, [129, 1, 5], [129, 300, 5]),
    (64, 14, 2, 16, [33], [50]),
    (128, 5, 1, 16, [1] * 40, list(range(1, 41))),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,n_q,n_kv,page,new,kv", APPEND)
def test_append_writes_its_places_and_no_other(d, n_q, n_kv, page, new, kv, bits):
    g = gen(d + page)
    pages = sum(-(-n // page) for n in kv) + 2
    cache = make_cache(g, pages, page, n_kv, d, bits)
    table = make_table(g, kv, page, pages)
    T = sum(new) if new else len(kv)
    qkv = rnd(g, T, (n_q + 2 * n_kv) * d).to(torch.bfloat16).to(DEV)
    q, k, v = qkv[:, :n_q * d], qkv[:, n_q * d:(n_q + n_kv) * d], qkv[:, (n_q + n_kv) * d:]
    cos, sin = rope_tables(max(kv), d)
    starts = starts_of(new) if new else None
    want = [t.clone() if t is not None else None for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    got = ci().rope_paged_append(q, k, v, cos, sin, cache, table.to(DEV), i32(kv), starts)
    want_q = torch.empty(T, n_q, d, dtype=torch.bfloat16, device=DEV)
    at = ref.nibbles(d)
    for t, b, pos in ref.tokens(kv, starts, T):
        want_q[t] = rotate(q[t].view(n_q, d), cos[pos], sin[pos])
        i = ref.page(cache, table, b, pos)
        kr = rotate(k[t].view(n_kv, d), cos[pos], sin[pos])
        for j, x in ((0, kr), (1, v[t].view(n_kv, d))):
            if bits == 16:
                want[j][i, :, pos % page] = x
            else:
                code, scale = ref.quantise(x)
                want[2 + j][i, :, pos % page] = scale
                row = torch.zeros(n_kv, d // 2, dtype=torch.int64, device=DEV)
                for c, (byte, shift) in enumerate(at):
                    row[:, byte] |= code[:, c] << shift
                want[j][i, :, pos % page] = row.to(torch.uint8)
    assert torch.equal(got, want_q)
    for have, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        assert (have is None and w is None) or torch.equal(have, w)
    # and back: every token of every sequence
    total = sum(kv)
    gk, gv = ci().paged_gather(cache, table.to(DEV), i32(kv), starts_of(kv), total)
    row = 0
    for b, n in enumerate(kv):
        wk, wv, _ = ref.sequence(cache, table, b, n)
        assert torch.equal(gk[row:row + n], wk.to(torch.bfloat16)) and torch.equal(gv[row:row + n], wv.to(torch.bfloat16))
        row += n


@pytest.mark.parametrize("bits", [16, 4])
def test_append_of_tokens_without_a_place(bits):
    g = gen(5)
    d, page, n_kv = 128, 16, 2
    cache = make_cache(g, 6, page, n_kv, d, bits)
    before = [t.clone() for t in (cache.k, cache.v)]
    # sequence 0: an unmapped page; 1: an id past the pool; 2: no tokens at all (padding of a fixed batch); 3: past the
    # table's row; 4: past the rotation tables; 5: a place
    table = i32([[0, -1], [1, 6], [2, 3], [4, 5], [0, 1], [2, 3]])
    kv = i32([17, 32, 0, 33, 21, 20])
    q, k, v = (rnd(g, 6, h * d).to(torch.bfloat16).to(DEV) for h in (4, n_kv, n_kv))
    cos, sin = rope_tables(33, d)
    got = ci().rope_paged_append(q, k, v, cos, sin, cache, table, kv)
    assert torch.equal(got[2], torch.zeros_like(got[2]))
    for t, pos in ((0, 16), (1, 31), (3, 32), (4, 20), (5, 19)):
        assert torch.equal(got[t], rotate(q[t].view(4, d), cos[pos], sin[pos]))
    changed = [(a != b).flatten(3).any(3) for a, b in zip((cache.k, cache.v), before)]
    for c in changed:
        where = c.any(1).nonzero().tolist()
        assert where == [[1, 4], [3, 3]]                # page and place of sequences 4 and 5
    short = ci().rope_paged_append(q, k, v, cos[:20], sin[:20], cache, table, kv)
    assert torch.equal(short[4], torch.zeros_like(short[4])) and torch.equal(short[5], got[5])


def test_rows_behind_the_last_sequence_are_left_alone():
    g = gen(6)
    d, page = 64, 16
    cache = make_cache(g, 4, page, 1, d, 16)
    table, kv, starts = i32([[0, 1], [2, 3]]), i32([20, 7]), i32([0, 4, 6])
    q, k, v = (rnd(g, 9, h * d).to(torch.bfloat16).to(DEV) for h in (2, 1, 1))
    cos, sin = rope_tables(32, d)
    out = torch.full((9, 2, d), 7.0, dtype=torch.bfloat16, device=DEV)
    ci().rope_paged_append(q, k, v, cos, sin, cache, table, kv, starts, out=out)
    assert bool((out[6:] == 7).all()) and not bool((out[:6] == 7).any())
    o = torch.full((9, 2 * d), 7.0, dtype=torch.bfloat16, device=DEV)
    ci().paged_attention(out, cache, table, kv, starts, out=o)
    assert bool((o[6:] == 7).all()) and not bool((o[:6] == 7).any())


def test_append_of_what_is_not_finite_into_4_bits():
    d = 128
    cache = ci().PagedKVCache(1, 16, 1, d, 4, DEV)
    v = torch.zeros(4, d, dtype=torch.bfloat16, device=DEV)
    v[:, 64:] = 3.0                                     # the second group: one value, a step of zero
    v[1, 5], v[2, 6], v[3, 7] = float("nan"), float("inf"), 2.5
    k = v.clone()
    cos, sin = torch.ones(16, d, dtype=torch.bfloat16, device=DEV), torch.zeros(16, d, dtype=torch.bfloat16, device=DEV)
    ci().rope_paged_append(k, k, v, cos, sin, cache, i32([[0]]), i32([4]), i32([0, 4]))
    gk, gv = ci().paged_gather(cache, i32([[0]]), i32([4]), i32([0, 4]), 4)
    for x in (gk, gv):
        x = x[:, 0]
        assert torch.equal(x[[0, 3]], v[[0, 3]])
        assert bool(x[1:3, :64].isnan().all())
    assert torch.equal(gv[:, 0, 64:], v[:, 64:])
    assert bool(gk[1:3, 0, 64:].isnan().all())          # the rotation's 0 times NaN, 0 times infinity


# ---------------------------------------------------------------------------------------------- attention

def check_attention(q, cache, table, kv, new=None, window=0, sinks=0, scale=None, **more):
    starts = starts_of(new) if new else None
    got = ci().paged_attention(q, cache, table.to(DEV), i32(kv), starts, window=window, sinks=sinks, scale=scale, **more)
    want, bound = ref.attention(q.view(q.shape[0], -1, cache.head_dim), cache, table, kv, starts, window, sinks, scale)
    err = (got.double().view_as(want) - want).abs()
    assert bool((err <= bound).all()), (float((err - bound).max()), float(err.max()))
    return got


STEPS = [  # d, group, n_kv, page, tokens of each sequence, window, sinks
    (128, 1, 2, 64, [1, 2, 63, 64, 65, 300], 0, 0),
    (128, 4, 2, 16, [700, 1, 33], 0, 0),
    (128, 8, 1, 128, [1500], 0, 0),
    (64, 7, 3, 32, [129, 0, 128, 5], 0, 0),
    (64, 1, 5, 16, [40], 0, 0),
    (256, 2, 2, 64, [257, 31], 0, 0),
    (256, 5, 1, 16, [100, 1], 0, 0),
    (128, 16, 1, 32, [333, 64], 0, 0),                  # two groups of eight rows
    (64, 20, 1, 64, [90], 0, 0),                        # a group of rows that is not full
    (256, 12, 1, 32, [70, 3], 0, 0),
    (128, 4, 2, 64, [1000, 30, 257], 100, 0),
    (128, 4, 2, 64, [1000, 30, 257], 100, 4),
    (64, 2, 2, 16, [500, 499, 64], 1, 1),
    (64, 2, 2, 16, [500, 499, 64], 64, 200),            # the first tokens reach into the window
    (256, 1, 1, 128, [400], 129, 130),
    (128, 1, 1, 16, [400, 2], 5000, 3),                 # a window longer than the sequence
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,group,n_kv,page,kv,window,sinks", STEPS)
def test_decode_step(d, group, n_kv, page, kv, window, sinks, bits):
    g = gen(d + group + len(kv))
    pages = sum(-(-n // page) for n in kv) + 1
    cache, table = make_cache(g, pages, page, n_kv, d, bits), make_table(g, kv, page, pages)
    q = (2 * rnd(g, len(kv), group * n_kv, d)).to(torch.bfloat16).to(DEV)
    check_attention(q, cache, table, kv, window=window, sinks=sinks)


MANY = [  # d, group, n_kv, page, new tokens, tokens, window, sinks
    (128, 2, 2, 64, [3, 1, 8], [100, 1, 8], 0, 0),
    (128, 4, 1, 16, [2, 0, 5, 1], [300, 7, 5, 65], 0, 0),
    (64, 1, 2, 32, [17, 40], [17, 200], 0, 0),
    (64, 3, 1, 64, [50], [150], 30, 5),
    (256, 1, 1, 16, [20, 3], [33, 3], 0, 0),
    (128, 7, 1, 128, [37, 1], [37, 400], 10, 2),
    (128, 1, 1, 16, [200], [200], 0, 0),                # a whole prompt
    (128, 4, 1, 64, [130, 65], [400, 65], 0, 0),        # parts of prompts
    (128, 4, 1, 32, [150], [700], 128, 4),
    (64, 8, 1, 16, [70, 1, 33], [70, 300, 90], 0, 0),
    (256, 2, 1, 64, [140], [300], 0, 0),
    (64, 1, 1, 128, [300], [300], 1, 0),
    (128, 6, 1, 64, [100], [130], 40, 3),               # heads that do not divide the rows of a tile
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,group,n_kv,page,new,kv,window,sinks", MANY)
def test_several_new_tokens(d, group, n_kv, page, new, kv, window, sinks, bits):
    g = gen(sum(new) + d)
    pages = sum(-(-n // page) for n in kv) + 1
    cache, table = make_cache(g, pages, page, n_kv, d, bits), make_table(g, kv, page, pages)
    q = (2 * rnd(g, sum(new), group * n_kv, d)).to(torch.bfloat16).to(DEV)
    a = check_attention(q, cache, table, kv, new, window=window, sinks=sinks)
    b = check_attention(q, cache, table, kv, new, window=window, sinks=sinks, max_q_len=max(new))
    assert a.shape == b.shape == (sum(new), group * n_kv * d)


LONG = [  # few new tokens of a long sequence, whose keys are shared among the multiprocessors
    (128, 4, 2, 64, [40, 3, 70], [5000, 900, 70], 0, 0),
    (64, 1, 3, 128, [130], [4100], 0, 0),
    (256, 8, 1, 32, [17, 9, 90], [3000, 20, 100], 0, 0),
    (128, 5, 1, 16, [30] * 40, [30 + 61 * i for i in range(40)], 0, 0),
    (64, 2, 1, 64, [150], [9000], 6000, 300),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,group,n_kv,page,new,kv,window,sinks", LONG)
def test_new_tokens_of_long_sequences(d, group, n_kv, page, new, kv, window, sinks, bits):
    g = gen(sum(kv) + d)
    pages = sum(-(-n // page) for n in kv) + 1
    cache, table = make_cache(g, pages, page, n_kv, d, bits), make_table(g, kv, page, pages)
    q = (2 * rnd(g, sum(new), group * n_kv, d)).to(torch.bfloat16).to(DEV)
    a = check_attention(q, cache, table, kv, new, window=window, sinks=sinks)
    b = ci().paged_attention(q, cache, table.to(DEV), i32(kv), starts_of(new), max_q_len=max(new), window=window, sinks=sinks)
    assert torch.equal(a, b)                            # the same sums every time


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("said", [1, 20, 10 ** 6])
def test_a_max_q_len_that_is_not_true(said, bits):
    g = gen(said)
    kv, new = [200, 90, 7], [150, 65, 0]
    cache, table = make_cache(g, 20, 16, 1, 64, bits), make_table(g, kv, 16, 20)
    q = rnd(g, 215, 2, 64).to(torch.bfloat16).to(DEV)
    check_attention(q, cache, table, kv, new, max_q_len=said)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [[130, 40], [2, 9]])
def test_first_tokens_that_fill_tiles(new, bits):
    """More first tokens than window, the window a few tokens, sequences that end in the first tokens."""
    g = gen(41)
    kv = [1500, 60]
    cache, table = make_cache(g, 60, 32, 2, 128, bits), make_table(g, kv, 32, 60)
    q = rnd(g, sum(new), 4, 128).to(torch.bfloat16).to(DEV)
    for window, sinks in ((3, 700), (1, 128), (200, 129), (1400, 1000)):
        check_attention(q, cache, table, kv, new, window=window, sinks=sinks)


@pytest.mark.parametrize("bits", [16, 4])
def test_more_sequences_than_threads_and_uneven_lengths(bits):
    g = gen(9)
    kv = [(37 * i) % 90 for i in range(300)] + [2000]
    pages = sum(-(-n // 16) for n in kv)
    cache, table = make_cache(g, pages, 16, 1, 64, bits), make_table(g, kv, 16, pages)
    q = rnd(g, len(kv), 2, 64).to(torch.bfloat16).to(DEV)
    a = check_attention(q, cache, table, kv)
    assert torch.equal(a, ci().paged_attention(q, cache, table.to(DEV), i32(kv)))       # the same sums every time
    assert bool((a[0] == 0).all())                      # no tokens, nothing seen


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [None, [5, 3], [200, 150]])
def test_what_nobody_sees_reaches_nobody(new, bits):
    """Infinities and NaN behind the end of a sequence, on pages that it does not have and outside every window."""
    g = gen(11)
    page, d = 32, 128
    kv = [310, 170]
    cache = make_cache(g, 40, page, 1, d, bits)
    table = make_table(g, kv, page, 40)
    T = sum(new) if new else 2
    q = rnd(g, T, 4, d).to(torch.bfloat16).to(DEV)
    args = dict(window=40, sinks=3)
    a = check_attention(q, cache, table, kv, new, **args)
    b = check_attention(q, cache, table, kv, new)
    used = set(table.flatten().tolist())
    big = [float("nan"), float("inf"), -float("inf")]
    for target, j0 in ((b, None), (a, 3)):
        spoiled = make_cache(gen(0), 40, page, 1, d, bits, fill=False)
        for x, y in zip((spoiled.k, spoiled.v, spoiled.k_scale, spoiled.v_scale), (cache.k, cache.v, cache.k_scale, cache.v_scale)):
            if x is None:
                continue
            x.copy_(y)
            if x.dtype != torch.bfloat16:
                continue
            for i in set(range(40)) - used:
                x[i] = big[i % 3]
            for s, n in enumerate(kv):
                x[table[s, n // page], :, n % page:] = big[s]           # the rest of the last page
                if j0 is not None:
                    first = n - (new[s] if new else 1) - 40
                    for j in range(j0, first):
                        x[table[s, j // page], :, j % page] = big[j % 3]
        got = ci().paged_attention(q, spoiled, table.to(DEV), i32(kv), starts_of(new) if new else None, **(args if j0 else {}))
        assert torch.equal(got, target)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [None, [3, 2], [90, 70]])
def test_positions_without_a_page(new, bits):
    """A hole in the table, an id past the pool, lengths past the table's row, and fewer tokens than new ones."""
    g = gen(13)
    cache = make_cache(g, 12, 16, 2, 64, bits)
    table = torch.tensor([[0, -1, 2, 3, 4, 5], [6, 12, 2 ** 31 - 1, 9, 10, 11]], dtype=torch.int32)
    T = sum(new) if new else 2
    q = rnd(g, T, 4, 64).to(torch.bfloat16).to(DEV)
    check_attention(q, cache, table, [90, 96], new)
    check_attention(q, cache, table, [90, 130], new)    # past the row
    got = check_attention(q, cache, table, [1, 0], new)
    if new:
        assert bool((got[:new[0] - 1] == 0).all())      # positions below zero
    check_attention(q, cache, torch.full_like(table, -1), [90, 96], new)
    check_attention(q, cache, table, [30, 20], new, window=5)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [None, [150]])
def test_values_far_from_1(new, bits):
    """Keys, queries and values of 1e-6 and of 1e6, and values that grow along the sequence by 2^40."""
    g = gen(19)
    kv, d = [400], 128
    T = new[0] if new else 1
    table = make_table(g, kv, 32, 14)
    for kq, kk, kv_ in ((1e-6, 1e6, 1.0), (1e3, 1e-3, 1e6), (1.0, 1.0, 1e-6), (1.0, 1.0, None)):
        cache = ci().PagedKVCache(14, 32, 1, d, bits, DEV)
        pos = torch.arange(kv[0], dtype=torch.float64)
        grow = (2.0 ** (pos / 10.0 - 20.0))[:, None] if kv_ is None else kv_
        k, v = (kk * rnd(g, kv[0], d)).to(torch.bfloat16).to(DEV), (grow * rnd(g, kv[0], d)).to(torch.bfloat16).to(DEV)
        one, none = torch.ones(400, d, dtype=torch.bfloat16, device=DEV), torch.zeros(400, d, dtype=torch.bfloat16, device=DEV)
        ci().rope_paged_append(k, k, v, one, none, cache, table.to(DEV), i32(kv), i32([0, 400]))
        q = (kq * rnd(g, T, 4, d)).to(torch.bfloat16).to(DEV)
        check_attention(q, cache, table, kv, new)


def test_strides_scale_and_out():
    g = gen(15)
    kv, d = [100, 37, 5], 128
    cache, table = make_cache(g, 12, 16, 2, d, 16), make_table(g, kv, 16, 12)
    wide = rnd(g, 3, 9 * d).to(torch.bfloat16).to(DEV)
    q = wide[:, d:5 * d]                                # a column slice
    a = check_attention(q, cache, table, kv, scale=0.2)
    odd = rnd(g, 3 * 4 * d + 1).to(torch.bfloat16).to(DEV)[1:].view(3, 4, d)
    check_attention(odd, cache, table, kv)              # rows that are not 16-byte aligned
    turned = rnd(g, 4, 3, d).to(torch.bfloat16).to(DEV).transpose(0, 1)
    check_attention(turned, cache, table, kv, scale=-0.1)
    assert bool((check_attention(q, cache, table, kv, scale=0.0) == check_attention(-q, cache, table, kv, scale=0.0)).all())
    room = torch.full((3, 6 * d), 3.0, dtype=torch.bfloat16, device=DEV)
    out = room[:, d:5 * d]
    assert ci().paged_attention(q, cache, table.to(DEV), i32(kv), scale=0.2, out=out) is not None
    assert torch.equal(out, a) and bool((room[:, :d] == 3).all()) and bool((room[:, 5 * d:] == 3).all())
    part = torch.zeros(3, 40, dtype=torch.int32, device=DEV)
    part[:, 7:7 + table.shape[1]] = table.to(DEV)       # a slice of a wider table
    assert torch.equal(ci().paged_attention(q, cache, part[:, 7:7 + table.shape[1]], i32(kv), scale=0.2), a)


def test_offsets_past_32_bits():
    """Pages whose first byte, and whose first element, lies past 2^32."""
    d, page, n_kv = 256, 128, 8
    pages = (1 << 32) // (page * n_kv * d) + 4
    c = ci()
    cache = c.PagedKVCache.from_tensors(*(torch.empty(pages, n_kv, page, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)))
    g = gen(17)
    for x in (cache.k, cache.v):
        x[-3:] = rnd(g, 3, n_kv, page, d).to(torch.bfloat16).to(DEV)
        x[:3] = 0.0
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32)
    q, k, v = (rnd(g, 1, h * d).to(torch.bfloat16).to(DEV) for h in (n_kv, n_kv, n_kv))
    cos, sin = rope_tables(300, d)
    qr = c.rope_paged_append(q, k, v, cos, sin, cache, table.to(DEV), i32([300]))
    assert torch.equal(cache.v[pages - 2, :, 299 - 256], v.view(n_kv, d))
    check_attention(qr, cache, table, [300])
    new = rnd(g, 150, n_kv, d).to(torch.bfloat16).to(DEV)
    check_attention(new, cache, table, [300], [150])
    assert bool((cache.k[:3] == 0).all())


@pytest.mark.parametrize("bits", [16, 4])
def test_a_captured_step_goes_by_the_lengths_of_its_replay(bits):
    """Append and attention captured once, replayed as the sequences grow, two graphs at once on two streams."""
    c = ci()
    d, page, n_q, n_kv, B = 128, 16, 4, 2, 3
    cos, sin = rope_tables(64, d)
    sets = []
    for seed in (1, 2):
        g = gen(seed)
        s = dict(cache=make_cache(g, 12, page, n_kv, d, bits), table=make_table(g, [64] * B, page, 12).to(DEV),
                 kv=i32([5, 16, 31]), q=rnd(g, B, n_q * d).to(torch.bfloat16).to(DEV),
                 k=rnd(g, B, n_kv * d).to(torch.bfloat16).to(DEV), v=rnd(g, B, n_kv * d).to(torch.bfloat16).to(DEV))
        sets.append(s)

    def step(s):
        s["kv"].add_(1)
        q = c.rope_paged_append(s["q"], s["k"], s["v"], cos, sin, s["cache"], s["table"], s["kv"])
        return c.paged_attention(q, s["cache"], s["table"], s["kv"])

    eager = []
    for s in sets:
        keep = {n: (s[n].clone() if n == "kv" else None) for n in s}
        pages = [x.clone() if x is not None else None for x in (s["cache"].k, s["cache"].v, s["cache"].k_scale, s["cache"].v_scale)]
        eager.append([step(s).clone() for _ in range(6)])
        s["kv"].copy_(keep["kv"])
        for x, y in zip((s["cache"].k, s["cache"].v, s["cache"].k_scale, s["cache"].v_scale), pages):
            if x is not None:
                x.copy_(y)
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(s)
        graphs.append((graph, stream, out))
    for i in range(6):
        for graph, stream, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), want in zip(graphs, eager):
            assert torch.equal(out, want[i])


def test_calls_on_another_stream():
    g = gen(21)
    kv, d = [500, 80], 64
    cache, table = make_cache(g, 40, 16, 1, d, 16), make_table(g, kv, 16, 40)
    q = rnd(g, 2, 4, d).to(torch.bfloat16).to(DEV)
    want = check_attention(q, cache, table, kv)
    streams = [torch.cuda.Stream() for _ in range(2)]
    t, n = table.to(DEV), i32(kv)
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ci().paged_attention(q, cache, t, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ---------------------------------------------------------------------------------------------- logits

def bf16_close(got, want):
    """One rounding to bf16 (half a step, 2^-8) of a float32 result (a few roundings of 2^-24 of what was added up)."""
    want = want.to(got.device)
    same = torch.isinf(want) & (got.double() == want)
    err = (got.double() - want).abs()
    return bool((same | (err <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * (want.abs() + 40))).all())


LOGITS = [(1, 1000, 5, 0, False), (3, 4097, 40, 7, True), (2, 8192, 0, 3, True), (5, 32, 100, 1, False), (2, 31, 9, 2, True),
          (1, 1, 3, 1, True), (4, 12000, 3000, 300, True), (2, 16400, 50, 1100, False),
          (3, 2051, 10, 40, True), (2, 100003, 700, 512, True), (64, 20011, 30, 5, True)]


@pytest.mark.parametrize("B,V,L,n_bias,masked", LOGITS)
def test_adjust_logits(B, V, L, n_bias, masked):
    g = gen(V + L)
    logits = (4 * rnd(g, B, V)).to(torch.bfloat16)
    tok = torch.randint(-2, V + 2, (B, L), generator=g)
    tok = torch.where(torch.rand(B, L, generator=g) < 0.6, tok % max(1, min(V, 7)), tok)        # the same tokens again and again
    lens = torch.tensor([max(0, L - 3 * b) for b in range(B)], dtype=torch.int32)
    prompt = torch.tensor([L // (b + 2) for b in range(B)], dtype=torch.int32)
    r, f, p = 0.7 + torch.rand(B, generator=g), torch.rand(B, generator=g), torch.rand(B, generator=g) - 0.5
    ids = torch.randint(-1, V + 1, (B, n_bias), generator=g)
    if n_bias > 2:
        ids[:, 1] = ids[:, 2] = ids[:, 0]               # the same token more than once
    bias = 3 * rnd(g, B, n_bias)
    mask = torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=g).to(torch.int32) if masked else None
    dev = [None if x is None else x.to(DEV) for x in (logits, tok, lens, prompt, r, p, f, ids, bias, mask)]
    got = ci().adjust_logits(*dev[:8], dev[8], dev[9])
    want = ref.adjust(logits, tok, lens, prompt, r, p, f, ids, bias, mask)
    assert bf16_close(got, want)
    assert torch.equal(got, ci().adjust_logits(*dev[:8], dev[8], dev[9]))
    inplace = dev[0].clone()
    assert ci().adjust_logits(inplace, *dev[1:], out=inplace) is not None and torch.equal(inplace, got)
    for only in ({"tokens": 1, "lens": 2, "repetition": 4}, {"tokens": 1, "lens": 2, "prompt_lens": 3, "frequency": 6},
                 {"bias_ids": 7, "bias": 8}, {"mask": 9}, {}):
        host = [logits, tok, lens, prompt, r, p, f, ids, bias, mask]
        kw = {n: i for n, i in only.items() if host[i] is not None}
        a = ci().adjust_logits(dev[0], **{n: dev[i] for n, i in kw.items()})
        names = {"tokens": "tok"}
        assert bf16_close(a, ref.adjust(logits, **{names.get(n, n): host[i] for n, i in kw.items()}))


@pytest.mark.parametrize("shift", range(8))
def test_adjust_logits_wherever_rows_start(shift):
    """Rows that start on every even address of a 16-byte word, the output on another."""
    g = gen(shift)
    V, ld = 2100 + shift, 2200 + 3 * shift
    room = torch.full((3 * ld + 16,), 9.0, dtype=torch.bfloat16, device=DEV)
    x = room[shift:shift + 3 * ld].view(3, ld)[:, :V]
    x.copy_((4 * rnd(g, 3, V)).to(torch.bfloat16))
    tok = torch.randint(0, V, (3, 20), generator=g)
    tok[:, :4] = torch.tensor([0, V - 1, -1, V])
    lens, mask = torch.full((3,), 20, dtype=torch.int32), torch.randint(-2 ** 31, 2 ** 31, (3, -(-V // 32)), generator=g).to(torch.int32)
    f = torch.rand(3, generator=g)
    want = ref.adjust(x.cpu(), tok, lens, frequency=f, mask=mask)
    args = dict(tokens=tok.to(DEV), lens=lens.to(DEV), frequency=f.to(DEV), mask=mask.to(DEV))
    assert bf16_close(ci().adjust_logits(x, **args), want)
    other = torch.full((3 * (V + 5) + 16,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = other[3:3 + 3 * (V + 5)].view(3, V + 5)[:, 2:2 + V]
    assert bf16_close(ci().adjust_logits(x, out=out, **args), want)
    ci().adjust_logits(x, out=x, **args)
    assert bf16_close(x, want)
    assert bool((room[:shift] == 9).all()) and bool((room[shift:shift + 3 * ld].view(3, ld)[:, V:] == 9).all())
    assert bool((other[3:3 + 3 * (V + 5)].view(3, V + 5)[:, :2] == 7).all()) and bool((other[3:3 + 3 * (V + 5)].view(3, V + 5)[:, 2 + V:] == 7).all())


def test_adjust_logits_of_strided_rows_and_extremes():
    V = 64
    wide = torch.zeros(2, 3 * V, dtype=torch.bfloat16, device=DEV)
    x = wide[:, 3:3 + V]
    x[0, 0], x[0, 1], x[0, 2], x[0, 3] = float("nan"), float("inf"), -float("inf"), -3.3895e38
    mask = torch.full((2, 2), -1, dtype=torch.int32, device=DEV)
    mask[1] = 0                                         # nothing is allowed
    mask[0, 0] = -2                                     # token 0, the NaN, is not
    got = ci().adjust_logits(x, mask=mask)
    assert torch.equal(got[0, 1:], x[0, 1:]) and bool((got[1] == -float("inf")).all()) and float(got[0, 0]) == -float("inf")
    out = torch.full((2, 3 * V), 5.0, dtype=torch.bfloat16, device=DEV)
    ci().adjust_logits(x, mask=mask, out=out[:, 5:5 + V])
    assert torch.equal(out[:, 5:5 + V], got) and bool((out[:, :5] == 5).all()) and bool((out[:, 5 + V:] == 5).all())
    hist = torch.arange(10, device=DEV).view(1, 10).repeat(2, 3)[:, 5:25]
    one = torch.ones(2, device=DEV)
    a = ci().adjust_logits(x, hist, i32([20, 20]), presence=one)
    assert float(a[0, 2]) == -float("inf") and float(a[1, 4]) == -1.0 and float(a[1, 20]) == 0.0
    assert ci().adjust_logits(x, hist, i32([2 ** 31 - 1, -5]), presence=one)[1].eq(0).all()     # lengths outside the row


# ---------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("bits", [16, 4])
def test_a_run_of_them(bits):
    """Prompts of three lengths, then steps that grow past their pages: append, attention, adjusted logits, the token picked."""
    c, g = ci(), gen(31)
    B, d, n_q, n_kv, page, V = 3, 64, 4, 2, 16, 512
    new = [37, 130, 5]
    E = (0.7 * rnd(g, V, (n_q + 2 * n_kv) * d)).to(torch.bfloat16).to(DEV)
    W = (0.2 * rnd(g, n_q * d, V)).to(torch.bfloat16).to(DEV)
    cos, sin = rope_tables(200, d)
    cache = make_cache(g, 20, page, n_kv, d, bits)
    table = make_table(g, [n + 20 for n in new], page, 20)
    history = torch.zeros(B, 200, dtype=torch.int64, device=DEV)
    for b, n in enumerate(new):
        history[b, :n] = torch.randint(0, V, (n,), generator=g).to(DEV)
    kv = torch.tensor(new, dtype=torch.int32, device=DEV)
    prompt_lens = kv.clone()
    r, p = torch.full((B,), 1.3, device=DEV), torch.full((B,), 0.2, device=DEV)
    mask = torch.randint(-2 ** 31, 2 ** 31, (B, V // 32), generator=g).to(torch.int32).to(DEV)
    tok, pos, done = torch.zeros(B, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    picked, ticket = torch.zeros(B, 10, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    starts = starts_of(new)
    ids = torch.cat([history[b, :n] for b, n in enumerate(new)])
    for step in range(5):
        x = E[ids]
        q, k, v = x[:, :n_q * d], x[:, n_q * d:(n_q + n_kv) * d], x[:, (n_q + n_kv) * d:]
        q = c.rope_paged_append(q, k, v, cos, sin, cache, table.to(DEV), kv, starts)
        o = c.paged_attention(q, cache, table.to(DEV), kv, starts, max_q_len=max(new) if step == 0 else 1)
        want, bound = ref.attention(q, cache, table, kv.tolist(), starts)
        assert bool(((o.double().view_as(want) - want).abs() <= bound).all())
        last = o if step else o[(starts[1:] - 1).long()]
        logits = last @ W
        got = c.adjust_logits(logits, history, kv, prompt_lens, repetition=r, presence=p, mask=mask)
        assert bf16_close(got, ref.adjust(logits.cpu(), history.cpu(), kv.cpu(), prompt_lens.cpu(), r.cpu(), p.cpu(), mask=mask.cpu()))
        c.ops.greedy_step(got, tok, pos, done, picked, ticket)
        assert torch.equal(tok, got.float().argmax(1)) and torch.equal(picked[:, step + 1], tok)
        history[torch.arange(B), kv.long()] = tok
        kv += 1
        starts, ids = None, tok.clone()
    gk, _ = c.paged_gather(cache, table.to(DEV), kv - 1, starts_of((kv - 1).tolist()), int((kv - 1).sum()))
    assert gk.shape == (int((kv - 1).sum()), n_kv, d)


def test_outputs_that_overlap_inputs():
    c, g = ci(), gen(33)
    d, T = 64, 4
    cache = make_cache(g, 4, 16, 1, d, 16)
    table, kv = i32([[0], [1], [2], [3]]), i32([3, 1, 9, 16])
    cos, sin = rope_tables(16, d)
    qkv = rnd(g, T, 4 * d).to(torch.bfloat16).to(DEV)
    q, k, v = qkv[:, :2 * d], qkv[:, 2 * d:3 * d], qkv[:, 3 * d:]
    own = q.contiguous()
    want = c.rope_paged_append(q, k, v, cos, sin, cache, table, kv)
    assert torch.equal(c.rope_paged_append(own, k, v, cos, sin, cache, table, kv, out=own).view_as(want), want)      # all of q
    flat = torch.zeros(3 * T * d, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        c.rope_paged_append(flat[:2 * T * d].view(T, 2 * d), k, v, cos, sin, cache, table, kv, out=flat[d:d + 2 * T * d].view(T, 2 * d))
    with pytest.raises(ValueError, match="overlaps"):
        c.rope_paged_append(qkv.view(2 * T, 2 * d)[:T], k, v, cos, sin, cache, table, kv, out=qkv.view(2 * T, 2 * d)[:T])
    want = c.paged_attention(q, cache, table, kv)
    assert torch.equal(c.paged_attention(q, cache, table, kv, out=qkv[:, 2 * d:]), want)        # other columns of the same rows
    with pytest.raises(ValueError, match="overlaps"):
        c.paged_attention(q, cache, table, kv, out=q)
    with pytest.raises(ValueError, match="overlaps"):
        c.paged_attention(q, cache, table, kv, out=qkv[:, d:3 * d])
    x = rnd(g, 3, 100).to(torch.bfloat16).to(DEV)
    with pytest.raises(ValueError, match="overlaps"):
        c.adjust_logits(x[:2], out=x[1:])


def test_a_tensor_on_the_wrong_device():
    c, g = ci(), gen(35)
    cache = make_cache(g, 4, 16, 1, 64, 16)
    q, table, kv = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV), i32([[0], [1]]), i32([3, 1])
    for args in ((q.cpu(), cache, table, kv), (q, cache, table.cpu(), kv), (q, cache, table, kv.cpu())):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            c.paged_attention(*args)
    host = c.PagedKVCache(4, 16, 1, 64, device="cpu")
    with pytest.raises(RuntimeError):
        c.paged_attention(q, host, table, kv)


@pytest.mark.parametrize("bits", [16, 4])
def test_prompts_in_a_graph_beside_eager_ones(bits):
    """A captured call of prompts and steps, replayed with other lengths on its stream while another stream makes the same calls."""
    c, g = ci(), gen(37)
    B, d, n_q, n_kv, page = 4, 128, 4, 1, 32
    cache, table = make_cache(g, 80, page, n_kv, d, bits), make_table(g, [600] * B, page, 80)
    q = rnd(g, 400, n_q, d).to(torch.bfloat16).to(DEV)
    t, kv, starts = table.to(DEV), i32([500, 40, 300, 100]), starts_of([150, 1, 90, 100])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph, o = torch.cuda.CUDAGraph(), torch.full((400, n_q * d), 7.0, dtype=torch.bfloat16, device=DEV)
    c.paged_attention(q, cache, t, kv, starts, out=o)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        c.paged_attention(q, cache, t, kv, starts, out=o)
    for lens, new in (([500, 40, 300, 100], [150, 1, 90, 100]), ([600, 2, 1, 17], [280, 2, 1, 17]), ([0, 0, 0, 590], [0, 0, 0, 399])):
        kv.copy_(i32(lens))
        starts.copy_(starts_of(new))
        o.fill_(7.0)
        torch.cuda.synchronize()
        eager = [c.paged_attention(q, cache, t, kv, starts, out=torch.full_like(o, 7.0)) for _ in range(3)]
        with torch.cuda.stream(side):
            graph.replay()
        eager += [c.paged_attention(q, cache, t, kv, starts, out=torch.full_like(o, 7.0)) for _ in range(3)]
        torch.cuda.synchronize()
        want, bound = ref.attention(q, cache, table, lens, starts)
        n = sum(new)
        assert bool(((o[:n].double().view_as(want[:n]) - want[:n]).abs() <= bound[:n]).all()) and bool((o[n:] == 7).all())
        assert all(torch.equal(e, o) for e in eager)
    assert _status() is None


def _status():
    return ci().check_status()
