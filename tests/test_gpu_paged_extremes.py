"""GPU: the operators over a paged cache with extreme lengths."""
import pytest
import torch

from test_gpu_paged import DEV, ci, gen, i32, make_cache, rnd, rope_tables, starts_of

pytestmark = pytest.mark.gpu


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
