"""GPU: attention over a paged cache under windows with first tokens, at the places where the window leaves the tiles of those."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import DEV, ci, gen, i32, make_cache, make_table, rnd, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,group,new,kv", [(128, 2, [300], [300]), (64, 1, [600], [650]), (64, 8, [100, 90], [190, 150]), (256, 4, [150], [260]),
                                            (128, 5, [200], [2500])])
def test_first_tokens_stay_seen_where_the_window_leaves_them(d, group, new, kv, bits):
    """A prompt's first query tile still has them in its window, the second one not."""
    g = gen(d + group)
    pages = sum(-(-n // 16) for n in kv) + 1
    cache, table = make_cache(g, pages, 16, 1, d, bits), make_table(g, kv, 16, pages)
    q = rnd(g, sum(new), group, d).to(torch.bfloat16).to(DEV)
    for window, sinks in ((20, 3), (100, 1), (64, 130), (37, 300), (150, 40)) + (((2350, 4), (2290, 140)) if kv[0] == 2500 else ()):
        got = ci().paged_attention(q, cache, table.to(DEV), i32(kv), starts_of(new), window=window, sinks=sinks)
        want, bound = ref.attention(q, cache, table, kv, starts_of(new), window, sinks)
        over = (got.double().view_as(want) - want).abs() > bound
        assert not bool(over.any()), (window, sinks, over.flatten(1).any(1).nonzero().flatten().tolist()[:10])


@pytest.mark.parametrize("bits", [16, 4])
def test_a_table_without_pages(bits):
    """No token has a page: attention and gather give zeros, an append rotates and writes nothing."""
    g = gen(bits)
    cache = make_cache(g, 3, 16, 1, 64, bits)
    before = [x.clone() for x in (cache.k, cache.v)]
    table = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    one, none = torch.ones(200, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(200, 64, dtype=torch.bfloat16, device=DEV)
    for new, kv in ((None, [5, 0]), ([100, 3], [150, 3])):
        starts = starts_of(new) if new else None
        T = sum(new) if new else 2
        q, k = rnd(g, T, 2, 64).to(torch.bfloat16).to(DEV), rnd(g, T, 1, 64).to(torch.bfloat16).to(DEV)
        assert bool((ci().paged_attention(q, cache, table, i32(kv), starts) == 0).all())
        rotated = ci().rope_paged_append(q, k, k, one, none, cache, table, i32(kv), starts)
        assert torch.equal(rotated[0], q[0]) and all(torch.equal(x, y) for x, y in zip((cache.k, cache.v), before))
        assert all(bool((x == 0).all()) for x in ci().paged_gather(cache, table, i32(kv), starts, T))
