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
