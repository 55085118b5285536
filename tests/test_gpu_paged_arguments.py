"""GPU: what a caller may give the operators over a paged cache, where prompts go: scales, strides, outputs, many heads, mixed batches."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import DEV, check_attention, ci, gen, i32, make_cache, make_table, rnd, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,group", [(64, 3), (128, 2), (256, 1)])
def test_scales_of_prompts(d, group, bits):
    """Negative ones, the caller's, and zero: the mean of what a row sees."""
    g = gen(d)
    new, kv = [150, 90], [400, 90]
    cache, table = make_cache(g, 20, 32, 2, d, bits), make_table(g, kv, 32, 20)
    q = rnd(g, sum(new), group * 2, d).to(torch.bfloat16).to(DEV)
    starts = starts_of(new)
    for scale in (-0.1, 0.3, -d ** -0.5, 1e-4, 0.0, 2.0):
        for args in (dict(), dict(window=70, sinks=2)):
            got = ci().paged_attention(q, cache, table.to(DEV), i32(kv), starts, scale=scale, **args)
            # scale q . k = |scale| (-q) . k; the bound holds |scale| times a sum of moduli, so it is asked for with |scale|
            want, bound = ref.attention(-q if scale < 0 else q, cache, table, kv, starts, scale=abs(scale), **args)
            assert bool(((got.double().view_as(want) - want).abs() <= bound).all()), (scale, args)
            other = ci().paged_attention(-q, cache, table.to(DEV), i32(kv), starts, scale=-scale, **args)
            assert torch.equal(got, other), (scale, args)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_strides_and_outputs_of_prompts(d, bits):
    """Queries as columns of a projection, rows that have to be copied, outputs as columns of a wider matrix, rows that overlap."""
    g = gen(d + 1)
    new, kv, n_q = [130, 1, 70], [200, 300, 70], 4
    T = sum(new)
    cache, table = make_cache(g, 40, 16, 2, d, bits), make_table(g, kv, 16, 40)
    wide = rnd(g, T, 9 * d).to(torch.bfloat16).to(DEV)
    a = check_attention(wide[:, d:5 * d], cache, table, kv, new)
    assert torch.equal(a, check_attention(wide[:, d:5 * d].contiguous(), cache, table, kv, new))
    odd = rnd(g, T * n_q * d + 1).to(torch.bfloat16).to(DEV)[1:].view(T, n_q, d)
    check_attention(odd, cache, table, kv, new)
    turned = rnd(g, n_q, T, d).to(torch.bfloat16).to(DEV).transpose(0, 1)
    check_attention(turned, cache, table, kv, new)
    same = rnd(g, 1, n_q, d).to(torch.bfloat16).to(DEV).expand(T, n_q, d)
    check_attention(same, cache, table, kv, new)
    room = torch.full((T, 6 * d), 3.0, dtype=torch.bfloat16, device=DEV)
    out = room[:, d:5 * d]
    ci().paged_attention(wide[:, d:5 * d], cache, table.to(DEV), i32(kv), starts_of(new), out=out)
    assert torch.equal(out, a) and bool((room[:, :d] == 3).all()) and bool((room[:, 5 * d:] == 3).all())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("group", [100, 128, 129, 200])
def test_many_heads_that_share_a_key_head(group, bits):
    """Up to 128 of them are rows of one tile; more go to the kernel of the few, whatever the number of tokens."""
    g = gen(group)
    new, kv, d = [5, 40, 1], [5, 90, 33], 64
    cache, table = make_cache(g, 12, 16, 1, d, bits), make_table(g, kv, 16, 12)
    q = rnd(g, sum(new), group, d).to(torch.bfloat16).to(DEV)
    starts = starts_of(new)
    for args in (dict(), dict(window=20, sinks=2)):
        got = ci().paged_attention(q, cache, table.to(DEV), i32(kv), starts, **args)
        want, bound = ref.attention(q, cache, table, kv, starts, args.get("window", 0), args.get("sinks", 0), few=64 if group <= 128 else 10 ** 9)
        assert bool(((got.double().view_as(want) - want).abs() <= bound).all())


@pytest.mark.parametrize("bits", [16, 4])
def test_prompts_and_steps_of_long_sequences_in_one_batch(bits):
    g = gen(3)
    new, kv, d = [1, 200, 1, 1, 64, 0, 17, 1], [5000, 200, 1, 2300, 900, 40, 17, 130], 128
    pages = sum(-(-n // 64) for n in kv) + 1
    cache, table = make_cache(g, pages, 64, 2, d, bits), make_table(g, kv, 64, pages)
    q = rnd(g, sum(new), 8, d).to(torch.bfloat16).to(DEV)
    a = check_attention(q, cache, table, kv, new, max_q_len=200)
    assert torch.equal(a, check_attention(q, cache, table, kv, new))
    check_attention(q, cache, table, kv, new, window=300, sinks=5)
