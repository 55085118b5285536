"""GPU: adjust_logits where the result is not finite: masked tokens are -infinity, no other is, and finite logits stay finite."""
import pytest
import torch

import paged_reference as ref
from test_gpu_paged import DEV, ci, gen, rnd

pytestmark = pytest.mark.gpu


def equal(got, want):
    """Infinities where the definition has them, with their sign, and nowhere else; the rest within half a step of bf16 (2^-8) of a
    float32 result (a few roundings of 2^-24 of what was added up, 40 at most)."""
    got, want = got.double().cpu(), want.cpu()
    far = want.isinf()
    assert torch.equal(got.isinf(), far), (got.isinf() != far).nonzero()[:8].tolist()
    assert torch.equal(got[far], want[far])
    return bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * (want.abs() + 40))[~far].all())


@pytest.mark.parametrize("B,V", [(1, 1), (2, 31), (3, 33), (2, 2047), (2, 2048), (3, 2049), (3, 4097), (2, 8192), (1, 32000), (64, 8193), (40, 50257), (2, 131071)])
@pytest.mark.parametrize("kind", ["random", "one bit", "all but one"])
def test_masks(B, V, kind):
    g = gen(B * V)
    logits = (4 * rnd(g, B, V)).to(torch.bfloat16)
    words = -(-V // 32)
    if kind == "random":
        mask = torch.randint(-2 ** 31, 2 ** 31, (B, words), generator=g).to(torch.int32)
    else:
        bits = torch.zeros(B, words * 32, dtype=torch.int64)
        bits[torch.arange(B), torch.randint(0, V, (B,), generator=g)] = 1
        if kind == "all but one":
            bits = 1 - bits
        mask = (bits.view(B, words, 32) << torch.arange(32)).sum(2)
        mask = torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).to(torch.int32)
    allowed = (mask.long()[:, :, None] >> torch.arange(32) & 1).flatten(1)[:, :V].bool()
    want = logits.double().masked_fill(~allowed, -float("inf"))
    got = ci().adjust_logits(logits.to(DEV), mask=mask.to(DEV))
    assert torch.equal(got.double().cpu(), want)
    x = logits.to(DEV)
    ci().adjust_logits(x, mask=mask.to(DEV), out=x)
    assert torch.equal(x, got)


@pytest.mark.parametrize("shift", range(8))
@pytest.mark.parametrize("V", [2100, 16391])
def test_masks_wherever_rows_start(shift, V):
    """Every even address of a 16-byte word, the output on another: masks' words straddle the loads."""
    g = gen(shift + V)
    B, ld = 3, V + 100 + 3 * shift
    room = torch.full((B * ld + 16,), 9.0, dtype=torch.bfloat16, device=DEV)
    x = room[shift:shift + B * ld].view(B, ld)[:, :V + shift]
    x.copy_((4 * rnd(g, B, V + shift)).to(torch.bfloat16))
    V = V + shift
    tok = torch.randint(0, V, (B, 30), generator=g)
    tok[:, :4] = torch.tensor([0, V - 1, -1, V])
    lens, f = torch.full((B,), 30, dtype=torch.int32), torch.rand(B, generator=g)
    ids, bias = torch.randint(0, V, (B, 9), generator=g), 3 * rnd(g, B, 9)
    mask = torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=g).to(torch.int32)
    want = ref.adjust(x.cpu(), tok, lens, frequency=f, bias_ids=ids, bias=bias, mask=mask)
    args = dict(tokens=tok.to(DEV), lens=lens.to(DEV), frequency=f.to(DEV), bias_ids=ids.to(DEV), bias=bias.to(DEV), mask=mask.to(DEV))
    assert equal(ci().adjust_logits(x, **args), want)
    other = torch.full((B * (V + 5) + 16,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = other[3:3 + B * (V + 5)].view(B, V + 5)[:, 2:2 + V]
    ci().adjust_logits(x, out=out, **args)
    assert equal(out, want)


def test_infinite_biases_and_logits():
    """-infinity and +infinity as biases and as logits, a NaN from both; a token that is not allowed is -infinity all the same."""
    x = torch.zeros(1, 100, dtype=torch.bfloat16, device=DEV)
    inf = float("inf")
    x[0, 3], x[0, 4], x[0, 5] = inf, -inf, inf
    ids = torch.tensor([[1, 2, 5, 6, 6, 7]], device=DEV)
    bias = torch.tensor([[inf, -inf, -inf, inf, -inf, inf]], device=DEV)
    mask = torch.full((1, 4), -1, dtype=torch.int32, device=DEV)
    mask[0, 0] = ~(1 << 7)
    got = ci().adjust_logits(x, bias_ids=ids, bias=bias, mask=mask)[0]
    assert float(got[1]) == inf and float(got[2]) == -inf and float(got[3]) == inf and float(got[4]) == -inf
    assert bool(got[5].isnan()) and bool(got[6].isnan()) and float(got[7]) == -inf and bool((got[8:] == 0).all())
