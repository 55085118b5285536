"""GPU: the bounded waits between the roles of the prompts' kernel, made to run out: the call ends, its code is reported, nothing is left in
flight, and the next call is right."""
import pytest
import torch

from comp_inference_b200 import _lib
from test_gpu_paged import DEV, ci, gen, i32, make_cache, make_table, rnd, starts_of

pytestmark = pytest.mark.gpu

CODES = {16: (20, 21, 15, 13, 11, 12, 16, 22), 4: (20, 21, 17, 18, 13, 11, 12, 19, 22)}


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_wait_that_runs_out(d, bits):
    """One role after the other gives up at its first wait, the others when theirs are as short as two milliseconds; 220 pieces, so that
    blocks have several."""
    g = gen(d)
    new, kv = [70] * 218 + [300, 130], [70 + i % 90 for i in range(218)] + [900, 150]
    page = 32
    pages = sum(-(-n // page) for n in kv) + 1
    cache, table = make_cache(g, pages, page, 1, d, bits), make_table(g, kv, page, pages).to(DEV)
    q = rnd(g, sum(new), 1, d).to(torch.bfloat16).to(DEV)
    lens, starts = i32(kv), starts_of(new)
    want = ci().paged_attention(q, cache, table, lens, starts, max_q_len=300)
    ci().check_status()
    lib = _lib.load()
    for code in CODES[bits]:
        lib.ci_paged_set_wait_limit(500, code)
        try:
            ci().paged_attention(q, cache, table, lens, starts, max_q_len=300)
            torch.cuda.synchronize()
        finally:
            lib.ci_paged_set_wait_limit(0, 0)
        with pytest.raises(RuntimeError, match=f"status {code}"):
            ci().check_status()
        ci().check_status()                             # cleared
        assert torch.equal(ci().paged_attention(q, cache, table, lens, starts, max_q_len=300), want), code
        ci().check_status()
