"""What the operators over a paged cache and adjust_logits refuse, before anything reaches a GPU (no GPU here at all: tensors of the
right shapes on the CPU are refused for their device, last)."""
import ctypes as C

import pytest
import torch

import comp_inference_b200 as ci
from comp_inference_b200 import _lib

BF, I32 = torch.bfloat16, torch.int32


def bf(*shape):
    return torch.zeros(*shape, dtype=BF)


def i32(*shape):
    return torch.zeros(*shape, dtype=I32)


def cache(bits=16, d=128, n_kv=2, page=16, pages=4):
    return ci.PagedKVCache(pages, page, n_kv, d, bits, device="cpu")


def test_what_is_right_is_refused_for_its_device_alone():
    c, table, kv = cache(), i32(3, 2), i32(3)
    for call in (lambda: ci.paged_attention(bf(3, 4, 128), c, table, kv),
                 lambda: ci.paged_attention(bf(5, 512), c, table, kv, i32(4), max_q_len=3, window=7, sinks=2, scale=0.1),
                 lambda: ci.rope_paged_append(bf(3, 512), bf(3, 256), bf(3, 2, 128), bf(9, 128), bf(9, 128), c, table, kv),
                 lambda: ci.paged_gather(cache(4), table, kv, i32(4), 6),
                 lambda: ci.adjust_logits(bf(3, 50), torch.zeros(3, 5, dtype=torch.int64), kv, kv, mask=i32(3, 2))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


@pytest.mark.parametrize("args,words", [
    (dict(bits=8), "8 bits"), (dict(d=96), "head dimension 96"), (dict(page=24), "24 tokens"), (dict(pages=0), "a cache of"),
])
def test_caches(args, words):
    with pytest.raises(ValueError, match=words):
        cache(**args)


def test_pages_of_the_caller():
    make = ci.PagedKVCache.from_tensors
    k, codes, scale = bf(4, 2, 16, 128), torch.zeros(4, 2, 16, 64, dtype=torch.uint8), bf(4, 2, 16, 2, 2)
    assert make(k, k.clone()).bits == 16 and make(codes, codes.clone(), scale, scale.clone()).bits == 4
    for bad in ((k, bf(4, 2, 32, 128)), (k[:, :, ::2], k[:, :, ::2]), (codes, codes), (k, k, scale, scale), (codes, codes, scale, None),
                (codes, codes, scale, bf(4, 2, 16, 1, 2)), (bf(4, 2, 128), bf(4, 2, 128)), (bf(4 * 2 * 16 * 128 + 1)[1:].view(4, 2, 16, 128), k)):
        with pytest.raises(ValueError):
            make(*bad)
    for bad in ((k.float(), k.float()), (k, codes), (codes, codes, scale.float(), scale)):
        with pytest.raises(RuntimeError):
            make(*bad)


@pytest.mark.parametrize("change,kind", [
    (dict(q=bf(3, 3, 128)), ValueError), (dict(q=bf(3, 500)), ValueError), (dict(q=bf(3, 4, 64)), ValueError),
    (dict(q=bf(4, 4, 128)), ValueError), (dict(q=bf(3, 4, 128).float()), RuntimeError), (dict(q=bf(512)), ValueError),
    (dict(table=i32(6)), ValueError), (dict(table=i32(3, 2).long()), RuntimeError), (dict(table=i32(2, 3).t()), ValueError),
    (dict(table=i32(1, 2).expand(3, 2)), ValueError), (dict(kv=i32(2)), ValueError), (dict(kv=i32(3).long()), RuntimeError),
    (dict(kv=i32(6)[::2]), ValueError), (dict(starts=i32(3)), ValueError), (dict(starts=i32(4).long()), RuntimeError),
    (dict(window=-1), ValueError), (dict(sinks=-2), ValueError), (dict(max_q_len=-1), ValueError), (dict(out=bf(3, 500)), ValueError),
    (dict(out=bf(512, 3).t()), ValueError), (dict(out=bf(3, 512).float()), RuntimeError), (dict(out=bf(3, 516)[:, :512]), ValueError),
])
def test_attention(change, kind):
    a = dict(q=bf(3, 4, 128), table=i32(3, 2), kv=i32(3), starts=None)
    a.update(change)
    with pytest.raises(kind) as e:
        ci.paged_attention(a.pop("q"), cache(), a.pop("table"), a.pop("kv"), a.pop("starts"), **a)
    assert "CUDA tensor" not in str(e.value)


@pytest.mark.parametrize("change,kind", [
    (dict(k=bf(3, 3, 128)), ValueError), (dict(v=bf(2, 256)), ValueError), (dict(cos=bf(9, 64)), ValueError),
    (dict(sin=bf(8, 128)), ValueError), (dict(cos=bf(9, 256)[:, ::2]), ValueError), (dict(cos=bf(9, 128).float()), RuntimeError),
    (dict(v=bf(3, 256).half()), RuntimeError), (dict(out=bf(3, 4, 64)), ValueError), (dict(out=bf(4, 3, 128).transpose(0, 1)), ValueError),
])
def test_append(change, kind):
    a = dict(q=bf(3, 512), k=bf(3, 256), v=bf(3, 256), cos=bf(9, 128), sin=bf(9, 128), out=None)
    a.update(change)
    with pytest.raises(kind) as e:
        ci.rope_paged_append(a["q"], a["k"], a["v"], a["cos"], a["sin"], cache(), i32(3, 2), i32(3), out=a["out"])
    assert "CUDA tensor" not in str(e.value)


def test_gather():
    for total in (-1, 4):
        with pytest.raises(ValueError):
            ci.paged_gather(cache(), i32(3, 2), i32(3), None, total)


@pytest.mark.parametrize("args,kind", [
    (dict(logits=bf(50)), ValueError), (dict(logits=bf(50, 2).t()), ValueError), (dict(logits=bf(2, 50).float()), RuntimeError),
    (dict(lens=i32(2)), ValueError), (dict(tokens=torch.zeros(2, 5, dtype=torch.int64)), ValueError),
    (dict(tokens=torch.zeros(3, 5, dtype=torch.int64), lens=i32(2)), ValueError), (dict(tokens=i32(2, 5), lens=i32(2)), RuntimeError),
    (dict(tokens=torch.zeros(1, 1, dtype=torch.int64).expand(2, 1 << 20), lens=i32(2)), ValueError),
    (dict(presence=torch.zeros(2)), ValueError), (dict(bias=torch.zeros(2, 3)), ValueError),
    (dict(bias=torch.zeros(2, 3), bias_ids=torch.zeros(2, 4, dtype=torch.int64)), ValueError),
    (dict(mask=i32(2, 1)), ValueError), (dict(mask=i32(3, 2)), ValueError), (dict(mask=torch.zeros(2, 2)), RuntimeError),
    (dict(out=bf(2, 51)), ValueError), (dict(out=bf(2, 50).float()), RuntimeError),
])
def test_logits(args, kind):
    with pytest.raises(kind) as e:
        ci.adjust_logits(**{"logits": bf(2, 50), **args})
    assert "CUDA tensor" not in str(e.value)


# ------------------------------------------------------------------------------ the C entry points: codes, not exceptions

def descriptors(**change):
    c = _lib.PagedCache(k=4096, v=4096, k_scale=4096, v_scale=4096, num_pages=4, page_size=16, n_kv=2, head_dim=128, bits=16)
    b = _lib.PagedBatch(block_table=4096, kv_lens=4096, q_starts=None, B=3, max_pages=2, T=3, table_stride=2)
    for name, value in change.items():
        setattr(c if hasattr(c, name) else b, name, value)
    return c, b


BAD = [dict(k=None), dict(v=4104), dict(bits=8), dict(bits=4, k_scale=None), dict(head_dim=100), dict(page_size=8), dict(num_pages=0),
       dict(n_kv=0), dict(n_kv=65536), dict(num_pages=0x7FFFFFFF, n_kv=65535), dict(block_table=None), dict(kv_lens=None),
       dict(B=(1 << 20) + 1), dict(T=(1 << 30) + 1), dict(max_pages=1 << 27, table_stride=1 << 27), dict(table_stride=1)]


@pytest.mark.parametrize("change", BAD)
def test_c_descriptors(change):
    lib = _lib.load()
    c, b = (C.byref(x) for x in descriptors(**change))
    assert lib.ci_rope_paged_append(c, b, 4096, 512, 4096, 256, 4096, 256, 4, 4096, 4096, 9, 4096, None) != 0
    assert lib.ci_paged_gather(c, b, 4096, 4096, None) != 0
    assert lib.ci_paged_attention(c, b, 4096, 512, 4, 0, 0, 0, 1.0, 4096, 1 << 40, 4096, 512, None) != 0


def test_c_arguments():
    lib = _lib.load()
    c, b = (C.byref(x) for x in descriptors())
    assert lib.ci_paged_attention(c, b, 4096, 512, 3, 0, 0, 0, 1.0, 4096, 1 << 40, 4096, 512, None) != 0        # heads
    assert lib.ci_paged_attention(c, b, 4098, 512, 4, 0, 0, 0, 1.0, 4096, 1 << 40, 4096, 512, None) != 0        # alignment
    assert lib.ci_paged_attention(c, b, 4096, 516, 4, 0, 0, 0, 1.0, 4096, 1 << 40, 4096, 512, None) != 0
    assert lib.ci_paged_attention(c, b, None, 512, 4, 0, 0, 0, 1.0, 4096, 1 << 40, 4096, 512, None) != 0
    assert lib.ci_paged_attention(c, b, 4096, 512, 4, 0, 0, 0, 1.0, None, 1 << 40, 4096, 512, None) != 0        # workspace
    assert lib.ci_rope_paged_append(c, b, 4096, 512, 4096, 256, 4096, 256, 0, 4096, 4096, 9, 4096, None) != 0
    assert lib.ci_rope_paged_append(c, b, 4096, 512, 4096, 256, 4096, 256, 4, 4096, 4096, 9, 4104, None) != 0
    assert lib.ci_paged_gather(c, b, None, 4096, None) != 0
    for call in (lambda c, b: lib.ci_paged_gather(c, b, 4096, 4096, None), lambda c, b: lib.ci_paged_attention(
            c, b, 4096, 512, 4, 0, 0, 0, 1.0, 4096, 1 << 40, 4096, 512, None)):
        assert call(None, b) != 0 and call(c, None) != 0
    good = dict(d_in=4096, d_out=4096, ld_in=50, ld_out=50, B=2, V=50)
    for bad in (dict(d_in=None), dict(V=0), dict(ld_in=49), dict(ld_out=49), dict(B=65536), dict(d_in=4097), dict(d_tokens=4096, L=5),
                dict(d_tokens=4096, d_lens=4096, L=5, ld_tokens=4), dict(d_tokens=4096, d_lens=4096, L=1 << 20, ld_tokens=1 << 20),
                dict(n_bias=3), dict(n_bias=3, d_bias_ids=4096, d_bias=4096, ld_bias=2), dict(d_mask=4096, ld_mask=1)):
        assert lib.ci_adjust_logits(C.byref(_lib.LogitAdjust(**{**good, **bad})), None) != 0
    assert lib.ci_adjust_logits(None, None) != 0
