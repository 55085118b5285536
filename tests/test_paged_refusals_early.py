"""Refusals of the operators over a paged cache come before anything is queued (no GPU here: what is right is refused for its device)."""
import ctypes as C

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import comp_inference_b200 as ci
from comp_inference_b200 import _lib
from test_paged_refusals import bf, cache, descriptors, i32


class Calls(TorchDispatchMode):
    """What torch is asked to run."""

    def __enter__(self):
        self.names = []
        return super().__enter__()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name())
        return func(*args, **(kwargs or {}))


def turned(*shape):
    """Heads in another order than rows: what a call has to copy."""
    return bf(shape[1], shape[0], *shape[2:]).transpose(0, 1)


def test_the_mode_sees_copies():
    with Calls() as calls:
        turned(3, 4, 128).contiguous()
    assert any("clone" in n or "copy" in n for n in calls.names)


@pytest.mark.parametrize("call", [
    lambda: ci.paged_attention(turned(3, 4, 128), cache(), i32(3, 2), i32(3), window=-1),
    lambda: ci.paged_attention(turned(3, 4, 128), cache(), i32(3, 2), i32(3), out=bf(3, 500)),
    lambda: ci.paged_attention(turned(3, 4, 128), cache(), i32(3, 2), i32(2)),
    lambda: ci.paged_attention(turned(3, 4, 128), cache(), i32(3, 2), i32(3)),
    lambda: ci.rope_paged_append(turned(3, 4, 128), turned(3, 2, 128), turned(3, 3, 128), bf(9, 128), bf(9, 128), cache(), i32(3, 2), i32(3)),
    lambda: ci.rope_paged_append(turned(3, 4, 128), turned(3, 2, 128), turned(3, 2, 128), bf(9, 128), bf(8, 128), cache(), i32(3, 2), i32(3)),
    lambda: ci.rope_paged_append(turned(3, 4, 128), turned(3, 2, 128), turned(3, 2, 128), bf(9, 128), bf(9, 128), cache(), i32(3, 2), i32(3)),
])
def test_nothing_is_copied_for_a_refused_call(call):
    turned(2, 2, 64)
    with Calls() as calls, pytest.raises((ValueError, RuntimeError)):
        call()
    assert not any("clone" in n or "copy" in n or "contiguous" in n for n in calls.names), calls.names


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39, 3e38])
def test_a_scale_that_is_not_finite(scale):
    """3e38 is not in the exponentials' base.  (A NaN made prompts the mean of their values.)"""
    with pytest.raises(ValueError, match="scale"):
        ci.paged_attention(bf(3, 4, 128), cache(), i32(3, 2), i32(3), scale=scale)
    c, b = (C.byref(x) for x in descriptors())
    assert _lib.load().ci_paged_attention(c, b, 4096, 512, 4, 0, 0, 0, scale, 4096, 1 << 40, 4096, 512, None) == -1
    assert b"scale" in _lib.load().ci_last_error()


def test_a_pool_that_the_prompts_kernel_cannot_index():
    """Refused for that, not for what its first kernel met."""
    lib = _lib.load()
    c, b = (C.byref(x) for x in descriptors(num_pages=(1 << 24) + 1, page_size=128, n_kv=1, q_starts=4096, T=500))
    assert lib.ci_paged_attention(c, b, 4096, 512, 4, 0, 0, 0, 1.0, 4096, 1 << 40, 4096, 512, None) == -1
    assert b"2^31" in lib.ci_last_error()


def test_a_table_without_pages_is_no_argument_error():
    """(Its pointer is null; what is refused is its device.)"""
    for call in (lambda: ci.paged_attention(bf(3, 4, 128), cache(), i32(3, 0), i32(3)), lambda: ci.paged_gather(cache(), i32(3, 0), i32(3))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    c, b = (C.byref(x) for x in descriptors(block_table=None, max_pages=0, table_stride=0, T=(1 << 30) + 1))
    assert _lib.load().ci_paged_gather(c, b, 4096, 4096, None) == -1 and b"null" not in _lib.load().ci_last_error()
