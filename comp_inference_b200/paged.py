"""Serving over a paged key/value cache: new tokens into it, attention over it, and the logits before a token is picked.

One layer's cache is a pool of pages, [num_pages, n_kv, page_size, row] for keys and for values; the caller's block table
says which pages hold a sequence, so sequences of any lengths share a pool and grow a page at a time.  A call takes the
new tokens of a whole ragged batch, one behind the other:

    block_table  int32 [B, pages]   row b: the pages of sequence b in order; an id outside the pool names no page
    kv_lens      int32 [B]          tokens of each sequence, the new ones among them
    q_starts     int32 [B + 1]      sequence b's new tokens are rows q_starts[b] .. q_starts[b + 1] - 1, its last ones;
                                    None: one new token per sequence (a decode step)

All three live on the GPU and are read when the kernels run: nothing waits for them, and a captured call goes by what they
hold when its graph is replayed.  Rows behind the last sequence are left as they were (undefined in an output that the call
makes itself: a padded batch whose later stages read them passes ``out``).  No counterpart in the reference,
which leaves cache, attention and sampling to Hugging Face's ``generate`` (tests/test_rans_pytorch_runtime.py:89-118).

Calls are queued on the current stream of the cache's device, whichever device is current.  A kernel whose internal wait ran
out leaves a code that ``check_status`` raises.  Argument errors raise ValueError or RuntimeError before anything is queued.

    cache = PagedKVCache(num_pages=4096, page_size=64, n_kv=8, head_dim=128, bits=4)       # one for each layer
    # prompts: T rows, q_starts says whose
    q = rope_paged_append(q, k, v, cos, sin, cache, block_table, kv_lens, q_starts)
    o = paged_attention(q, cache, block_table, kv_lens, q_starts, max_q_len=longest)
    # a decode step: one row per sequence, kv_lens already counts it
    q = rope_paged_append(q, k, v, cos, sin, cache, block_table, kv_lens)
    o = paged_attention(q, cache, block_table, kv_lens)
    logits = adjust_logits(logits, tokens, lens, prompt_lens, repetition=r, mask=allowed)   # before ops.greedy_step
"""
import torch

from . import _lib


class PagedKVCache:
    """Keys and values of one layer.  ``bits=16``: rows of ``head_dim`` bf16 (64, 128 or 256).  ``bits=4``: rows of codes,
    two to a byte, in ``k`` and ``v`` and, for each 64 channels, a step and a lowest value (bf16) in ``k_scale`` and
    ``v_scale`` [num_pages, n_kv, page_size, head_dim / 64, 2]: 72 bytes for a head of 128 instead of 256.  Pages of 16, 32, 64
    or 128 tokens.

    A code c stands for lowest + step * c.  The 32-bit word p of a row of codes belongs to group p % G (G = head_dim / 64)
    and holds channels 8 * (p // G) .. + 7 of it, channel i of those in bits 4 * (i // 2) + 16 * (i % 2)."""

    def __init__(self, num_pages, page_size, n_kv, head_dim, bits=16, device="cuda"):
        if bits not in (16, 4):
            raise ValueError(f"a cache of {bits} bits; 16 or 4")
        shape = (int(num_pages), int(n_kv), int(page_size))
        scale = [None, None]
        if bits == 16:
            pages = [torch.zeros(*shape, head_dim, dtype=torch.bfloat16, device=device) for _ in range(2)]
        else:
            pages = [torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device) for _ in range(2)]
            scale = [torch.zeros(*shape, head_dim // 64, 2, dtype=torch.bfloat16, device=device) for _ in range(2)]
        self._set(*pages, *scale)

    @classmethod
    def from_tensors(cls, k, v, k_scale=None, v_scale=None):
        """A cache over pages that the caller owns (a view of a larger pool, another layer's share)."""
        cache = cls.__new__(cls)
        cache._set(k, v, k_scale, v_scale)
        return cache

    def _set(self, k, v, k_scale, v_scale):
        self._handle = _lib.host().PagedCache(k, v, k_scale, v_scale)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.bits = 4 if k.dtype == torch.uint8 else 16
        self.num_pages, self.n_kv, self.page_size = k.shape[:3]
        self.head_dim = k.shape[3] * (2 if self.bits == 4 else 1)


def rope_paged_append(q, k, v, cos, sin, cache, block_table, kv_lens, q_starts=None, out=None):
    """Rotary embedding of the new tokens' queries and keys (rotate-half convention, bf16 tables [positions, head_dim] as
    ops.rope_kv takes them), and their keys and values into the pages, in one kernel; returns the rotated queries
    [T, n_q, head_dim].  q, k, v: bf16 [T, heads, head_dim] or [T, heads * head_dim], column slices of a fused
    projection included.

    A cache of 4 bits takes of each 64 channels (keys: after rotation and rounding to bf16) lowest = min, step =
    bf16((max - min) / 15) and code = round((x - lowest) / step); a NaN, or a span that is not finite, makes the group NaN.
    ``out``: all of a contiguous q, or a contiguous tensor apart from q, k and v.
    Tokens whose position is negative or past the tables get zero queries and go nowhere; so do keys and values whose
    position has no page.  No two tokens of a call may go to the same place."""
    return cache._handle.append(q, k, v, cos, sin, block_table, kv_lens, q_starts, out)


def paged_gather(cache, block_table, kv_lens, starts=None, total=None):
    """The last starts[b + 1] - starts[b] tokens of every sequence read back from the pages: (keys, values), bf16
    [total, n_kv, head_dim], zeros where there is no page.  ``total``: the rows of the result, starts[-1] (default: one token
    per sequence)."""
    return cache._handle.gather(block_table, kv_lens, starts, len(block_table) if total is None else int(total))


def paged_attention(q, cache, block_table, kv_lens, q_starts=None, max_q_len=0, window=0, sinks=0, scale=None, out=None):
    """softmax(scale * q . K^T) . V of the new tokens over the pages of their sequence, keys of later tokens left out;
    q [T, n_q, head_dim] or [T, n_q * head_dim], n_q a multiple of the cache's heads; returns [T, n_q * head_dim].

    ``window`` > 0: a token at position i sees positions j with i - j < window, and those with j < ``sinks``.  A token that
    sees nothing (no tokens, no pages) gets zeros.  ``max_q_len``: no sequence has more new tokens than that, 0 if it is not
    known; it chooses between kernels, and a longer sequence is served all the same.  ``scale``: a finite number, head_dim ** -0.5 if not given.
    ``out``: rows that do not overlap q, 16-byte aligned (columns of a wider matrix included).

    A NaN or +infinity among a token's scores makes its row NaN, -infinity is a weight of 0, nothing but -infinity NaN (0 / 0).
    Where several new tokens of one sequence stand in one call, an infinity or a NaN in a value that one of them sees may reach the
    others, the earlier ones and, under a window, the later ones too; what lies behind a sequence's end, outside everyone's
    window or on no page reaches nobody.  In a cache of 4 bits the values of 128 neighbouring positions then share a power of two: steps
    below 2^-25 of the largest value among them, or 2^-90 of the largest so far, lose bits."""
    return cache._handle.attention(q, block_table, kv_lens, q_starts, max_q_len, window, sinks, scale, out)


def adjust_logits(logits, tokens=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None,
                  bias_ids=None, bias=None, mask=None, out=None):
    """bf16 logits [B, V] as a sampler adjusts them before it picks, in one kernel, fp32 with one rounding at the end:

        x / repetition[b] where x > 0, x * repetition[b] elsewhere, for tokens of the history tokens[b, :lens[b]]
        - frequency[b] * count - presence[b] * (count > 0), count over its generated part tokens[b, prompt_lens[b]:lens[b]]
        + the sum of bias[b, i] over the i with bias_ids[b, i] == token
        -inf for tokens whose bit (token % 32 of mask[b, token // 32]) is 0

    tokens, bias_ids int64; lens, prompt_lens, mask int32; the rest float32.  What is not given is left out; without
    prompt_lens all of the history counts; ids outside [0, V) are passed over; histories of less than 2^20 tokens.  ``out`` may
    be ``logits``; otherwise it does not overlap them."""
    return _lib.host().adjust_logits(logits, tokens, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias, mask, out)
