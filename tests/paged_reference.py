"""Plain 64-bit forms of the paged-cache operators and of the logit adjustments, for the tests: page by page and token by
token, on any device."""
import math

import torch


def nibbles(d):
    """(byte, shift) of every channel's code in a row of d / 2 bytes."""
    G = d // 64
    out = []
    for c in range(d):
        group, inside = divmod(c, 64)
        bit = 32 * (inside // 8 * G + group) + 4 * (inside % 8 // 2) + 16 * (inside % 2)
        out.append(divmod(bit, 8))
    return out


def codes_of(rows):
    """uint8 [..., d / 2] -> int64 codes [..., d]."""
    at = nibbles(rows.shape[-1] * 2)
    return torch.stack([rows[..., byte].long() >> shift & 15 for byte, shift in at], -1)


def values(codes, scale):
    """float64 values of rows of codes with their (step, lowest)."""
    c = codes_of(codes).double().unflatten(-1, (-1, 64))
    return (scale[..., 1:].double() + scale[..., :1].double() * c).flatten(-2)


def quantise(x):
    """What 4 bits make of bf16 rows [..., d]: (codes [..., d] int64, scale [..., d / 64, 2] bf16), in the float32 arithmetic that the
    definition names."""
    g = x.float().unflatten(-1, (-1, 64))
    low = g.amin(-1, keepdim=True)
    step = ((g.amax(-1, keepdim=True) - low) / 15).to(torch.bfloat16).float()
    code = torch.where(step > 0, torch.round((g - low) / step), torch.zeros_like(g)).clamp(0, 15)
    return code.flatten(-2).long(), torch.cat((step, low), -1).to(torch.bfloat16)


def tokens(kv_lens, q_starts, T):
    """(row, sequence, position) of every new token."""
    kv = [int(n) for n in kv_lens]
    if q_starts is None:
        return [(b, b, n - 1) for b, n in enumerate(kv)]
    s = [int(n) for n in q_starts]
    return [(t, b, kv[b] - (s[b + 1] - s[b]) + t - s[b]) for b in range(len(kv)) for t in range(s[b], s[b + 1]) if t < T]


def page(cache, table, b, pos):
    """Page of a position or None."""
    if pos < 0 or pos >= table.shape[1] * cache.page_size:
        return None
    i = int(table[b, pos // cache.page_size])
    return i if 0 <= i < cache.num_pages else None


def sequence(cache, table, b, n):
    """(keys, values, there) of positions 0 .. n - 1: float64 [n, n_kv, d] and which of them have a page."""
    P = cache.page_size
    there = torch.tensor([page(cache, table, b, j) is not None for j in range(n)], dtype=torch.bool, device=cache.k.device)
    out = []
    for rows, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = torch.zeros(n, cache.n_kv, cache.head_dim, dtype=torch.float64, device=rows.device)
        for j in range(0, n, P):
            i = page(cache, table, b, j)
            if i is None:
                continue
            m = min(P, n - j)
            y = rows[i, :, :m].double() if cache.bits == 16 else values(rows[i, :, :m], scale[i, :, :m])
            x[j:j + m] = y.transpose(0, 1)
        out.append(x)
    return out[0], out[1], there


def attention(q, cache, table, kv_lens, q_starts=None, window=0, sinks=0, scale=None, few=64):
    """(result, bound) float64 [T, n_q, d]: the result, and how far one that rounds each weight (4 bits: times its step) and
    the result to bf16 may be from it.  Half a step of bf16 is 2^-8 relative: 2^-8 (sum of p |v| + |o|); for 4 bits
    |v - middle| in the place of |v|, the middle of a group being code 8, where the few new tokens' kernel rounds the weights'
    products with steps alone; the prompts' kernel (more than `few` query rows of a sequence and key head) has weights, values
    and keys of 4 bits in fp16, half a step 2^-11: 2 |v| for the first two and the change of p by the third, whose scores are
    off by 2^-11 scale sum |q k|; a sixty-fourth more for products of roundings; and for sums in float32
    2^-18 of the sum of p times the largest thing added up, |v| or (4 bits) step * 143 and |lowest|."""
    T, n_q, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(T, n_q, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    per_seq = {}
    for t, b, pos in tokens(kv_lens, q_starts, T):
        if pos < 0:
            continue
        if b not in per_seq:
            per_seq = {b: sequence(cache, table, b, max(0, int(kv_lens[b])))}
            if cache.bits == 4:
                P, ids = cache.page_size, range(0, max(0, int(kv_lens[b])))
                low = torch.zeros_like(per_seq[b][1])
                step = torch.zeros_like(low)
                for j in ids:
                    i = page(cache, table, b, j)
                    if i is not None:
                        low[j] = cache.v_scale[i, :, j % P, :, 1].double().repeat_interleave(64, -1)
                        step[j] = cache.v_scale[i, :, j % P, :, 0].double().repeat_interleave(64, -1)
                extra = (low, step)
        k, v, there = per_seq[b]
        j = torch.arange(k.shape[0], device=q.device)
        seen = (j <= pos) & there
        if window:
            seen &= (pos - j < window) | (j < sinks)
        if not bool(seen.any()):
            continue
        k, v = k[seen], v[seen]
        if cache.bits == 4:
            lowv, stepv = extra[0][seen], extra[1][seen]
        for h in range(n_q):
            g = h // (n_q // cache.n_kv)
            p = torch.softmax(scale * (k[:, g] @ q[t, h].double()), 0)
            out[t, h] = p @ v[:, g]
            if cache.bits == 16:
                a, big = p @ v[:, g].abs(), p @ v[:, g].abs()
            else:
                a, big = p @ (v[:, g] - lowv[:, g] - 8 * stepv[:, g]).abs(), p @ (143 * stepv[:, g] + lowv[:, g].abs())
                if q_starts is not None and (int(q_starts[b + 1]) - int(q_starts[b])) * (n_q // cache.n_kv) > few:
                    ds = scale * (k[:, g].abs() @ q[t, h].double().abs())       # p_j changes by at most (e^(2 max ds) - 1) p_j
                    a = (2 * (p @ v[:, g].abs()) + (p * 2 * ds.max()) @ (v[:, g] - out[t, h]).abs()) / 8
            bound[t, h] = 2.0 ** -8 * (a + out[t, h].abs()) * (1 + 2.0 ** -6) + 2.0 ** -18 * big
    return out, bound


def adjust(logits, tok=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None,
           mask=None):
    """float64 [B, V]."""
    out = logits.double().clone()
    V = out.shape[1]
    for b in range(out.shape[0]):
        x = out[b]
        if tok is not None:
            n = max(0, min(int(lens[b]), tok.shape[1]))
            p = 0 if prompt_lens is None else max(0, min(int(prompt_lens[b]), n))
            history = [int(i) for i in tok[b, :n]]
            for i in set(history):
                if 0 <= i < V and repetition is not None:
                    x[i] = x[i] / float(repetition[b]) if x[i] > 0 else x[i] * float(repetition[b])
            new = [i for i in history[p:] if 0 <= i < V]
            for i in set(new):
                if frequency is not None:
                    x[i] -= float(frequency[b]) * new.count(i)
                if presence is not None:
                    x[i] -= float(presence[b])
        if bias is not None:
            for i, w in zip(bias_ids[b].tolist(), bias[b].tolist()):
                if 0 <= i < V:
                    x[i] += w
        if mask is not None:
            for i in range(V):
                if not int(mask[b, i // 32]) >> i % 32 & 1:
                    x[i] = -math.inf
    return out
