"""The operators of a serving step over a paged key/value cache, as a list of measurable cases.

A layer's cache is a pool of pages; row b of a block table names the pages of sequence b in order, kv_lens[b] counts
its tokens, the new ones among them, and the new tokens of all sequences lie one behind the other in q, k and v
(sequence b's are rows q_starts[b] .. q_starts[b + 1] - 1, its last ones; without q_starts there is one per sequence).

    append     rotary embedding of the new tokens, their keys and values written to the pages in bf16 or in 4 bits
               (ops.rope_paged_append); a 4-bit cache is read back with ops.paged_gather
    attention  new tokens against the pages of their sequence: causal, over all of it or over a window of the last
               tokens and a few first ones; bf16 or 4-bit pages (ops.paged_attention)
    logits     repetition, presence and frequency penalties, sparse biases and a bit mask of allowed tokens
               (ops.adjust_logits)

A 4-bit page holds, for each token and head, head_dim codes of 4 bits and for each 64 channels a step and a lowest
value, both bf16; a code c stands for lowest + step * c.  The 32-bit word p of a row of codes belongs to group p % G
(G = head_dim / 64) and holds channels 8 * (p // G) .. + 7 of it, channel i of those in bits 4 * (i // 2) + 16 * (i % 2).

Head counts and widths are those of the repository's benchmark (32 heads of 128) and tests, and generic ones of grouped
heads; sequences run from one token to the tens of thousands.
"""
import math

import torch

own = False

GROUP = 64


def listed():
    def case(name, kind, **more):
        return {"name": name, "kind": kind, **more}

    return [
        # a step of eight sequences into a 4-bit cache, read back: the smallest call, launches count
        case("append4_step_b8", "append", bits=4, B=8, n_q=32, n_kv=32, d=128, page=64, q_lo=1, q_hi=1, kv_lo=1, kv_hi=130),
        # prompts of odd lengths, grouped heads
        case("append_prompts", "append", bits=16, B=5, n_q=32, n_kv=8, d=128, page=64, q_lo=37, q_hi=4001, kv_lo=37, kv_hi=4001),
        # prompts and parts of prompts in one batch into 4 bits
        case("append4_prompts", "append", bits=4, B=9, n_q=32, n_kv=8, d=128, page=32, q_lo=1, q_hi=4096, kv_lo=700, kv_hi=5000),
        # a decode step of one short sequence, as many heads of keys as of queries: latency
        case("step_b1", "attention", bits=16, B=1, n_q=32, n_kv=32, d=128, page=64, q_lo=1, q_hi=1, kv_lo=513, kv_hi=513,
             window=0, sinks=0),
        # a decode step of a batch whose sequences are of very different lengths
        case("step_b32_ragged", "attention", bits=16, B=32, n_q=32, n_kv=8, d=128, page=64, q_lo=1, q_hi=1, kv_lo=1,
             kv_hi=16000, window=0, sinks=0),
        # a step of long chats that keep a window and the first tokens; seven queries a head of keys, small pages
        case("step_window", "attention", bits=16, B=16, n_q=28, n_kv=4, d=64, page=16, q_lo=1, q_hi=1, kv_lo=5000,
             kv_hi=40000, window=4096, sinks=4),
        # the prompts of a small batch
        case("prompts_b4", "attention", bits=16, B=4, n_q=32, n_kv=32, d=128, page=64, q_lo=1, q_hi=4096, kv_lo=1, kv_hi=4096,
             window=0, sinks=0),
        # one long prompt under a window
        case("prompt_window", "attention", bits=16, B=1, n_q=32, n_kv=8, d=128, page=128, q_lo=16001, q_hi=16001,
             kv_lo=16001, kv_hi=16001, window=4096, sinks=4),
        # a decode step of many long sequences, which 4 bits make room for
        case("step4_b32_long", "attention", bits=4, B=32, n_q=32, n_kv=8, d=128, page=64, q_lo=1, q_hi=1, kv_lo=2000,
             kv_hi=32000, window=0, sinks=0),
        # the next parts of long prompts over a 4-bit cache
        case("prompts4_on_cache", "attention", bits=4, B=3, n_q=32, n_kv=8, d=128, page=64, q_lo=400, q_hi=1024, kv_lo=3500,
             kv_hi=8000, window=0, sinks=0),
        # one sequence over the benchmark's vocabulary, penalties alone
        case("logits_b1", "logits", B=1, V=32000, hist_lo=600, hist_hi=600, biases=0, mask=False),
        # a large batch with every kind of adjustment
        case("logits_b64", "logits", B=64, V=131072, hist_lo=1, hist_hi=4096, biases=32, mask=True),
    ]


# What a drawn case may cost at most: under the largest listed ones.
MAX_FLOPS, MAX_BYTES = 6e11, 3e8


def _size(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "logits"])
    if kind == "logits":
        B = _size(rng, 1, 64)
        hi = _size(rng, 1, 4096)
        return {"kind": kind, "B": B, "V": _size(rng, 1000, 131072), "hist_lo": _size(rng, 1, hi), "hist_hi": hi,
                "biases": rng.choice([0, 1, 32, 300]), "mask": rng.random() < 0.6}
    group = rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
    n_kv = rng.choice([h for h in (1, 2, 4, 5, 8, 16, 32) if h * group <= 64])
    case = {"kind": kind, "bits": rng.choice([16, 4]), "B": _size(rng, 1, 64), "n_q": n_kv * group, "n_kv": n_kv,
            "d": rng.choice([64, 128, 128, 256]), "page": rng.choice([16, 32, 64, 128])}
    step = rng.random() < 0.5                           # a decode step, or prompts and parts of prompts
    case["q_hi"] = 1 if step else _size(rng, 2, 4096)
    case["q_lo"] = 1 if step else _size(rng, 1, case["q_hi"])
    case["kv_hi"] = max(case["q_hi"], _size(rng, 1, 40000))
    case["kv_lo"] = _size(rng, 1, case["kv_hi"])
    if kind == "attention":
        windowed = rng.random() < 0.5
        case["window"] = _size(rng, 1, 8192) if windowed else 0
        case["sinks"] = rng.choice([0, 1, 4, 64, 130]) if windowed else 0

    def dear():
        w = work(case)
        return w["flops"] > MAX_FLOPS or max(w["bytes"], _cost(case)) > MAX_BYTES

    while case["B"] > 1 and dear():
        case["B"] = (case["B"] + 1) // 2
    while dear():
        case["kv_hi"] = max(1, case["kv_hi"] * 3 // 4)
        case["q_hi"] = min(case["q_hi"], case["kv_hi"])
        case["q_lo"], case["kv_lo"] = min(case["q_lo"], case["q_hi"]), min(case["kv_lo"], case["kv_hi"])
    return case


def _spread(lo, hi, n, turn):
    """n lengths over the logarithm of [lo, hi], the first of them hi; the same in every run."""
    return [max(lo, min(hi, round(lo * (hi / lo) ** ((1.0 - turn * i) % 1.0 if i else 1.0)))) for i in range(n)]


def _lengths(case):
    """New tokens and all tokens of every sequence."""
    q = _spread(case["q_lo"], case["q_hi"], case["B"], 0.381966)
    kv = _spread(case["kv_lo"], case["kv_hi"], case["B"], 0.618034)
    return q, [max(a, b) for a, b in zip(q, kv)]


def _row_bytes(case):
    """Bytes of one token's key, or value, of one head."""
    d = case["d"]
    return 2 * d if case["bits"] == 16 else d // 2 + 4 * (d // GROUP)


def _cost(case):
    """Bytes of the cache that the sequences fill."""
    return 2 * sum(_lengths(case)[1]) * case["n_kv"] * _row_bytes(case)


# ------------------------------------------------------------------------------------------------ inputs

def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def _pool(case, seed_gen):
    """Pages of keys and values as earlier steps left them (keys have channels that stand out, as rotated keys do),
    a block table over them in scattered order, and the lengths."""
    B, n_kv, d, page, bits = (case[k] for k in ("B", "n_kv", "d", "page", "bits"))
    q_len, kv_len = _lengths(case)
    need = [-(-n // page) for n in kv_len]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=seed_gen, device="cuda").to(torch.int32)
    table = torch.full((B, max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    offset = 3.0 * (torch.rand(n_kv, 1, d, generator=seed_gen, device="cuda") < 0.05) * torch.randn(
        n_kv, 1, d, generator=seed_gen, device="cuda")
    s = {"table": table, "kv_lens": torch.tensor(kv_len, dtype=torch.int32, device="cuda"),
         "q_lens": q_len, "kv_list": kv_len}
    chunk = max(1, (1 << 26) // (n_kv * page * d))
    for name, shift in (("k", offset), ("v", torch.zeros_like(offset))):
        parts = []
        for p in range(0, pages, chunk):
            x = torch.randn(min(chunk, pages - p), n_kv, page, d, generator=seed_gen, device="cuda")
            x = (x + shift).to(torch.bfloat16)
            parts.append(_quantise(x) if bits == 4 else (x,))
        s[name] = torch.cat([x[0] for x in parts])
        s[name + "_scale"] = torch.cat([x[1] for x in parts]) if bits == 4 else None
    return s


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "logits":
        B, V = case["B"], case["V"]
        lens = _spread(case["hist_lo"], case["hist_hi"], B, 0.381966)
        L = max(lens)
        s["logits"] = (4.0 * torch.randn(B, V, generator=gen, device="cuda")).to(torch.bfloat16)
        # text repeats itself: half of a history comes from a few hundred tokens
        few = torch.randint(0, V, (256,), generator=gen, device="cuda")
        hist = torch.randint(0, V, (B, L), generator=gen, device="cuda")
        again = few[torch.randint(0, 256, (B, L), generator=gen, device="cuda")]
        s["tokens"] = torch.where(torch.rand(B, L, generator=gen, device="cuda") < 0.5, again, hist)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["prompt_lens"] = torch.tensor([n // 3 for n in lens], dtype=torch.int32, device="cuda")
        s["repetition"] = 1.0 + 0.3 * torch.rand(B, generator=gen, device="cuda")
        s["presence"] = 0.5 * torch.rand(B, generator=gen, device="cuda")
        s["frequency"] = 0.2 * torch.rand(B, generator=gen, device="cuda")
        n = case["biases"]
        s["bias_ids"] = torch.randint(0, V, (B, n), generator=gen, device="cuda") if n else None
        s["bias"] = 5.0 * torch.randn(B, n, generator=gen, device="cuda") if n else None
        s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32)), generator=gen, device="cuda").to(torch.int32) \
            if case["mask"] else None
        return s
    s.update(_pool(case, gen))
    T, n_q, n_kv, d = sum(s["q_lens"]), case["n_q"], case["n_kv"], case["d"]
    s["q_starts"] = None if case["q_hi"] == 1 else _starts(s["q_lens"])
    qkv = torch.randn(T, (n_q + 2 * n_kv) * d, generator=gen, device="cuda").to(torch.bfloat16)
    if case["kind"] == "attention":
        s["q"] = qkv[:, :n_q * d].contiguous().view(T, n_q, d)
        s["longest"] = max(s["q_lens"])
    else:
        # one projection's output, its columns split into the heads
        s["q"], s["k_new"], s["v_new"] = qkv[:, :n_q * d], qkv[:, n_q * d:(n_q + n_kv) * d], qkv[:, (n_q + n_kv) * d:]
        inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
        angle = torch.outer(torch.arange(max(s["kv_list"]), dtype=torch.float64, device="cuda"), inv)
        angle = torch.cat((angle, angle), 1)
        s["cos"], s["sin"] = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
        s["kv_starts"] = _starts(s["kv_list"])
    if own:
        import comp_inference_b200 as ci
        s["cache"] = ci.PagedKVCache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _words(d):
    """For each channel of a head: the byte of its code in a row and the shift inside the byte."""
    G = d // GROUP
    c = torch.arange(d, device="cuda")
    group, inside = c // GROUP, c % GROUP
    bit = 32 * ((inside // 8) * G + group) + 4 * (inside % 8 // 2) + 16 * (inside % 2)
    return bit // 8, bit % 8


def _quantise(x):
    """bf16 [..., d] -> codes uint8 [..., d / 2], (step, lowest) bf16 [..., d / 64, 2]."""
    d = x.shape[-1]
    g = x.float().unflatten(-1, (d // GROUP, GROUP))
    low = g.amin(-1, keepdim=True)
    step = ((g.amax(-1, keepdim=True) - low) / 15.0).to(torch.bfloat16).float()
    code = torch.where(step > 0, torch.round((g - low) / step), torch.zeros_like(g)).clamp(0, 15).flatten(-2).to(torch.uint8)
    byte, shift = _words(d)
    first = torch.argsort(byte * 8 + shift)             # channels in the order of their nibbles
    return code[..., first[0::2]] | code[..., first[1::2]] << 4, torch.cat((step, low), -1).to(torch.bfloat16)


def _values(codes, scale):
    """What 4-bit rows stand for, float32."""
    d = codes.shape[-1] * 2
    byte, shift = _words(d)
    c = (codes[..., byte] >> shift.to(torch.uint8) & 15).float().unflatten(-1, (d // GROUP, GROUP))
    return (scale[..., 1:].float() + scale[..., :1].float() * c).flatten(-2)


def _slots(s, lengths):
    """Sequence and position of the last lengths[b] tokens of every sequence, in order."""
    seq = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), torch.tensor(lengths, device="cuda"))
    first = torch.tensor([kv - n for kv, n in zip(s["kv_list"], lengths)], device="cuda")
    begin = torch.tensor([0] + lengths, device="cuda").cumsum(0)[:-1]
    pos = torch.arange(seq.numel(), device="cuda") - begin[seq] + first[seq]
    return seq, pos


def _plain_append(s):
    case = s["case"]
    d, page = case["d"], case["page"]
    seq, pos = _slots(s, s["q_lens"])
    cos, sin = s["cos"][pos][:, None].float(), s["sin"][pos][:, None].float()

    def rotate(x):
        x = x.float().unflatten(-1, (-1, d))
        return (x * cos + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1) * sin).to(torch.bfloat16)

    q, k, v = rotate(s["q"]), rotate(s["k_new"]), s["v_new"].unflatten(-1, (-1, d))
    where = (s["table"][seq, pos // page].long(), slice(None), pos % page)
    if case["bits"] == 16:
        s["k"][where], s["v"][where] = k, v
        return [q, s["k"], s["v"]]
    for name, x in (("k", k), ("v", v)):
        s[name][where], s[name + "_scale"][where] = _quantise(x)
    seq, pos = _slots(s, s["kv_list"])
    where = (s["table"][seq, pos // page].long(), slice(None), pos % page)
    return [q] + [_values(s[n][where], s[n + "_scale"][where]).to(torch.bfloat16) for n in ("k", "v")]


def _rows(s, name, pages, at):
    """Keys or values of one sequence at positions `at`, float32 [n_kv, len(at), d]."""
    page = s["case"]["page"]
    where = (pages[at // page].long(), slice(None), at % page)
    x = s[name][where].float() if s["case"]["bits"] == 16 else _values(s[name][where], s[name + "_scale"][where])
    return x.transpose(0, 1)


def _plain_attention(s):
    case = s["case"]
    n_kv, d, window, sinks = case["n_kv"], case["d"], case["window"], case["sinks"]
    out, row = [], 0
    for b, (n, kv) in enumerate(zip(s["q_lens"], s["kv_list"])):
        q = s["q"][row:row + n].float().unflatten(1, (n_kv, -1)).permute(1, 2, 0, 3)       # [n_kv, group, n, d]
        row += n
        o = torch.empty_like(q)
        for i in range(0, n, 1024):                     # queries of a long prompt, some at a time
            pos = torch.arange(kv - n + i, kv - n + min(i + 1024, n), device="cuda")
            lo = max(0, kv - n + i - window + 1) if window else 0
            at = torch.cat((torch.arange(min(sinks, lo), device="cuda"),
                            torch.arange(lo, kv - n + min(i + 1024, n), device="cuda")))
            k, v = _rows(s, "k", s["table"][b], at), _rows(s, "v", s["table"][b], at)
            seen = at[None] <= pos[:, None]
            if window:
                seen &= (pos[:, None] - at[None] < window) | (at[None] < sinks)
            scores = q[:, :, i:i + 1024] @ k.transpose(1, 2)[:, None] * d ** -0.5
            scores.masked_fill_(~seen, -math.inf)
            scores = (scores - scores.amax(-1, keepdim=True)).exp_()
            o[:, :, i:i + 1024] = scores @ v[:, None] / scores.sum(-1, keepdim=True)
        out.append(o.permute(2, 0, 1, 3).flatten(1).to(torch.bfloat16))
    return torch.cat(out)


def _plain_logits(s):
    B, V = s["logits"].shape
    x = s["logits"].float()
    at = torch.arange(s["tokens"].shape[1], device="cuda")[None]
    there, new = at < s["lens"][:, None], at >= s["prompt_lens"][:, None]
    seen = torch.zeros_like(x).scatter_add_(1, s["tokens"], there.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, s["tokens"], (there & new).float())
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"], s["bias"])
    if s["mask"] is not None:
        v = torch.arange(V, device="cuda")
        x = x.masked_fill(s["mask"][:, v // 32] >> (v % 32).to(torch.int32) & 1 == 0, -math.inf)
    return x.to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "logits": _plain_logits}[kind](s)
    import comp_inference_b200 as ci
    if kind == "logits":
        return ci.adjust_logits(s["logits"], s["tokens"], s["lens"], s["prompt_lens"], repetition=s["repetition"],
                                presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"], bias=s["bias"],
                                mask=s["mask"])
    if kind == "attention":
        return ci.paged_attention(s["q"], s["cache"], s["table"], s["kv_lens"], s["q_starts"], max_q_len=s["longest"],
                                  window=s["case"]["window"], sinks=s["case"]["sinks"])
    q = ci.rope_paged_append(s["q"], s["k_new"], s["v_new"], s["cos"], s["sin"], s["cache"], s["table"], s["kv_lens"],
                             s["q_starts"])
    if s["case"]["bits"] == 16:
        return [q, s["cache"].k, s["cache"].v]
    k, v = ci.paged_gather(s["cache"], s["table"], s["kv_lens"], s["kv_starts"], sum(s["kv_list"]))
    return [q, k, v]


# ------------------------------------------------------------------------------------------------ bounds

def work(case):
    """Each input once and each output once; a product and a sum for every channel of a visible pair, twice."""
    if case["kind"] == "logits":
        B, V = case["B"], case["V"]
        hist = sum(_spread(case["hist_lo"], case["hist_hi"], B, 0.381966))
        return {"bytes": 4 * B * V + 8 * hist + 12 * B * case["biases"] + (B * -(-V // 32) * 4 if case["mask"] else 0),
                "flops": 2 * B * V}
    n_q, n_kv, d = case["n_q"], case["n_kv"], case["d"]
    q_len, kv_len = _lengths(case)
    T = sum(q_len)
    if case["kind"] == "append":
        moved = 2 * T * (2 * n_q + 2 * n_kv) * d + 2 * T * n_kv * _row_bytes(case) + 4 * min(T, max(kv_len)) * d
        if case["bits"] == 4:                           # and read back
            moved += 2 * sum(kv_len) * n_kv * (_row_bytes(case) + 2 * d)
        return {"bytes": moved, "flops": 3 * T * (n_q + n_kv) * d}
    window, sinks = case["window"], case["sinks"]
    pairs = rows = 0
    for n, kv in zip(q_len, kv_len):
        first = kv - n
        if not window:
            pairs += n * first + n * (n + 1) // 2
            rows += kv
            continue
        pos = torch.arange(first, kv, dtype=torch.int64)
        begin = (pos - window + 1).clamp(min=0)
        pairs += int((pos + 1 - begin + begin.clamp(max=sinks)).sum())
        lo = max(0, first - window + 1)
        rows += kv - lo + min(lo, sinks)
    return {"bytes": 4 * T * n_q * d + 2 * rows * n_kv * _row_bytes(case) + 4 * (rows // case["page"] + 1), "flops": 4 * pairs * n_q * d}


# ------------------------------------------------------------------------------------------------ definitions in 64 bits

def _exact_rows(s, name, b, n):
    """Keys or values of the first n tokens of sequence b, float64 [n, n_kv, d], page by page."""
    case = s["case"]
    page, d = case["page"], case["d"]
    ids = s["table"][b, :-(-n // page)].tolist()
    if case["bits"] == 16:
        return torch.cat([s[name][i].transpose(0, 1) for i in ids])[:n].double()
    words = torch.cat([s[name][i].transpose(0, 1) for i in ids])[:n].contiguous().view(torch.int32).long()     # [n, n_kv, d / 8]
    scale = torch.cat([s[name + "_scale"][i].transpose(0, 1) for i in ids])[:n].double()
    G = d // GROUP
    out = torch.empty(n, case["n_kv"], d, dtype=torch.float64, device="cuda")
    for p in range(d // 8):
        step, low = scale[:, :, p % G, 0], scale[:, :, p % G, 1]
        for i in range(8):
            code = words[:, :, p] >> (4 * (i // 2) + 16 * (i % 2)) & 15
            out[:, :, p % G * GROUP + p // G * 8 + i] = low + step * code
    return out


def _exact_attention(s):
    case = s["case"]
    n_q, n_kv, d, window, sinks = (case[k] for k in ("n_q", "n_kv", "d", "window", "sinks"))
    out = torch.empty(sum(s["q_lens"]), n_q, d, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, kv) in enumerate(zip(s["q_lens"], s["kv_list"])):
        k, v = _exact_rows(s, "k", b, kv), _exact_rows(s, "v", b, kv)
        j = torch.arange(kv, device="cuda")
        for i0 in range(0, n, 2048):
            i = torch.arange(i0, min(n, i0 + 2048), device="cuda")[:, None] + kv - n
            hidden = j > i
            if window:
                hidden |= (j <= i - window) & (j >= sinks)
            rows = slice(row + i0, row + min(n, i0 + 2048))
            for h in range(n_q):
                g = h // (n_q // n_kv)
                score = s["q"][rows, h].double() @ k[:, g].T / math.sqrt(d)
                out[rows, h] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v[:, g]
        row += n
    return out.flatten(1)


def _exact_quantised(x):
    """float64 [..., d] -> what its 4-bit form stands for."""
    g = x.to(torch.bfloat16).double().unflatten(-1, (-1, GROUP))
    low, high = g.aminmax(dim=-1, keepdim=True)
    step = ((high - low) / 15).to(torch.bfloat16).double()
    return (low + step * ((g - low) / step.where(step > 0, 1.0)).round().clamp(0, 15)).flatten(-2)


def _exact_append(s):
    case = s["case"]
    n_kv, d, page = case["n_kv"], case["d"], case["page"]
    q_out, k_new, v_new, row = [], [], [], 0
    for n, kv in zip(s["q_lens"], s["kv_list"]):
        c, si = (s[t][kv - n:kv, :d // 2].double()[:, None] for t in ("cos", "sin"))
        c2, si2 = (s[t][kv - n:kv, d // 2:].double()[:, None] for t in ("cos", "sin"))
        for src, dst in (("q", q_out), ("k_new", k_new)):
            x = s[src][row:row + n].double().view(n, -1, d)
            a, z = x[..., :d // 2], x[..., d // 2:]
            dst.append(torch.cat((a * c - z * si, z * c2 + a * si2), -1))
        v_new.append(s["v_new"][row:row + n].double().view(n, n_kv, d))
        row += n
    if case["bits"] == 16:
        k, v = s["k"].double(), s["v"].double()
        for b, (n, kv) in enumerate(zip(s["q_lens"], s["kv_list"])):
            ids = s["table"][b].tolist()
            for t in range(n):
                p, at = ids[(kv - n + t) // page], (kv - n + t) % page
                k[p, :, at], v[p, :, at] = k_new[b][t], v_new[b][t]
        return [torch.cat(q_out), k, v]
    k, v = [], []
    for b, (n, kv) in enumerate(zip(s["q_lens"], s["kv_list"])):
        for name, fresh, dst in (("k", k_new[b], k), ("v", v_new[b], v)):
            dst.append(torch.cat((_exact_rows(s, name, b, kv)[:kv - n], _exact_quantised(fresh))))
    return [torch.cat(q_out), torch.cat(k), torch.cat(v)]


def _exact_logits(s):
    out = s["logits"].double()
    for b in range(out.shape[0]):
        n, p = int(s["lens"][b]), int(s["prompt_lens"][b])
        ids, count = torch.unique(s["tokens"][b, :n], return_counts=True)
        x = out[b, ids]
        out[b, ids] = torch.where(x > 0, x / s["repetition"][b].double(), x * s["repetition"][b].double())
        ids, count = torch.unique(s["tokens"][b, p:n], return_counts=True)
        out[b, ids] -= s["frequency"][b].double() * count + s["presence"][b].double()
        if s["bias"] is not None:
            out[b].index_add_(0, s["bias_ids"][b], s["bias"][b].double())
        if s["mask"] is not None:
            bits = (s["mask"][b][:, None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).flatten()
            out[b][bits[:out.shape[1]] == 0] = -math.inf
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[case["kind"]](s)
