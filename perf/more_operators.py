"""The operators of a server's step around the paged cache, as timed cases.

A case is one call, or a run of calls that belong together, that a host
serving several sequences makes for one layer, or at the end of a step:

  append     the step's queries and keys rotated by their positions, keys and
             values written into one layer's cache, and the rows of the pages
             that changed read back through their slots; a cache of 8 bits
             (a scale for each page and head) or of 4
  attention  a step's queries over a layer's cache of 4 bits: single tokens or
             prompt rows, with capped scores, distance biases, windows or
             bidirectional prefixes
  logprobs   of a step's logits: the log probabilities of given tokens, the
             entropy of each row and its most likely tokens

Pages hold `block` tokens of every KV head. In 4 bits a value is code * sub *
scale: codes -8 .. 7, a signed 8-bit sub for each token and 32 dims, a bfloat16
scale for each token and head. Codes (plus 8) lie eight to a 32-bit word, elements
0, 2, 4, 6, 1, 3, 5, 7 from the lowest nibble up, along the dims of a key and along the
tokens of a value's dim. Of 32 dims, the value of largest magnitude is -8 steps
(of two equal ones the negative); a step is sub * scale; the scale is the largest
step over 127, rounded up to bfloat16, a sub the step over the scale, rounded up.

Request lengths are spread by their logarithm and depend on the case alone.
"""
import math
import random

import torch

own = False

# heads, KV heads and head_dim of layers (listed by the model class they are of)
HEADS_05B = {"heads": 14, "kv_heads": 2, "head_dim": 64}
HEADS_8B = {"heads": 32, "kv_heads": 8, "head_dim": 128}
HEADS_32B = {"heads": 40, "kv_heads": 8, "head_dim": 128}
PLAIN = {"cap": 0.0, "window": 0, "slopes": False, "prefix": False}
BASE = 500000.0  # of the rotation's frequencies


def listed():
    return [
        # the new token of every sequence of a small server, 8-bit cache: latency of two launches
        {"name": "append8_step_64_8b", "kind": "append", "bits": 8, **HEADS_8B, "requests": 64, "block": 32, "max_len": 8192,
         "max_add": 1, "rot": 128, "neighbours": True},
        # prompt chunks, the longest of odd length behind a cached context
        {"name": "append8_prompts_32b", "kind": "append", "bits": 8, **HEADS_32B, "requests": 5, "block": 64, "max_len": 500,
         "max_add": 2047, "rot": 128, "neighbours": False},
        # the same two into a cache of 4 bits
        {"name": "append4_step_64_8b", "kind": "append", "bits": 4, **HEADS_8B, "requests": 64, "block": 32, "max_len": 8192,
         "max_add": 1, "rot": 128, "neighbours": True},
        {"name": "append4_prompts_32b", "kind": "append", "bits": 4, **HEADS_32B, "requests": 5, "block": 64, "max_len": 500,
         "max_add": 2047, "rot": 128, "neighbours": False},
        # a single user early in a conversation: latency
        {"name": "step_1_600_8b", "kind": "attention", **HEADS_8B, **PLAIN, "requests": 1, "block": 32, "max_len": 600,
         "max_add": 1},
        # a decode step of a batch with ragged lengths
        {"name": "step_64_8192_8b", "kind": "attention", **HEADS_8B, **PLAIN, "requests": 64, "block": 16,
         "max_len": 8191, "max_add": 1},
        # one very long context
        {"name": "step_1_131072_8b", "kind": "attention", **HEADS_8B, **PLAIN, "requests": 1, "block": 64,
         "max_len": 131071, "max_add": 1},
        # a usual prompt of a small model, of odd length
        {"name": "prompt_1_509_0.5b", "kind": "attention", **HEADS_05B, **PLAIN, "requests": 1, "block": 16,
         "max_len": 0, "max_add": 509},
        # prompts of a 32B model whose heads have distance biases and whose
        # beginnings see each other both ways, the largest case
        {"name": "prompts_3_4096_32b", "kind": "attention", **HEADS_32B, **PLAIN, "slopes": True, "prefix": True,
         "requests": 3, "block": 64, "max_len": 1000, "max_add": 4096},
        # the answer's next token of a single user: latency
        {"name": "logprobs_1_151936", "kind": "logprobs", "rows": 1, "vocab": 151936, "given": 1, "top": 5, "masked": False},
        # a batch whose answers have to follow a grammar: most tokens are masked; an odd vocabulary
        {"name": "logprobs_64_32003", "kind": "logprobs", "rows": 64, "vocab": 32003, "given": 2, "top": 20, "masked": True},
        # the tokens of a prompt, scored
        {"name": "logprobs_500_151936", "kind": "logprobs", "rows": 500, "vocab": 151936, "given": 1, "top": 20,
         "masked": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "append", "attention", "attention", "attention", "attention", "logprobs", "logprobs"])
    if kind == "logprobs":
        vocab = _log_int(rng, 100, 262000)
        return {"kind": kind, "rows": _log_int(rng, 1, min(4000, 76000000 // vocab)), "vocab": vocab,
                "given": rng.randint(1, 4), "top": rng.choice([0, 1, 5, rng.randint(1, 64)]), "masked": rng.random() < 0.4}
    case = {"kind": kind, "block": rng.choice([16, 32, 64, 128]), "kv_heads": rng.choice([1, 2, 4, 8]),
            "head_dim": rng.choice([32, 64, 96, 128, 128, 192, 256])}
    width = case["kv_heads"] * case["head_dim"]
    case["heads"] = case["kv_heads"] * rng.randint(1, 8)
    if kind == "append":
        n = _log_int(rng, 1, 128)
        return {**case, "bits": rng.choice([4, 8]), "requests": n, "max_len": _log_int(rng, 1, 8192),
                "max_add": rng.choice([1, _log_int(rng, 2, (1 << 22) // width // n)]), "neighbours": rng.random() < 0.5,
                "rot": rng.choice([case["head_dim"], case["head_dim"], case["head_dim"] // 2, case["head_dim"] // 2 - 10])}
    case = {**case, "cap": rng.choice([0.0, 0.0, 30.0]), "window": rng.choice([0, 0, _log_int(rng, 16, 8192)]),
            "slopes": rng.random() < 0.3, "prefix": rng.random() < 0.3}
    if rng.random() < 0.6:  # single tokens, or a few drafted ones
        n = _log_int(rng, 1, 64)
        return {**case, "requests": n, "max_len": _log_int(rng, 16, min(131072, (1 << 28) // width // n)),
                "max_add": rng.choice([1, 1, rng.randint(2, 8)])}
    n = _log_int(rng, 1, 8)
    # no more work than the largest listed case
    most = int(math.sqrt(1.2e9 * 128 / n / case["heads"] / max(case["head_dim"], 128)))
    add = _log_int(rng, 9, min(4096, most))
    return {**case, "requests": n, "max_add": add, "max_len": rng.choice([0, _log_int(rng, 1, add)])}


# ---- inputs -----------------------------------------------------------------


def _lengths(case):
    """(cached tokens, new tokens) of each request; the first has the longest."""
    n = case["requests"]
    rng = random.Random("%d %d %d %d" % (n, case["block"], case["max_len"], case["max_add"]))

    def spread(most):
        return [most] + [_log_int(rng, max(1, most // 16), most) if most else 0 for _ in range(n - 1)]

    return spread(case["max_len"]), spread(case["max_add"])


def _blocks(tokens, block):
    return -(-tokens // block)


class State:
    pass


ORDER = [0, 2, 4, 6, 1, 3, 5, 7]  # elements of a word, from the lowest nibble up


def _pack(codes):
    """Codes -8 .. 7 along the last axis to bytes of two."""
    n = (codes + 8).to(torch.uint8).unflatten(-1, (-1, 8))[..., ORDER].unflatten(-1, (4, 2))
    return (n[..., 0] | (n[..., 1] << 4)).flatten(-2)


def _unpack(data):
    """The codes of _pack's bytes, as int8."""
    n = torch.stack([data & 15, data >> 4], -1).flatten(-2).unflatten(-1, (-1, 8))
    back = [ORDER.index(e) for e in range(8)]
    return (n[..., back].to(torch.int8) - 8).flatten(-2)


def _quantize4(x):
    """(codes, subs, scales) of rows [..., head_dim], f32; scales are f32 that bfloat16 holds."""
    g = x.unflatten(-1, (-1, 32))
    top, low = g.amax(-1), g.amin(-1)
    step = torch.where(-low >= top, -low, -top) * 0.125
    most = step.abs().amax(-1)
    scale = torch.where(most < 2.0 ** -103, 0.0, (most.double() / 127).float())
    scale = ((scale.view(torch.int32) + 0xffff) & -0x10000).view(torch.float32)
    size = torch.ceil(step.abs().double() / torch.where(scale > 0, scale, 1.0).double()[..., None]).clamp(1, 127)
    sub = torch.where(step < 0, -size, size)
    x = g.double() / (sub * torch.where(scale > 0, scale, 1.0).double()[..., None])[..., None]
    codes = torch.round(x).clamp(-8, 7).flatten(-2)
    return codes.to(torch.int8), sub.to(torch.int8), scale


def _random_pages(pages, heads, block, dim, gen):
    """Rows [page, head, token, dim] with uneven channels and tokens."""
    x = torch.randn(pages, heads, block, dim, device="cuda", generator=gen)
    x *= torch.exp(0.5 * torch.randn(heads, 1, dim, device="cuda", generator=gen))
    return x * torch.exp(0.3 * torch.randn(pages, heads, block, 1, device="cuda", generator=gen))


def _cache(case, pages, transposed, gen):
    """Codes, subs (none for 8 bits) and scales of random rows."""
    kv, dim, block = case["kv_heads"], case["head_dim"], case["block"]
    step, parts = max(1, (1 << 25) // (kv * dim * block)), []
    for first in range(0, pages, step):
        x = _random_pages(min(step, pages - first), kv, block, dim, gen)
        if case.get("bits") == 8:
            scale = torch.clamp(x.abs().amax((2, 3)) / 127, min=1e-20)
            codes, sub = torch.round(x / scale[..., None, None]).clamp(-127, 127).to(torch.int8), scale
            parts.append(((codes.transpose(2, 3) if transposed else codes).contiguous(), sub, scale))
        else:
            codes, sub, scale = _quantize4(x)
            parts.append((_pack(codes.transpose(2, 3) if transposed else codes).contiguous(),
                          sub.transpose(2, 3).contiguous(), scale.to(torch.bfloat16)))
    return [torch.cat(x) for x in zip(*parts)]


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _prepare_logprobs(s, case, gen):
    rows, vocab = case["rows"], case["vocab"]
    # a few likely tokens over a broad rest, as logits are; rounded, so that some are equal
    x = 2.2 * torch.randn(rows, vocab, device="cuda", generator=gen)
    peaks = torch.randint(vocab, (rows, 12), device="cuda", generator=gen)
    x.scatter_add_(1, peaks, 9 * torch.rand(rows, 12, device="cuda", generator=gen))
    x = torch.round(x * 1024) / 1024
    s.token = torch.randint(vocab, (rows, case["given"]), device="cuda", generator=gen)
    s.token[:, 0] = torch.where(torch.arange(rows, device="cuda") % 3 > 0, peaks[:, 0], s.token[:, 0])
    s.token = s.token.to(torch.int32)
    if case["masked"]:
        # what a grammar allows: from nearly all tokens of a row to a few
        share = torch.exp(-7 * torch.rand(rows, 1, device="cuda", generator=gen))
        allowed = torch.rand(rows, vocab, device="cuda", generator=gen) < share
        allowed.scatter_(1, peaks, True)
        x.masked_fill_(~allowed, -math.inf)
    s.logits = x
    s.logprob = torch.empty(rows, case["given"], device="cuda")
    s.entropy = torch.empty(rows, device="cuda")
    s.top_id = torch.empty(rows, case["top"], device="cuda", dtype=torch.int32)
    s.top_logprob = torch.empty(rows, case["top"], device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = State()
    s.case = case
    if case["kind"] == "logprobs":
        _prepare_logprobs(s, case, gen)
        if own:
            _bind(s)
        return s
    length, add = _lengths(case)
    n, block = case["requests"], case["block"]
    kv, dim, heads = case["kv_heads"], case["head_dim"], case["heads"]
    held = [_blocks(x + a, block) for x, a in zip(length, add)]
    s.n_tok, s.max_blocks = sum(add), max(held) + 2
    s.n_pages = sum(held) + sum(held) // 8 + 4
    order = torch.randperm(s.n_pages, device="cuda", generator=gen).to(torch.int32)
    mine = torch.arange(s.max_blocks, device="cuda")[None, :] < _ints(held)[:, None]
    at = (torch.cumsum(mine.flatten().long(), 0) - 1).reshape(mine.shape)
    s.table = torch.where(mine, order[at.clamp(min=0)], -1).to(torch.int32).contiguous()
    s.kv_len = _ints([x + a for x, a in zip(length, add)])
    s.q_start = _ints([sum(add[:r]) for r in range(n + 1)])
    s.max_q, s.max_kv = max(add), max(x + a for x, a in zip(length, add))
    s.k, s.k_sub, s.k_scale = _cache(case, s.n_pages, False, gen)
    s.v, s.v_sub, s.v_scale = _cache(case, s.n_pages, True, gen)
    s.q = 1.3 * torch.randn(s.n_tok, heads, dim, device="cuda", generator=gen)
    s.out = torch.empty_like(s.q)
    if case["kind"] == "append":
        # the positions to read: of the pages that get new tokens
        first = [x // block * block for x in length]
        at = torch.cat([torch.arange(f, x + a) for f, x, a in zip(first, length, add)]).cuda()
        req = torch.cat([torch.full((x + a - f,), r) for r, (f, x, a) in enumerate(zip(first, length, add))]).cuda()
        s.slot = s.table[req, at // block].long() * block + at % block
        s.pos = torch.cat([torch.arange(x, x + a) for x, a in zip(length, add)]).cuda()
        s.out_k = torch.empty(len(at), kv, dim, device="cuda")
        s.out_v = torch.empty_like(s.out_k)
        # keys whose sizes differ from token to token
        size = torch.exp(0.4 * torch.randn(s.n_tok, kv, 1, device="cuda", generator=gen))
        s.new_k = size * torch.randn(s.n_tok, kv, dim, device="cuda", generator=gen)
        s.new_v = torch.randn(s.n_tok, kv, dim, device="cuda", generator=gen)
        rot = case["rot"]
        turn = BASE ** (-torch.arange(0, rot, 2, device="cuda").double() / rot)
        angle = torch.arange(s.max_kv, device="cuda").double()[:, None] * turn
        s.rope = torch.stack([torch.cos(angle), torch.sin(angle)], -1).float().contiguous()
    else:
        steps = torch.arange(1, heads + 1, device="cuda").float()
        s.slopes = torch.exp2(-8.0 * steps / heads) if case["slopes"] else None
        s.prefix = (s.kv_len // 3).to(torch.int32) if case["prefix"] else None
    if own:
        _bind(s)
    return s


# ---- the library's calls -------------------------------------------------------

_device = None


def _ptr(t):
    return t.data_ptr() if t is not None and t.numel() else None


def _bind(s):
    """The argument structures that a program keeps beside its buffers."""
    global _device
    import siphon_amd as sa
    if _device is None:
        _device = sa.Device(0)
    case = s.case
    if case["kind"] == "logprobs":
        s.args = sa.Logprobs(logits=_ptr(s.logits), ld=case["vocab"], n_rows=case["rows"], n_vocab=case["vocab"],
                             token=_ptr(s.token), n_token=case["given"], logprob=_ptr(s.logprob), entropy=_ptr(s.entropy),
                             n_top=case["top"], top_id=_ptr(s.top_id), top_logprob=_ptr(s.top_logprob))
        return
    sizes = dict(n_pages=s.n_pages, n_head_kv=case["kv_heads"], head_dim=case["head_dim"], block=case["block"])
    if case.get("bits") == 8:
        s.cache = sa.KvCache(k=_ptr(s.k), v=_ptr(s.v), k_scale=_ptr(s.k_scale), v_scale=_ptr(s.v_scale), **sizes)
    else:
        s.cache = sa.Kv4Cache(k=_ptr(s.k), v=_ptr(s.v), k_sub=_ptr(s.k_sub), v_sub=_ptr(s.v_sub), k_scale=_ptr(s.k_scale),
                              v_scale=_ptr(s.v_scale), **sizes)
    s.batch = sa.KvBatch(q_start=_ptr(s.q_start), kv_len=_ptr(s.kv_len), table=_ptr(s.table), n_req=case["requests"],
                         max_blocks=s.max_blocks, n_tok=s.n_tok, max_q=s.max_q, max_kv=s.max_kv)
    width, wide = case["kv_heads"] * case["head_dim"], case["heads"] * case["head_dim"]
    if case["kind"] == "append":
        s.rows = sa.KvRows(k=_ptr(s.new_k), ldk=width, v=_ptr(s.new_v), ldv=width, q=_ptr(s.q), ldq=wide, q_out=_ptr(s.out),
                           ldq_out=wide, n_head=case["heads"], rope=_ptr(s.rope), rope_len=s.max_kv, rope_dim=case["rot"],
                           rope_neighbours=case["neighbours"])
    else:
        s.attn = sa.AttnPaged(q=_ptr(s.q), ldq=wide, out=_ptr(s.out), ldo=wide, n_head=case["heads"],
                              kq_scale=1.0 / math.sqrt(case["head_dim"]), softcap=case["cap"], slopes=_ptr(s.slopes),
                              prefix=_ptr(s.prefix), window=case["window"])


def _own_run(s):
    case = s.case
    if case["kind"] == "logprobs":
        _device.logprobs_dev(s.args)
        return [s.logprob, s.entropy, s.top_id, s.top_logprob][:4 if case["top"] else 2]
    if case["kind"] == "attention":
        _device.attn_paged4_dev(s.cache, s.batch, s.attn)
        return s.out
    width = case["kv_heads"] * case["head_dim"]
    back = (s.slot.data_ptr(), s.slot.shape[0], s.out_k.data_ptr(), width, s.out_v.data_ptr(), width)
    if case["bits"] == 8:
        _device.kv_append_rope_dev(s.cache, s.batch, s.rows)
        _device.kv_read_dev(s.cache, *back)
    else:
        _device.kv4_append_dev(s.cache, s.batch, s.rows)
        _device.kv4_read_dev(s.cache, *back)
    return [s.out, s.out_k, s.out_v]


# ---- the plain forms ------------------------------------------------------------


def _rotate(x, s):
    """Rows [token, head, dim] turned by their positions; in 64 bits, as a
    code next to a border depends on the last bit, and rounded once."""
    rot = s.case["rot"]
    c, d = (y[:, None].double() for y in s.rope[s.pos].unbind(-1))
    y = x[..., :rot].double()
    y = y.unflatten(-1, (rot // 2, 2) if s.case["neighbours"] else (2, rot // 2))
    a, b = y.unbind(-1 if s.case["neighbours"] else -2)
    y = torch.stack([a * c - b * d, a * d + b * c], -1 if s.case["neighbours"] else -2).flatten(-2)
    return torch.cat([y.float(), x[..., rot:]], -1)


def _touched(s, rows):
    """Of the pages that get new tokens: their numbers [request, block], the new
    rows at their places [request, block, head, token, dim] and which of a
    page's tokens are new and which were there before."""
    block = s.case["block"]
    length, end = (s.kv_len - (s.q_start[1:] - s.q_start[:-1])).long(), s.kv_len.long()
    most = (s.max_q + block - 2) // block + 1
    # a request with fewer than `most` repeats its last
    b = torch.minimum(length[:, None] // block + torch.arange(most, device="cuda"), (end[:, None] - 1) // block)
    pos = b[:, :, None] * block + torch.arange(block, device="cuda")
    new, past = (pos >= length[:, None, None]) & (pos < end[:, None, None]), pos < length[:, None, None]
    row = (s.q_start[:-1].long()[:, None, None] + pos - length[:, None, None]).clamp(0, s.n_tok - 1)
    return torch.gather(s.table.long(), 1, b), rows[row].transpose(2, 3), new[:, :, None, :], past[:, :, None, :]


def _write8(codes, scales, rows, s, transposed):
    page, x, new, past = _touched(s, rows)
    was = codes[page].double()
    was = was.transpose(3, 4) if transposed else was
    new, past = new[..., None], past[..., None]
    old = torch.where(past.any(3, keepdim=True), scales[page].double()[..., None, None], 0.0)
    top = torch.where(new, x.abs(), 0.0).amax((3, 4), keepdim=True).double()
    scale = torch.maximum(old, (top / 127).float().double())
    floor = torch.where(scale > 0, scale, 1.0)
    x = torch.round(x.double() / floor).clamp(-127, 127)
    got = torch.where(new, x, torch.where(past & (scale > old), torch.round(was * old / floor), was))
    codes[page] = (got.transpose(3, 4) if transposed else got).to(torch.int8)
    scales[page] = scale[..., 0, 0].float()


def _write4(codes, subs, scales, rows, s, transposed):
    page, x, new, _ = _touched(s, rows)
    c, sub, scale = _quantize4(x)
    was = _unpack(codes[page])
    c = torch.where(new[..., None], c, was.transpose(3, 4) if transposed else was)
    codes[page] = _pack(c.transpose(3, 4) if transposed else c)
    subs[page] = torch.where(new[:, :, :, None], sub.transpose(3, 4), subs[page])
    scales[page] = torch.where(new, scale.to(torch.bfloat16), scales[page])


def _values(codes, subs, scales, case, transposed):
    """Rows [..., token, dim] of pages [..., head], as f32."""
    if case.get("bits") == 8:
        x = (codes.transpose(-1, -2) if transposed else codes).float()
        return x * scales[..., None, None]
    x = _unpack(codes)
    x = (x.transpose(-1, -2) if transposed else x).float()
    step = subs.transpose(-1, -2).float() * scales.float()[..., None]
    return x * step.repeat_interleave(32, -1)


def _append(s):
    k = _rotate(s.new_k, s)
    for codes, subs, scales, rows, transposed in ((s.k, s.k_sub, s.k_scale, k, False), (s.v, s.v_sub, s.v_scale, s.new_v, True)):
        if s.case["bits"] == 8:
            _write8(codes, scales, rows, s, transposed)
        else:
            _write4(codes, subs, scales, rows, s, transposed)
    outs, block = [_rotate(s.q, s)], s.case["block"]
    page, off = s.slot // block, s.slot % block
    for codes, subs, scales, transposed in ((s.k, s.k_sub, s.k_scale, False), (s.v, s.v_sub, s.v_scale, True)):
        rows = torch.empty_like(s.out_k)
        for i in range(0, len(page), 2048):  # whole pages are a lot of memory
            p = page[i:i + 2048]
            x = _values(codes[p], subs[p], scales[p], s.case, transposed)
            rows[i:i + 2048] = x[torch.arange(len(p), device="cuda"), :, off[i:i + 2048]]
        outs.append(rows)
    return outs


def _attention(s):
    case = s.case
    n, kv, dim, heads = (case[k] for k in ("requests", "kv_heads", "head_dim", "heads"))
    group, block = heads // kv, case["block"]
    cols = _blocks(s.max_kv, block)
    table = s.table[:, :cols].long().clamp(min=0)
    k = _values(s.k[table], s.k_sub[table], s.k_scale[table], case, False)
    v = _values(s.v[table], s.v_sub[table], s.v_scale[table], case, True)
    k = k.permute(0, 2, 4, 1, 3).reshape(n, kv, dim, cols * block)
    v = v.transpose(1, 2).reshape(n, kv, cols * block, dim)
    add = s.q_start[1:] - s.q_start[:-1]
    i = torch.arange(s.max_q, device="cuda")
    row = torch.where(i < add[:, None], s.q_start[:-1, None] + i, s.n_tok)
    q = s.q[row.clamp(max=s.n_tok - 1)].reshape(n, s.max_q, kv, group, dim).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(n, kv, group * s.max_q, dim), k) * (1.0 / math.sqrt(dim))
    score = score.reshape(n, kv, group, s.max_q, cols * block)
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    j = torch.arange(cols * block, device="cuda")
    away = (s.kv_len - add)[:, None, None] + i[:, None] - j
    if s.slopes is not None:
        score = score - s.slopes.reshape(1, kv, group, 1, 1) * away.abs()[:, None, None].float()
    seen = away >= 0
    if case["window"]:
        seen = seen & (away < case["window"])
    if s.prefix is not None:
        seen = seen | (j < s.prefix[:, None, None])
    seen = seen & (j < s.kv_len[:, None, None])
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1)
    o = torch.matmul(p.reshape(n, kv, group * s.max_q, cols * block), v).reshape(n, kv, group, s.max_q, dim)
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    out = torch.zeros(s.n_tok + 1, heads, dim, device="cuda")
    out[row] = o.permute(0, 3, 1, 2, 4).reshape(n, s.max_q, heads, dim)
    return out[:-1]


def _logprobs(s):
    x = s.logits
    d = x - x.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    entropy = log_total - (e * torch.where(e > 0, d, 0.0)).sum(1) / total
    outs = [torch.gather(d, 1, s.token.long()) - log_total[:, None], entropy]
    top = s.case["top"]
    if top:
        value, index = torch.sort(d, dim=1, descending=True, stable=True)
        outs += [index[:, :top].to(torch.int32), value[:, :top] - log_total[:, None]]
    return outs


def run(s):
    if own:
        return _own_run(s)
    return {"append": _append, "attention": _attention, "logprobs": _logprobs}[s.case["kind"]](s)


# ---- what a pass cannot do without ----------------------------------------------


def _visible(case, length, add):
    """(query-key pairs, keys that some query sees) of one request."""
    end = length + add
    window = case["window"] or end
    prefix = min(end // 3, end) if case["prefix"] else 0
    pairs = 0
    for p in range(length, end):
        lo = max(0, p - window + 1)
        pairs += p + 1 - lo + max(0, min(prefix, lo)) + max(0, prefix - (p + 1))
    lo = max(0, length - window + 1)
    return pairs, end - lo + min(prefix, lo)


def work(case):
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        # a maximum, an exponential and two sums a logit
        return {"bytes": 4 * n + case["rows"] * (8 * case["given"] + 4 + 8 * case["top"]), "flops": 5 * n}
    length, add = _lengths(case)
    dim, wide = case["head_dim"], case["heads"] * case["head_dim"]
    row = case["kv_heads"] * (dim if case.get("bits") == 8 else dim // 2 + dim // 32 + 2)  # bytes of a token's keys
    if case["kind"] == "append":
        width, new = case["kv_heads"] * dim, sum(add)
        back = sum(x + a - x // case["block"] * case["block"] for x, a in zip(length, add))
        return {"bytes": 2 * (4 * width + row) * (new + back) + 8 * back + (8 * wide + 4 * case["rot"]) * new,
                "flops": 3 * case["rot"] * (case["heads"] + case["kv_heads"]) * new}
    pairs, keys = (sum(x) for x in zip(*(_visible(case, x, a) for x, a in zip(length, add))))
    return {"bytes": 2 * row * keys + 8 * wide * sum(add), "flops": 4 * wide * pairs}


# ---- the same in 64 bits ----------------------------------------------------------


def _exact_rotate(x, s):
    rot, y = s.case["rot"], x.double()
    out = y.clone()
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if s.case["neighbours"] else (i, i + rot // 2)
        c, d = s.rope[s.pos, i, 0].double()[:, None], s.rope[s.pos, i, 1].double()[:, None]
        out[..., a] = y[..., a] * c - y[..., b] * d
        out[..., b] = y[..., a] * d + y[..., b] * c
    return out


def _exact_codes(data, axis_tokens):
    """Codes of packed bytes, one element of each word at a time."""
    word = data.long().reshape(*data.shape[:-1], -1, 4)
    out = torch.empty(*data.shape[:-1], data.shape[-1] * 2, dtype=torch.float64, device=data.device)
    for e in range(8):
        nibble = e // 2 + 4 * (e % 2)
        out[..., e::8] = (word[..., nibble // 2] >> (4 * (nibble % 2))) % 16 - 8
    return out.transpose(-1, -2) if axis_tokens else out


def _exact_page(codes, subs, scales, page, case, transposed):
    """Values [head, token, dim] of a page."""
    if case.get("bits") == 8:
        x = codes[page].double()
        return (x.transpose(-1, -2) if transposed else x) * scales[page].double()[..., None, None]
    x = _exact_codes(codes[page], transposed)
    for g in range(case["head_dim"] // 32):
        x[..., 32 * g:32 * g + 32] *= (subs[page][..., g, :].double() * scales[page].double())[..., None]
    return x


def _exact_new8(codes, scales, page, x, lo, transposed):
    """A page's values [head, token, dim] up to its last new token; x: its new rows [head, token, dim]."""
    old = codes[page].double()
    old = (old.transpose(1, 2) if transposed else old)[:, :lo]
    was = scales[page].double()[:, None, None] * (lo > 0)
    step = torch.maximum(was, (x.abs().amax((1, 2), keepdim=True) / 127.0).float().double())
    old = torch.where(step > was, torch.round(old * was / step), old)
    return step * torch.cat([old, torch.round(x / step)], 1)


def _exact_new4(x):
    """The values that rows [head, token, dim] become."""
    size, out = [], torch.empty_like(x)
    for g in range(x.shape[-1] // 32):
        part = x[..., 32 * g:32 * g + 32]
        size.append(part.abs().amax(-1) / 8)
    scale = (torch.stack(size).amax(0) / 127).float()
    up = scale.to(torch.bfloat16).double()  # to the nearest, then up where that is below
    up = torch.where(up < scale.double(), up + torch.exp2(torch.floor(torch.log2(up)) - 7), up)
    for g, most in enumerate(size):
        part = x[..., 32 * g:32 * g + 32]
        minus = (part == -8 * most[..., None]).any(-1)
        sub = torch.ceil(most / up).clamp(1, 127) * torch.where(minus, 1.0, -1.0)
        step = (sub * up)[..., None]
        out[..., 32 * g:32 * g + 32] = torch.round(part / step).clamp(-8, 7) * step
    return out


def _exact_append(case, seed):
    s = prepare(case, seed)
    block, table = case["block"], s.table.tolist()
    k = _exact_rotate(s.new_k, s).float()
    outs = [_exact_rotate(s.q, s)]
    for codes, subs, scales, rows, transposed in ((s.k, s.k_sub, s.k_scale, k, False), (s.v, s.v_sub, s.v_scale, s.new_v, True)):
        parts, first = [], 0
        for r, (length, add) in enumerate(zip(*_lengths(case))):
            for b in range(length // block, _blocks(length + add, block)):
                lo, hi = max(length - b * block, 0), min(length + add - b * block, block)
                at = first + b * block + lo - length
                x = rows[at:at + hi - lo].double().transpose(0, 1)
                if case["bits"] == 8:
                    parts.append(_exact_new8(codes, scales, table[r][b], x, lo, transposed))
                else:
                    old = _exact_page(codes, subs, scales, table[r][b], case, transposed)[:, :lo]
                    parts.append(torch.cat([old, _exact_new4(x)], 1))
            first += add
        outs.append(torch.cat(parts, 1).transpose(0, 1))
    return outs


def _exact_logprobs(case, seed):
    s = prepare(case, seed)
    x = s.logits.double()
    lse = torch.logsumexp(x, 1, keepdim=True)
    p = torch.exp(x - lse)
    outs = [(x.gather(1, s.token.long()) - lse), -torch.where(p > 0, p * (x - lse), 0.0).sum(1)]
    if case["top"]:
        ids, left = [], x.clone()
        for _ in range(case["top"]):
            # the first of the largest; what was taken comes last of all (NaN equals nothing)
            best = torch.where(left.isnan(), -math.inf, left).amax(1, keepdim=True)
            index = (left == best).to(torch.uint8).argmax(1, keepdim=True)
            ids.append(index)
            left.scatter_(1, index, math.nan)
        ids = torch.cat(ids, 1)
        outs += [ids.to(torch.int32), x.gather(1, ids) - lse]
    return outs


def exact(case, seed):
    if case["kind"] == "logprobs":
        return _exact_logprobs(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, seed)
    s = prepare(case, seed)
    block, table = case["block"], s.table.tolist()
    outs, first = [], 0
    group = case["heads"] // case["kv_heads"]
    for r, (x, a) in enumerate(zip(*_lengths(case))):
        pages = torch.tensor(table[r][:_blocks(x + a, block)], device="cuda")
        keys = _exact_page(s.k, s.k_sub, s.k_scale, pages, case, False)
        values = _exact_page(s.v, s.v_sub, s.v_scale, pages, case, True)
        at = torch.arange(x, x + a, device="cuda")[:, None]
        j = torch.arange(x + a, device="cuda")[None, :]
        hidden = (j > at) | (j <= at - (case["window"] or x + a))
        if case["prefix"]:
            hidden &= j >= (x + a) // 3
        out = torch.empty(a, case["heads"], case["head_dim"], device="cuda", dtype=torch.float64)
        for h in range(case["heads"]):
            k = keys[:, h // group].flatten(0, 1)[:x + a]
            v = values[:, h // group].flatten(0, 1)[:x + a].contiguous()
            score = torch.mm(s.q[first:first + a, h].double(), k.t().contiguous()) / math.sqrt(case["head_dim"])
            if case["cap"]:
                score = torch.tanh(score / case["cap"]) * case["cap"]
            if case["slopes"]:
                score -= s.slopes[h].double() * (at - j).abs()
            score[hidden] = -math.inf
            out[:, h] = torch.mm(torch.softmax(score, 1), v)
        outs.append(out)
        first += a
    return torch.cat(outs)
