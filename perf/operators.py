"""The operators of the shared 8-bit KV cache, as timed cases.

A case is one call, or a run of calls that belong together, that a host
serving several sequences makes of the paged cache:

  plan       a step's bookkeeping on the device: the pages of ended requests
             go back to the free list, new ones are taken, and the block
             table, row starts, lengths, slots and positions come out
  append     the step's keys and values into one layer's cache (8-bit codes,
             a scale for each page and head), and the rows of the pages that
             changed read back through their slots
  read       whole sequences read back through their slots
  attention  a step's queries over one layer's cache: single tokens or
             prompt rows, with capped scores, distance biases, windows or
             bidirectional prefixes

A page holds `block` tokens of every KV head. Keys are [page][head][token][dim]
and values [page][head][dim][token], as in the f16 cache of the decode
attention. A code times its page's and head's scale is the value it stands for.
Request lengths are spread by their logarithm and depend on the case alone.
"""
import math
import random

import torch

own = False

# heads, KV heads and head_dim of layers (listed by the model class they are of)
HEADS_05B = {"heads": 14, "kv_heads": 2, "head_dim": 64}
HEADS_1B = {"heads": 32, "kv_heads": 4, "head_dim": 64}
HEADS_8B = {"heads": 32, "kv_heads": 8, "head_dim": 128}
HEADS_32B = {"heads": 40, "kv_heads": 8, "head_dim": 128}
HEADS_WIDE = {"heads": 16, "kv_heads": 8, "head_dim": 256}
PLAIN = {"cap": 0.0, "window": 0, "slopes": False, "prefix": False}


def _kv(heads):
    return {k: heads[k] for k in ("kv_heads", "head_dim")}


def listed():
    return [
        # one decode step of a small server: latency of one launch
        {"name": "plan_step_64", "kind": "plan", "requests": 64, "block": 32, "max_len": 8192, "max_add": 1, "ended": 3},
        # a busy server's step with many prompts in it
        {"name": "plan_prompts_1000", "kind": "plan", "requests": 1000, "block": 16, "max_len": 2000, "max_add": 257,
         "ended": 90},
        # the new token of every sequence of a small server
        {"name": "append_step_64_8b", "kind": "append", **_kv(HEADS_8B), "requests": 64, "block": 32, "max_len": 8192,
         "max_add": 1},
        # prompt chunks, the longest of odd length behind a cached context
        {"name": "append_prompts_8b", "kind": "append", **_kv(HEADS_8B), "requests": 5, "block": 64, "max_len": 500,
         "max_add": 2047},
        # a short conversation of a small model moved off the device
        {"name": "read_1_600_1b", "kind": "read", **_kv(HEADS_1B), "requests": 1, "block": 16, "max_len": 600,
         "max_add": 0},
        # a few long ones
        {"name": "read_4_7000_8b", "kind": "read", **_kv(HEADS_8B), "requests": 4, "block": 64, "max_len": 7001,
         "max_add": 0},
        # a single user early in a conversation: latency
        {"name": "step_1_600_8b", "kind": "attention", **HEADS_8B, **PLAIN, "requests": 1, "block": 32, "max_len": 600,
         "max_add": 1},
        # a decode step of a batch with ragged lengths
        {"name": "step_64_8192_8b", "kind": "attention", **HEADS_8B, **PLAIN, "requests": 64, "block": 16,
         "max_len": 8191, "max_add": 1},
        # one very long context
        {"name": "step_1_131072_8b", "kind": "attention", **HEADS_8B, **PLAIN, "requests": 1, "block": 64,
         "max_len": 131071, "max_add": 1},
        # wide heads with capped scores and a sliding window
        {"name": "step_16_capped_window", "kind": "attention", **HEADS_WIDE, **PLAIN, "cap": 50.0, "window": 4096,
         "requests": 16, "block": 32, "max_len": 16000, "max_add": 1},
        # a usual prompt of a small model, of odd length
        {"name": "prompt_1_509_0.5b", "kind": "attention", **HEADS_05B, **PLAIN, "requests": 1, "block": 16,
         "max_len": 0, "max_add": 509},
        # prompts of a 32B model whose heads have distance biases and whose
        # beginnings see each other both ways, the largest case
        {"name": "prompts_3_4096_32b", "kind": "attention", **HEADS_32B, **PLAIN, "slopes": True, "prefix": True,
         "requests": 3, "block": 64, "max_len": 1000, "max_add": 4096},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "read", "attention", "attention", "attention", "attention"])
    case = {"kind": kind, "block": rng.choice([16, 32, 64, 128])}
    if kind == "plan":
        n = _log_int(rng, 1, 1500)
        return {**case, "requests": n, "max_len": _log_int(rng, 30, 16384),
                "max_add": rng.choice([1, _log_int(rng, 2, 260)]), "ended": rng.randint(0, n // 4)}
    case = {**case, "kv_heads": rng.choice([1, 2, 4, 8]), "head_dim": rng.choice([64, 80, 96, 128, 256])}
    width = case["kv_heads"] * case["head_dim"]
    if kind == "read":
        n = _log_int(rng, 1, 16)
        return {**case, "requests": n, "max_len": _log_int(rng, 16, (1 << 24) // width // n), "max_add": 0}
    if kind == "append":
        n = _log_int(rng, 1, 128)
        return {**case, "requests": n, "max_len": _log_int(rng, 1, 8192),
                "max_add": rng.choice([1, _log_int(rng, 2, (1 << 22) // width // n)])}
    group = rng.randint(1, 8)
    case = {**case, "heads": case["kv_heads"] * group, "cap": rng.choice([0.0, 0.0, 30.0]),
            "window": rng.choice([0, 0, _log_int(rng, 16, 8192)]), "slopes": rng.random() < 0.3,
            "prefix": rng.random() < 0.3}
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

    length, add = spread(case["max_len"]), spread(case["max_add"])
    for r in rng.sample(range(n), case.get("ended", 0)):
        add[r] = -1
    return length, add


def _blocks(tokens, block):
    return -(-tokens // block)


class State:
    pass


def _codes(pages, heads, block, dim, transposed, gen):
    """Codes and scales of random rows with uneven channels."""
    size = torch.exp(0.5 * torch.randn(heads, dim, device="cuda", generator=gen))
    shape = (pages, heads, dim, block) if transposed else (pages, heads, block, dim)
    x = torch.randn(shape, device="cuda", generator=gen)
    x.mul_(size[None, :, :, None] if transposed else size[None, :, None, :])
    scale = torch.clamp(x.abs().amax((2, 3)) / 127, min=1e-20)
    x.div_(scale[:, :, None, None]).round_().clamp_(-127, 127)
    return x.to(torch.int8), scale


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = State()
    s.case = case
    length, add = _lengths(case)
    n, block = case["requests"], case["block"]
    new = [max(a, 0) for a in add]
    before = [_blocks(x, block) for x in length]
    after = [_blocks(x + a, block) for x, a in zip(length, new)]
    s.n_tok, s.max_blocks = sum(new), max(after) + 2
    total = sum(after)
    s.n_pages = total + total // 8 + 4
    order = torch.randperm(s.n_pages, device="cuda", generator=gen).to(torch.int32)
    s.length, s.add = _ints(length), _ints(add)
    # cached blocks take pages of the front of the order in request order
    held = before if case["kind"] == "plan" else after
    col = torch.arange(s.max_blocks, device="cuda")
    mine = col[None, :] < _ints(held)[:, None]
    at = (torch.cumsum(mine.flatten().long(), 0) - 1).reshape(mine.shape)
    s.table = torch.where(mine, order[at.clamp(min=0)], -1).to(torch.int32).contiguous()
    if case["kind"] == "plan":
        used = sum(before)
        s.free = torch.cat([order[used:], order[:used] * 0 - 1]).contiguous()
        s.n_free = _ints([s.n_pages - used])
        s.q_start, s.kv_len = torch.empty(n + 1, dtype=torch.int32, device="cuda"), torch.empty_like(s.length)
        s.slot = torch.empty(s.n_tok, dtype=torch.int64, device="cuda")
        s.pos = torch.empty(s.n_tok, dtype=torch.int32, device="cuda")
        s.n_free_out, s.status = _ints([0]), _ints([0])
    else:
        s.kv_len = _ints([x + a for x, a in zip(length, new)])
        s.q_start = _ints([sum(new[:r]) for r in range(n + 1)])
        s.max_q, s.max_kv = max(new), max(x + a for x, a in zip(length, new))
        kv, dim = case["kv_heads"], case["head_dim"]
        s.k, s.k_scale = _codes(s.n_pages, kv, block, dim, False, gen)
        s.v, s.v_scale = _codes(s.n_pages, kv, block, dim, True, gen)
        if case["kind"] in ("append", "read"):
            # the positions to read: of the pages that get new tokens, or all
            first = [x // block * block if case["kind"] == "append" else 0 for x in length]
            at = torch.cat([torch.arange(f, x + a) for f, x, a in zip(first, length, new)]).cuda()
            req = torch.cat([torch.full((x + a - f,), r) for r, (f, x, a) in enumerate(zip(first, length, new))]).cuda()
            s.slot = s.table[req, at // block].long() * block + at % block
            s.out_k = torch.empty(len(at), kv, dim, device="cuda")
            s.out_v = torch.empty_like(s.out_k)
        if case["kind"] == "append":
            # keys whose sizes differ from token to token, so that scales grow
            size = torch.exp(0.4 * torch.randn(s.n_tok, kv, 1, device="cuda", generator=gen))
            s.new_k = size * torch.randn(s.n_tok, kv, dim, device="cuda", generator=gen)
            s.new_v = torch.randn(s.n_tok, kv, dim, device="cuda", generator=gen)
        if case["kind"] == "attention":
            heads = case["heads"]
            s.q = 1.3 * torch.randn(s.n_tok, heads, dim, device="cuda", generator=gen)
            s.out = torch.empty_like(s.q)
            steps = torch.arange(1, heads + 1, device="cuda").float()
            s.slopes = torch.exp2(-8.0 * steps / heads) if case["slopes"] else None
            s.prefix = (s.kv_len // 3).to(torch.int32) if case["prefix"] else None
    if own:
        _bind(s)
    return s


# ---- the library's calls -------------------------------------------------------

_device = None


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _bind(s):
    """The argument structures that a program keeps beside its buffers."""
    global _device
    import siphon_amd as sa
    if _device is None:
        _device = sa.Device(0)
    case = s.case
    if case["kind"] == "plan":
        s.plan = sa.KvPlan(len=_ptr(s.length), add=_ptr(s.add), free_pages=_ptr(s.free), n_free=_ptr(s.n_free),
                           n_req=case["requests"], n_tok=s.n_tok, n_pages=s.n_pages, max_blocks=s.max_blocks,
                           block=case["block"], table=_ptr(s.table), q_start=_ptr(s.q_start), kv_len=_ptr(s.kv_len),
                           slot=_ptr(s.slot), pos=_ptr(s.pos), n_free_out=_ptr(s.n_free_out), status=_ptr(s.status))
        return
    s.cache = sa.KvCache(k=_ptr(s.k), v=_ptr(s.v), k_scale=_ptr(s.k_scale), v_scale=_ptr(s.v_scale), n_pages=s.n_pages,
                         n_head_kv=case["kv_heads"], head_dim=case["head_dim"], block=case["block"])
    s.batch = sa.KvBatch(q_start=_ptr(s.q_start), kv_len=_ptr(s.kv_len), table=_ptr(s.table), n_req=case["requests"],
                         max_blocks=s.max_blocks, n_tok=s.n_tok, max_q=s.max_q, max_kv=s.max_kv)
    if case["kind"] == "attention":
        width = case["heads"] * case["head_dim"]
        s.attn = sa.AttnPaged(q=_ptr(s.q), ldq=width, out=_ptr(s.out), ldo=width, n_head=case["heads"],
                              kq_scale=1.0 / math.sqrt(case["head_dim"]), softcap=case["cap"], slopes=_ptr(s.slopes),
                              prefix=_ptr(s.prefix), window=case["window"])


def _own_run(s):
    case = s.case
    if case["kind"] == "plan":
        _device.kv_plan_dev(s.plan)
        return [s.table, s.q_start, s.kv_len, s.slot, s.pos, s.free, s.n_free_out, s.status]
    if case["kind"] == "attention":
        _device.attn_paged_dev(s.cache, s.batch, s.attn)
        return s.out
    width = case["kv_heads"] * case["head_dim"]
    if case["kind"] == "append":
        _device.kv_append_dev(s.cache, s.batch, s.new_k.data_ptr(), width, s.new_v.data_ptr(), width)
    _device.kv_read_dev(s.cache, s.slot.data_ptr(), s.slot.shape[0], s.out_k.data_ptr(), width, s.out_v.data_ptr(),
                        width)
    return [s.out_k, s.out_v]


# ---- the plain forms ------------------------------------------------------------


def _plan(s):
    block, n = s.case["block"], s.case["requests"]
    add, ended = s.add.clamp(min=0).long(), s.add < 0
    length = s.length.long()
    before = (length + block - 1) // block
    kv_len = torch.where(ended, 0, length + add)
    after = torch.where(ended, before, (length + add + block - 1) // block)
    col = torch.arange(s.max_blocks, device="cuda")[None, :]
    # the free list with the pages of ended requests behind its entries
    back = (ended[:, None] & (col < before[:, None])).flatten()
    n_free = s.n_free.long()
    place = torch.where(back, n_free + torch.cumsum(back.long(), 0) - 1, s.n_pages)
    free = torch.cat([s.free, s.free.new_zeros(1)])
    free.scatter_(0, place, torch.where(back, s.table.flatten(), 0))
    n_back = back.long().sum()
    need = after - before
    start = torch.cumsum(need, 0) - need
    n_out = n_free + n_back - need.sum()
    taken = (col >= before[:, None]) & (col < after[:, None])
    rank = start[:, None] + col - before[:, None]
    page = free[(n_free + n_back - 1 - rank).clamp(0, s.n_pages)]
    table = torch.where(taken, page, s.table)
    index = torch.arange(s.n_pages, device="cuda")
    kept = torch.where((index >= n_free) & (index < n_out), free[:-1], s.free)
    q_end = torch.cumsum(add, 0)
    q_start = torch.cat([q_end.new_zeros(1), q_end])
    t = torch.arange(s.n_tok, device="cuda")
    r = torch.searchsorted(q_end, t, right=True).clamp(max=n - 1)
    live = t < q_end[-1]
    pos = length[r] + t - q_start[r]
    slot = table[r, (pos // block).clamp(0, s.max_blocks - 1)].long() * block + pos % block
    return [table, q_start.int(), kv_len.int(), torch.where(live, slot, -1), torch.where(live, pos, -1).int(), kept,
            n_out.int(), torch.zeros_like(s.status)]


def _quantize_into(codes, scales, rows, s, transposed):
    """Writes the rows of new tokens into the codes and scales of their pages."""
    block, dim = s.case["block"], s.case["head_dim"]
    length = (s.kv_len - (s.q_start[1:] - s.q_start[:-1])).long()
    end = s.kv_len.long()
    most = (s.max_q + block - 2) // block + 1
    # blocks with new tokens; a request with fewer than `most` repeats its last
    b = torch.minimum(length[:, None] // block + torch.arange(most, device="cuda"), (end[:, None] - 1) // block)
    page = torch.gather(s.table.long(), 1, b)
    pos = b[:, :, None] * block + torch.arange(block, device="cuda")
    new, past = (pos >= length[:, None, None]) & (pos < end[:, None, None]), pos < length[:, None, None]
    row = (s.q_start[:-1].long()[:, None, None] + pos - length[:, None, None]).clamp(0, s.n_tok - 1)
    x = rows[row].permute(0, 1, 3, 2, 4).double()  # [request, block, head, token, dim]
    was = codes[page].double()
    if transposed:
        was = was.transpose(3, 4)
    new, past = new[:, :, None, :, None], past[:, :, None, :, None]
    top = torch.where(new, x.abs(), 0.0).amax((3, 4))
    fresh = (b * block >= length[:, None])[:, :, None]
    old = torch.where(fresh, 0.0, scales[page].double())
    scale = torch.maximum(old, (top / 127).float().double())
    wide, floor = scale[..., None, None], torch.where(scale > 0, scale, 1.0)[..., None, None]
    x = torch.round(x / floor).clamp(-127, 127)
    kept = torch.where(wide > old[..., None, None], torch.round(was * old[..., None, None] / floor), was)
    got = torch.where(new, x, torch.where(past, kept, was))
    if transposed:
        got = got.transpose(3, 4)
    codes[page] = got.to(torch.int8)
    scales[page] = scale.float()


def _read(s):
    block = s.case["block"]
    page, off = s.slot // block, s.slot % block
    k = s.k[page, :, off, :].float() * s.k_scale[page][:, :, None]
    v = s.v[page, :, :, off].float() * s.v_scale[page][:, :, None]
    return [k, v]


def _attention(s):
    case = s.case
    n, kv, dim, heads = (case[k] for k in ("requests", "kv_heads", "head_dim", "heads"))
    group, block = heads // kv, case["block"]
    cols = _blocks(s.max_kv, block)
    table = s.table[:, :cols].long().clamp(min=0)
    k = s.k[table].float() * s.k_scale[table][..., None, None]
    v = s.v[table].float() * s.v_scale[table][..., None, None]
    k = k.permute(0, 2, 4, 1, 3).reshape(n, kv, dim, cols * block)
    v = v.permute(0, 2, 1, 4, 3).reshape(n, kv, cols * block, dim)
    add = s.q_start[1:] - s.q_start[:-1]
    i = torch.arange(s.max_q, device="cuda")
    live = i < add[:, None]
    row = torch.where(live, s.q_start[:-1, None] + i, s.n_tok)
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


def run(s):
    if own:
        return _own_run(s)
    kind = s.case["kind"]
    if kind == "plan":
        return _plan(s)
    if kind == "attention":
        return _attention(s)
    if kind == "append":
        _quantize_into(s.k, s.k_scale, s.new_k, s, False)
        _quantize_into(s.v, s.v_scale, s.new_v, s, True)
    return _read(s)


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
    length, add = _lengths(case)
    new = [max(a, 0) for a in add]
    if case["kind"] == "plan":
        blocks = [_blocks(x + a, case["block"]) - x // case["block"] for x, a in zip(length, new)]
        ended = sum(_blocks(x, case["block"]) for x, a in zip(length, add) if a < 0)
        return {"bytes": 4 * (4 * case["requests"] + 2 * sum(blocks) + 2 * ended) + 12 * sum(new), "flops": 0}
    width = case["kv_heads"] * case["head_dim"]
    if case["kind"] != "attention":
        first = [x // case["block"] * case["block"] if case["kind"] == "append" else 0 for x in length]
        rows = sum(x + a - f for x, a, f in zip(length, new, first))
        return {"bytes": 2 * width * 5 * ((sum(new) if case["kind"] == "append" else 0) + rows) + 8 * rows, "flops": 0}
    pairs, keys = (sum(x) for x in zip(*(_visible(case, x, a) for x, a in zip(length, new))))
    wide = case["heads"] * case["head_dim"]
    return {"bytes": 2 * width * keys + 8 * wide * sum(new), "flops": 4 * wide * pairs}


# ---- the same in 64 bits ----------------------------------------------------------


def _exact_append(codes, scales, rows, s, transposed):
    """{page: values [head, token, dim]} of the pages with new tokens, in f64."""
    block = s.case["block"]
    got, first = {}, 0
    table = s.table.tolist()
    for r, (length, add) in enumerate(zip(*_lengths(s.case))):
        for b in range(length // block, _blocks(length + add, block)):
            page, lo = table[r][b], max(length - b * block, 0)
            hi = min(length + add - b * block, block)
            at = first + b * block + lo - length
            x = rows[at:at + hi - lo].double().transpose(0, 1)
            old = codes[page].double()
            old = (old.transpose(1, 2) if transposed else old)[:, :lo]
            was = scales[page].double()[:, None, None] * (lo > 0)
            step = torch.maximum(was, (x.abs().amax((1, 2), keepdim=True) / 127.0).float().double())
            old = torch.where(step > was, torch.round(old * was / step), old)
            got[page] = step * torch.cat([old, torch.round(x / step)], 1)
        first += add
    return got


def exact(case, seed):
    s = prepare(case, seed)
    length, add = _lengths(case)
    block = case["block"]
    if case["kind"] == "plan":
        return None
    if case["kind"] == "append":
        outs = []
        for codes, scales, rows, transposed in ((s.k, s.k_scale, s.new_k, False), (s.v, s.v_scale, s.new_v, True)):
            got = _exact_append(codes, scales, rows, s, transposed)
            outs.append(torch.stack([got[x // block][:, x % block] for x in s.slot.tolist()]))
        return outs
    table = s.table.tolist()
    keys, values = [], []
    for r, (x, a) in enumerate(zip(length, add)):
        pages = torch.tensor(table[r][:_blocks(x + a, block)], device="cuda")
        k = s.k[pages].double() * s.k_scale[pages].double()[:, :, None, None]
        v = s.v[pages].double() * s.v_scale[pages].double()[:, :, None, None]
        keys.append(torch.cat(list(k), 1)[:, :x + a])
        values.append(torch.cat(list(v.transpose(2, 3)), 1)[:, :x + a])
    if case["kind"] == "read":
        return [torch.cat(keys, 1).transpose(0, 1), torch.cat(values, 1).transpose(0, 1)]
    outs, first = [], 0
    group = case["heads"] // case["kv_heads"]
    for r, (x, a) in enumerate(zip(length, add)):
        at = torch.arange(x, x + a, device="cuda")[:, None]
        j = torch.arange(x + a, device="cuda")[None, :]
        hidden = (j > at) | (j <= at - (case["window"] or x + a))
        if case["prefix"]:
            hidden &= j >= (x + a) // 3
        out = torch.empty(a, case["heads"], case["head_dim"], device="cuda", dtype=torch.float64)
        for h in range(case["heads"]):
            q = s.q[first:first + a, h].double()
            score = torch.mm(q, keys[r][h // group].t().contiguous()) / math.sqrt(case["head_dim"])
            if case["cap"]:
                score = torch.tanh(score / case["cap"]) * case["cap"]
            if case["slopes"]:
                score -= s.slopes[h].double() * (at - j).abs()
            score[hidden] = -math.inf
            out[:, h] = torch.mm(torch.softmax(score, 1), values[r][h // group])
        outs.append(out)
        first += a
    return torch.cat(outs)
