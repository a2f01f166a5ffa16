"""What the paged 8-bit cache operators and the token scorer are measured on.

`run` computes an operator in its plain form (elementary torch operations in 32 bits) where `own` is
false, and through diffusorrt_b200.kernels where it is true. The operators:

  plan    block tables and slot maps from the request lengths (kernels.plan_cache)
  append  rows of K and V written into the 8-bit cache, and the blocks they touched read back
          (kernels.append_cache_q8, kernels.read_cache_q8)
  attend  attention over the 8-bit cache (kernels.attend_cache_q8)
  score   log probabilities of given tokens, entropy, rank, alternatives (kernels.select_logprobs)

Cache layout: K [blocks, kv heads, block, dim], V [blocks, kv heads, block / 16, dim, 16], int8 or
float8_e4m3fn, with one float32 scale for each block and head of K and of V.
"""
from __future__ import annotations

import math
import random

import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One serving step of 64 requests, a new token each: what runs before every forward.
        dict(name="plan_step", op="plan", requests=64, count_min=1, count_max=1, start_max=8192, block=32,
             finished=0.05, shape=1),
        # The prompts of a full batch admitted at once: a quarter of a million rows get their slots.
        dict(name="plan_prompts", op="plan", requests=509, count_min=1, count_max=1024, start_max=2000, block=16,
             finished=0.1, shape=2),
        # A token for each of 64 requests joins blocks that hold tokens already (K/V heads of the 0.6B model).
        dict(name="append_step", op="append", requests=64, count_min=1, count_max=1, start_max=500, kv_heads=8, dim=128,
             block=32, code="int8", type="bf16", shape=3),
        # Two prompts' K and V enter the cache (K/V heads of the 7B model), ends inside of blocks.
        dict(name="append_prompts", op="append", requests=2, count_min=7001, count_max=8100, start_max=40, kv_heads=4,
             dim=128, block=64, code="e4m3", type="bf16", shape=4),
        # The smallest call: one token of one short request.
        dict(name="attend_one", op="attend", requests=1, rows_min=1, rows_max=1, len_min=37, len_max=37, heads=16,
             kv_heads=8, dim=128, block=32, code="int8", type="bf16", mask_block=1, pad=0, shape=5),
        # Single-token decoding of a batch with lengths of every size, an empty request and padding rows.
        dict(name="attend_batch", op="attend", requests=64, rows_min=1, rows_max=1, len_min=0, len_max=8192, heads=16,
             kv_heads=8, dim=128, block=64, code="e4m3", type="bf16", mask_block=1, pad=5, shape=6),
        # One token over a long context (heads of the 7B model).
        dict(name="attend_long", op="attend", requests=1, rows_min=1, rows_max=1, len_min=130001, len_max=130001,
             heads=28, kv_heads=4, dim=128, block=64, code="int8", type="bf16", mask_block=1, pad=0, shape=7),
        # A denoising step: each request's active block of 32 positions against its prefix.
        dict(name="attend_windows", op="attend", requests=8, rows_min=32, rows_max=32, len_min=600, len_max=4608,
             heads=16, kv_heads=8, dim=128, block=32, code="int8", type="bf16", mask_block=32, pad=0, shape=8),
        # Prompt chunks behind cached prefixes (heads of the 7B model), odd ends, block mask.
        dict(name="attend_prompts", op="attend", requests=2, rows_min=1900, rows_max=2600, len_min=4000, len_max=7000,
             heads=28, kv_heads=4, dim=128, block=128, code="e4m3", type="fp16", mask_block=8, pad=3, shape=9),
        # The score of one answered token, with five alternatives.
        dict(name="score_one", op="score", rows=1, vocab=151936, top=5, type="fp32", temperature=0.0, exclude=-1),
        # One block's tokens under a temperature, the mask token left out.
        dict(name="score_block", op="score", rows=32, vocab=151936, top=20, type="fp32", temperature=0.7,
             exclude=151669),
        # The masked rows of a batch of canvases, bf16 logits, ten alternatives each.
        dict(name="score_batch", op="score", rows=1005, vocab=152064, top=10, type="bf16", temperature=0.0, exclude=-1),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "score"])
    shape = rng.randrange(1 << 30)
    if op == "plan":
        requests = _log(rng, 1, 509)
        top = _log(rng, 1, 1024)
        return dict(op=op, requests=requests, count_min=rng.choice([0, 1, 1]), count_max=top, start_max=_log(rng, 1, 8192),
                    block=rng.choice([16, 32, 64, 128]), finished=rng.choice([0.0, 0.1]), shape=shape)
    if op == "append":
        requests = _log(rng, 1, 96)
        most = max(1, 16000 // requests)
        top = _log(rng, 1, most)
        return dict(op=op, requests=requests, count_min=rng.randint(0, top), count_max=top, start_max=rng.randint(0, 500),
                    kv_heads=rng.choice([1, 2, 4, 5, 8]), dim=rng.choice([64, 128]), block=rng.choice([16, 32, 64, 128]),
                    code=rng.choice(["int8", "e4m3"]), type=rng.choice(["bf16", "fp16"]), shape=shape)
    if op == "score":
        rows = _log(rng, 1, 1005)
        return dict(op=op, rows=rows, vocab=_log(rng, 1000, 152064), top=rng.randint(0, 20),
                    type=rng.choice(["fp32", "bf16", "fp16"]), temperature=rng.choice([0.0, 0.2, 0.7, 1.3]),
                    exclude=rng.choice([-1, 7]))
    kind = rng.choice(["decode", "window", "prompt"])
    heads, kv_heads = rng.choice([(16, 8), (28, 4), (8, 8), (32, 4), (12, 1), (15, 5), (2, 1)])
    common = dict(op=op, heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), block=rng.choice([16, 32, 64, 128]),
                  code=rng.choice(["int8", "e4m3"]), type=rng.choice(["bf16", "fp16"]),
                  mask_block=rng.choice([0, 1, 1, 8, 32]), pad=rng.choice([0, 0, 3]), shape=shape)
    if kind == "decode":
        requests = _log(rng, 1, 64)
        longest = _log(rng, 1, min(130001, 524288 // requests // max(1, kv_heads // 4)))
        return dict(common, requests=requests, rows_min=1, rows_max=1, len_min=rng.randint(0, longest), len_max=longest)
    if kind == "window":
        requests = _log(rng, 1, 12)
        rows = _log(rng, 2, 64)
        longest = _log(rng, rows, 6000)
        return dict(common, requests=requests, rows_min=rng.randint(1, rows), rows_max=rows,
                    len_min=rng.randint(rows, longest), len_max=longest)
    rows = _log(rng, 65, 2600)
    longest = _log(rng, rows, 7000)
    return dict(common, requests=rng.randint(1, 2), rows_min=rng.randint(65, rows), rows_max=rows,
                len_min=rng.randint(rows, longest), len_max=longest)


def _ragged(case):
    """The case's own lengths: (rows, length) of each request for attend, (start, count) otherwise."""
    rng = random.Random(case["shape"])
    out = []
    for r in range(case["requests"]):
        if case["op"] == "attend":
            n = rng.randint(case["rows_min"], case["rows_max"])
            lo, hi = case["len_min"], case["len_max"]
            length = 0 if lo == 0 and r == 1 else max(n, _log(rng, max(1, lo), max(1, hi)))
            out.append((n, length))
        else:
            done = case["op"] == "plan" and rng.random() < case["finished"]
            start = rng.randint(0, case["start_max"])
            out.append((start, -1 if done else rng.randint(case["count_min"], case["count_max"])))
    return out


def _up(a, b):
    return -(-a // b)


# ----------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _codes(gen, shape, code, spread):
    """Codes as a quantized cache holds them: near normal, some values at the ends."""
    x = torch.randn(shape, generator=gen, device="cuda")
    if code == "int8":
        return (x * (36.0 * spread)).round_().clamp_(-127, 127).to(torch.int8)
    return (x * (120.0 * spread)).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(gen, shape, code):
    unit = 1 / 36.0 if code == "int8" else 1 / 120.0
    return torch.exp(torch.randn(shape, generator=gen, device="cuda") * 0.3) * unit


def _tables(gen, held, width, blocks):
    """Tables whose blocks lie in a shuffled order, as after some time of serving; unused entries are -1."""
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((len(held), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, h in enumerate(held):
        tables[r, :h] = order[at:at + h]
        at += h
    return tables, order, at


def prepare(case, seed):
    gen = _gen(seed)
    s = dict(case=case)
    if case["op"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=gen, device="cuda") * 2.5
        x[:, : max(1, vocab // 500)] += 4.0  # the head of the vocabulary is likelier
        s["logits"] = x.to(TYPE[case["type"]])
        tok = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        best = s["logits"].float().argmax(1)
        s["tokens"] = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.6, best, tok).to(torch.int32)
        return s
    ragged = _ragged(case)
    block = case["block"]
    if case["op"] == "plan":
        held = [_up(a, block) for a, _ in ragged]
        need = sum(max(0, _up(a + c, block) - h) for (a, c), h in zip(ragged, held) if c >= 0)
        width = max(max(h, _up(a + max(c, 0), block)) for (a, c), h in zip(ragged, held)) + 1
        blocks = sum(held) + need + 17
        tables, order, at = _tables(gen, held, width, blocks)
        head = blocks // 3
        s.update(start=_ints([a for a, _ in ragged]), count=_ints([c for _, c in ragged]), held=_ints(held), tables=tables,
                 ring=torch.roll(torch.cat([order[at:], torch.zeros(at, dtype=torch.int32, device="cuda")]), head),
                 ring_state=_ints([head, blocks - at]), max_rows=sum(max(c, 0) for _, c in ragged) + 3)
        s.update(held_out=torch.empty_like(s["held"]), ring_state_out=torch.empty_like(s["ring_state"]))
        return s
    heads, dim, code = case["kv_heads"], case["dim"], case["code"]
    total = [a + c if case["op"] == "append" else c for a, c in ragged]
    held = [_up(n, block) for n in total]
    blocks = max(1, sum(held)) + 3
    tables, _, _ = _tables(gen, held, max(1, max(held)), blocks)
    s["tables"], s["lengths"] = tables, _ints(total)
    s["k_cache"] = _codes(gen, (blocks, heads, block, dim), code, 1.0)
    s["v_cache"] = _codes(gen, (blocks, heads, block // 16, dim, 16), code, 1.0)
    s["k_scale"] = _scales(gen, (blocks, heads), code)
    s["v_scale"] = _scales(gen, (blocks, heads), code)
    typ = TYPE[case["type"]]
    if case["op"] == "append":
        rows = sum(c for _, c in ragged)
        host, touched = tables.cpu(), []
        slots = []
        for r, (a, c) in enumerate(ragged):
            slots += [int(host[r, p // block]) * block + p % block for p in range(a, a + c)]
            if c:
                touched += [int(host[r, b]) for b in range(a // block, _up(a + c, block))]
        # the rows come as slices of one fused projection [rows, K and V, heads, dim]
        kv = torch.randn(max(1, rows), 2, heads, dim, generator=gen, device="cuda")
        kv *= torch.exp(torch.randn(1, 1, 1, dim, generator=gen, device="cuda") * 0.5)
        s["kv"] = kv[:rows].to(typ)
        s["slots"] = _ints(slots)
        s["read"] = (_ints(touched)[:, None] * block + torch.arange(block, dtype=torch.int32, device="cuda")).reshape(-1)
        # the blocks' earlier tokens have a smaller spread than the rows, so most of their scales grow
        s["k_scale"] *= 0.8
        s["v_scale"] *= 0.8
        return s
    rows = sum(n for n, _ in ragged)
    starts = [0]
    for n, _ in ragged:
        starts.append(starts[-1] + n)
    s["row_start"] = _ints(starts)
    s["q"] = (torch.randn(rows + case["pad"], case["heads"], dim, generator=gen, device="cuda") * 2).to(typ)
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(rows + case["pad"], case["heads"], dtype=torch.float32, device="cuda")
    s["max_rows"] = case["rows_max"]
    return s


# ------------------------------------------------------------------------------------- plain forms
def _plain_plan(s):
    block, max_rows = s["case"]["block"], s["max_rows"]
    start, count, held, tables, ring = (s[k].long() for k in ("start", "count", "held", "tables", "ring"))
    head, free = s["ring_state"].long()
    width, cap = tables.shape[1], ring.numel()
    live = count >= 0
    n = count.clamp(min=0)
    need = torch.where(live, (torch.div(start + n + block - 1, block, rounding_mode="floor") - held).clamp(min=0), 0)
    gone = torch.where(live, 0, held)
    before = torch.cumsum(need, 0) - need
    back = torch.cumsum(gone, 0) - gone
    j = torch.arange(width, device=start.device)
    new = (j >= held[:, None]) & (j < (held + need)[:, None])
    tables = torch.where(new, ring[(head + before[:, None] + j - held[:, None]) % cap], tables)
    freed = (j < gone[:, None])
    at = torch.where(freed, (head + free + back[:, None] + j) % cap, cap)
    longer = torch.cat([ring, ring[:1]])
    longer.scatter_(0, at.reshape(-1), tables.reshape(-1))
    row_start = torch.cat([torch.zeros_like(n[:1]), torch.cumsum(n, 0)])
    t = torch.arange(max_rows, device=start.device)
    r = torch.searchsorted(row_start[1:].contiguous(), t, right=True).clamp(max=n.numel() - 1)
    p = start[r] + t - row_start[r]
    used = t < row_start[-1]
    slot = tables[r, torch.div(p, block, rounding_mode="floor").clamp(0, width - 1)] * block + p % block
    moved = torch.stack([(head + need.sum()) % cap, free - need.sum() + gone.sum()])
    out = dict(row_start=row_start, slots=torch.where(used, slot, -1), positions=torch.where(used, p, -1),
               lengths=torch.where(live, start + n, 0), held=torch.where(live, held + need, 0), ring_state=moved, tables=tables,
               ring=longer[:-1])
    return {k: v.to(torch.int32) for k, v in out.items()}


def _as_codes(x, code):
    if code == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _over(x, y):
    return torch.where(y > 0, x / torch.where(y > 0, y, torch.ones_like(y)), torch.zeros_like(x))


def _plain_append_one(x, slots, cache, scale, case, is_v):
    """x [rows, heads, dim] f32 into cache (codes) with scale [blocks, heads]: in place."""
    block, code = case["block"], case["code"]
    blocks = cache.shape[0]
    b = torch.div(slots, block, rounding_mode="floor")
    off = slots % block
    amax = torch.zeros(blocks, x.shape[1], device=x.device).index_reduce_(0, b, x.abs().amax(2), "amax")
    first = torch.full((blocks,), block, dtype=torch.long, device=x.device).scatter_reduce_(0, b, off, "amin")
    touched, kept = (first < block)[:, None], (first > 0)[:, None]
    fresh = torch.maximum(amax / QMAX[code], torch.where(kept, scale, torch.zeros_like(scale)))
    fresh = torch.where(touched, fresh, scale)
    grew = touched & kept & (fresh > scale)
    ratio = torch.where(grew, _over(scale, fresh), torch.ones_like(scale))
    ratio = ratio[:, :, None, None, None] if is_v else ratio[:, :, None, None]
    cache.copy_(_as_codes(cache.float() * ratio, code))
    q = _as_codes(_over(x, fresh[b][:, :, None].expand_as(x)), code)
    raw, q = (t.view(torch.int8) for t in (cache, q))
    if is_v:
        raw[b, :, torch.div(off, 16, rounding_mode="floor"), :, off % 16] = q
    else:
        raw[b, :, off] = q
    scale.copy_(fresh)


def _token_major(cache, is_v):
    """Codes as [blocks, block, heads, dim] in 32 bits."""
    x = cache.float()
    if is_v:
        b, h, g, d, _ = x.shape
        return x.permute(0, 2, 4, 1, 3).reshape(b, g * 16, h, d)
    return x.permute(0, 2, 1, 3)


def _plain_append(s):
    case, slots = s["case"], s["slots"].long()
    read = s["read"].long()
    block = case["block"]
    out = {}
    for i, name in enumerate(("k", "v")):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        if slots.numel():
            _plain_append_one(s["kv"][:, i].float(), slots, cache, scale, case, name == "v")
        b = torch.div(read, block, rounding_mode="floor")
        values = _token_major(cache, name == "v")[b, read % block] * scale[b][:, :, None]
        out[name], out[name + "_scale"] = values.to(TYPE[case["type"]]), scale
    return out


def _limits(pos, length, mask_block):
    """How many keys a query at `pos` of a request with `length` tokens sees."""
    if mask_block == 0:
        lim = length.expand_as(pos)
    else:
        lim = torch.minimum((torch.div(pos, mask_block, rounding_mode="floor") + 1) * mask_block, length)
    return torch.where(pos >= 0, lim, torch.zeros_like(lim))


def _plain_attend(s):
    case = s["case"]
    hq, hk, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    rows, lengths, requests = case["rows_max"], s["lengths"].long(), case["requests"]
    width = s["tables"].shape[1]
    table = s["tables"].long().clamp(min=0)

    def values(name):  # [requests, kv heads, width * block, dim]
        x = _token_major(s[name + "_cache"], name == "v") * s[name + "_scale"][:, None, :, None]
        return x[table].reshape(requests, width * block, hk, dim).permute(0, 2, 1, 3)

    first = s["row_start"].long()
    n = first[1:] - first[:-1]
    i = torch.arange(rows, device=n.device)
    row = (first[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    has = i < n[:, None]
    q = s["q"].float()[row].reshape(requests, rows, hk, hq // hk, dim).permute(0, 2, 3, 1, 4).reshape(requests, hk, -1, dim)
    x = q @ values("k").transpose(2, 3) * (1 / math.sqrt(dim))
    x = x.reshape(requests, hk, hq // hk, rows, width * block)
    lim = _limits(lengths[:, None] - n[:, None] + i, lengths[:, None], case["mask_block"])
    seen = torch.arange(width * block, device=n.device) < lim[:, :, None]
    x = torch.where(seen[:, None, None], x, torch.full_like(x, -math.inf))
    top = x.amax(4, keepdim=True)
    x = torch.exp(x - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = x.sum(4, keepdim=True)
    o = (x.reshape(requests, hk, -1, width * block) @ values("v")).reshape(requests, hk, hq // hk, rows, dim)
    o = torch.where(total > 0, o / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros_like(o))
    lse = (top + torch.log(total))[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(requests, rows, hq, dim).to(s["q"].dtype)
    lse = lse.permute(0, 3, 1, 2).reshape(requests, rows, hq)
    out, lses = s["out"].clone(), s["lse"].clone()
    out[row[has]], lses[row[has]] = o[has], lse[has]
    return dict(out=out, lse=lses)


def _plain_score(s):
    case = s["case"]
    x = s["logits"].float()
    rows, vocab = x.shape
    j = torch.arange(vocab, device=x.device)
    if case["exclude"] >= 0:
        x = torch.where(j == case["exclude"], torch.full_like(x, -math.inf), x)
    tok = s["tokens"].long()[:, None]
    mine = x.gather(1, tok)
    rank = ((x > mine) | ((x == mine) & (j < tok))).sum(1)
    order = torch.sort(x, dim=1, descending=True, stable=True)  # equal values: the lowest index first
    ids, best = order.indices[:, : case["top"]], order.values[:, : case["top"]]
    unit = 1 / case["temperature"] if case["temperature"] > 0 else 1.0
    top = x.amax(1, keepdim=True)
    z = (x - top) * unit
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    inner = torch.where(e > 0, e * z, torch.zeros_like(z)).sum(1, keepdim=True)
    entropy = (log_total - inner / total)[:, 0]
    listed_ = torch.isfinite(best)
    return dict(logprob=((mine - top) * unit - log_total)[:, 0], entropy=entropy, rank=rank.to(torch.int32),
                top_token=torch.where(listed_, ids, -1).to(torch.int32), top_logprob=(best - top) * unit - log_total)


_PLAIN = dict(plan=_plain_plan, append=_plain_append, attend=_plain_attend, score=_plain_score)


# ------------------------------------------------------------------------------------ framework's
def _own_plan(s):
    from diffusorrt_b200 import kernels

    p = kernels.plan_cache(s["start"], s["count"], s["held"], s["tables"], s["ring"], s["ring_state"],
                           block_size=s["case"]["block"], max_rows=s["max_rows"], held_out=s["held_out"],
                           ring_state_out=s["ring_state_out"])
    return dict(row_start=p.row_start, slots=p.slots, positions=p.positions, lengths=p.lengths, held=p.held,
                ring_state=p.ring_state, tables=s["tables"], ring=s["ring"])


def _own_append(s):
    from diffusorrt_b200 import kernels

    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    kernels.append_cache_q8(s["kv"][:, 0], s["kv"][:, 1], s["slots"], *cache)
    k, v = kernels.read_cache_q8(s["read"], *cache, dtype=TYPE[s["case"]["type"]])
    return dict(k=k, k_scale=s["k_scale"], v=v, v_scale=s["v_scale"])


def _own_attend(s):
    from diffusorrt_b200 import kernels

    out, lse = kernels.attend_cache_q8(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["tables"],
                                       s["lengths"], s["row_start"], mask_block=s["case"]["mask_block"],
                                       max_rows=s["max_rows"], out=s["out"], lse=s["lse"])
    return dict(out=out, lse=lse)


def _own_score(s):
    from diffusorrt_b200 import kernels

    case = s["case"]
    p = kernels.select_logprobs(s["logits"], s["tokens"], top=case["top"], temperature=case["temperature"],
                                exclude_token=case["exclude"])
    return dict(logprob=p.logprob, entropy=p.entropy, rank=p.rank, top_token=p.top_token, top_logprob=p.top_logprob)


_OWN = dict(plan=_own_plan, append=_own_append, attend=_own_attend, score=_own_score)


def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


# ------------------------------------------------------------------------------------------- work
def _visible(case, n, length):
    """Key positions that the n rows of a request of this length see, summed; and the most that one sees."""
    b, total, most = case["mask_block"], 0, 0
    for i in range(n):
        p = length - n + i
        lim = 0 if p < 0 else length if b == 0 else min(length, (p // b + 1) * b)
        total, most = total + lim, max(most, lim)
    return total, most


def work(case):
    if case["op"] == "score":
        size = 4 if case["type"] == "fp32" else 2
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * size + case["rows"] * (16 + 8 * case["top"]), flops=n * 5)
    ragged, block = _ragged(case), case["block"]
    if case["op"] == "plan":
        rows = sum(max(c, 0) for _, c in ragged)
        new = sum(max(0, _up(a + c, block) - _up(a, block)) for a, c in ragged if c >= 0)
        gone = sum(_up(a, block) for a, c in ragged if c < 0)
        seen = sum(_up(a + c, block) - a // block for a, c in ragged if c > 0)
        return dict(bytes=24 * len(ragged) + 8 * (new + gone) + 4 * seen + 8 * rows, flops=4 * rows + 8 * len(ragged))
    heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "append":
        rows = sum(c for _, c in ragged)
        back = block * sum(_up(a + c, block) - a // block for a, c in ragged if c)
        one = heads * dim * 2  # K and V
        return dict(bytes=rows * one * 3 + back * one * 3, flops=rows * one * 3 + back * one)
    seen = [_visible(case, n, length) for n, length in ragged]
    rows = sum(n for n, _ in ragged)
    return dict(bytes=sum(m for _, m in seen) * heads * dim * 2 + rows * case["heads"] * (dim * 4 + 4),
                flops=4 * dim * case["heads"] * sum(t for t, _ in seen))


# ------------------------------------------------------------------------------------------ exact
def _nearest(x, code):
    """The nearest value that a code stands for (ties to even), in 64 bits."""
    if code == "int8":
        return x.round().clamp(-127, 127)
    step = 2.0 ** (torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_append(case, s):
    """Block by block: the definition on the block's tokens, in 64 bits."""
    block, most = case["block"], QMAX[case["code"]]
    out = {}
    for i, name in enumerate(("k", "v")):
        cache, scale = s[name + "_cache"].cpu(), s[name + "_scale"].cpu().double()
        held = cache.float().double()
        if name == "v":
            held = held.permute(0, 1, 2, 4, 3).reshape(cache.shape[0], cache.shape[1], block, case["dim"])
        x = s["kv"][:, i].cpu().double()
        by_block = {}
        for row, slot in enumerate(s["slots"].tolist()):
            by_block.setdefault(slot // block, []).append((slot % block, row))
        for b, run_ in by_block.items():
            off, row = [o for o, _ in run_], [r for _, r in run_]
            mine = x[row].permute(1, 0, 2)  # heads, tokens, dim
            new = mine.abs().amax((1, 2)) / most
            if min(off) > 0:
                new = torch.maximum(new, scale[b])
                held[b] = _nearest(held[b] * (scale[b] / new)[:, None, None], case["code"])
            held[b][:, off] = _nearest(mine / new[:, None, None], case["code"])
            scale[b] = new
        read = s["read"].cpu().long()
        values = held[read // block, :, read % block] * scale[read // block][:, :, None]
        out[name], out[name + "_scale"] = values, scale
    return out


def _exact_attend(case, s):
    out, lse = s["out"].double(), s["lse"].double()
    dim, block, group = case["dim"], case["block"], case["heads"] // case["kv_heads"]
    first = s["row_start"].tolist()
    tables, lengths = s["tables"].cpu(), s["lengths"].tolist()
    for r, length in enumerate(lengths):
        ids = tables[r, : _up(length, block)].long().cuda()
        rows = slice(first[r], first[r + 1])
        n = first[r + 1] - first[r]
        at = torch.arange(length - n, length, device="cuda")
        for h in range(case["kv_heads"]):
            k = s["k_cache"][ids, h].double() * s["k_scale"][ids, h].double()[:, None, None]
            v = s["v_cache"][ids, h].double() * s["v_scale"][ids, h].double()[:, None, None, None]
            k = k.reshape(-1, dim)[:length]
            v = v.transpose(2, 3).reshape(-1, dim)[:length]
            for g in range(h * group, (h + 1) * group):
                x = s["q"][rows, g].double() @ k.T / math.sqrt(dim)
                if case["mask_block"]:
                    end = (at // case["mask_block"] + 1) * case["mask_block"]
                    x.masked_fill_(torch.arange(length, device="cuda")[None] >= end[:, None], -math.inf)
                x.masked_fill_((at < 0)[:, None], -math.inf)
                total = torch.logsumexp(x, 1)
                out[rows, g] = torch.nan_to_num(torch.exp(x - total[:, None])) @ v
                lse[rows, g] = total
    return dict(out=out, lse=lse)


def _exact_score(case, s):
    x = s["logits"].double()
    if case["exclude"] >= 0:
        x[:, case["exclude"]] = -math.inf
    if case["temperature"] > 0:
        x /= case["temperature"]
    lp = x - torch.logsumexp(x, 1, keepdim=True)
    entropy = -torch.where(torch.isfinite(lp), torch.exp(lp) * lp, torch.zeros_like(lp)).sum(1)
    best = torch.topk(lp, case["top"], 1).values
    return dict(logprob=lp.gather(1, s["tokens"].long()[:, None])[:, 0], entropy=entropy, rank=None, top_token=None,
                top_logprob=best)


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    return dict(append=_exact_append, attend=_exact_attend, score=_exact_score)[case["op"]](case, s)
