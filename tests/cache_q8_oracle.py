"""Plain restatements (Python loops, float64) of the paged 8-bit cache operators and the token scorer."""
from __future__ import annotations

import math

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def plan(start, count, held, tables, ring, ring_state, block, max_rows):
    """drt_cache_plan on Python lists (tables and ring are copied): a dict of its outputs."""
    tables, ring, held = [list(t) for t in tables], list(ring), list(held)
    head, free = ring_state
    width = len(tables[0]) if tables else 1
    need, status = [], 0
    for s, c, h in zip(start, count, held):
        if s < 0 or c < -1 or h < 0 or h > width:
            status = -4
        need.append(max(0, -(-(s + c) // block) - h) if c >= 0 else 0)
    gone = [h if c < 0 else 0 for c, h in zip(count, held)]
    if not 0 <= head < len(ring) or not 0 <= free <= len(ring):
        status = -4
    if status == 0 and any(c >= 0 and s + c > width * block for s, c in zip(start, count)):
        status = -2
    if status == 0 and sum(max(c, 0) for c in count) > max_rows:
        status = -3
    if status == 0 and free - sum(need) + sum(gone) > len(ring):
        status = -4
    if status == 0 and sum(need) > free:
        status = sum(need) - free
    if status != 0:
        return dict(row_start=[0] * (len(start) + 1), slots=[-1] * max_rows, positions=[-1] * max_rows,
                    lengths=[max(0, s) for s in start], held=held, ring_state=[head, free], status=status, tables=tables,
                    ring=ring)
    taken, back = 0, []
    for r, n in enumerate(need):
        for i in range(n):
            tables[r][held[r] + i] = ring[(head + taken) % len(ring)]
            taken += 1
        back += tables[r][:gone[r]]
    for i, b in enumerate(back):
        ring[(head + free + i) % len(ring)] = b
    row_start, slots, positions, lengths = [0], [], [], []
    for r, (s, c) in enumerate(zip(start, count)):
        held[r] = held[r] + need[r] if c >= 0 else 0
        lengths.append(s + c if c >= 0 else 0)
        for p in range(s, s + max(c, 0)):
            slots.append(tables[r][p // block] * block + p % block)
            positions.append(p)
        row_start.append(len(slots))
    pad = [-1] * (max_rows - len(slots))
    return dict(row_start=row_start, slots=slots + pad, positions=positions + pad, lengths=lengths, held=held,
                ring_state=[(head + taken) % len(ring), free - taken + len(back)], status=0, tables=tables, ring=ring)


def to_code(x, dtype):
    """Nearest code (ties to even, saturating, NaN to 0) of f32 values."""
    x = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf).clamp(-QMAX[dtype], QMAX[dtype])
    return x.round().to(torch.int8) if dtype == torch.int8 else x.to(torch.float8_e4m3fn)


def token_major(cache, is_v):
    """Codes [blocks, heads, block, dim] as f32."""
    x = cache.float()
    return x.permute(0, 1, 2, 4, 3).reshape(x.shape[0], x.shape[1], -1, x.shape[3]) if is_v else x


def append(x, slots, cache, scale, is_v):
    """Rows x [rows, heads, dim] into copies of cache and scale, in f32 steps: codes equal bit for bit."""
    dtype = cache.dtype
    held, scale = token_major(cache, is_v).clone(), scale.clone()
    block = held.shape[2]
    x = x.float()
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= held.shape[0] * block:
            t += 1
            continue
        b, off, m = slots[t] // block, slots[t] % block, 1
        while off + m < block and t + m < len(slots) and slots[t + m] == slots[t] + m:
            m += 1
        for h in range(x.shape[1]):
            rows = x[t:t + m, h]
            mag = rows.abs()
            amax = torch.where(torch.isfinite(mag), mag, torch.zeros_like(mag)).max()
            old = scale[b, h] if off > 0 else torch.tensor(0.0)
            s = torch.maximum(amax / QMAX[dtype], old)
            if off > 0 and s > old:
                held[b, h] = to_code(held[b, h] * (old / s), dtype).float()
            codes = torch.zeros_like(rows) if s == 0 else rows / s
            held[b, h, off:off + m] = to_code(codes, dtype).float()
            scale[b, h] = s
        t += m
    return held, scale


def limit(p, length, mask_block, origin):
    if p < 0:
        return 0
    if mask_block == 0:
        return length
    if p < origin:
        return min(origin, length)
    return min(origin + ((p - origin) // mask_block + 1) * mask_block, length)


def attend(q, k_cache, v_cache, k_scale, v_scale, tables, lengths, row_start, mask_block, origin, scale, out, lse):
    """(out, lse, tol_out, tol_lse) in float64 on the CPU; the tolerances bound the operator's rounding errors.

    u = 2^-24. A score is an f32 sum of dim exact products (each addition off by at most 2u of the sum of
    magnitudes B, allowing for truncation) and three products with scales: |ds| <= (2 dim + 6) u B, with
    B = scale ks sum |q k|. The reference maximum subtracted and the exponential's argument cost u times their size
    and ex2.approx 2^-22; p is then off by e = 2 (max |ds| + 4 u max |s|) + 2^-21 relative, twice for numerator and
    denominator. Each weight is rounded to f16: 2^-11 of itself or 2^-25 of the largest weight. O is an f32 sum
    over at most n keys. Then one rounding to the output type."""
    u = 2.0 ** -24
    out, lse = out.double().clone(), lse.double().clone()
    tol_out, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    eps = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal
    dim = q.shape[2]
    group = q.shape[1] // k_cache.shape[1]
    kc, vc = token_major(k_cache, False).double(), token_major(v_cache, True).double()
    block = kc.shape[2]
    for r in range(len(lengths)):
        n = row_start[r + 1] - row_start[r]
        blocks = [int(tables[r][j]) for j in range(-(-lengths[r] // block))]
        good = torch.tensor([0 <= b < kc.shape[0] for b in blocks], dtype=torch.bool)
        ids = torch.tensor([b if 0 <= b < kc.shape[0] else 0 for b in blocks], dtype=torch.long)
        shown = good.repeat_interleave(block)[:lengths[r]]
        for h in range(k_cache.shape[1]):
            k = (kc[ids, h] * k_scale[ids, h].double()[:, None, None]).reshape(-1, dim)[:lengths[r]]
            v = (vc[ids, h] * v_scale[ids, h].double()[:, None, None]).reshape(-1, dim)[:lengths[r]]
            vs = v_scale[ids, h].double().repeat_interleave(block)[:lengths[r]]
            for i in range(n):
                lim = limit(lengths[r] - n + i, lengths[r], mask_block, 0 if origin is None else origin[r])
                see = shown[:lim].nonzero()[:, 0]
                for g in range(h * group, (h + 1) * group):
                    row = row_start[r] + i
                    if see.numel() == 0:
                        out[row, g], lse[row, g] = 0.0, -math.inf
                        continue
                    qq = q[row, g].double()
                    s = (k[see] @ qq) * scale
                    B = (k[see].abs() @ qq.abs()).max() * scale
                    total = torch.logsumexp(s, 0)
                    p = torch.exp(s - total)
                    out[row, g], lse[row, g] = p @ v[see], total
                    ds = (2 * dim + 6) * u * B
                    e = 2 * (ds + 4 * u * s.abs().max()) + 2.0 ** -21
                    size = p @ v[see].abs()
                    w = (p * vs[see]).max()  # the largest weight, in the output's units per code
                    code = QMAX[k_cache.dtype]
                    tol_out[row, g] = (eps * out[row, g].abs() + (2 * e + 2.0 ** -11 + see.numel() * 2 * u) * size
                                       + see.numel() * 2.0 ** -25 * w * code + tiny)
                    tol_lse[row, g] = ds + 8 * u * (s.abs().max() + total.abs() + 1) + 2.0 ** -21 + see.numel() * 2 * u
    return out, lse, tol_out, tol_lse


def score(logits, tokens, top, temperature, exclude):
    """Per row (logprob, entropy, rank, top tokens, top log probabilities) in float64 on the CPU."""
    res = []
    for x, t in zip(logits.double(), tokens):
        x = x.clone()
        if exclude >= 0:
            x[exclude] = -math.inf
        z = x / temperature if temperature > 0 else x
        none = bool((x == -math.inf).all())
        # the maximum is taken off first: beside logits of 3e38 a logarithm of a sum has no bits left
        d = z - z[~torch.isnan(z)].max() if not none else z
        lp = d - torch.logsumexp(d, 0) if not none else z
        inner = torch.where(torch.isfinite(lp) | torch.isnan(lp), torch.exp(lp) * lp, torch.zeros_like(lp)).sum()
        given = 0 <= t < x.numel()
        idx = torch.arange(x.numel())
        rank = int(((x > x[t]) | ((x == x[t]) & (idx < t))).sum()) if given else -1
        order = sorted((i for i in range(x.numel()) if x[i] > -math.inf), key=lambda i: (-float(x[i]), i))[:top] if top else []
        ids = order + [-1] * (top - len(order))
        res.append((float(lp[t]) if given else -math.inf, 0.0 if none else float(-inner), rank, ids,
                    [float(lp[i]) if i >= 0 else -math.inf for i in ids]))
    return res
