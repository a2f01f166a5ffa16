"""The paged 8-bit K/V cache on the GPU: block tables, append, read back and attention against plain
loops in float64 (tests/cache_q8_oracle.py), one by one and as a serving step runs them together."""
from __future__ import annotations

import math
import random

import pytest

torch = pytest.importorskip("torch")

import cache_q8_oracle as oracle  # noqa: E402

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def kernels():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from diffusorrt_b200 import build

    build.build()
    from diffusorrt_b200 import kernels as k

    return k


def ints(v, device="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=device)


def bits(t):
    return t.view(torch.int8) if t.dtype == E4 else t


def random_cache(seed, blocks, heads, block, dim, code):
    g = torch.Generator().manual_seed(seed)
    spread = 36.0 if code == I8 else 120.0

    def codes(shape):
        return oracle.to_code(torch.randn(shape, generator=g) * spread, code)

    k, v = codes((blocks, heads, block, dim)), codes((blocks, heads, block // 16, dim, 16))
    ks, vs = (torch.exp(torch.randn(blocks, heads, generator=g) * 0.4) / spread for _ in range(2))
    return k, v, ks, vs


def cuda(*ts):
    return [t.cuda() for t in ts]


# ------------------------------------------------------------------------------------------ plan
def check_plan(kernels, start, count, held, tables, ring, state, block, max_rows, in_place=True):
    want = oracle.plan(start, count, held, tables, ring, state, block, max_rows)
    n, width = len(start), len(tables[0]) if tables else 1
    t, rg = ints(tables).reshape(n, width), ints(ring)
    h, st = ints(held).reshape(n), ints(state)
    more = {} if in_place else dict(held_out=torch.full_like(h, 7), ring_state_out=torch.full_like(st, 7))
    p = kernels.plan_cache(ints(start).reshape(n), ints(count).reshape(n), h, t, rg, st, block_size=block, max_rows=max_rows, **more)
    got = dict(row_start=p.row_start, slots=p.slots, positions=p.positions, lengths=p.lengths, held=p.held,
               ring_state=p.ring_state, tables=t, ring=rg)
    assert int(p.status[0]) == want["status"]
    for name, x in got.items():
        w = want[name] if n or name != "tables" else []
        assert x.reshape(-1).tolist() == ints(w).reshape(-1).tolist(), name
    if in_place:
        assert p.held is h and p.ring_state is st
    else:
        assert h.tolist() == list(held) and st.tolist() == list(state)
    return want


def serving_state(seed, requests, block, count_max, start_max, finished, spare=5):
    rng = random.Random(seed)
    start = [rng.randint(0, start_max) for _ in range(requests)]
    count = [-1 if rng.random() < finished else rng.randint(0, count_max) for _ in range(requests)]
    held = [-(-s // block) + rng.choice([0, 0, 1]) for s in start]
    need = sum(max(0, -(-(s + c) // block) - h) for s, c, h in zip(start, count, held) if c >= 0)
    width = max(max(h, -(-(s + max(0, c)) // block)) for s, c, h in zip(start, count, held)) + 1
    ids = list(range(sum(held) + need + spare))
    rng.shuffle(ids)
    tables, at = [], 0
    for h in held:
        tables.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    head = rng.randrange(len(ids))
    ring = [0] * len(ids)
    for i, b in enumerate(ids[at:]):
        ring[(head + i) % len(ring)] = b
    return start, count, held, tables, ring, [head, len(ids) - at], sum(max(0, c) for c in count)


@pytest.mark.parametrize("seed,requests,block,count_max,start_max,finished,pad", [
    (0, 1, 16, 1, 0, 0.0, 0), (1, 7, 32, 40, 100, 0.3, 5), (2, 64, 64, 1, 900, 0.1, 0), (3, 33, 16, 200, 50, 0.2, 1),
    (4, 1500, 16, 3, 60, 0.1, 9), (5, 700, 128, 60, 1000, 0.5, 0), (6, 5, 16, 3000, 10, 0.0, 17), (7, 40, 32, 0, 70, 0.0, 4)])
def test_plan(kernels, seed, requests, block, count_max, start_max, finished, pad):
    *state, rows = serving_state(seed, requests, block, count_max, start_max, finished)
    check_plan(kernels, *state, block, rows + pad, in_place=seed % 2 == 0)


def test_plan_many_requests_and_rows(kernels):
    *state, rows = serving_state(11, 5000, 16, 4, 30, 0.1)
    assert rows > 4096
    check_plan(kernels, *state, 16, rows + 3)


def test_plan_uneven_requests(kernels):
    """Fewer rows than requests, nearly all of them one request's, as one launch writes them."""
    start, count, held, tables, ring, state, _ = serving_state(12, 900, 16, 0, 40, 0.1, spare=200)
    tables = [row + [-1] * 45 for row in tables]
    count[17], count[400], count[880] = 600, 33, 1
    for max_rows in (634, 900, 901):
        check_plan(kernels, start, count, held, tables, ring, state, 16, max_rows)


def test_plan_without_requests(kernels):
    check_plan(kernels, [], [], [], [], [3, 4], [1, 2], 16, 3)


def test_plan_refusals_change_nothing(kernels):
    base = dict(start=[5, 40], count=[20, 3], held=[1, 3], tables=[[4, -1, -1, -1], [1, 2, 3, -1]], ring=[9, 8, 7, 0],
                state=[1, 1], block=16, max_rows=23)

    def status(**change):
        a = dict(base, **change)
        return check_plan(kernels, a["start"], a["count"], a["held"], a["tables"], a["ring"], a["state"], a["block"],
                          a["max_rows"])["status"]

    assert status() == 0
    assert status(state=[0, 0]) == 1          # a block is missing
    assert status(count=[60, 3]) == -2        # 65 tokens in four blocks of 16
    assert status(max_rows=22) == -3
    assert status(start=[-1, 40]) == -4
    assert status(count=[-2, 3]) == -4
    assert status(held=[5, 3]) == -4
    assert status(state=[4, 1]) == -4
    assert status(count=[20, -1], state=[1, 4]) == -4   # more free blocks than the ring holds
    assert status(max_rows=5000, state=[0, 0]) == 1     # the slots of a refused call with many rows


def test_plan_again_takes_nothing(kernels):
    """A window planned anew for its next denoising step keeps its blocks; so does a call that grows nothing."""
    tables, ring, st, held = ints([[3, -1, -1], [5, 6, -1]]), ints([0, 1, 2, 4]), ints([0, 4]), ints([1, 2])
    args = (ints([10, 20]), ints([32, 8]), held, tables, ring, st)
    a = kernels.plan_cache(*args, block_size=16, max_rows=64)
    first = [a.slots.tolist(), tables.tolist(), st.tolist(), held.tolist()]
    b = kernels.plan_cache(*args, block_size=16, max_rows=64)
    assert [b.slots.tolist(), tables.tolist(), st.tolist(), held.tolist()] == first
    assert st.tolist() == [2, 2] and held.tolist() == [3, 2]


# ------------------------------------------------------------------------------------------ append and read
def check_append(kernels, cache, k, v, slots, views=None):
    kc, vc, ks, vs = cache
    want_k, want_ks = oracle.append(k, slots, kc, ks, False)
    want_v, want_vs = oracle.append(v, slots, vc, vs, True)
    dev = cuda(kc, vc, ks, vs)
    dk, dv = views(k, v) if views else cuda(k, v)
    kernels.append_cache_q8(dk, dv, ints(slots), *dev)
    for got, want, is_v in ((dev[0], want_k, False), (dev[1], want_v, True)):
        assert torch.equal(oracle.token_major(got.cpu(), is_v).nan_to_num(nan=999.0), want.nan_to_num(nan=999.0))
    assert torch.equal(dev[2].cpu(), want_ks) and torch.equal(dev[3].cpu(), want_vs)
    return dev


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("heads,block,dim,typ,runs", [
    (2, 16, 64, BF, [(0, 0, 1)]), (1, 32, 128, HF, [(2, 5, 27), (0, 0, 32), (3, 31, 1)]), (3, 64, 128, BF, [(1, 17, 30)]),
    (2, 128, 64, HF, [(0, 0, 128), (2, 100, 28), (1, 0, 3)]), (5, 16, 128, BF, [(3, 15, 1), (1, 1, 15), (0, 0, 16)])])
def test_append(kernels, code, heads, block, dim, typ, runs):
    """Runs (block, offset, rows): new blocks, full ones, tails, single tokens; the codes equal bit for bit."""
    cache = random_cache(heads * block + dim, 4, heads, block, dim, code)
    g = torch.Generator().manual_seed(block)
    slots = [b * block + o + i for b, o, n in runs for i in range(n)]
    k, v = (torch.randn(len(slots), heads, dim, generator=g).to(typ) * s for s in (1.0, 6.0))
    check_append(kernels, cache, k.to(typ), v.to(typ), slots)


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("typ", [BF, HF])
def test_append_ties(kernels, code, typ):
    """Values between two codes: the f32 quotient decides, over 2,400 (block, head) scales of many sizes; zeros keep their signs."""
    block, heads, blocks = 16, 4, 300
    g = torch.Generator().manual_seed(7)
    cache = random_cache(7, blocks, heads, block, 64, code)

    def rows():
        top = torch.exp2(torch.rand(blocks, 1, heads, 1, generator=g) * 24 - 14).to(typ).float()  # of each block and head
        step = torch.randint(-254, 255, (blocks, block, heads, 64), generator=g).float()
        step[:, 3, :, 5] = 254
        x = (top * step / 254).to(typ)
        x[:, 7, :, 9] = -0.0
        return x.reshape(blocks * block, heads, 64)

    check_append(kernels, cache, rows(), rows(), list(range(blocks * block)))


def test_append_many_rows_and_skipped_slots(kernels):
    """Over 1024 rows a CTA looks for runs in 32 rows; slots of -1 and beyond the cache split runs and write nothing."""
    block, blocks = 32, 50
    cache = random_cache(1, blocks, 2, block, 64, I8)
    order = list(range(blocks))
    random.Random(0).shuffle(order)
    slots = [b * block + i for b in order[:40] for i in range(block)]
    slots[0:3] = [-1, -1, blocks * block]
    slots[700] = -1
    slots += [-1] * 5
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(len(slots), 2, 64, generator=g).to(BF) for _ in range(2))
    # the run after the gap at 700 lies in the same block as the one before it: its own call
    cut = slots[700 + 1:700 + block - 700 % block]
    slots[701:701 + len(cut)] = [-1] * len(cut)
    check_append(kernels, cache, k, v, slots)


def test_append_strided_and_misaligned(kernels):
    cache = random_cache(5, 3, 2, 16, 64, E4)
    g = torch.Generator().manual_seed(3)
    slots = list(range(16, 29))
    k, v = (torch.randn(13, 2, 64, generator=g).to(HF) for _ in range(2))

    def fused(k, v):  # slices of one projection
        x = torch.zeros(13, 5, 64, dtype=HF, device="cuda")
        x[:, 1:3], x[:, 3:5] = k.cuda(), v.cuda()
        return x[:, 1:3], x[:, 3:5]

    def odd(k, v):    # rows that start two bytes off a 16-byte boundary
        x = torch.zeros(2, 13, 2, 67, dtype=HF, device="cuda")
        x[0, :, :, 1:65], x[1, :, :, 1:65] = k.cuda(), v.cuda()
        return x[0, :, :, 1:65], x[1, :, :, 1:65]

    check_append(kernels, cache, k, v, slots, fused)
    check_append(kernels, cache, k, v, slots, odd)


@pytest.mark.parametrize("code", [I8, E4])
def test_append_extreme_values(kernels, code):
    """Zeros, the smallest numbers, infinities, NaN: none of them spoils the block's other values."""
    cache = random_cache(6, 3, 1, 16, 64, code)
    k = torch.zeros(20, 1, 64)
    k[3, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 2.0])
    k[16:] = 1e-38
    k[17, 0, 5] = -3e-39
    v = torch.full((20, 1, 64), 3e38)
    v[2, 0, 9] = math.nan
    check_append(kernels, cache, k.to(BF), v.to(BF), list(range(20)))
    only = torch.full((1, 1, 64), math.inf).to(BF)
    check_append(kernels, cache, only, torch.zeros(1, 1, 64).to(BF), [16])


def test_append_nothing(kernels):
    cache = random_cache(7, 2, 2, 16, 64, I8)
    empty = torch.zeros(0, 2, 64).to(BF)
    check_append(kernels, cache, empty, empty, [])


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("heads,block,dim,typ", [(2, 16, 64, BF), (3, 64, 128, HF), (1, 128, 128, torch.float32)])
def test_read(kernels, code, heads, block, dim, typ):
    """Aligned groups, odd orders, repeated and missing slots: scale * code rounded once."""
    kc, vc, ks, vs = random_cache(block, 4, heads, block, dim, code)
    rng = random.Random(block)
    slots = list(range(block, 2 * block)) + [rng.randrange(4 * block) for _ in range(21)] + [-1, 4 * block, 0, 0] + list(range(3, 19))
    k, v = kernels.read_cache_q8(ints(slots), *cuda(kc, vc, ks, vs), dtype=typ)
    for got, cache, scale, is_v in ((k, kc, ks, False), (v, vc, vs, True)):
        full = oracle.token_major(cache, is_v)
        want = torch.zeros(len(slots), heads, dim)
        for i, s in enumerate(slots):
            if 0 <= s < 4 * block:
                want[i] = full[s // block, :, s % block] * scale[s // block][:, None]
        assert torch.equal(got.cpu(), want.to(typ))


# ------------------------------------------------------------------------------------------ attention
def attend_case(seed, requests, heads, kv_heads, dim, block, code, typ, pad=0, blocks_extra=2, poison=False):
    """requests: (rows, length) each. Everything on the CPU; the caller moves it."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // block) for _, n in requests]
    blocks = sum(held) + blocks_extra
    cache = random_cache(seed, blocks, kv_heads, block, dim, code)
    order = torch.randperm(blocks, generator=g).tolist()
    width = max(1, max(held))
    tables, at = [], 0
    for h in held:
        tables.append(order[at:at + h] + [-1] * (width - h))
        at += h
    if poison:  # codes behind the last token, and scales of blocks that nobody holds
        k, v, ks, vs = cache
        for (_, n), h, row in zip(requests, held, tables):
            if n % block:
                b, o = row[h - 1], n % block
                bad = torch.full((1,), 0x7f, dtype=torch.int8)  # e4m3's NaN
                bits(k)[b, :, o:] = bad
                for t in range(o, block):
                    bits(v)[b, :, t // 16, :, t % 16] = bad
        for b in order[at:]:
            ks[b], vs[b] = math.nan, math.inf
    rows = sum(n for n, _ in requests)
    q = (torch.randn(rows + pad, heads, dim, generator=g) * 2).to(typ)
    starts = [0]
    for n, _ in requests:
        starts.append(starts[-1] + n)
    return q, cache, tables, [n for _, n in requests], starts


def check_attend(kernels, case, mask_block=1, origin=None, scale=None, max_rows=0, views=None, stream=None):
    q, cache, tables, lengths, starts = case
    out0, lse0 = torch.full_like(q, 3.0), torch.full(q.shape[:2], 5.0)
    use = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    want, want_lse, tol, tol_lse = oracle.attend(q, *cache, tables, lengths, starts, mask_block, origin, use, out0, lse0)
    dev = cuda(*cache)
    dq, out = views(q, out0) if views else (q.cuda(), out0.cuda())
    lse = lse0.cuda()
    got, got_lse = kernels.attend_cache_q8(dq, *dev, ints(tables), ints(lengths), ints(starts), mask_block=mask_block,
                                           origin=None if origin is None else ints(origin), scale=scale, max_rows=max_rows,
                                           out=out, lse=lse, stream=stream)
    torch.cuda.synchronize()
    assert got is out and got_lse is lse
    got, got_lse = got.cpu().double(), got_lse.cpu().double()
    off = (got - want).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol.clamp(min=1e-30)).max()):.3g} of the tolerance"
    inf = want_lse == -math.inf
    assert torch.equal(inf, got_lse == -math.inf)
    assert bool(((got_lse - want_lse).abs()[~inf] <= tol_lse[~inf]).all())
    last = starts[-1]
    assert bool((got[last:] == 3.0).all()) and bool((got_lse[last:] == 5.0).all())
    return got


@pytest.mark.parametrize("code", [I8, E4])
@pytest.mark.parametrize("typ", [BF, HF])
@pytest.mark.parametrize("dim,block", [(64, 16), (64, 128), (128, 16), (128, 32), (128, 64), (128, 128)])
def test_attend_single_tokens(kernels, code, typ, dim, block):
    """One row per request: lengths 1, around tiles and blocks, an empty request, padding rows."""
    requests = [(1, n) for n in (1, 15, 16, 17, 63, 64, 65, 0, 129, 300, 2)]
    check_attend(kernels, attend_case(dim + block, requests, 8, 4, dim, block, code, typ, pad=3))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (8, 1), (28, 4), (15, 5), (40, 1), (12, 2)])
def test_attend_head_layouts(kernels, heads, kv_heads):
    requests = [(1, 70), (3, 130), (0, 40), (9, 9)]
    check_attend(kernels, attend_case(heads, requests, heads, kv_heads, 64, 32, I8, BF))


@pytest.mark.parametrize("mask_block,origin", [(0, None), (1, None), (3, None), (8, [5, 100, 0, 7]), (32, None), (32, [200, 33, 1, 0]),
                                               (1, [16, 0, 40, 3])])
def test_attend_masks(kernels, mask_block, origin):
    """Causal, block and full masks, blocks counted from an origin inside, at and behind the rows."""
    requests = [(33, 100), (7, 64), (20, 20), (1, 50)]
    check_attend(kernels, attend_case(7, requests, 4, 2, 128, 32, E4, BF), mask_block, origin)


def test_attend_rows_before_the_first_token(kernels):
    """More rows than tokens: the rows before position 0 see nothing."""
    for mask_block in (0, 1, 4):
        check_attend(kernels, attend_case(8, [(5, 3), (4, 0), (2, 2), (70, 60)], 4, 2, 64, 16, I8, HF), mask_block)


@pytest.mark.parametrize("code", [I8, E4])
def test_attend_ignores_what_is_masked(kernels, code):
    """NaN codes behind a request's end, NaN and infinite scales of blocks that it does not hold."""
    requests = [(1, 1), (1, 17), (4, 77), (33, 130), (1, 0)]
    for dim in (64, 128):
        check_attend(kernels, attend_case(9, requests, 4, 2, dim, 32, code, BF, pad=2, poison=True))


def test_attend_bad_table_entries_hide_their_tokens(kernels):
    q, cache, tables, lengths, starts = attend_case(10, [(1, 100), (3, 40), (2, 32)], 4, 2, 128, 16, I8, BF)
    tables[0][2], tables[0][6], tables[1][0] = -1, 10 ** 6, 2 ** 31 - 1
    tables[2][0] = tables[2][1] = -5
    check_attend(kernels, (q, cache, tables, lengths, starts), 0)


def test_attend_length_beyond_the_table(kernels):
    """A length that the table cannot hold is taken as the table's."""
    q, cache, tables, lengths, starts = attend_case(11, [(1, 64)], 2, 2, 64, 16, I8, BF)
    got, _ = kernels.attend_cache_q8(q.cuda(), *cuda(*cache), ints(tables), ints([10 ** 9]), ints(starts))
    want, _ = kernels.attend_cache_q8(q.cuda(), *cuda(*cache), ints(tables), ints([64]), ints(starts))
    assert torch.equal(got, want)


@pytest.mark.parametrize("code", [I8, E4])
def test_attend_scales_of_every_size(kernels, code):
    """Block scales spread over 30 orders of magnitude, zero scales, and very large and small queries."""
    q, cache, tables, lengths, starts = attend_case(12, [(1, 150), (4, 260), (2, 33)], 4, 2, 128, 16, code, BF)
    k, v, ks, vs = cache
    g = torch.Generator().manual_seed(1)
    vs.copy_(10 ** (torch.rand(vs.shape, generator=g) * 30 - 15))
    vs[tables[0][1]] = 0.0
    vs[tables[2][0]] = vs[tables[2][1]] = vs[tables[2][2]] = 0.0   # this request's values are all zero
    ks[tables[1][3]] = 0.0
    q[1], q[2] = q[1] * 1e-30, (q[2].float() * 20).to(BF)
    check_attend(kernels, (q, cache, tables, lengths, starts), 0)


def test_attend_large_queries_take_one_key(kernels):
    """Scores in the thousands: one probability is 1 and the rest vanish."""
    q, cache, tables, lengths, starts = attend_case(13, [(1, 200), (5, 90)], 4, 2, 64, 32, E4, HF)
    check_attend(kernels, ((q * 200).to(HF), cache, tables, lengths, starts), 1, scale=1.0)


def test_attend_strides_and_misaligned_rows(kernels):
    case = attend_case(14, [(2, 70), (1, 33)], 4, 2, 64, 16, I8, BF, pad=1)

    def fused(q, out):
        x = torch.zeros(q.shape[0], 9, 64, dtype=BF, device="cuda")
        x[:, 2:6] = q.cuda()
        y = torch.zeros(4, q.shape[0], 64, dtype=BF, device="cuda").transpose(0, 1)
        y.copy_(out.cuda())
        return x[:, 2:6], y

    def odd(q, out):
        x = torch.zeros(q.shape[0], 4, 67, dtype=BF, device="cuda")
        x[:, :, 1:65] = q.cuda()
        return x[:, :, 1:65], out.cuda()

    for views in (fused, odd):
        check_attend(kernels, case, views=views)


def test_attend_long_axis_is_split_and_joined(kernels):
    """Long requests beside short ones: many shares of one unit, several units of one share."""
    for requests in ([(1, 9001)], [(1, 5000), (1, 3), (2, 700), (1, 64), (1, 1)], [(1, 100)] * 150 + [(1, 4000)]):
        check_attend(kernels, attend_case(15, requests, 4, 2, 64, 64, I8, BF), max_rows=2)


@pytest.mark.parametrize("dim,code,heads,rows", [(128, E4, 16, 1), (64, I8, 16, 1), (128, I8, 40, 1), (128, E4, 32, 5)])
def test_attend_many_units_and_tiles_to_a_share(kernels, dim, code, heads, rows):
    """More work than the GPU has warps: each goes through several units, of one tile and of many."""
    rng = random.Random(dim + heads)
    requests = [(rng.choice([1, rows]), rng.choice([0, 3, 64, 65, 200, 700, 1400])) for _ in range(120)]
    check_attend(kernels, attend_case(21, requests, heads, 16 if heads < 32 else 8, dim, 64, code, BF), max_rows=rows)


@pytest.mark.parametrize("mask_block", [0, 1, 32])
@pytest.mark.parametrize("dim,code,typ", [(128, I8, BF), (128, E4, HF), (64, E4, BF), (64, I8, HF)])
def test_attend_many_rows(kernels, mask_block, dim, code, typ):
    """Windows and prompt chunks beside single tokens."""
    requests = [(150, 190), (1, 70), (64, 64), (32, 333), (0, 5), (17, 400)]
    check_attend(kernels, attend_case(16, requests, 6, 2, dim, 32, code, typ, pad=4), mask_block)


@pytest.mark.parametrize("dim,code,typ", [(128, I8, BF), (64, E4, HF)])
def test_attend_rows_about_the_limit_between_the_kernels(kernels, dim, code, typ):
    """31 to 33 rows of a kv head, bounds that leave one kernel out, and a small request among large ones."""
    for heads, requests in ((8, [(8, 300), (5, 77), (8, 2000), (1, 64)]), (11, [(3, 300), (3, 1500)]), (31, [(1, 700), (1, 9)])):
        case = attend_case(23, requests, heads, 1 if heads > 8 else 2, dim, 64, code, typ)
        for bound in (0, max(n for n, _ in requests)):
            check_attend(kernels, case, max_rows=bound)
    check_attend(kernels, attend_case(24, [(32, 900), (32, 1290), (4, 70), (32, 333)], 8, 2, dim, 64, code, typ), 32, max_rows=32)


@pytest.mark.parametrize("dim,code,typ,heads,kv_heads", [(128, E4, BF, 4, 2), (64, I8, HF, 3, 1), (128, I8, HF, 2, 2)])
def test_attend_many_rows_over_long_prefixes(kernels, dim, code, typ, heads, kv_heads):
    """Units of many key tiles, cut between shares and joined; one and two row tiles; rows that the tile does not fill."""
    requests = [(129, 2500), (40, 3001), (0, 9), (7, 1100), (260, 260), (64, 640)]
    case = attend_case(22, requests, heads, kv_heads, dim, 128, code, typ, pad=2)
    for mask_block in (1, 32):
        check_attend(kernels, case, mask_block, origin=[100, 0, 0, 2000, 64, 7])


def test_attend_bound_on_rows_changes_nothing_but_speed(kernels):
    """max_rows is a hint: requests with more rows are served all the same."""
    case = attend_case(17, [(40, 100), (3, 80)], 8, 2, 128, 32, I8, BF)
    for bound in (0, 1, 5, 1000):
        check_attend(kernels, case, max_rows=bound)


def test_attend_same_bits_again(kernels):
    q, cache, tables, lengths, starts = attend_case(18, [(1, 3000), (33, 700), (1, 20)], 8, 2, 128, 64, E4, BF)
    args = (q.cuda(), *cuda(*cache), ints(tables), ints(lengths), ints(starts))
    a, b = (kernels.attend_cache_q8(*args) for _ in range(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dim", [64, 128])
def test_attend_most_requests(kernels, dim):
    """16,384 requests, the most that a call takes: empty ones between single tokens and windows, by one kernel and by both."""
    rng = random.Random(dim)
    requests = [(0, 0)] * 16384
    for r in rng.sample(range(16384), 60):
        requests[r] = (rng.choice([1, 3]), rng.choice([5, 70, 300]))
    for r in (0, 7001, 16383):
        requests[r] = (40, 200)
    case = attend_case(25, requests, 2, 1, dim, 64, I8, BF)
    check_attend(kernels, case)
    check_attend(kernels, attend_case(26, [(n if n < 9 else 1, m) for n, m in requests], 2, 1, dim, 64, E4, HF), max_rows=3)


def test_blocks_beyond_four_gigabytes(kernels):
    """The same rows through the first and the last blocks of a cache whose codes pass 32-bit offsets: the same bits."""
    heads, block, dim, blocks = 8, 128, 128, 35_000  # 4.6 GB each of K and V
    cache = kernels.cache_q8(blocks, heads, block, dim, dtype=I8)
    g = torch.Generator().manual_seed(8)
    k, v, q = (torch.randn(300, n, dim, generator=g).to(BF).cuda() for n in (heads, heads, 2 * heads))
    got = []
    for ids in ([0, 1, 2], [blocks - 1, blocks - 3, blocks - 2]):
        slots = torch.cat([torch.arange(block) + b * block for b in ids])[:300].to(torch.int32).cuda()
        kernels.append_cache_q8(k, v, slots, *cache)
        back = kernels.read_cache_q8(slots, *cache)
        tables, lengths = ints([ids]), ints([300])
        many = kernels.attend_cache_q8(q, *cache, tables, lengths, ints([0, 300]))
        few = kernels.attend_cache_q8(q[-2:], *cache, tables, lengths, ints([0, 2]), max_rows=2)
        got.append((*back, *many, *few))
    assert float(got[0][0].abs().max()) > 1
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_attend_nothing(kernels):
    q, cache, tables, lengths, starts = attend_case(19, [(1, 5)], 2, 2, 64, 16, I8, BF)
    out, lse = kernels.attend_cache_q8(q.cuda()[:0], *cuda(*cache), ints(tables), ints(lengths), ints([0, 0]))
    assert out.shape[0] == 0 and lse.shape[0] == 0
    out, _ = kernels.attend_cache_q8(q.cuda(), *cuda(*cache), ints(tables)[:0], ints([]).reshape(0), ints([0]))
    assert bool((out == 0).all())


def test_attend_on_another_stream_and_in_two_graphs(kernels):
    """Another stream with tensors made here; two graphs captured with their own scratch, replayed at once."""
    case = attend_case(20, [(1, 2000), (2, 90)], 8, 2, 128, 32, I8, BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    check_attend(kernels, case, stream=side)
    q, cache, tables, lengths, starts = case
    fixed = (*cuda(*cache), ints(tables), ints(lengths), ints(starts))
    want = kernels.attend_cache_q8(q.cuda(), *fixed)
    graphs, outs, queries = [], [], [q.cuda(), q.cuda() * 0.5]
    torch.cuda.synchronize()
    for x in queries:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kernels.attend_cache_q8(x, *fixed))
        graphs.append(graph)
    half = kernels.attend_cache_q8(queries[1], *fixed)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], want[0]) and torch.equal(outs[1][0], half[0])


# ------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("code", [I8, E4])
def test_serving_steps(kernels, code):
    """Prompts, a denoised block planned and written anew, single tokens, a finished request whose blocks the next
    one takes: plan, append and attention as a server runs them. Each row's attention is checked against the
    values that the cache holds (read back), and those against what was appended, to a code's rounding."""
    heads, kv_heads, dim, block, width, blocks = 8, 2, 64, 16, 12, 30
    cache = kernels.cache_q8(blocks, kv_heads, block, dim, dtype=code)
    tables = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    held, ring, state = ints([0, 0, 0]), torch.arange(blocks, dtype=torch.int32, device="cuda"), ints([0, blocks])
    g = torch.Generator().manual_seed(4)
    length, kept = [0, 0, 0], [[], [], []]
    free = blocks
    for step, (count, commit, mask_block) in enumerate([
            ([40, 0, 17], True, 1), ([32, 5, 1], False, 32), ([32, 5, 1], True, 32), ([1, 1, 1], True, 1), ([1, -1, 1], True, 1),
            ([0, 90, 3], True, 0)]):
        if count[1] == -1:
            length[1], kept[1] = 0, []
        rows = sum(max(0, c) for c in count)
        p = kernels.plan_cache(ints(length), ints(count), held, tables, ring, state, block_size=block, max_rows=rows + 2)
        assert int(p.status[0]) == 0
        k, v = (torch.randn(rows + 2, kv_heads, dim, generator=g).to(BF) for _ in range(2))
        q = torch.randn(rows + 2, heads, dim, generator=g).to(BF)
        kernels.append_cache_q8(k.cuda(), v.cuda(), p.slots, *cache)
        total = p.lengths.tolist()
        starts = p.row_start.tolist()
        for r in range(3):
            new = [(k[i], v[i]) for i in range(starts[r], starts[r + 1])]
            now = kept[r] + new
            assert total[r] == (len(now) if count[r] >= 0 else 0)
            if now and count[r] >= 0:
                at = kernels.plan_cache(ints([0]), ints([len(now)]), held[r:r + 1].clone(), tables[r:r + 1].clone(), ring.clone(),
                                        state.clone(), block_size=block, max_rows=len(now)).slots
                rk, rv = kernels.read_cache_q8(at, *cache, dtype=torch.float32)
                scale = torch.stack([cache[2], cache[3]])[:, (at // block).long()].cpu()
                for got, want, s in ((rk, [a for a, _ in now], scale[0]), (rv, [b for _, b in now], scale[1])):
                    want = torch.stack(want).float()
                    # half a code's step at the current scale for the last rounding, as much for each earlier one
                    # (at most one per append to the block, at a smaller scale); e4m3: half a step of the value
                    # (2^-4 relative, or half the smallest step 2^-9)
                    roundings = step + 1
                    one = 0.5 * s[:, :, None] if code == I8 else torch.maximum(want.abs() * 2.0 ** -4, s[:, :, None] * 2.0 ** -10)
                    assert bool(((got.cpu() - want).abs() <= roundings * one * 1.25 + 1e-6).all())
            if commit and count[r] >= 0:
                kept[r], length[r] = now, len(now)
        host = [t.cpu() for t in cache]
        check_attend(kernels, (q, host, tables.tolist(), total, starts), mask_block)
        free = blocks - sum(held.tolist())
        assert int(state[1]) == free
    ids = [b for r in range(3) for b in tables[r, :int(held[r])].tolist()]
    head = int(state[0])
    rest = [int(ring[(head + i) % blocks]) for i in range(free)]
    assert sorted(ids + rest) == list(range(blocks))


def test_captured_step(kernels):
    """Plan, append and attention captured once and replayed with other lengths, counts and rows."""
    kv_heads, dim, block = 2, 64, 16
    cache = kernels.cache_q8(20, kv_heads, block, dim)
    tables = torch.full((2, 8), -1, dtype=torch.int32, device="cuda")
    held, ring, state = ints([0, 0]), torch.arange(20, dtype=torch.int32, device="cuda"), ints([0, 20])
    start, count = ints([0, 0]), ints([0, 0])
    k, v, q = (torch.zeros(24, h, dim, dtype=BF, device="cuda") for h in (kv_heads, kv_heads, 4))

    def step():
        p = kernels.plan_cache(start, count, held, tables, ring, state, block_size=block, max_rows=24)
        kernels.append_cache_q8(k, v, p.slots, *cache)
        return (p, *kernels.attend_cache_q8(q, *cache, tables, p.lengths, p.row_start))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p, out, lse = step()
    g = torch.Generator().manual_seed(9)
    lengths = [0, 0]
    for counts in ([20, 3], [1, 1], [0, 16], [1, 1]):
        start.copy_(ints(lengths))
        count.copy_(ints(counts))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        lengths = [a + b for a, b in zip(lengths, counts)]
        assert int(p.status[0]) == 0 and p.lengths.tolist() == lengths
        starts = p.row_start.tolist()
        want, want_lse, tol, _ = oracle.attend(q.cpu(), *(t.cpu() for t in cache), tables.tolist(), lengths, starts, 1, None,
                                               1 / 8, out.cpu(), lse.cpu())
        n = starts[-1]
        assert bool(((out.cpu().double() - want).abs()[:n] <= tol[:n]).all())
