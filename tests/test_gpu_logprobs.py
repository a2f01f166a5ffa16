"""The token scorer on the GPU against float64 (tests/cache_q8_oracle.py)."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

import cache_q8_oracle as oracle  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kernels():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from diffusorrt_b200 import build

    build.build()
    from diffusorrt_b200 import kernels as k

    return k


def close(got, want, tol):
    if math.isnan(want):
        return math.isnan(got)
    return got == want if math.isinf(want) else abs(got - want) <= tol


def check(kernels, x, tokens, top=0, temperature=0.0, exclude=-1, view=None, **more):
    """u = 2^-24: z = (x - m) / T is off by 2u of itself, e^z by that times |z| plus 2^-21 (ex2.approx and the
    reference's rounding), and terms weigh e^z, where |z| e^z <= 1: S is off by 2^-20 relative and the f32 sums
    over a lane's terms (under 2^7 roundings each) by 2^-17 at most; the entropy sum weighs its terms by |z| <= 40
    wherever e^z counts in f32. The result is rounded once more."""
    want = oracle.score(x, tokens, top, temperature, exclude)
    dev = view(x) if view else x.cuda()
    p = kernels.select_logprobs(dev, torch.tensor(tokens, dtype=torch.int32, device="cuda"), top=top, temperature=temperature,
                                exclude_token=exclude, **more)
    torch.cuda.synchronize()
    p = [t.cpu().tolist() for t in p]
    for r, (lp, ent, rank, ids, lps) in enumerate(want):
        tol = 2.0 ** -17 + 2.0 ** -23 * (abs(lp) if math.isfinite(lp) else 0)
        assert close(p[0][r], lp, tol), (r, p[0][r], lp)
        assert close(p[1][r], ent, 40 * 2.0 ** -18), (r, p[1][r], ent)
        assert p[2][r] == rank and p[3][r] == ids, (r, p[2][r], rank, p[3][r], ids)
        for a, b in zip(p[4][r], lps):
            assert close(a, b, 2.0 ** -17 + 2.0 ** -23 * (abs(b) if math.isfinite(b) else 0))


def rows(seed, n, vocab, typ=torch.float32, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, vocab, generator=g) * spread).to(typ), torch.randint(0, vocab, (n,), generator=g).tolist()


@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab,top,temperature", [(1, 1, 0.0), (7, 9, 0.5), (100, 32, 0.0), (1023, 5, 1.5), (1024, 3, 0.7),
                                                   (2049, 0, 0.0), (5000, 20, 0.2), (40001, 32, 0.0)])
def test_sizes_and_types(kernels, typ, vocab, top, temperature):
    """bf16 and f16 rows hold many equal logits: ranks and alternatives go by the lowest id."""
    x, tokens = rows(vocab, 3, vocab, typ)
    check(kernels, x, tokens, top, temperature)


def test_many_rows(kernels):
    x, tokens = rows(1, 300, 4111)
    check(kernels, x, tokens, 4, exclude=17)


@pytest.mark.parametrize("exclude", [0, 5, 2047, 2048, 4094])
def test_excluded_token(kernels, exclude):
    x, tokens = rows(2, 4, 4095, torch.bfloat16)
    x[:, exclude] = 30.0
    tokens[0] = exclude
    check(kernels, x, tokens, 6, 0.9, exclude)


def test_strides_and_row_index(kernels):
    """Rows that begin inside a 16-byte vector, and gathered rows, one of them twice."""
    for typ in (torch.float32, torch.bfloat16):
        x, tokens = rows(3, 5, 3001, typ)

        def odd(x):
            y = torch.full((5, 3007), 90.0, dtype=typ, device="cuda")
            y[:, 3:3004] = x.cuda()
            return y[:, 3:3004]

        check(kernels, x, tokens, 7, view=odd)
        low = x.clone()
        low[:, ::2] = -math.inf
        check(kernels, low, [0, 2, 4, 3000, 1], 7, view=odd)
        pick = [4, 0, 0, 2]
        check(kernels, x[pick], tokens[:4], 7, view=lambda _: odd(x),
              row_index=torch.tensor(pick, dtype=torch.int32, device="cuda"))


def test_row_index_outside_the_logits(kernels):
    """Such a row reads nothing and scores nothing; its neighbours are as ever."""
    x, tokens = rows(9, 3, 5000, torch.bfloat16)
    index = torch.tensor([1, -1, 3, 2**31 - 1, 0], dtype=torch.int32, device="cuda")
    given = torch.tensor([5, 6, 7, 8, tokens[0]], dtype=torch.int32, device="cuda")
    p = kernels.select_logprobs(x.cuda(), given, top=3, row_index=index)
    q = kernels.select_logprobs(x.cuda()[[1, 0]], given[[0, 4]], top=3)
    for a, b in zip(p, q):
        assert torch.equal(a[[0, 4]], b)
    for r in (1, 2, 3):
        assert p.logprob[r] == -math.inf and p.entropy[r] == 0 and p.rank[r] == -1
        assert p.top_token[r].tolist() == [-1] * 3 and p.top_logprob[r].tolist() == [-math.inf] * 3


def test_equal_logits(kernels):
    """More equal logits than the candidate list holds: the lowest ids win."""
    x = torch.zeros(3, 30000)
    x[1, 100:] = -1.0
    x[2, ::3] = 2.0
    check(kernels, x, [29999, 5, 4], 20)


@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16])
def test_fewer_segments_than_alternatives(kernels, typ):
    """Rows whose alternatives are bounded by lanes' maxima: equal ones, all in one lane, hardly any, none."""
    x, _ = rows(10, 7, 6001, typ)
    x[0] = 0.5
    x[1, 40:] = -math.inf
    x[2] = -math.inf
    x[3] = -5.0
    x[3, 3000:3040] = torch.arange(40).to(typ) / 8
    x[4, 1:] = -math.inf
    x[5, ::2] = math.nan
    x[5, 1::2] = 1.0
    check(kernels, x[[0, 1, 2, 3, 4, 6]], [6000, 3, 5, 3001, 0, 17], 32, exclude=3002)
    p = kernels.select_logprobs(x.cuda(), torch.zeros(7, dtype=torch.int32, device="cuda"), top=32)
    # a NaN is no alternative
    assert p.top_token[5].tolist() == list(range(1, 65, 2)) and bool(torch.isnan(p.logprob[5]))


def test_masked_infinite_and_nan_logits(kernels):
    x, _ = rows(4, 8, 2500)
    x[0] = -math.inf                         # nothing can be drawn
    x[1] = -math.inf
    x[1, 2400] = -5.0                        # one token only
    x[2, 5:] = -math.inf
    x[3] = torch.finfo(torch.float32).min    # every logit the type's lowest value
    x[4, 10] = math.nan
    x[5, 20] = math.inf
    x[6, :] = -math.inf
    x[6, 3] = math.nan
    x[7, 1:] = torch.finfo(torch.float32).min
    check(kernels, x[:4], [3, 2400, 7, 9], 6)
    check(kernels, x[7:], [0], 6)
    p = kernels.select_logprobs(x[4:7].cuda(), torch.tensor([1, 20, 3], dtype=torch.int32, device="cuda"), top=3)
    assert bool(torch.isnan(p.logprob).all()) and bool(torch.isnan(p.entropy).all())
    assert p.rank.tolist()[1] == 0
    assert p.top_token[1, 0].item() == 20 and 10 not in p.top_token[0].tolist() and p.top_token[2].tolist() == [-1, -1, -1]


def test_tokens_outside_the_vocabulary(kernels):
    x, _ = rows(5, 3, 600)
    check(kernels, x, [-1, 600, 599], 2)


def test_no_rows(kernels):
    p = kernels.select_logprobs(torch.zeros(0, 50, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), top=3)
    assert p.logprob.numel() == 0 and tuple(p.top_token.shape) == (0, 3)


def test_full_vocabulary_batch_stream_and_graph(kernels):
    """A serving batch at the 0.6B model's vocabulary: on another stream, and captured and replayed with new logits."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(40, 151936, device="cuda", generator=g) * 3
    tok = x.argmax(1).to(torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def want(x):
        lp = torch.log_softmax(x.double(), 1)
        return lp.gather(1, tok.long()[:, None])[:, 0], -(lp.exp() * lp).sum(1), torch.topk(lp, 5, 1)

    def compare(p, x):
        lp, ent, best = want(x)
        assert float((p.logprob.double() - lp).abs().max()) <= 2.0 ** -17 + 2.0 ** -23 * float(lp.abs().max())
        assert float((p.entropy.double() - ent).abs().max()) <= 40 * 2.0 ** -18
        assert torch.equal(p.top_token.long(), best.indices)

    p = kernels.select_logprobs(x, tok, top=5, stream=side)
    torch.cuda.synchronize()
    compare(p, x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = kernels.select_logprobs(x, tok, top=5)
    x.copy_(torch.randn(x.shape, device="cuda", generator=g) * 2)
    graph.replay()
    torch.cuda.synchronize()
    compare(p, x)
