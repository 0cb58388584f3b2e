"""Log probabilities of given tokens, ranks, entropy and alternatives.

Tolerances, from the formulas.  Ranks and tokens are whole numbers and compared exactly.  S is a sum of exponentials that are off by at
most 2^-21 of themselves (argument |d| <= 16 rounded twice: 2 * 16 * 1.45 * 2^-24, and 2^-22 for the function; smaller terms count less),
added in float32 by a thread in at most V / 512 + 16 additions (V / 512 * 2^-24 of the sum) and joined in float64.  So log S is off by
at most e = 2^-20 + V 2^-33, and a log probability by that and one rounding, 2^-24 of it.  T is such a sum of p d with |d| <= 200 p-weighted:
off by e of the sum of |p d|, so the entropy by e (1 + 2 T / S) and one rounding."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
NAN, INF = float("nan"), float("inf")


def ops():
    from slipstream_b200 import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def expected(logits, tokens, top):
    """(log p, entropy, ranks, top log p, top tokens, sum of p |d|) in 64 bits; rows that have NaN or nothing are not for this."""
    z = logits.to(F64)
    log_p = torch.log_softmax(z, dim=1)
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(dim=1)
    own = z.gather(1, tokens[:, None].long())
    index = torch.arange(z.shape[1], device=z.device)
    ranks = 1 + ((z > own) | ((z == own) & (index < tokens[:, None]))).sum(dim=1)
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
    d = torch.where(p > 0, p * (z.amax(dim=1, keepdim=True) - z), torch.zeros_like(p)).sum(dim=1)
    return log_p.gather(1, tokens[:, None].long())[:, 0], entropy, ranks.int(), log_p.gather(1, order), order.int(), d


def close(got, ref, off):
    finite = torch.isfinite(ref)
    assert torch.equal(got[~finite].to(F64), ref[~finite])
    assert torch.all((got.to(F64) - ref).abs()[finite] <= (off + ref.abs() * 2.0 ** -23)[finite])


def check(got, logits, tokens, top):
    v = logits.shape[1]
    lp, entropy, ranks, top_lp, top_tokens, d = expected(logits, tokens, top)
    e = torch.full_like(lp, 2.0 ** -20 + v * 2.0 ** -33)
    assert got.packed.shape == (len(tokens), 3 + 2 * top) and got.top_tokens.shape == got.top_logprobs.shape == (len(tokens), top)
    assert got.ranks.dtype == got.top_tokens.dtype == torch.int32
    close(got.logprobs, lp, e)
    close(got.entropy, entropy, e * (1 + 2 * d))
    assert torch.equal(got.ranks, ranks) and torch.equal(got.top_tokens, top_tokens)
    close(got.top_logprobs, top_lp, e[:, None].expand_as(top_lp))


VOCABULARIES = [1, 2, 3, 5, 7, 8, 9, 31, 64, 100, 511, 1000, 2047, 2049, 4096, 8193, 16387, 32003, 50257, 65537, 151936]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocabulary", VOCABULARIES)
def test_token_logprobs(vocabulary, dtype):
    o = ops()
    for rows, pad, shift, wide in [(1, 0, 0, True), (3, 0, 0, False), (9, 5, 1, True), (70, 3, 3, False), (150, 8, 0, True), (400 if vocabulary < 60000 else 299, 0, 0, False)]:
        g = gen(vocabulary + rows)
        logits = (torch.randn(rows, vocabulary + pad, generator=g, device=DEV) * 3).to(dtype)[:, shift:shift + vocabulary]
        tokens = torch.randint(0, vocabulary, (rows,), generator=g, device=DEV)
        tokens[0], tokens[-1] = 0, vocabulary - 1
        for top in {0, 1, min(5, vocabulary), min(20, vocabulary), min(64, vocabulary)}:
            check(o.token_logprobs(logits, tokens if wide else tokens.int(), top=top), logits, tokens, top)
    o.check_errors(torch.device(DEV))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 5, 40, 200, 600])
def test_ties_and_masks(rows, dtype):
    """Few distinct values, so that nearly everything ties; rows of one value; nearly everything masked; both zeros; falling and rising
    rows and rows whose largest values all stand in one thread's vectors, where the bound on the alternatives keeps out the least."""
    o = ops()
    for vocabulary in (70, 1003, 20011, 152064):
        g = gen(rows + vocabulary)
        logits = torch.randint(-3, 4, (rows, vocabulary), generator=g, device=DEV).float()
        logits[0] = 2.5
        logits[rows // 2] = torch.where(torch.rand(vocabulary, generator=g, device=DEV) < 0.999, torch.full((vocabulary,), -INF, device=DEV), logits[rows // 2])
        logits[rows // 2, 1] = 0.5
        logits[rows // 3, ::3] = -0.0
        logits[rows // 3, 1::3] = 0.0
        if rows > 4:
            line = torch.linspace(-50, 30, vocabulary, device=DEV)
            logits[1], logits[2] = line, line.flip(0)
            for v, r in ((4, 3), (8, 4)):  # vectors of one thread: 512 of them apart, in a row that one or several blocks share
                logits[r] = -2.0
                first = torch.arange(vocabulary, device=DEV)
                hot = (first // v) % 512 == 3
                logits[r, hot] = 5 + torch.rand(int(hot.sum()), generator=g, device=DEV)
        logits = logits.to(dtype)
        tokens = torch.randint(0, vocabulary, (rows,), generator=g, device=DEV)
        tokens[rows // 2] = 1
        for top in (0, 1, 20, 64):
            check(o.token_logprobs(logits, tokens, top=top), logits, tokens, top)
    o.check_errors(torch.device(DEV))


def test_token_at_every_place_of_a_small_row():
    """Ranks where the token stands in the head, the vectors or the tail of a row, with equal values on both sides."""
    o = ops()
    for dtype in (F32, BF16):
        for vocabulary in (13, 40):
            for shift in range(8):
                logits = torch.randint(0, 3, (vocabulary, vocabulary + 8), generator=gen(shift), device=DEV).to(dtype)[:, shift:shift + vocabulary]
                tokens = torch.arange(vocabulary, device=DEV)
                check(o.token_logprobs(logits, tokens, top=13), logits, tokens, 13)


def test_far_values():
    """Offsets and spreads at which a careless sum would overflow, cancel or vanish."""
    o, g = ops(), gen(1)
    for vocabulary in (1000, 40000):
        logits = torch.randn(8, vocabulary, generator=g, device=DEV)
        logits[1] += 1e4
        logits[2] -= 1e4
        logits[3] *= 1e3
        logits[4] *= 1e30
        logits[5, 17] = 200.0
        logits[6] = 1e38
        logits[6, 5] = -3e38
        logits[7] = -3e38
        tokens = torch.full((8,), 17, device=DEV)
        check(o.token_logprobs(logits, tokens, top=20), logits, tokens, 20)


def test_masked_tokens_and_rows_without_any():
    o = ops()
    for rows, vocabulary in ((6, 500), (6, 60000), (400, 60000)):
        logits = torch.full((rows, vocabulary), -INF, device=DEV)
        logits[0, 3], logits[0, 8] = 1.0, 2.0
        logits[2, vocabulary - 1] = -5.0
        logits[3, :] = NAN
        logits[4, 10] = NAN
        logits[4, 11] = 1.0
        logits[5, 10] = INF
        tokens = torch.zeros(rows, dtype=torch.int64, device=DEV)
        tokens[0], tokens[2], tokens[4] = 8, vocabulary - 1, 11
        got = o.token_logprobs(logits, tokens, top=4)
        lp = torch.log_softmax(torch.tensor([1.0, 2.0], dtype=F64, device=DEV), dim=0)
        assert abs(float(got.logprobs[0] - lp[1])) < 1e-6 and abs(float(got.entropy[0] + (lp.exp() * lp).sum())) < 1e-6 and int(got.ranks[0]) == 1
        assert got.top_tokens[0].tolist() == [8, 3, 0, 1] and got.top_logprobs[0, 2:].tolist() == [-INF, -INF]
        assert float(got.logprobs[2]) == 0.0 and float(got.entropy[2]) == 0.0 and got.top_tokens[2].tolist() == [vocabulary - 1, 0, 1, 2]
        # nothing but masked tokens; NaN; infinity: no numbers, and the order is still that of the values
        for r in (1, 3, 4, 5):
            assert torch.isnan(got.logprobs[r]) and torch.isnan(got.entropy[r]) and torch.isnan(got.top_logprobs[r]).all(), r
        assert got.top_tokens[1].tolist() == [0, 1, 2, 3] and int(got.ranks[1]) == 1
        assert got.top_tokens[3].tolist() == [-1] * 4 and int(got.ranks[3]) == 0
        assert got.top_tokens[4].tolist() == [11, 0, 1, 2] and int(got.ranks[4]) == 1
        assert got.top_tokens[5].tolist() == [10, 0, 1, 2]
        plain = o.token_logprobs(logits, tokens)
        assert torch.equal(plain.packed[:, :3].nan_to_num(7.0), got.packed[:, :3].nan_to_num(7.0))


def test_tokens_that_are_none_or_outside():
    o = ops()
    device = torch.device(DEV)
    logits = torch.randn(3, 1000, generator=gen(2), device=DEV)
    tokens = torch.tensor([5, -1, 7], device=DEV)
    got = o.token_logprobs(logits, tokens, top=3)
    assert torch.isnan(got.logprobs[1]) and int(got.ranks[1]) == 0 and torch.isfinite(got.entropy).all() and torch.isfinite(got.top_logprobs).all()
    o.check_errors(device)
    for bad in (1000, 2 ** 40):
        got = o.token_logprobs(logits, torch.tensor([5, bad, 7], device=DEV), top=3)
        assert torch.isnan(got.logprobs[1]) and int(got.ranks[1]) == 0 and torch.isfinite(got.logprobs[[0, 2]]).all()
        with pytest.raises(o.KernelError, match="token id"):
            o.check_errors(device)
    o.check_errors(device)


def test_alternatives_hold_what_the_token_says():
    """The token's own log probability is bit for bit that of the alternative at its rank."""
    o = ops()
    for rows, dtype in ((2, F32), (300, BF16)):
        logits = (torch.randn(rows, 30000, generator=gen(rows), device=DEV) * 3).to(dtype)
        first = o.token_logprobs(logits, torch.zeros(rows, dtype=torch.int32, device=DEV), top=20)
        for place in (0, 3, 19):
            got = o.token_logprobs(logits, first.top_tokens[:, place].contiguous(), top=0)
            assert (got.ranks == place + 1).all() and torch.equal(got.logprobs, first.top_logprobs[:, place])


def test_on_another_stream_and_in_graphs():
    o = ops()
    logits, tokens = torch.randn(12, 50257, generator=gen(3), device=DEV), torch.arange(12, device=DEV)
    torch.cuda.synchronize()
    now = o.token_logprobs(logits, tokens, top=5).packed
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        there = o.token_logprobs(logits, tokens, top=5).packed
    side.synchronize()
    assert torch.equal(there, now)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = o.token_logprobs(logits, tokens, top=5).packed
        graphs.append((graph, out))
    logits.copy_(torch.randn(12, 50257, generator=gen(4), device=DEV))
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    replayed = [out.clone() for _, out in graphs]
    now = o.token_logprobs(logits, tokens, top=5).packed
    assert torch.equal(replayed[0], now) and torch.equal(replayed[1], now)


def test_rows_past_32_bits():
    """A row that starts beyond 2^31 elements."""
    o = ops()
    stride = 2 ** 31 // 5 + 7
    store = torch.empty(7 * stride, dtype=BF16, device=DEV)
    logits = torch.as_strided(store, (7, 1001), (stride, 1))
    logits.copy_(torch.randn(7, 1001, generator=gen(5), device=DEV))
    tokens = torch.arange(7, device=DEV)
    check(o.token_logprobs(logits, tokens, top=5), logits, tokens, 5)


def test_refusals_and_empty_calls():
    o = ops()
    err = o.KernelError
    x, t = torch.zeros(4, 100, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for call in (lambda: o.token_logprobs(x.half(), t), lambda: o.token_logprobs(x.cpu(), t), lambda: o.token_logprobs(x, t.cpu()), lambda: o.token_logprobs(x[0], t),
                 lambda: o.token_logprobs(x.t(), t), lambda: o.token_logprobs(x[:, :0], t), lambda: o.token_logprobs(x, t[:3]), lambda: o.token_logprobs(x, t.float()),
                 lambda: o.token_logprobs(x, t[:, None]), lambda: o.token_logprobs(x, t, top=-1), lambda: o.token_logprobs(x, t, top=65), lambda: o.token_logprobs(x[:, :5], t, top=6),
                 lambda: o.token_logprobs(x, torch.zeros(8, dtype=torch.int64, device=DEV)[::2])):
        before = o.launch_count()
        with pytest.raises(err):
            call()
        assert o.launch_count() == before
    none = o.token_logprobs(x[:0], t[:0], top=2)
    assert none.packed.shape == (0, 7) and none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 2)
    before = o.launch_count()
    got = o.token_logprobs(x, t, top=2)
    assert o.launch_count() == before + 1 and got.top_tokens.tolist() == [[0, 1]] * 4
    with pytest.raises(TypeError):
        o.token_logprobs(x, t, top="two")
