"""`logprobs.log_probs` against a plain 64-bit implementation: every kind of logits, row lengths around the vector, tile and cluster
sizes, strided and misaligned rows, masks, ties, orders that defeat the pruning of alternatives, rows that have no probabilities.

Tolerances. The kernel takes l - m exactly rounded (one rounding, 2^-24 relative), e^d by an approximation of 2 units (2^-22) of an
argument rounded twice (d log2 e: 2^-23 |d| absolute in the exponent's natural units), and sums with at most 200 roundings of 2^-24 in
a row (a thread's entries of a tile, its tiles, 8 + 4 levels of joining with a rescaling each): relative errors of S and T below
2^-22 + 2^-23 * 40 + 212 * 2^-24 < 2.1e-5 at the very worst (terms with |d| > 40 weigh nothing at the sizes here: V e^-40 < 1e-12). That is the absolute
error of ln S. log p adds a rounding of each of its two parts; H = ln S - T / S two relative errors of |T / S| <= ln V + 1 on top."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
SUM = 2.1e-5
FR = 24


def reference(x, tok, top, fr=FR):
    """Lists from a row of logits (Python's floats hold int64 logits of 53 bits) on the host, in 64 bits."""
    n, V = x.shape
    masked = x <= -(1 << 62) if x.dtype == torch.int64 else x == -math.inf
    z = (x - x.amax(1, keepdim=True)).double() * 2.0 ** -fr if x.dtype == torch.int64 else x.double()
    z = z.masked_fill(masked, -math.inf)
    alive = (z.amax(1) < math.inf) & (z.amax(1) > -math.inf)
    logp = torch.log_softmax(z, 1)
    ent = -(logp.exp() * logp).masked_fill(masked, 0.0).sum(1)
    order = torch.sort(x.masked_fill(masked, -(1 << 62)) if x.dtype == torch.int64 else x.double(), dim=1, descending=True, stable=True).indices
    ids = order[:, :top]
    ids = torch.cat([ids, torch.full((n, top - ids.shape[1]), -1, dtype=torch.long)], 1)
    none = (ids < 0) | masked.gather(1, ids.clamp(min=0))
    tl = logp.gather(1, ids.clamp(min=0)).masked_fill(none, -math.inf)
    ids = ids.masked_fill(none, -1)
    inside = (tok >= 0) & (tok < V)
    t = tok.clamp(0, V - 1)[:, None]
    rank = torch.where(inside & alive, (order == t).int().argmax(1) + 1, 0)
    lp = torch.where(inside & alive, logp.gather(1, t)[:, 0], math.nan)
    nan = ~alive
    return (lp, ent.masked_fill(nan, math.nan), rank, ids.masked_fill(nan[:, None], -1), tl.masked_fill(nan[:, None], math.nan))


def same(got, want, V):
    lp, ent, rank, ids, tl = want
    assert torch.equal(got.rank.cpu(), rank)
    assert torch.equal(got.top_ids.cpu(), ids)
    for g, w, size in ((got.logp, lp, 0.0), (got.top_logp, tl, 0.0), (got.entropy, ent, math.log(V) + 1)):
        g = g.double().cpu()
        fin = torch.isfinite(w)
        assert torch.equal(torch.isnan(g), torch.isnan(w)) and torch.equal(g[~fin & ~torch.isnan(w)], w[~fin & ~torch.isnan(w)])
        err, tol = (g - w)[fin].abs(), SUM * (1 + 2 * size) + 2.0 ** -22 * w[fin].abs()
        assert (err <= tol).all(), float((err - tol).max())


def make(n, V, kind, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, V, generator=g) * spread
    tok = torch.randint(V, (n,), generator=g)
    if kind == "int64":
        return (x.double() * 2.0 ** FR).round().long(), tok
    return x.to(getattr(torch, kind)), tok


KINDS = ("int64", "float32", "bfloat16")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,V,top", [(1, 1, 1), (3, 2, 5), (2, 7, 7), (5, 31, 32), (4, 1023, 3), (2, 2048, 20), (3, 2049, 0), (1, 40001, 32),
                                     (70, 5000, 8), (1, 128256, 20), (2, 128257, 1), (9, 70003, 5), (700, 300, 2)])
def test_against_64_bits(n, V, top, kind):
    from bitexact_llm_b200.logprobs import log_probs
    x, tok = make(n, V, kind, n + V)
    same(log_probs(x.cuda(), tok.cuda(), top), reference(x, tok, top), V)


@pytest.mark.parametrize("kind", KINDS)
def test_strided_and_misaligned_rows(kind):
    from bitexact_llm_b200.logprobs import log_probs
    x, tok = make(6, 9000, kind, 3)
    for a, b in ((0, 8999), (1, 9000), (3, 4100), (5, 6), (7, 2055)):
        part = x[::2, a:b]
        dev = x.cuda()[::2, a:b]
        t = tok[:3] % (b - a)
        same(log_probs(dev, t.cuda(), 6), reference(part, t, 6), b - a)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V", [700, 30011, 128256])
def test_masks_and_orders(kind, V):
    """Masked rows (one entry, few, a half, all but the first), constant rows, ascending and descending ones, ties across the row."""
    from bitexact_llm_b200.logprobs import log_probs
    low = -(1 << 62) if kind == "int64" else -math.inf
    base, tok = make(12, V, kind, V)
    x = base.clone()
    g = torch.Generator().manual_seed(1)
    x[0] = low
    x[0, V // 3] = base[0, 0]
    x[1][torch.rand(V, generator=g) < 0.999] = low
    x[2][torch.rand(V, generator=g) < 0.5] = low
    x[3, 0] = low
    x[4] = 0
    x[5] = base[5].sort().values
    x[6] = base[6].sort(descending=True).values
    x[7] = (torch.arange(V) % 7).to(x.dtype)
    x[8, : V // 2] = low
    x[9] = low
    x[10] = base[10].sort().values
    x[10, ::2] = low
    tok[0], tok[1], tok[8], tok[11] = V // 3, int((x[1] > low).nonzero()[-1]) if (x[1] > low).any() else 0, 1, V
    if kind == "int64":
        x[9] -= 5
        x[3, 0] = -(1 << 63)
    else:
        x[6, V // 2] = -0.0
    for top in (1, 20, 32):
        same(log_probs(x.cuda(), tok.cuda(), top), reference(x, tok, top), V)


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
def test_rows_without_probabilities(kind):
    from bitexact_llm_b200.logprobs import log_probs
    x, tok = make(5, 6000, kind, 2)
    x[0, 17] = math.nan
    x[1, 5999] = math.inf
    x[2] = -math.inf
    x[3] = -math.inf
    x[3, 40] = math.nan
    r = log_probs(x.cuda(), tok.cuda(), 4)
    for bad in range(4):
        assert r.rank[bad] == 0 and (r.top_ids[bad] == -1).all()
        assert torch.isnan(r.logp[bad]) and torch.isnan(r.entropy[bad]) and torch.isnan(r.top_logp[bad]).all()
    same(log_probs(x[4:].cuda(), tok[4:].cuda(), 4), reference(x[4:], tok[4:], 4), 6000)
    assert torch.isfinite(r.logp[4])


def test_extremes_and_other_points():
    """int64: values at both ends of the type, other binary points; float: values at the ends of the range."""
    from bitexact_llm_b200.logprobs import log_probs
    x = torch.full((3, 900), -(1 << 61), dtype=torch.long)
    x[0, 5], x[0, 6] = (1 << 62) + 3, (1 << 62) + 3 - (1 << 24)
    x[1, 7] = (1 << 63) - 1
    x[2, 8], x[2, 9] = -(1 << 62) + 1, -(1 << 63)
    tok = torch.tensor([6, 7, 9])
    r = log_probs(x.cuda(), tok.cuda(), 3)
    z = math.log1p(math.exp(-1.0))
    assert r.rank.tolist() == [2, 1, 900] and r.top_ids[:, 0].tolist() == [5, 7, 0] and r.top_ids[0].tolist() == [5, 6, 0]
    assert abs(float(r.logp[0]) + 1 + z) < SUM and abs(float(r.logp[1])) < SUM and r.logp[2] == -math.inf
    for fr in (0, 8, 16, 30, 40):
        x, tok = make(3, 3000, "float32", fr, 4.0)
        q = (x.double() * 2.0 ** fr).round().long()
        same(log_probs(q.cuda(), tok.cuda(), 4, fr=fr), reference(q, tok, 4, fr), 3000)
    big = torch.tensor([[3.0e38, -3.0e38, 1.0, -math.inf]]).cuda()
    r = log_probs(big, torch.tensor([1]).cuda(), 4)
    assert r.logp[0] == -math.inf and r.entropy[0] == 0 and r.top_ids.tolist() == [[0, 2, 1, -1]]


def test_no_tokens_no_rows_and_the_same_bits_again():
    from bitexact_llm_b200.logprobs import log_probs
    x, tok = make(40, 50000, "float32", 4)
    x, tok = x.cuda(), tok.cuda()
    r = log_probs(x, None, 3)
    assert r.logp is None and r.rank is None
    full = log_probs(x, tok, 3)
    assert torch.equal(r.entropy, full.entropy) and torch.equal(r.top_ids, full.top_ids)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(log_probs(x, tok, 3), full))
    empty = log_probs(x[:0], tok[:0], 3)
    assert empty.logp.shape == (0,) and empty.top_ids.shape == (0, 3)


def test_in_a_graph_and_on_another_stream():
    from bitexact_llm_b200.logprobs import log_probs
    x, tok = make(8, 20000, "int64", 5)
    dev, t = x.cuda(), tok.cuda()
    want = log_probs(dev, t, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = log_probs(dev, t, 5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = log_probs(dev, t, 5)
    x2, t2 = make(8, 20000, "int64", 6)
    dev.copy_(x2)
    t.copy_(t2)
    g.replay()
    same(got, reference(x2, t2, 5), 20000)


def test_of_an_engine_against_the_integer_log_p():
    """The same rows through `int_logp` (integer-defined, 2^-40): the float form agrees to its own tolerance."""
    from bitexact_llm_b200.exact.consts import ln_table
    from bitexact_llm_b200.logprobs import log_probs
    from bitexact_llm_b200.vllm_plugin import rl
    x, tok = make(20, 128256, "int64", 7)
    q = (x >> 8).cuda()                                     # 16 fractional bits, as int8 mode has
    want = rl.int_logp(q, tok.cuda(), ln_table(40, "cuda"), 16)
    # the integer rule's own error: entries of the table are off by 2^-45, its interpolation by (2^-12)^2 / 8
    assert ((log_probs(q, tok.cuda(), fr=16).logp.double() - want).abs() < SUM + 2.0 ** -22 * want.abs() + 1e-8).all()


def test_refusals():
    from bitexact_llm_b200.logprobs import log_probs
    x, tok = make(4, 100, "float32")
    dev, t = x.cuda(), tok.cuda()
    for bad in (lambda: log_probs(dev.double(), t), lambda: log_probs(dev[0], t), lambda: log_probs(dev.t(), t[:1]),
                lambda: log_probs(dev, t[:3]), lambda: log_probs(dev, t.int()), lambda: log_probs(dev, t, 33), lambda: log_probs(dev, t, -1),
                lambda: log_probs(dev, t, fr=41), lambda: log_probs(x, t), lambda: log_probs(dev, tok), lambda: log_probs(dev[:, :0], t),
                lambda: log_probs(dev[:1].expand(4, 100), t)):
        with pytest.raises(ValueError):
            bad()
