"""Keys and values in 4 bits: the rows that `gqa_store4` keeps against the definition in 64 bits, bit for bit, and `gqa_attention4` against a
plain 64-bit attention over the entries that the cache holds.

Tolerances of the attention. 32-bit: scores are sums of dim products in fp32 (relative to the sum of magnitudes: (dim + 16) 2^-24), weights
e^s with |s| <= S give e^s (1 + (S + 2) 2^-23) on top, sums of n weights (n / 64 + 70) 2^-24 more: with dim <= 300, S <= 60 and n <= 3000 an
output is off by less than 300 * 2^-24 * 60 * 2 ... of the largest |value|, 2.2e-3 at worst and in practice 1e-6; the tests hold the
errors to `F32` = 3e-5 of the largest magnitude of a row's values, which random signs keep by far. bf16: weights are rounded to 11 bits (2^-12
relative each, so the weighted mean moves by at most 2^-12 of the largest |value|, twice where the sum of the weights is not the rounded one's),
the exponentials are off by 2^-21, the output by 2^-8: 2^-11 of the largest |value| + 2^-8 of the output. The kernel of tall tiles
holds the codes of a value relative to the largest exponent of the sequence's values: what it loses is below 2^-36 of that one's entries."""

import math
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = ("bfloat16", "float32")
F32 = 3e-5
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
SCALES = torch.tensor([(c & 7) * 2.0 ** -9 if c < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10) for c in range(127)], dtype=torch.float64)


def kept(x):
    """The definition, in 64 bits: the entries that a row x [..., n] is kept as."""
    n = x.shape[-1]
    x = torch.nn.functional.pad(x.double().cpu(), (0, -n % 16)).clamp(-2.0 ** 127, 2.0 ** 127)
    most = x.abs().amax(-1, keepdim=True)
    e = torch.where(most > 0, torch.floor(torch.log2(most.clamp(min=2.0 ** -200))) - 10, -100.0).clamp(-100, 117)
    b = (x / 2.0 ** e).unflatten(-1, (-1, 16))
    s = torch.searchsorted(6 * SCALES, b.abs().amax(-1).contiguous())
    step = SCALES[s][..., None]
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])            # even codes first: the nearest, ties to them
    gap = (b.abs()[..., None] - GRID[order] * step[..., None]).abs()
    y = GRID[order][gap.argmin(-1)] * step * torch.sign(b)
    return (y.flatten(-2) * 2.0 ** e)[..., :n]


def spec(heads, kv_heads, dim, vdim, window=0, scale=None):
    return SimpleNamespace(heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, window=window, scale=scale or dim ** -0.5)


def rows(M, G, n, dtype, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(M, G, n, generator=g) * torch.exp(torch.randn(M, G, 1, generator=g)) * gain).to(getattr(torch, dtype))


# ---------------------------------------------------------------- rows

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,G,dim,vdim,page", [(1, 1, 1, 1, 64), (3, 2, 16, 40, 64), (5, 1, 64, 64, 128), (64, 8, 128, 128, 64), (70, 3, 24, 80, 192),
                                               (513, 2, 128, 64, 64), (1500, 1, 100, 130, 128), (600, 1, 512, 512, 64)])
def test_rows_are_kept_as_defined(M, G, dim, vdim, page, dtype):
    from bitexact_llm_b200.hybrid import ops
    sp = spec(G, G, dim, vdim)
    k, v = rows(M, G, dim, dtype, M), rows(M, G, vdim, dtype, M + 1, 0.2)
    nb = -(-M // page) + 2
    cache = ops.gqa_cache4(sp, nb, page, "cuda")
    slot = torch.randperm(nb * page, generator=torch.Generator().manual_seed(3))[:M]
    slot[M // 2:] = torch.arange(M - M // 2) + 5            # a run that begins off every boundary
    if M > 4:
        slot[: M // 2] = torch.arange(M // 2) + (nb * page - M // 2)
    ops.gqa_store4(k.cuda(), v.cuda(), slot.cuda(), cache)
    a, b = ops.gqa_read4(cache, sp, slot.cuda(), k.dtype)
    assert torch.equal(a.double().cpu(), kept(k)) and torch.equal(b.double().cpu(), kept(v))
    # nothing else was written
    rest = torch.ones(nb * page, dtype=torch.bool)
    rest[slot] = False
    empty = rest.nonzero()[:, 0][:2000].cuda()
    a, b = ops.gqa_read4(cache, sp, empty, torch.float32)
    assert not a.any() and not b.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_and_many_rows_leave_the_same_bytes(dtype):
    from bitexact_llm_b200.hybrid import ops
    sp = spec(2, 2, 128, 96)
    M = 700
    k, v = rows(M, 2, 128, dtype, 1).cuda(), rows(M, 2, 96, dtype, 2).cuda()
    slot = (torch.arange(M) + 64 * 3 + 7).cuda()
    one, many = (ops.gqa_cache4(sp, 16, 64, "cuda") for _ in range(2))
    ops.gqa_store4(k, v, slot, many)
    for i in range(0, M, 300):
        ops.gqa_store4(k[i:i + 300], v[i:i + 300], slot[i:i + 300], one)
    assert torch.equal(one, many) and one.any()


def test_extremes_ties_and_strides():
    from bitexact_llm_b200.hybrid import ops
    dim = 48
    x = torch.zeros(14, 1, dim)
    x[1] = torch.arange(dim) / 7.0
    x[2] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 6) * 1.5     # every tie, at a step of 1.5
    x[3] = -x[2]
    x[4] = x[2] * 2.0 ** -120
    x[5] = x[2] * 2.0 ** 120
    x[6, 0, 0], x[6, 0, 20], x[6, 0, 40] = 1.0, 2.0 ** -18, 2.0 ** -40              # blocks far below the row's largest entry
    x[7] = 1e-42
    x[8] = 3.3e38
    x[9] = 1e-30
    x[10, 0, 47] = -1e-3
    x[11] = 2.0 ** torch.arange(dim).float()
    x[12] = torch.linspace(-1, 1, dim)
    x[13] = 448 * 6
    wide = torch.zeros(14, 3, 2 * dim)
    wide[:, 1:2, 5:5 + dim] = x
    k = wide.cuda()[:, 1:2, 5:5 + dim]
    sp = spec(1, 1, dim, dim)
    cache = ops.gqa_cache4(sp, 2, 64, "cuda")
    slot = torch.arange(14).cuda() * 9
    ops.gqa_store4(k, -k, slot, cache)
    a, b = ops.gqa_read4(cache, sp, slot, torch.float32)
    assert torch.equal(a.double().cpu(), kept(x)) and torch.equal(b.double().cpu(), kept(-x))
    assert (a[5] / a[2] == 2.0 ** 120).logical_or(a[2] == 0).all() and torch.isfinite(a).all()


@pytest.mark.parametrize("M", [40, 700])
def test_padding_rows_and_rows_that_are_not_numbers(M):
    from bitexact_llm_b200.hybrid import ops
    sp = spec(2, 2, 64, 64)
    k, v = rows(M, 2, 64, "bfloat16", 1), rows(M, 2, 64, "bfloat16", 2)
    k[3, 0, 5], v[7, 1, 9], v[9, 0, 60] = math.nan, math.inf, -math.inf
    slot = torch.arange(M) + 1
    slot[11], slot[12], slot[13] = -1, 20 * 64, 1 << 40
    cache = ops.gqa_cache4(sp, 20, 64, "cuda")
    ops.gqa_store4(k.cuda(), v.cuda(), slot.cuda(), cache)
    a, b = (t.double().cpu() for t in ops.gqa_read4(cache, sp, slot.cuda(), torch.float32))
    for m, g in ((3, 0), (7, 1), (9, 0)):
        assert torch.isnan(a[m, g]).all() and not b[m, g].any()
        k[m, g], a[m, g], v[m, g], b[m, g] = 0, 0, 0, 0
    for m in (11, 12, 13):
        assert not a[m].any() and not b[m].any()
        k[m], v[m] = 0, 0
    assert torch.equal(a, kept(k)) and torch.equal(b, kept(v))


# ---------------------------------------------------------------- attention

def batch(sp, page, lens, new, dtype, seed, extra=1):
    """A cache of sequences of `lens` tokens on scattered pages, junk behind them, and queries for their last `new` tokens.
    -> q, cache, bt, seq, pos, keys and values held [S][tokens, G, entries]."""
    from bitexact_llm_b200.hybrid import ops
    T, G, S = getattr(torch, dtype), sp.kv_heads, len(lens)
    g = torch.Generator().manual_seed(seed)
    nblk = -(-max(lens) // page) + extra
    nb = S * nblk + 1
    cache = ops.gqa_cache4(sp, nb, page, "cuda")
    # everything is full of large values first: what lies behind a sequence must not matter
    junk = torch.arange(nb * page).cuda()
    ops.gqa_store4((1e4 * torch.randn(nb * page, G, sp.dim, generator=g)).to(T).cuda(), (1e6 * torch.randn(nb * page, G, sp.vdim, generator=g)).to(T).cuda(), junk, cache)
    bt = (torch.randperm(nb - 1, generator=g)[: S * nblk] + 1).view(S, nblk)
    held = []
    for s, n in enumerate(lens):
        t = torch.arange(n)
        slot = (bt[s, t // page] * page + t % page).cuda()
        k, v = torch.randn(n, G, sp.dim, generator=g).to(T).cuda(), (torch.randn(n, G, sp.vdim, generator=g) * 0.5).to(T).cuda()
        ops.gqa_store4(k, v, slot, cache)
        held.append(tuple(x.double().cpu() for x in ops.gqa_read4(cache, sp, slot, torch.float32)))
    per, M = sp.heads // G, sum(new)
    q = torch.full((G, M, per, (sp.dim + 7) // 8 * 8), 7.0).to(T)
    q[..., : sp.dim] = torch.randn(G, M, per, sp.dim, generator=g).to(T)
    seq = torch.repeat_interleave(torch.arange(S), torch.tensor(new))
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)])
    return q.cuda(), cache, bt.int().cuda(), seq.cuda(), pos.cuda(), held


def tiles_of(new, per):
    out, row, tall = [], 0, max(1, 128 // per)
    for s, n in enumerate(new):
        out += [[s, row + t, min(tall, n - t)] for t in range(0, n, tall)]
        row += n
    return torch.tensor(out, dtype=torch.int32).cuda()


def attention(q, sp, seq, pos, held, sink):
    G, M, per, _ = q.shape
    q = q[..., : sp.dim].double().cpu()
    out, big = torch.zeros(M, G, per, sp.vdim, dtype=torch.float64), torch.zeros(M, 1)
    for m in range(M):
        p, (k, v) = int(pos[m]), held[int(seq[m])]
        lo = max(0, p - sp.window + 1) if sp.window else 0
        z = torch.einsum("ghd,tgd->ght", q[:, m], k[lo:p + 1]) * sp.scale
        if sink is not None:
            z = torch.cat([z, sink.double().cpu().view(G, per, 1)], 2)
        w = torch.softmax(z, 2)[..., : p + 1 - lo]
        out[m] = torch.einsum("ght,tgd->ghd", w, v[lo:p + 1])
        big[m] = v[lo:p + 1].abs().amax()
    return out.flatten(1), big


def close(got, want, big, dtype):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    tol = F32 * big if dtype == "float32" else 2.0 ** -11 * big + 2.0 ** -8 * want.abs()
    err = (got - want).abs()
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()))


def run(sp, page, lens, new, dtype, seed, sink=False, tiles=False, variant=0, bt64=False):
    from bitexact_llm_b200.hybrid import ops
    q, cache, bt, seq, pos, held = batch(sp, page, lens, new, dtype, seed)
    s = torch.randn(sp.heads, generator=torch.Generator().manual_seed(seed)).cuda() if sink else None
    t = tiles_of(new, sp.heads // sp.kv_heads) if tiles else None
    out = ops.gqa_attention4(q, sp, cache, bt.long() if bt64 else bt, seq, pos, s, t, variant)
    want, big = attention(q, sp, seq, pos, held, s)
    close(out[:, : sp.heads * sp.vdim], want, big, dtype)


VARIANTS = (0, 1)
SHAPES = [(1, 1, 64, 64), (4, 1, 64, 64), (8, 2, 128, 128), (16, 2, 128, 64), (6, 3, 64, 128), (5, 5, 10, 13), (12, 2, 80, 100), (24, 2, 128, 128),
          (20, 1, 64, 64), (32, 1, 40, 64), (4, 2, 200, 96), (2, 1, 300, 260)]


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,vdim", SHAPES)
def test_single_tokens(heads, kv_heads, dim, vdim, dtype, variant):
    sp = spec(heads, kv_heads, dim, vdim)
    run(sp, 64, [1, 2, 63, 64, 65, 300, 130], [1] * 7, dtype, heads + dim, sink=heads % 2 == 0, variant=variant, bt64=heads % 3 == 0)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
def test_windows_and_pages(window, dtype, variant):
    run(spec(8, 2, 64, 128, window), 192, [1, 70, 191, 192, 193, 900], [1] * 6, dtype, window, sink=window == 5, variant=variant)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch_size,n", [(1, 3000), (2, 1500), (40, 200), (1, 64), (1, 65)])
def test_split_over_keys(batch_size, n, dtype):
    run(spec(8, 2, 128, 128), 64, [n] * batch_size, [1] * batch_size, dtype, n, sink=True)


@pytest.mark.parametrize("dtype,variant", [("bfloat16", 0), ("bfloat16", 1), ("bfloat16", 2), ("float32", 0)])
@pytest.mark.parametrize("heads,kv_heads,dim,vdim,window", [(4, 1, 64, 64, 0), (8, 2, 128, 128, 0), (6, 2, 128, 64, 33), (5, 5, 20, 30, 0), (16, 1, 64, 128, 70),
                                                            (136, 1, 64, 64, 0), (24, 2, 64, 64, 0)])
def test_prompt_portions(heads, kv_heads, dim, vdim, window, dtype, variant):
    """Whole prompts, portions behind a context, single tokens and a padding row among the tiles."""
    run(spec(heads, kv_heads, dim, vdim, window), 128, [150, 70, 33, 1, 260, 64], [150, 31, 1, 1, 130, 64], dtype, heads + window, sink=heads == 8, tiles=True, variant=variant)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[100], [3, 1, 40]])
def test_a_short_portion_behind_a_long_context(new, dtype):
    """Few tiles: their keys are split."""
    run(spec(8, 2, 128, 64), 64, [2500, 700, 1800][: len(new)], new, dtype, 5, sink=True, tiles=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("variant", VARIANTS)
def test_large_and_small_magnitudes(variant, dtype):
    """Keys and values far from 1, values of very different size in one sequence, queries of any size; weights of one key."""
    from bitexact_llm_b200.hybrid import ops
    sp = spec(4, 2, 64, 64)
    T, n = getattr(torch, dtype), 200
    g = torch.Generator().manual_seed(0)
    for gq, gk, gv in ((1e-6, 1e5, 1e8), (3e7, 1e-8, 1e-9), (1.0, 1.0, 1e30), (60.0, 1.0, 1.0)):
        k, v = (torch.randn(n, 2, 64, generator=g) * gk).to(T).cuda(), torch.randn(n, 2, 64, generator=g) * gv
        v *= 10.0 ** torch.randint(-4, 1, (n, 1, 1), generator=g)
        q = (torch.randn(2, 1, 2, 64, generator=g) * gq).to(T).cuda()
        cache, slot = ops.gqa_cache4(sp, 5, 64, "cuda"), torch.arange(n).cuda() + 64
        ops.gqa_store4(k, v.to(T).cuda(), slot, cache)
        held = [tuple(x.double().cpu() for x in ops.gqa_read4(cache, sp, slot, torch.float32))]
        bt, seq, pos = torch.arange(1, 5, dtype=torch.int32).cuda()[None], torch.zeros(1, dtype=torch.long).cuda(), torch.tensor([n - 1]).cuda()
        want, big = attention(q, sp, seq, pos, held, None)
        close(ops.gqa_attention4(q, sp, cache, bt, seq, pos, None, None, variant), want, big, dtype)
        many = q.expand(2, 90, 2, 64).contiguous()          # the same row in a tile of 90 tokens
        t = torch.tensor([[0, 0, 64], [0, 64, 26]], dtype=torch.int32).cuda()
        got = ops.gqa_attention4(many, sp, cache, bt, seq.expand(90).contiguous(), pos.expand(90).contiguous(), None, t, variant)
        close(got, want.expand(90, -1), big, dtype)


@pytest.mark.parametrize("dtype,variant", [("bfloat16", 0), ("bfloat16", 1), ("bfloat16", 2), ("float32", 0)])
@pytest.mark.parametrize("per", [1, 4])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("keys,values", [(1.0, 1e25), (1e20, 1.0), (1e20, 1e25)])
def test_large_tokens_cost_nothing_to_rows_that_do_not_see_them(keys, values, window, per, dtype, variant):
    """Tiles, tall ones and short ones, in which some tokens are larger by powers that no number of 16 bits spans: rows in front of them,
    or behind them by more than the window, keep the accuracy of their own values."""
    from bitexact_llm_b200.hybrid import ops
    sp, T, n, G, before = spec(2 * per, 2, 64, 128, window), getattr(torch, dtype), 300, 2, 70
    big = [100, 163, 164, 250, 299]
    k, v = rows(n, G, 64, dtype, 5).float(), rows(n, G, 128, dtype, 6).float()
    k[big] *= keys
    v[big] *= values
    cache, slot = ops.gqa_cache4(sp, 6, 64, "cuda"), torch.arange(n).cuda() + 64
    ops.gqa_store4(k.to(T).cuda(), v.to(T).cuda(), slot, cache)
    held = [tuple(x.double().cpu() for x in ops.gqa_read4(cache, sp, slot, torch.float32))]
    bt, M = torch.arange(1, 6, dtype=torch.int32).cuda()[None], n - before
    q = torch.randn(G, M, per, 64, generator=torch.Generator().manual_seed(7)).to(T)
    seq, pos = torch.zeros(M, dtype=torch.long).cuda(), torch.arange(before, n).cuda()
    want, size = attention(q, sp, seq, pos, held, None)
    for tall in (128 // per, 8 // per):
        t = torch.tensor([[0, i, min(tall, M - i)] for i in range(0, M, tall)], dtype=torch.int32).cuda()
        close(ops.gqa_attention4(q.cuda(), sp, cache, bt, seq, pos, None, t, variant)[:, : 2 * per * 128], want, size, dtype)


@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_a_number_stays_with_those_who_see_it(dtype, variant):
    from bitexact_llm_b200.hybrid import ops
    sp = spec(4, 2, 64, 64, 50)
    T, n, G = getattr(torch, dtype), 140, 2
    k, v = rows(n, G, 64, dtype, 1), rows(n, G, 64, dtype, 2)
    k[40, 0, 3], v[90, 1, 60] = math.nan, math.inf
    cache, slot = ops.gqa_cache4(sp, 4, 64, "cuda"), torch.arange(n).cuda() + 64
    ops.gqa_store4(k.cuda(), v.cuda(), slot, cache)
    q = torch.randn(G, n, 2, 64, generator=torch.Generator().manual_seed(3)).to(T).cuda()
    q[1, 5] = math.nan
    bt = torch.arange(1, 4, dtype=torch.int32).cuda()[None]
    seq, pos = torch.zeros(n, dtype=torch.long).cuda(), torch.arange(n).cuda()
    t = torch.tensor([[0, i, min(64, n - i)] for i in range(0, n, 64)], dtype=torch.int32).cuda()
    # two tiles of 64 and more rows, and single tokens
    for tiles in (None, t):
        out = ops.gqa_attention4(q, sp, cache, bt, seq, pos, None, tiles, variant).view(n, G, 2, 64).float().cpu()
        bad = torch.zeros(n, G, dtype=torch.bool)
        bad[40:90, 0] = True
        bad[90:, 1] = True
        bad[5, 1] = True
        assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_that_are_none_and_positions_beyond_the_table(dtype):
    """Page numbers outside the cache read page 0, positions are held to the table, a row in front of the sequence sees nothing."""
    from bitexact_llm_b200.hybrid import ops
    sp = spec(2, 1, 64, 64)
    q, cache, bt, seq, pos, held = batch(sp, 64, [100, 128], [1, 1], dtype, 1, extra=0)
    sink = torch.zeros(2).cuda()
    bad = bt.clone()
    bad[0, 0], bad[0, 1] = -5, 10 ** 6
    zero = bt.clone()
    zero[0] = 0
    a, b = (ops.gqa_attention4(q, sp, cache, t, seq, pos, None) for t in (bad, zero))
    assert torch.equal(a, b)
    far = pos.clone()
    far[1] = 10 ** 7
    assert torch.equal(ops.gqa_attention4(q, sp, cache, bt, seq, far, None)[1], ops.gqa_attention4(q, sp, cache, bt, seq, pos, None)[1])
    far[0] = -1
    for s in (None, sink):
        assert not ops.gqa_attention4(q, sp, cache, bt, seq, far, s)[0].any()


def test_the_same_bits_again_and_in_a_graph():
    from bitexact_llm_b200.hybrid import ops
    sp = spec(8, 2, 128, 128)
    q, cache, bt, seq, pos, held = batch(sp, 64, [500, 90, 1000], [1, 1, 1], "bfloat16", 1)
    want = ops.gqa_attention4(q, sp, cache, bt, seq, pos, None)
    for _ in range(5):
        assert torch.equal(ops.gqa_attention4(q, sp, cache, bt, seq, pos, None), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.gqa_attention4(q, sp, cache, bt, seq, pos, None)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    k, v = (torch.randn(3, 2, 128, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in (1, 2))
    slot = bt.long()[seq, pos // 64] * 64 + pos % 64
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.gqa_store4(k, v, slot, cache)
        got = ops.gqa_attention4(q, sp, cache, bt, seq, pos, None)
    k.mul_(0.5)
    g.replay()
    for s in range(3):
        held[s][0][-1], held[s][1][-1] = kept(k[s]), kept(v[s])
    want, big = attention(q, sp, seq, pos, held, None)
    close(got, want, big, "bfloat16")


def test_offsets_beyond_32_bits():
    """Pages behind 4 GB of cache."""
    from bitexact_llm_b200.hybrid import ops
    sp = spec(8, 8, 128, 128)
    nb = (5 << 30) // (8 * 9344)
    cache = ops.gqa_cache4(sp, nb, 64, "cuda")
    n = 100
    k, v = rows(n, 8, 128, "bfloat16", 1), rows(n, 8, 128, "bfloat16", 2)
    slot = torch.arange(n) + (nb - 2) * 64
    ops.gqa_store4(k.cuda(), v.cuda(), slot.cuda(), cache)
    held = [tuple(x.double().cpu() for x in ops.gqa_read4(cache, sp, slot.cuda(), torch.float32))]
    assert torch.equal(held[0][0], kept(k))
    q = rows(8, 1, 128, "bfloat16", 3).view(8, 1, 1, 128).cuda()
    bt, seq, pos = torch.tensor([[nb - 2, nb - 1]]).cuda(), torch.zeros(1, dtype=torch.long).cuda(), torch.tensor([n - 1]).cuda()
    want, big = attention(q, sp, seq, pos, held, None)
    close(ops.gqa_attention4(q, sp, cache, bt, seq, pos, None), want, big, "bfloat16")


def test_nothing():
    from bitexact_llm_b200.hybrid import ops
    sp = spec(2, 1, 64, 64)
    cache = ops.gqa_cache4(sp, 1, 64, "cuda")
    z = torch.zeros(0, dtype=torch.long, device="cuda")
    ops.gqa_store4(torch.zeros(0, 1, 64, device="cuda"), torch.zeros(0, 1, 64, device="cuda"), z, cache)
    assert ops.gqa_read4(cache, sp, z, torch.float32)[0].shape == (0, 1, 64)
    assert ops.gqa_attention4(torch.zeros(1, 0, 2, 64, device="cuda"), sp, cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), z, z, None).shape == (0, 128)


def test_refusals():
    from bitexact_llm_b200.hybrid import ops
    sp = spec(4, 2, 64, 64)
    cache = ops.gqa_cache4(sp, 3, 64, "cuda")
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device="cuda")
    slot = z(5, t=torch.int64)
    k = z(5, 2, 64)
    for bad in (lambda: ops.gqa_cache4(sp, 3, 16, "cuda"), lambda: ops.gqa_cache4(sp, 3, 96, "cuda"), lambda: ops.gqa_store4(k, z(5, 1, 64), slot, cache),
                lambda: ops.gqa_store4(k, k.float(), slot, cache), lambda: ops.gqa_store4(k.half(), k.half(), slot, cache),
                lambda: ops.gqa_store4(k, k, slot[:4], cache), lambda: ops.gqa_store4(k, k, slot.int(), cache),
                lambda: ops.gqa_store4(k, k, slot, cache[:, :1]), lambda: ops.gqa_store4(k, z(5, 2, 128), slot, cache),
                lambda: ops.gqa_store4(z(5, 2, 128)[..., ::2], k, slot, cache), lambda: ops.gqa_store4(k, k, slot, cache.cpu()),
                lambda: ops.gqa_read4(cache, sp, slot.int(), torch.float32), lambda: ops.gqa_read4(cache, sp, slot, torch.float16),
                lambda: ops.gqa_read4(cache, spec(4, 2, 128, 64), slot, torch.float32)):
        with pytest.raises(ValueError):
            bad()
    q, bt, pos = z(2, 5, 2, 64), z(1, 3, t=torch.int32), slot
    good = dict(q=q, spec=sp, cache=cache, bt=bt, seq=slot, pos=pos, sink=None)
    ops.gqa_attention4(**good)
    for change in (dict(q=q.half()), dict(q=z(1, 5, 2, 64)), dict(q=z(2, 5, 3, 64)), dict(q=z(2, 5, 2, 56)), dict(q=z(2, 2, 5, 64).transpose(1, 2)),
                   dict(cache=cache.view(torch.int8)), dict(bt=bt.float()), dict(bt=z(3, 2, t=torch.int32).t()), dict(seq=slot[:4]), dict(pos=slot.int()),
                   dict(tiles=z(1, 3, t=torch.int64)), dict(tiles=z(1, 4, t=torch.int32)), dict(sink=z(4)), dict(sink=z(3, t=torch.float32)),
                   dict(cache=cache.cpu()), dict(pos=slot.cpu())):
        with pytest.raises(ValueError):
            ops.gqa_attention4(**{**good, **change})
    for variant in (9, -1):
        with pytest.raises(RuntimeError):
            ops.gqa_attention4(**{**good, "variant": variant})
    with pytest.raises(RuntimeError):                       # no matrix instructions in 32 bits
        ops.gqa_attention4(**{**good, "q": q.float(), "variant": 3})
