"""`gqa_attention4` over tiles whose keys are split over CTAs, and over what only some of its kernels meet (tolerances: test_cache4_gpu.py); the
decisions of `gqa_store4` where they are closest."""

import math

import pytest
import torch

from test_cache4_gpu import SCALES, attention, batch, close, kept, rows, spec, tiles_of

pytestmark = pytest.mark.gpu
FORMS = [("bfloat16", 0), ("bfloat16", 1), ("bfloat16", 2), ("float32", 0)]


@pytest.mark.parametrize("dtype,variant", FORMS)
@pytest.mark.parametrize("new", [16, 3, 1])
def test_what_is_not_a_number_is_seen_behind_a_split(new, dtype, variant):
    """The last `new` tokens of 2500 (16 of them: a tall tile in four parts), a window that ends among them."""
    from bitexact_llm_b200.hybrid import ops
    n, bad_key, bad_value = 2500, 700, 2500 - (new + 1) // 2
    sp = spec(8, 2, 128, 64, n - new // 2 - bad_key)
    q, cache, bt, seq, pos, held = batch(sp, 64, [n], [new], dtype, 3)
    k, v = rows(2, 2, 128, dtype, 1), rows(2, 2, 64, dtype, 2)
    k[0, 0, 3], v[1, 1, 60] = math.nan, math.inf
    for g, at in ((0, bad_key), (1, bad_value)):                # (the other head's row is stored again)
        slot = torch.tensor([int(bt[0, at // 64]) * 64 + at % 64]).cuda()
        a, b = (t.to(getattr(torch, dtype)) for t in ops.gqa_read4(cache, sp, slot, torch.float32))
        a[0, g], b[0, g] = k[g, g].cuda(), v[g, g].cuda()
        ops.gqa_store4(a, b, slot, cache)
        for old, now in zip(held[0], ops.gqa_read4(cache, sp, slot, torch.float32)):
            old[at] = now[0].double().cpu()
    want, big = attention(q, sp, seq, pos, held, None)
    bad = torch.zeros(new, 2, dtype=torch.bool)
    bad[:, 0] = pos.cpu() - sp.window < bad_key
    bad[:, 1] = pos.cpu() >= bad_value
    assert bad.any(0).all() and (new < 3 or not bad.all(0).any())
    for tiles in (None, tiles_of([new], 4)):
        got = ops.gqa_attention4(q, sp, cache, bt, seq, pos, None, tiles, variant).view(new, 2, -1)
        assert torch.isnan(got.cpu()[bad]).all()
        ok = ~bad
        close(got.cpu()[ok], want.view(new, 2, -1)[ok], big.double().expand(new, 2)[ok][:, None], dtype)


@pytest.mark.parametrize("dtype,variant", FORMS)
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("new", [16, 3])
def test_rows_that_see_nothing_behind_a_split(new, window, dtype, variant):
    """Rows in front of their sequence (position -1) in a tile with others of a long one: zeros, with a sink or without."""
    from bitexact_llm_b200.hybrid import ops
    sp = spec(8, 2, 128, 64, window)
    q, cache, bt, seq, pos, held = batch(sp, 64, [2500], [new], dtype, 4)
    none = (new + 1) // 2
    for sink in (None, torch.randn(8, generator=torch.Generator().manual_seed(1)).cuda()):
        want, big = attention(q, sp, seq, pos, held, sink)
        at = pos.clone()
        at[:none] = -1
        for tiles in (None, tiles_of([new], 4)):
            got = ops.gqa_attention4(q, sp, cache, bt, seq, at, sink, tiles, variant)
            assert not got[:none].any()
            close(got[none:], want[none:], big[none:], dtype)


@pytest.mark.parametrize("dtype,variant", FORMS)
@pytest.mark.parametrize("lens,new,tiles", [([2500], [40], [[0, 5, 16]]),                                     # one tall tile in parts
                                            ([2500], [40], [[0, 3, 2], [0, 8, 30]]),                          # a short one beside it
                                            ([300, 90, 200], [80, 1, 60], [[0, 0, 32], [1, 80, 1], [2, 100, 32]]),
                                            ([200], [20], [[0, 7, 1]]),
                                            ([200], [20], [])])
def test_rows_in_no_tile_are_left_as_they_were(lens, new, tiles, dtype, variant):
    """Through the C entry, into an output that is filled already and has columns of its own behind the heads."""
    from bitexact_llm_b200 import _native as nv
    from bitexact_llm_b200.hybrid import ops
    sp = spec(8, 2, 128, 64)
    q, cache, bt, seq, pos, held = batch(sp, 64, lens, new, dtype, 6)
    lib, M, wide = nv.float_lib(), sum(new), 8 * 64 + 24
    t = torch.tensor(tiles + [[0, 0, M]], dtype=torch.int32).cuda()          # (the last one is not given: a pointer to no tiles)
    out = torch.full((M, wide), 3.0, dtype=q.dtype, device="cuda")
    need = lib.bxf_gqa_attention_scratch(M, 8, 2, 64)
    scratch = torch.full((need,), 255, dtype=torch.uint8, device="cuda")     # NaN
    rc = lib.bxf_gqa_attention4(ops.code(q), q.data_ptr(), q.shape[3], M, 8, 2, 128, 64, cache.data_ptr(), 64, cache.shape[0], bt.data_ptr(), 0,
                                bt.stride(0), bt.shape[1], seq.data_ptr(), pos.data_ptr(), t.data_ptr(), len(tiles), 0, None, sp.scale,
                                out.data_ptr(), wide, scratch.data_ptr(), need, variant, nv.stream())
    nv.check(rc, "bxf_gqa_attention4")
    mine = torch.zeros(M, dtype=torch.bool)
    for _, row, n in tiles:
        mine[row:row + n] = True
    assert (out[:, 8 * 64:] == 3).all() and (out.cpu()[~mine] == 3).all()
    want, big = attention(q, sp, seq, pos, held, None)
    if tiles:
        close(out[:, :8 * 64].cpu()[mine], want[mine], big[mine], dtype)


@pytest.mark.parametrize("dtype,variant", FORMS)
@pytest.mark.parametrize("keys", [1.0, 1e6])
@pytest.mark.parametrize("per,far", [(4, 26), (4, 20), (1, 26)])
def test_small_values_beside_a_large_one_without_weight(per, far, keys, dtype, variant):
    """One token's values are 2^far times the others', and no row gives it any weight: what the others lose is told by fp16's smallest step.

    A tall tile keeps a weight as 2^6 w 2^(e - E) in fp16: off by at most 2^-25 where that is subnormal, so w 2^(e - E) by 2^-31. A
    token's entries are below 2^11 in units of its own power of two, the largest token's largest entry is at least 2^10: each token adds at
    most 2^-30 of that to a sum of weights that is at least the number of tokens that weigh 1 (all of them, here). In operands that hold the powers
    of two, scale times 2^(e - E) is off by 2^-25, times a code of at most 6, and that product by 2^-25: 7 * 2^-25 / 2^10 < 2^-32 of it.
    So the mean is off by less than 2^-30 of the largest token's largest entry, beside the tolerances of every row."""
    from bitexact_llm_b200.hybrid import ops
    sp, T, n, G = spec(2 * per, 2, 64, 64), getattr(torch, dtype), 400, 2
    k, v = torch.zeros(n, G, 64), rows(n, G, 64, "float32", 8)
    v = v / v.abs().amax(-1, keepdim=True)
    large = 70
    k[large] = -keys                                        # scores 0 for the others, below -1000 for it
    v[large] *= 2.0 ** far
    cache, slot = ops.gqa_cache4(sp, 8, 64, "cuda"), torch.arange(n).cuda() + 64
    ops.gqa_store4(k.to(T).cuda(), v.to(T).cuda(), slot, cache)
    held = [tuple(x.double().cpu() for x in ops.gqa_read4(cache, sp, slot, torch.float32))]
    first = 30
    M = n - first
    q = torch.full((G, M, per, 64), 200.0).to(T).cuda()
    bt, seq, pos = torch.arange(1, 8, dtype=torch.int32).cuda()[None], torch.zeros(M, dtype=torch.long).cuda(), torch.arange(first, n).cuda()
    want, big = attention(q, sp, seq, pos, held, None)
    own = held[0][1][torch.arange(n) != large].abs().amax()
    tol = 2.0 ** -30 * big + (2.0 ** -11 * own + 2.0 ** -8 * want.abs() if dtype == "bfloat16" else 3e-5 * own)
    for tall in (128 // per, 8 // per):
        t = torch.tensor([[0, i, min(tall, M - i)] for i in range(0, M, tall)], dtype=torch.int32).cuda()
        got = ops.gqa_attention4(q, sp, cache, bt, seq, pos, None, t, variant)[:, :2 * per * 64].double().cpu()
        err = (got - want).abs()
        assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype,variant", FORMS)
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("n,extra", [(2500, 1), (100, 40)])
def test_sinks_of_no_weight(n, extra, window, dtype, variant):
    """A sink of -infinity is none: rows are as without it, and zeros where they see nothing; the table as wide as the context or far wider."""
    from bitexact_llm_b200.hybrid import ops
    sp, new, none = spec(8, 2, 128, 64, window), 16, 5
    q, cache, bt, seq, pos, held = batch(sp, 64, [n], [new], dtype, 4, extra)
    sink = torch.randn(8, generator=torch.Generator().manual_seed(1)).cuda()
    sink[::2] = -math.inf
    want, big = attention(q, sp, seq, pos, held, sink)
    for tiles in (None, tiles_of([new], 4), torch.tensor([[0, i, 1] for i in range(new)], dtype=torch.int32).cuda()):
        got = ops.gqa_attention4(q, sp, cache, bt, seq, pos, sink, tiles, variant)
        close(got, want, big, dtype)
        at = pos.clone()
        at[:none] = -1
        got = ops.gqa_attention4(q, sp, cache, bt, seq, at, sink, tiles, variant)
        assert not got[:none].any()
        close(got[none:], want[none:], big[none:], dtype)


@pytest.mark.parametrize("variant", (0, 1, 2))
@pytest.mark.parametrize("ldq,shift", [(20, 0), (21, 0), (24, 1), (24, 4), (64, 3)])
def test_queries_of_any_stride_and_alignment(ldq, shift, variant):
    """Rows that no 16-byte copy can take."""
    from bitexact_llm_b200.hybrid import ops
    sp = spec(8, 2, 20, 30)
    lens, new = [200, 90], [40, 3]
    q, cache, bt, seq, pos, held = batch(sp, 64, lens, new, "bfloat16", 4)
    want, big = attention(q, sp, seq, pos, held, None)
    room = torch.full((q.shape[0] * q.shape[1] * q.shape[2] * ldq + shift,), 9.0, dtype=q.dtype, device="cuda")
    wide = room[shift:].view(*q.shape[:3], ldq)
    wide[..., :20] = q[..., :20]
    for tiles in (None, tiles_of(new, 4)):
        close(ops.gqa_attention4(wide, sp, cache, bt, seq, pos, None, tiles, variant)[:, :240], want, big, "bfloat16")


@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
@pytest.mark.parametrize("few", [True, False])
def test_entries_beside_a_tie(few, dtype):
    """Every scale, every tie of its steps and the numbers up to five next to it, both signs; and blocks whose largest entry is beside six steps."""
    from bitexact_llm_b200.hybrid import ops
    T = getattr(torch, dtype)

    def beside(x):
        """x and its neighbours: x [n] -> [n, 11]."""
        x, out = x.to(T), []
        for to in (torch.inf, -torch.inf):
            y = x
            for _ in range(5):
                y = torch.nextafter(y, torch.full_like(y, to))
                out.append(y)
        return torch.stack([x, *out], 1)

    scales = SCALES[8:113]                                  # up to 160: six steps are within a row whose largest magnitude is 1024 .. 2047
    entries = beside((scales[:, None] * torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)).flatten()).view(len(scales), -1)
    entries = torch.cat([entries, -entries], 1)
    entries = torch.nn.functional.pad(entries, (0, -entries.shape[1] % 15)).view(len(scales), -1, 15)
    blocks = torch.cat([(6 * scales).to(T)[:, None, None].expand(-1, entries.shape[1], 1), entries], 2).reshape(-1, 16)
    most = torch.nn.functional.pad(beside(6 * SCALES[1:113]).reshape(-1, 1), (0, 15))
    blocks = torch.cat([blocks, most])
    blocks = torch.nn.functional.pad(blocks, (0, 0, 0, -len(blocks) % 31)).view(-1, 31 * 16)
    x = torch.cat([torch.full((len(blocks), 16), 1500.0).to(T), blocks], 1)[:, None]
    x = x.repeat(1 if few else 20, 1, 1)
    sp, M = spec(1, 1, 512, 512), len(x)
    assert few == (M <= 512)
    slot = torch.arange(M).cuda() + 3
    cache = ops.gqa_cache4(sp, M // 64 + 2, 64, "cuda")
    ops.gqa_store4(x.cuda(), -x.cuda(), slot, cache)
    a, b = ops.gqa_read4(cache, sp, slot, torch.float32)
    assert torch.equal(a.double().cpu(), kept(x)) and torch.equal(b.double().cpu(), kept(-x))


@pytest.mark.parametrize("dtype,variant", FORMS)
@pytest.mark.parametrize("size", [2.0 ** 126, 2.0 ** -88])
@pytest.mark.parametrize("n,new", [(300, 40), (2500, 16), (2500, 1)])
def test_values_at_the_ends_of_the_range(n, new, size, dtype, variant):
    """Many keys of about the same weight: the sum of their values is beyond 32 bits, their mean is not; and the smallest values that have all their digits."""
    from bitexact_llm_b200.hybrid import ops
    sp, T = spec(8, 2, 128, 64), getattr(torch, dtype)
    g = torch.Generator().manual_seed(9)
    k, v = torch.randn(n, 2, 128, generator=g) * 0.1, (1 + 0.9 * torch.rand(n, 2, 64, generator=g)) * size
    v[..., ::3] *= -1
    nblk = -(-n // 64) + 1
    cache, slot = ops.gqa_cache4(sp, nblk + 1, 64, "cuda"), torch.arange(n).cuda() + 64
    ops.gqa_store4(k.to(T).cuda(), v.to(T).cuda(), slot, cache)
    held = [tuple(x.double().cpu() for x in ops.gqa_read4(cache, sp, slot, torch.float32))]
    q = torch.randn(2, new, 4, 128, generator=g).to(T).cuda()
    bt, seq, pos = torch.arange(1, nblk + 1, dtype=torch.int32).cuda()[None], torch.zeros(new, dtype=torch.long).cuda(), torch.arange(n - new, n).cuda()
    want, big = attention(q, sp, seq, pos, held, None)
    for tiles in (None, tiles_of([new], 4), torch.tensor([[0, i, 1] for i in range(new)], dtype=torch.int32).cuda()):
        close(ops.gqa_attention4(q, sp, cache, bt, seq, pos, None, tiles, variant), want, big.double(), dtype)
