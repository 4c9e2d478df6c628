"""Operators of a serving step, as cases to be timed: the tables of a step's token rows, key/value rows kept in 4 bits, attention
over them, and log probabilities of the tokens that come out.

A case is a dict of plain values; `op`:

  pages   the tables of a step from the requests' lengths: pages of finished requests go back to the pool, new ones are taken,
          every token row gets its sequence, position and cache slot
  store   rows of keys and values into the 4-bit cache, and what the cache then holds of them
  attend  grouped-query attention over the 4-bit cache, single tokens (`tokens` 0) or prompt portions
  score   log p of given tokens, entropy, rank and top alternatives of rows of logits

Lengths of ragged batches come from the case alone (`spread`), so that its work does not depend on the seed; everything else comes
from the seed. Where `own` is false, `run` computes the operators from elementary tensor operations in 32 bits; where it is true,
it makes the calls of the package.

The 4-bit cache is uint8 [pages, kv_heads, page / 64, block]. A block holds 64 tokens of one head; with K and V the entries of a
key and a value, each rounded up to a multiple of 64:

  key codes     [64 tokens][K / 2]          entry 2 i in the low half of byte i, 2 i + 1 in the high half
  key scales    [4][2][K / 16][8]           of token 16 a + 2 t + b and entries 16 j .. 16 j + 15 at [a][b][j][t]
  value codes   [V / 16][8][64 tokens]      [j][i][token]: entry 16 j + i in the low half, 16 j + i + 8 in the high half
  value scales  [V / 16][64 tokens]
  key exponents [64 tokens], value exponents [64 tokens]

A code is a sign and an index into 0, 0.5, 1, 1.5, 2, 3, 4, 6 (e2m1), a scale is an e4m3 byte, an exponent e stands for 2^(e - 127).
A row's exponent is that of its largest magnitude less 10, a block's scale the smallest that keeps its largest entry within 6
steps, a code the nearest (ties to the even one): entry = code * scale * 2^(e - 127)."""

import math
import random
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
VOCAB = 128256
FR = 24
TOKENS = 64                         # of a block of the 4-bit cache
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32, "int64": torch.int64}


def listed():
    return [
        # The first generated token of one chat user, with the alternatives an API shows.
        dict(name="score-1", op="score", rows=1, vocab=VOCAB, dtype="int64", top=5, masked=0.0),
        # The decode batch of the throughput benchmark, every request asking for the most alternatives.
        dict(name="score-256-top20", op="score", rows=256, vocab=VOCAB, dtype="int64", top=20, masked=0.0),
        # Evaluation of prompts: log p and entropy of every token, bf16 logits.
        dict(name="score-2000-bf16", op="score", rows=2000, vocab=VOCAB, dtype="bfloat16", top=0, masked=0.0),
        # Reinforcement learning: rows of float logits, a grammar that leaves half of the vocabulary.
        dict(name="score-700-f32", op="score", rows=700, vocab=VOCAB, dtype="float32", top=5, masked=0.5),
        # A decode step of 256 running requests, one in sixteen finished.
        dict(name="pages-256", op="pages", seqs=256, lo=64, hi=2000, new=1, page=64, drop=16),
        # An evaluation batch: a thousand requests in portions of up to 128 tokens.
        dict(name="pages-1000", op="pages", seqs=1000, lo=0, hi=4000, new=128, page=64, drop=10),
        # The keys and values of a decode step.
        dict(name="store-64", op="store", rows=64, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16"),
        # A chunk of prompts of the largest size that a session feeds at once, twice.
        dict(name="store-8192", op="store", rows=8192, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16"),
        # One user with a long chat: latency.
        dict(name="attend-1", op="attend", seqs=1, lo=2000, hi=2000, tokens=0, heads=32, kv_heads=8, dim=128, vdim=128, page=64,
             window=0, sink=False, dtype="bfloat16"),
        # The decode batch of the throughput benchmark at the 1B geometry, contexts of any length.
        dict(name="attend-256", op="attend", seqs=256, lo=64, hi=1100, tokens=0, heads=32, kv_heads=8, dim=64, vdim=64, page=64,
             window=0, sink=True, dtype="bfloat16"),
        # Long documents: what the 4-bit cache is for.
        dict(name="attend-64-long", op="attend", seqs=64, lo=8192, hi=8192, tokens=0, heads=32, kv_heads=8, dim=128, vdim=128,
             page=64, window=0, sink=False, dtype="bfloat16"),
        # Prompts of a batch, beginning to end.
        dict(name="attend-prompt-4x2048", op="attend", seqs=4, lo=1700, hi=2048, tokens=2048, heads=32, kv_heads=8, dim=128,
             vdim=128, page=64, window=0, sink=False, dtype="bfloat16"),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))
    op = rng.choice(["score", "score", "pages", "store", "attend", "attend", "attend"])
    if op == "score":
        vocab = rng.choice([VOCAB, log(500, 160000), log(500, 160000)])
        return dict(op=op, vocab=vocab, rows=log(1, min(4000, 30_000_000 // vocab)), dtype=rng.choice(["int64", "float32", "bfloat16"]),
                    top=rng.choice([0, 1, 3, 5, 20, 32]), masked=rng.choice([0.0, 0.0, 0.3, 0.95]))
    if op == "pages":
        seqs, new = log(1, 1000), rng.choice([1, 1, log(2, 128)])
        a, b = log(1, 4000), log(1, 4000)
        return dict(op=op, seqs=seqs, lo=min(a, b) - 1, hi=max(a, b), new=new, page=rng.choice([16, 64, 64, 128]), drop=rng.choice([0, 3, 16]))
    kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, rng.randint(20, 128)])
    c = dict(op=op, kv_heads=kv_heads, dim=dim, vdim=rng.choice([dim, dim, 64, rng.randint(20, 128)]), page=rng.choice([64, 64, 128]),
             dtype=rng.choice(["bfloat16"] * 4 + ["float32"]))
    if op == "store":
        return dict(c, rows=log(1, 8000))
    c.update(heads=kv_heads * rng.choice([1, 2, 4, 6, 8]), window=rng.choice([0, 0, log(10, 2000)]), sink=rng.choice([False, True]))
    slow = 32 if c["dtype"] == "float32" else 1
    if rng.random() < 0.6:
        seqs = log(1, 200)
        most = min(16000, 500_000 // seqs // slow + 20)
        a, b = log(1, most), log(1, most)
        return dict(c, seqs=seqs, tokens=0, lo=min(a, b), hi=max(a, b))
    seqs = rng.randint(1, 4)
    a, b = log(8, 1800 // slow), log(8, 1800 // slow)
    return dict(c, seqs=seqs, tokens=log(2, max(a, b)), lo=min(a, b), hi=max(a, b))


def spread(case):
    """The contexts of a case's sequences: lo .. hi in steps of the golden ratio, hi first."""
    lo, hi = case["lo"], case["hi"]
    return [hi - int((hi - lo) * ((0.6180339887498949 * i) % 1.0)) for i in range(case["seqs"])]


def fresh(case):
    """The new tokens of a case's sequences: of an attention case those at the end of the context, of a page case those behind it."""
    if case["op"] == "attend":
        return [min(n, max(1, case["tokens"])) for n in spread(case)]
    r = random.Random(case["seqs"])
    gone = dropped(case)
    return [0 if gone[i] else case["new"] if case["new"] == 1 else r.randint(0, case["new"]) for i in range(case["seqs"])]


def dropped(case):
    return [case["drop"] > 0 and i % case["drop"] == case["drop"] - 1 for i in range(case["seqs"])]


def up(n, m):
    return (n + m - 1) // m * m


# ---- the 4-bit form --------------------------------------------------------------------------------------------------

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SCALES = [(c & 7) * 2.0 ** -9 if c < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10) for c in range(127)]      # e4m3, 0 .. 448


def quantise(x):
    """x [..., n] -> codes uint8 [..., n up to 64], scales uint8 [..., that / 16], exponents uint8 [...]."""
    x = torch.nn.functional.pad(x.float(), (0, up(x.shape[-1], 64) - x.shape[-1]))
    most = x.abs().amax(-1)
    e = torch.clamp(torch.frexp(most).exponent.int() - 11, -100, 117)
    e = torch.where(most > 0, e, torch.full_like(e, -100))
    x = torch.ldexp(x, -e[..., None]).unflatten(-1, (-1, 16))
    table = torch.tensor(SCALES, device=x.device)
    s = torch.bucketize(x.abs().amax(-1), 6.0 * table).clamp_(max=126)
    step, mag = table[s][..., None], x.abs()
    code = mag > 0.25 * step
    code = code.to(torch.uint8)
    code += mag >= 0.75 * step
    code += mag > 1.25 * step
    code += mag >= 1.75 * step
    code += mag > 2.5 * step
    code += mag >= 3.5 * step
    code += mag > 5.0 * step
    code *= step > 0
    code += 8 * (x < 0).to(torch.uint8)
    return code.flatten(-2), s.to(torch.uint8), (e + 127).to(torch.uint8)


def blocks_of(k, v):
    """k [..., 64 tokens, dim], v [..., 64 tokens, vdim] -> blocks uint8 [..., bytes]."""
    (kc, ks, ke), (vc, vs, ve) = quantise(k), quantise(v)
    kc = kc[..., 0::2] | kc[..., 1::2] << 4
    ks = ks.unflatten(-2, (4, 8, 2)).transpose(-2, -3).transpose(-1, -2)             # [a][b][t][j] -> [a][b][j][t]
    vc = vc.unflatten(-1, (-1, 2, 8))
    vc = (vc[..., 0, :] | vc[..., 1, :] << 4).flatten(-2).transpose(-1, -2)
    vs = vs.transpose(-1, -2)
    flat = lambda t, n: t.reshape(*t.shape[:-n], -1)
    return torch.cat([flat(kc, 2), flat(ks, 4), flat(vc, 2), flat(vs, 2), ke, ve], -1)


def values_of(code, scale, e, grid, table):
    """codes, scales and exponents [..., n], [..., n / 16], [...] -> the entries that they stand for, in the tables' type."""
    v = grid[code.int()].unflatten(-1, (-1, 16)) * table[scale.int()][..., None]
    return torch.ldexp(v.flatten(-2), e.int()[..., None] - 127)


def entries_of(blocks, K, V):
    """blocks uint8 [..., bytes] -> keys [..., 64, K], values [..., 64, V] in 32 bits (K, V multiples of 64)."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=blocks.device)
    table = torch.tensor(SCALES + [math.nan], device=blocks.device)
    kc, ks, vc, vs, ke, ve = blocks.split([32 * K, 4 * K, 32 * V, 4 * V, 64, 64], -1)
    kc = kc.unflatten(-1, (64, -1))
    kc = torch.stack([kc & 15, kc >> 4], -1).flatten(-2)
    ks = ks.unflatten(-1, (4, 2, -1, 8)).transpose(-1, -2).transpose(-2, -3).flatten(-4, -2)
    vc = vc.unflatten(-1, (-1, 8, 64))
    vc = torch.stack([vc & 15, vc >> 4], -3).flatten(-4, -2).transpose(-1, -2)
    return values_of(kc, ks, ke, grid, table), values_of(vc, vs.unflatten(-1, (-1, 64)).transpose(-1, -2), ve, grid, table)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return SimpleNamespace(op=case["op"], **{"score": _score_inputs, "pages": _pages_inputs, "store": _store_inputs, "attend": _attend_inputs}[case["op"]](case, g))


def _score_inputs(case, g):
    n, V = case["rows"], case["vocab"]
    x = torch.randn(n, V, generator=g, device=DEV) * 2.5
    # a few tokens stand out, as they do behind a trained head
    at = torch.randint(V, (n, 8), generator=g, device=DEV)
    x.scatter_(1, at, 6.0 + 9.0 * torch.rand(n, 8, generator=g, device=DEV))
    hidden = torch.rand(V, generator=g, device=DEV) < case["masked"]
    hidden[0] = False
    tok = torch.where(torch.rand(n, generator=g, device=DEV) < 0.7, at[:, 0], torch.randint(V, (n,), generator=g, device=DEV))
    if case["dtype"] == "int64":
        x = torch.round(x.double() * 2.0 ** FR).long()
        x[:, hidden] = -(1 << 62)
    else:
        x = x.to(DTYPES[case["dtype"]])
        x[:, hidden] = -math.inf
    return dict(logits=x, tokens=tok, top=case["top"])


def _pages_inputs(case, g):
    lens, new, page = spread(case), fresh(case), case["page"]
    B = len(lens)
    nblk = max(-(-(a + b) // page) for a, b in zip(lens, new)) + 1
    held = torch.tensor([-(-a // page) for a in lens], device=DEV)
    used = sum(-(-a // page) for a in lens)
    need = sum(-(-(a + b) // page) + (-a // page) for a, b in zip(lens, new))
    # half as many pages again as the step takes, and room for those that come back
    pool = used + need + need // 2 + 8
    order = torch.randperm(pool, generator=g, device=DEV).int() + 1
    bt = torch.zeros(B, nblk, dtype=torch.int32, device=DEV)
    live = torch.arange(nblk, device=DEV)[None] < held[:, None]
    bt[live] = order[:used]
    free = torch.zeros(pool, dtype=torch.int32, device=DEV)
    free[:pool - used] = order[used:]
    return dict(lens=torch.tensor(lens, device=DEV), counts=torch.tensor(new, device=DEV), bt=bt, free=free, page=page,
                top=torch.tensor([pool - used], dtype=torch.int32, device=DEV), rows=up(sum(new), 64),
                drop=torch.tensor(dropped(case), device=DEV) if case["drop"] else None)


def _heads(case):
    return SimpleNamespace(heads=case.get("heads", case["kv_heads"]), kv_heads=case["kv_heads"], dim=case["dim"], vdim=case["vdim"],
                           window=case.get("window", 0), scale=case["dim"] ** -0.5)


def _keys(g, n, dim, shape):
    """Rows of keys: some channels are several times larger than the others, the same ones in every row."""
    gain = torch.exp(0.7 * torch.randn(dim, generator=g, device=DEV))
    return torch.randn(*shape, n, dim, generator=g, device=DEV) * gain


def _store_inputs(case, g):
    T, M, G, dim, vdim, page = DTYPES[case["dtype"]], case["rows"], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    pages = up(2 * M, page) // page + 1
    K, V = up(dim, 64), up(vdim, 64)
    # the rows of a step lie in runs of a page's slots
    first = torch.randperm(pages - 1, generator=g, device=DEV) + 1
    slot = (first[:, None] * page + torch.arange(page, device=DEV)).flatten()[:M] if M > 512 else first[torch.arange(M, device=DEV) % (pages - 1)] * page + \
        torch.arange(M, device=DEV) // (pages - 1)
    v = torch.randn(M, G, vdim, generator=g, device=DEV) * 0.5
    return dict(k=_keys(g, M, dim, (G,)).transpose(0, 1).to(T).contiguous(), v=v.to(T), slot=slot, spec=_heads(case),
                cache=torch.zeros(pages, G, page // TOKENS, 36 * (K + V) + 128, dtype=torch.uint8, device=DEV))


def _attend_inputs(case, g):
    T, G, dim, vdim, page = DTYPES[case["dtype"]], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    lens, new, per = spread(case), fresh(case), case["heads"] // case["kv_heads"]
    S, nblk, M = len(lens), -(-max(lens) // page), sum(new)
    K, V = up(dim, 64), up(vdim, 64)
    cache = torch.empty(S * nblk + 1, G, page // TOKENS, 36 * (K + V) + 128, dtype=torch.uint8, device=DEV)
    bt = (torch.randperm(S * nblk, generator=g, device=DEV) + 1).view(S, nblk).int()
    for s in range(0, S, max(1, 32768 // (nblk * page))):
        rows = bt[s:s + max(1, 32768 // (nblk * page))].flatten().long()
        shape = (len(rows), G, page // TOKENS)
        cache[rows] = blocks_of(_keys(g, TOKENS, dim, shape).to(T), (torch.randn(*shape, TOKENS, vdim, generator=g, device=DEV) * 0.5).to(T))
    cache[0] = cache[1]
    q = torch.zeros(G, M, per, up(dim, 8), dtype=T, device=DEV)
    q[..., :dim] = torch.randn(G, M, per, dim, generator=g, device=DEV)
    seq = torch.repeat_interleave(torch.arange(S), torch.tensor(new))
    pos = torch.cat([torch.arange(a - b, a) for a, b in zip(lens, new)])
    starts, tall = [sum(new[:i]) for i in range(S)], max(1, 128 // per)
    # where the rows of a sequence are, for the plain form; runs of a prompt's rows, for the kernels
    at = torch.full((S, max(new)), M)
    for s in range(S):
        at[s, :new[s]] = torch.arange(starts[s], starts[s] + new[s])
    tiles = [[s, starts[s] + t, min(tall, new[s] - t)] for s in range(S) for t in range(0, new[s], tall)]
    return dict(q=q, cache=cache, bt=bt, seq=seq.to(DEV), pos=pos.to(DEV), at=at.to(DEV), spec=_heads(case),
                tiles=torch.tensor(tiles, dtype=torch.int32, device=DEV) if case["tokens"] else None,
                sink=torch.randn(case["heads"], generator=g, device=DEV) if case["sink"] else None)


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(s):
    return {"score": _score, "pages": _pages, "store": _store, "attend": _attend}[s.op](s)


def _score(s):
    if own:
        from bitexact_llm_b200.logprobs import log_probs
        r = log_probs(s.logits, s.tokens, top=s.top, fr=FR)
        return dict(logp=r.logp, entropy=r.entropy, rank=r.rank, top_ids=r.top_ids, top_logp=r.top_logp)
    V, index = s.logits.shape[1], torch.arange(s.logits.shape[1], device=s.logits.device)
    if s.logits.dtype == torch.int64:
        raw = s.logits
        d = (raw - raw.amax(1, keepdim=True)).float() * 2.0 ** -FR
        gone, key = raw <= -(1 << 62), raw.clamp(-(1 << 43), 1 << 43)
    else:
        raw = s.logits.float() + 0.0
        d = raw - raw.amax(1, keepdim=True)
        bits = raw.view(torch.int32).long()
        gone, key = raw == -math.inf, torch.where(bits < 0, -2147483649 - bits, bits)
    e = torch.exp(d).masked_fill(gone, 0.0)
    total = e.sum(1)
    log_total = torch.log(total)
    entropy = log_total - (e * d).masked_fill(gone, 0.0).sum(1) / total
    t = s.tokens[:, None]
    given = lambda i: d.gather(1, i).masked_fill(gone.gather(1, i), -math.inf) - log_total[:, None]
    mine = raw.gather(1, t)
    rank = 1 + ((raw > mine) | ((raw == mine) & (index < t))).sum(1)
    best = torch.topk(key << 19 | (V - 1 - index), s.top, dim=1).values
    ids = V - 1 - (best & (1 << 19) - 1)
    top_logp = given(ids)
    ids = ids.masked_fill(gone.gather(1, ids), -1)
    return dict(logp=given(t)[:, 0], entropy=entropy, rank=rank, top_ids=ids, top_logp=top_logp)


def _pages(s):
    if own:
        from bitexact_llm_b200.pages import step_tables
        r = step_tables(s.lens, s.counts, s.bt, s.free, s.top, s.page, s.rows, drop=s.drop)
        return dict(seq=r.seq, pos=r.pos, slot=r.slot, last=r.last, lens=r.lens, top=r.top, status=r.status, bt=s.bt, free=s.free)
    B, nblk, pool = s.bt.shape[0], s.bt.shape[1], s.free.shape[0]
    dev, page = s.bt.device, s.page
    blocks = lambda n: (n + page - 1) // page
    drop = torch.zeros(B, dtype=torch.bool, device=dev) if s.drop is None else s.drop
    lens = s.lens.masked_fill(drop, 0)
    after, back = lens + s.counts, blocks(s.lens).masked_fill(~drop, 0)
    have, need = blocks(lens), blocks(after) - blocks(lens)
    j = torch.arange(nblk, device=dev)[None]
    # pages of finished requests onto the stack, a request's last page first
    place = s.top + (torch.cumsum(back, 0) - back + back - 1)[:, None] - j
    free = torch.cat([s.free, s.free[:1]]).scatter(0, torch.where(j < back[:, None], place, pool).flatten(), s.bt.flatten())[:pool]
    top = s.top + back.sum()
    # new pages from its end, in the order of requests and positions
    nth = (torch.cumsum(need, 0) - need - have)[:, None] + j
    new = (j >= have[:, None]) & (j < (have + need)[:, None])
    bt = torch.where(new, free[(top - 1 - nth).clamp(0, pool - 1)], s.bt)
    ends = torch.cumsum(s.counts, 0)
    i = torch.arange(s.rows, device=dev)
    live = i < ends[-1]
    seq = torch.searchsorted(ends, i, right=True).clamp(max=B - 1)
    pos = (lens - ends + s.counts)[seq] + i
    slot = bt[seq, (pos // page).clamp(0, nblk - 1)].long() * page + pos % page
    last = torch.where(s.counts > 0, ends - 1, -1)
    return dict(seq=seq.masked_fill(~live, 0), pos=pos.masked_fill(~live, 0), slot=slot.masked_fill(~live, -1), last=last, lens=after,
                top=(top - need.sum()).int(), status=torch.zeros(1, dtype=torch.int32, device=dev), bt=bt, free=free)


def _store(s):
    if own:
        from bitexact_llm_b200.hybrid import ops
        ops.gqa_store4(s.k, s.v, s.slot, s.cache)
        k, v = ops.gqa_read4(s.cache, s.spec, s.slot, s.k.dtype)
        return dict(k=k, v=v)
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=DEV)
    table = torch.tensor(SCALES + [math.nan], device=DEV)
    k, v = values_of(*quantise(s.k), grid, table), values_of(*quantise(s.v), grid, table)
    return dict(k=k[..., :s.spec.dim].to(s.k.dtype), v=v[..., :s.spec.vdim].to(s.v.dtype))


def _attend(s):
    sp, G, M, per = s.spec, *s.q.shape[:3]
    if own:
        from bitexact_llm_b200.hybrid import ops
        return ops.gqa_attention4(s.q, sp, s.cache, s.bt, s.seq, s.pos, s.sink, s.tiles)[:, :sp.heads * sp.vdim]
    S, T = s.at.shape
    k, v = entries_of(s.cache[s.bt.long()], up(sp.dim, 64), up(sp.vdim, 64))         # [S, blocks, G, block, 64, entries]
    k, v = (t.transpose(1, 2).flatten(2, 4) for t in (k, v))                         # [S, G, tokens, entries]
    q = torch.cat([s.q, s.q[:, :1]], 1)[..., :sp.dim].float()[:, s.at]               # [G, S, T, per, dim]; rows that are none read any
    q = q.transpose(0, 1).flatten(2, 3)
    pos = torch.cat([s.pos, s.pos[:1]])[s.at]
    key = torch.arange(k.shape[2], device=DEV)
    seen = key <= pos[..., None]
    if sp.window:
        seen &= key > pos[..., None] - sp.window
    score = (q @ k[..., :sp.dim].transpose(-1, -2)) * sp.scale
    score = score.unflatten(2, (T, per)).masked_fill(~seen[:, None, :, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    if s.sink is not None:
        sink = s.sink.view(1, G, 1, per, 1)
        most = torch.maximum(most, sink)
    p = torch.exp(score - most)
    total = p.sum(-1, keepdim=True)
    if s.sink is not None:
        total = total + torch.exp(sink - most)
    out = (p.flatten(2, 3) @ v[..., :sp.vdim]).unflatten(2, (T, per)) / total
    out = out.permute(0, 2, 1, 3, 4).flatten(2)                                      # [S, T, heads * vdim]
    rows = torch.empty(M + 1, out.shape[-1], device=DEV)
    rows[s.at.flatten()] = out.flatten(0, 1)
    return rows[:M].to(s.q.dtype)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    if case["op"] == "score":
        n, V = case["rows"], case["vocab"]
        return {"bytes": n * V * DTYPES[case["dtype"]].itemsize + n * (8 + 4 + 4 + 8 + 12 * case["top"]), "flops": 6 * n * V}
    if case["op"] == "pages":
        lens, new, gone, page = spread(case), fresh(case), dropped(case), case["page"]
        moved = sum(-(-(a + b) // page) + (-a // page) + (-(-a // page) if d else 0) for a, b, d in zip(lens, new, gone))
        # a decode row needs its page's entry, a prompt row shares it
        return {"bytes": 24 * up(sum(new), 64) + 33 * len(lens) + 8 * moved + 4 * len(lens), "flops": 0}
    K, V = case["dim"], case["vdim"]
    row = (K + V) // 2 + -(-K // 16) - (-V // 16) + 2
    if case["op"] == "store":
        n, size = case["rows"] * case["kv_heads"], DTYPES[case["dtype"]].itemsize
        return {"bytes": n * (2 * (K + V) * size + 2 * row) + 16 * case["rows"], "flops": 4 * n * (K + V)}
    pairs = keys = 0
    for a, b in zip(spread(case), fresh(case)):
        w = case["window"] or a
        pairs += sum(min(p + 1, w) for p in range(a - b, a))
        keys += min(a, w + b - 1)
    M, size = sum(fresh(case)), DTYPES[case["dtype"]].itemsize
    return {"bytes": keys * case["kv_heads"] * row + M * case["heads"] * (K + V) * size, "flops": 2 * pairs * case["heads"] * (K + V)}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"score": _exact_score, "pages": lambda s: None, "store": _exact_store, "attend": _exact_attend}[s.op](s)


def _exact_score(s):
    out = dict(logp=[], entropy=[], rank=None, top_ids=None, top_logp=[])
    for x, t in zip(s.logits.split(64), s.tokens.split(64)):
        z = x.double() * (2.0 ** -FR if x.dtype == torch.int64 else 1.0)
        z[z < -1e9] = -math.inf
        logp = torch.log_softmax(z, 1)
        out["logp"].append(logp.gather(1, t[:, None])[:, 0])
        out["entropy"].append(torch.special.entr(torch.softmax(z, 1)).sum(1))
        out["top_logp"].append(logp.sort(dim=1, descending=True).values[:, :s.top])
    return {k: v if v is None else torch.cat(v) for k, v in out.items()}


def _exact_rows(x):
    """The entries that the 4-bit form keeps of x [rows, n], from their nearest candidates."""
    n = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -n % 16))
    unit = torch.exp2(torch.floor(torch.log2(x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -140))).clamp(min=-90) - 10)
    x = (x / unit).unflatten(-1, (-1, 16))
    table = torch.tensor(SCALES, dtype=torch.float64, device=x.device)
    far = 6 * table - x.abs().amax(-1, keepdim=True)
    step = table[torch.where(far < 0, math.inf, far).argmin(-1)][..., None]
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)                  # even codes first: they win ties
    gap = (x.abs()[..., None] - grid[order] * step[..., None]).abs()
    y = grid[order[gap.argmin(-1)]] * step * torch.sign(x) * unit[..., None]
    return y.flatten(-2)[..., :n]


def _exact_store(s):
    part = lambda t: torch.cat([_exact_rows(c.flatten(0, 1)).view(c.shape) for c in t.split(256)])
    return dict(k=part(s.k), v=part(s.v))


def _exact_attend(s):
    sp, G, M, per = s.spec, *s.q.shape[:3]
    K, V, page = up(sp.dim, 64), up(sp.vdim, 64), s.cache.shape[2] * TOKENS
    e2m1 = torch.tensor([math.copysign(GRID[c & 7], -1.0 if c > 7 else 1.0) for c in range(16)], dtype=torch.float64, device=DEV)
    e4m3 = torch.tensor(SCALES + [math.nan], dtype=torch.float64, device=DEV)
    out = torch.empty(M, sp.heads * sp.vdim, dtype=torch.float64, device=DEV)
    seqs, pos = s.seq.tolist(), s.pos.tolist()
    begin = 0
    while begin < M:
        end = begin
        while end < M and seqs[end] == seqs[begin] and end - begin < 512:
            end += 1
        n = pos[end - 1] + 1
        tok = torch.arange(n, device=DEV)
        block = s.cache[s.bt[seqs[begin], tok // page].long(), :, tok % page // 64].long()       # [tokens, G, bytes]
        t = tok % 64

        def entry(width, code_at, high, scale_at, power_at):
            """Entries [tokens, G, width] whose code, scale and exponent lie at these bytes of the block."""
            take = lambda at: block.gather(2, at[:, None].expand(n, G, at.shape[1]))
            c = take(code_at) >> (4 * high) & 15
            return e2m1[c] * e4m3[take(scale_at)] * torch.exp2(take(power_at[:, None]).double() - 127)
        d, t1 = torch.arange(sp.dim, device=DEV), t[:, None]
        k = entry(sp.dim, t1 * (K // 2) + d // 2, d % 2, 32 * K + ((t1 // 16 * 2 + t1 % 2) * (K // 16) + d // 16) * 8 + t1 % 16 // 2, 36 * (K + V) + t)
        d = torch.arange(sp.vdim, device=DEV)
        v = entry(sp.vdim, 36 * K + (d // 16 * 8 + d % 8) * 64 + t1, d % 16 // 8, 36 * K + 32 * V + d // 16 * 64 + t1, 36 * (K + V) + 64 + t)
        q = s.q[:, begin:end, :, :sp.dim].double()
        p = s.pos[begin:end, None]
        hide = (tok > p) | ((tok <= p - sp.window) if sp.window else False)
        for g in range(G):
            z = torch.einsum("mhd,td->mht", q[g], k[:, g]) * sp.scale
            z = z.masked_fill(hide[:, None], -math.inf)
            if s.sink is not None:
                z = torch.cat([z, s.sink[g * per:(g + 1) * per].double()[None, :, None].expand(end - begin, per, 1)], 2)
            w = torch.softmax(z, 2)[..., :n]
            out[begin:end, g * per * sp.vdim:(g + 1) * per * sp.vdim] = torch.einsum("mht,td->mhd", w, v[:, g]).flatten(1)
        begin = end
    return out
