"""`decode.Session` with its pool on the device, host side: what a call that fails leaves behind. `step_tables` is played by plain
bookkeeping, the engine by one whose rows are sums over the cache."""

import pytest
import torch

from bitexact_llm_b200 import pages
from bitexact_llm_b200.decode import Session

PAGE = 4


def tables(lens, counts, bt, free, top, page, rows, drop=None, lens_out=None, top_out=None, status=None):
    """`pages.step_tables` in Python."""
    held = lambda n: -(-n // page)
    L, C, T = lens.tolist(), counts.tolist(), int(top)
    base = [0 if drop is not None and drop[b] else n for b, n in enumerate(L)]
    back = [p for b in range(len(L)) if drop is not None and drop[b] for p in bt[b, :held(L[b])].tolist()[::-1]]
    long = [s + n > bt.shape[1] * page for s, n in zip(base, C)]
    need = [0 if l else held(s + n) - held(s) for l, s, n in zip(long, base, C)]
    bad = pages.TOO_LONG if any(long) else 0
    bad |= pages.NO_PAGES if sum(need) > T + len(back) else 0
    bad |= pages.TOO_MANY_ROWS if sum(C) > rows else 0
    seq, pos, slot = (torch.full((rows,), v, dtype=torch.long) for v in (0, 0, -1))
    last = torch.full((len(L),), -1, dtype=torch.long)
    out, left = list(L), T
    if not bad:
        free[T:T + len(back)] = torch.tensor(back, dtype=torch.int32)
        left, r = T + len(back), 0
        for b, n in enumerate(C):
            for j in range(held(base[b]), held(base[b] + n)):
                left -= 1
                bt[b, j] = free[left]
            for p in range(base[b], base[b] + n):
                seq[r], pos[r], slot[r] = b, p, int(bt[b, p // page]) * page + p % page
                r += 1
            last[b] = r - 1 if n else -1
            out[b] = base[b] + n
    lens_out = torch.empty_like(lens) if lens_out is None else lens_out
    top_out = torch.empty_like(top) if top_out is None else top_out
    own = status is None
    status = torch.zeros(1, dtype=torch.int32) if own else status
    lens_out.copy_(torch.tensor(out))
    top_out.fill_(left)
    status |= bad
    return pages.StepTables(seq, pos, slot, last, lens_out, top_out, status)


class Engine:
    """A row of token p is the sum of (t + 1) * (position + 1) over the tokens up to p, as the cache holds them."""

    page, tiles_from, D, V = PAGE, 1 << 30, 1, 50
    dev = torch.device("cpu")
    failing = False

    def new_cache(self, n_seqs, n_blocks, bs):
        return [torch.zeros(n_blocks * bs)]

    def tile_table(self, runs, bs):
        return None

    def check(self):
        pass

    def forward(self, kvs, ids, pos, slot, bt, rmap, tiles=None):
        if self.failing:
            raise RuntimeError("no memory")
        kvs[0][slot[slot >= 0]] = (ids[slot >= 0] + 1).float()
        rows = []
        for s, p in zip(rmap.tolist(), pos.tolist()):
            t = torch.arange(p + 1)
            rows.append((kvs[0][bt[s].long()[t // PAGE] * PAGE + t % PAGE] * (t + 1)).sum())
        return torch.stack(rows)[:, None]


@pytest.fixture
def make(monkeypatch):
    monkeypatch.setattr(pages, "step_tables", tables)
    return lambda B, max_len, n: Session(Engine(), B, max_len, pages=n, on_device=True)


def state(ses):
    return ses.lens.tolist(), int(ses.pool.top)


def full(make):
    """Two sequences on all pages, and a decode step that found none left."""
    ses = make(3, 16, 4)
    ses.feed([(0, range(8)), (1, [7] * 8)])
    before = state(ses)
    ses.step(torch.tensor([1, 1, 1]))
    assert state(ses) == before
    ses.release(1)
    return ses


def test_feed_after_a_step_that_failed(make):
    ses, plain = full(make), Session(Engine(), 3, 16)
    plain.feed([(0, range(8))])
    entries = [(0, [9, 4]), (2, [5])]
    got, want = ses.feed(entries), plain.feed(entries)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and ses.lens.tolist() == [10, 0, 1] and int(ses.pool.top) == 0
    with pytest.raises(MemoryError):                       # the step's failure is told where it is asked for, once
        ses.check()
    ses.check()


def test_prefill_after_a_step_that_failed(make):
    ses = full(make)
    ses.release(0)
    prompts, lens = torch.arange(15).view(3, 5), torch.tensor([5, 2, 1])
    assert torch.equal(ses.prefill(prompts, lens), Session(Engine(), 3, 16).prefill(prompts, lens))
    assert state(ses) == ([5, 2, 1], 0)
    with pytest.raises(MemoryError):
        ses.check()


def test_feed_and_prefill_that_fail_change_nothing(make):
    ses, plain = make(3, 16, 4), Session(Engine(), 3, 16)
    for s in (ses, plain):
        s.feed([(0, range(3)), (1, [7] * 8)])
    before = state(ses)
    for entries, error in (([(2, range(5))], MemoryError), ([(1, [1] * 9)], ValueError)):
        with pytest.raises(error):
            ses.feed(entries)
        assert state(ses) == before
    ses.eng.failing = True
    with pytest.raises(RuntimeError):
        ses.feed([(0, [1, 2]), (2, [3])][:1])
    assert state(ses) == before
    ses.eng.failing = False
    entries = [(0, [1]), (2, [3])]
    assert all(torch.equal(a, b) for a, b in zip(ses.feed(entries), plain.feed(entries)))
    assert state(ses) == ([4, 8, 1], 0)
    ses.check()

    ses = make(2, 16, 4)
    prompts = torch.arange(10).view(2, 5)
    ses.eng.failing = True
    with pytest.raises(RuntimeError):
        ses.prefill(prompts)
    assert state(ses) == ([0, 0], 4)
    ses.eng.failing = False
    with pytest.raises(MemoryError):
        make(2, 16, 3).prefill(prompts)
    assert torch.equal(ses.prefill(prompts), Session(Engine(), 2, 16).prefill(prompts)) and state(ses) == ([5, 5], 0)
    ses.check()


def test_release_takes_what_a_list_takes(make):
    """As without a pool on the device: an index from the end, and IndexError beyond."""
    ses = make(3, 16, 4)
    ses.feed([(0, range(3)), (2, [7] * 8)])
    for seq in (3, -4):
        with pytest.raises(IndexError):
            ses.release(seq)
    assert state(ses) == ([3, 0, 8], 1)
    ses.release(-1)
    assert state(ses) == ([3, 0, 0], 3)
    ses.release(torch.tensor(0))
    assert state(ses) == ([0, 0, 0], 4)
