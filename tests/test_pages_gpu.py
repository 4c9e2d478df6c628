"""`pages.step_tables` and `DevicePages` against plain bookkeeping on the host (a list of free pages, as `decode.Session` keeps it):
whole numbers, compared exactly."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu


class Host:
    """The same pool in Python."""

    def __init__(self, B, blocks, pages, page, order=None):
        self.page, self.blocks = page, blocks
        self.free = (list(range(1, pages + 1)) if order is None else list(order))[::-1]
        self.bt, self.lens = [[0] * blocks for _ in range(B)], [0] * B

    def step(self, counts, rows, drop=None):
        """-> (seq, pos, slot, last) or the status."""
        held = lambda n: -(-n // self.page)
        bad = 0
        base = [0 if drop and drop[b] else n for b, n in enumerate(self.lens)]
        for b, n in enumerate(counts):
            bad |= 8 if n < 0 else 1 if base[b] + n > self.blocks * self.page else 0
        ok = [n if 0 <= n and base[b] + n <= self.blocks * self.page else None for b, n in enumerate(counts)]
        back = sum(held(self.lens[b]) for b in range(len(counts)) if drop and drop[b] and ok[b] is not None)
        need = sum(held(base[b] + n) - held(base[b]) for b, n in enumerate(ok) if n is not None)
        bad |= 2 if need > len(self.free) + back else 0
        bad |= 4 if sum(n for n in ok if n is not None) > rows else 0
        if bad:
            return bad
        for b in range(len(counts)):
            if drop and drop[b]:
                self.free += self.bt[b][:held(self.lens[b])][::-1]
        out = ([], [], [])
        last = []
        for b, n in enumerate(counts):
            for j in range(held(base[b]), held(base[b] + n)):
                self.bt[b][j] = self.free.pop()
            for i in range(base[b], base[b] + n):
                out[0].append(b)
                out[1].append(i)
                out[2].append(self.bt[b][i // self.page] * self.page + i % self.page)
            last.append(len(out[0]) - 1 if n else -1)
            self.lens[b] = base[b] + n
        for l, v in zip(out, (0, 0, -1)):
            l += [v] * (rows - len(l))
        return (*out, last)


def equal(dev, host, r, want):
    assert [t.tolist() for t in r[:4]] == list(want)
    assert dev.lens.tolist() == host.lens and dev.bt.tolist() == host.bt
    assert int(dev.top) == len(host.free) and dev.free[: len(host.free)].tolist() == host.free


@pytest.mark.parametrize("B,blocks,page,most,seed", [(1, 5, 16, 1, 0), (1, 40, 64, 700, 1), (3, 4, 1, 3, 2), (33, 9, 7, 40, 3), (256, 20, 64, 1, 4),
                                                     (257, 30, 16, 90, 5), (1024, 6, 64, 5, 6), (1500, 8, 64, 64, 7), (8192, 3, 16, 3, 8)])
def test_steps_against_the_host(B, blocks, page, most, seed):
    from bitexact_llm_b200.pages import DevicePages
    r = random.Random(seed)
    pages = B * blocks
    order = list(range(1, pages + 1))
    r.shuffle(order)
    dev, host = DevicePages(B, blocks, pages, page, "cuda", torch.tensor(order)), Host(B, blocks, pages, page, order)
    for step in range(6):
        drop = [r.random() < 0.25 for _ in range(B)] if step % 2 else None
        counts = []
        for b in range(B):
            room = blocks * page - (0 if drop and drop[b] else host.lens[b])
            counts.append(min(room, r.choice([0, 1, most, r.randint(0, most)])))
        rows = sum(counts) + r.choice([0, 1, 70])
        got = dev.step(torch.tensor(counts).cuda(), rows, None if drop is None else torch.tensor(drop).cuda())
        equal(dev, host, got, host.step(counts, rows, drop))
    assert int(dev.status) == 0


def test_errors_change_nothing_and_stay():
    from bitexact_llm_b200.pages import INVALID, NO_PAGES, TOO_LONG, TOO_MANY_ROWS, DevicePages
    dev, host = DevicePages(4, 3, 7, 8, "cuda"), Host(4, 3, 7, 8)
    c = lambda *n: torch.tensor(n).cuda()
    equal(dev, host, dev.step(c(20, 3, 0, 9), 40), host.step([20, 3, 0, 9], 40))
    keep = [t.clone() for t in (dev.lens, dev.bt, dev.free, dev.top)]
    for counts, rows, bits in (((5, 0, 0, 0), 40, TOO_LONG), ((4, 6, 24, 0), 40, NO_PAGES), ((1, 1, 1, 1), 3, TOO_MANY_ROWS),
                               ((0, -1, 0, 0), 40, INVALID), ((5, 0, 0, -2), 0, TOO_LONG | INVALID), ((1 << 40, 0, 0, 0), 40, TOO_LONG)):
        assert host.step(list(counts), rows) == bits
        r = dev.step(c(*counts), rows)
        assert int(dev.status) == bits, counts
        assert (r.slot == -1).all() and (r.last == -1).all() and not r.seq.any() and not r.pos.any()
        assert all(torch.equal(a, b) for a, b in zip(keep, (dev.lens, dev.bt, dev.free, dev.top)))
        with pytest.raises(MemoryError if bits & NO_PAGES else ValueError):
            dev.check()
    dev.check()
    # the pages of a request that is over serve the step itself
    d = torch.tensor([True, False, False, False]).cuda()
    equal(dev, host, dev.step(c(24, 6, 0, 0), 64, d), host.step([24, 6, 0, 0], 64, [1, 0, 0, 0]))
    # sticky: a bit stays through steps that are in order
    dev.step(c(99, 0, 0, 0), 99)
    dev.step(c(0, 0, 0, 0), 4)
    with pytest.raises(ValueError):
        dev.check()


def test_functional_form_again_and_strided_table():
    from bitexact_llm_b200.pages import step_tables
    lens, counts = torch.tensor([5, 0, 64]).cuda(), torch.tensor([60, 0, 1]).cuda()
    wide = torch.zeros(3, 9, dtype=torch.int32, device="cuda")
    bt = wide[:, 2:6]
    bt[0, 0], bt[2, 0] = 11, 12
    free, top = torch.arange(20, 40, dtype=torch.int32, device="cuda"), torch.tensor([10], dtype=torch.int32).cuda()
    a = step_tables(lens, counts, bt, free, top, 64, 70)
    b = step_tables(lens, counts, bt, free, top, 64, 70)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert a.lens.tolist() == [65, 0, 65] and int(a.top) == 8 and lens.tolist() == [5, 0, 64] and int(top) == 10
    assert bt.tolist() == [[11, 29, 0, 0], [0] * 4, [12, 28, 0, 0]] and not wide[:, :2].any() and not wide[:, 6:].any()
    assert a.slot[:61].tolist() == [11 * 64 + 5 + i if i < 59 else 29 * 64 + i - 59 for i in range(60)] + [28 * 64]
    assert a.last.tolist() == [59, -1, 60] and (a.slot[61:] == -1).all()


def test_in_a_graph():
    from bitexact_llm_b200.pages import DevicePages
    B = 5
    dev, host = DevicePages(B, 6, 30, 4, "cuda"), Host(B, 6, 30, 4)
    counts = torch.ones(B, dtype=torch.long, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = dev.step(counts, 8)
    for step in range(9):
        c = [1, 1, step % 2, 1, 0]
        counts.copy_(torch.tensor(c))
        g.replay()
        equal(dev, host, r, host.step(c, 8))


def test_nothing():
    from bitexact_llm_b200.pages import DevicePages
    dev = DevicePages(0, 3, 4, 16, "cuda")
    r = dev.step(torch.zeros(0, dtype=torch.long, device="cuda"), 5)
    assert (r.slot == -1).all() and int(dev.top) == 4
    dev = DevicePages(2, 3, 0, 16, "cuda")
    assert dev.step(torch.zeros(2, dtype=torch.long, device="cuda"), 0).seq.shape == (0,)
    dev.step(torch.ones(2, dtype=torch.long, device="cuda"), 2)
    with pytest.raises(MemoryError):
        dev.check()


def test_refusals():
    from bitexact_llm_b200.pages import step_tables
    z = lambda *s, t=torch.int64: torch.zeros(*s, dtype=t, device="cuda")
    lens, bt, free, top = z(3), z(3, 4, t=torch.int32), z(9, t=torch.int32), z(1, t=torch.int32)
    good = dict(lens=lens, counts=z(3), bt=bt, free=free, top=top, page=16, rows=4)
    step_tables(**good)
    for change in (dict(lens=lens.int()), dict(counts=z(2)), dict(counts=z(6)[::2]), dict(bt=bt.long()), dict(bt=bt.t()), dict(bt=bt[:2]),
                   dict(free=free.long()), dict(free=z(18, t=torch.int32)[::2]), dict(top=z(2, t=torch.int32)), dict(top=z(1)), dict(page=0),
                   dict(rows=-1), dict(drop=z(3)), dict(drop=z(2, t=torch.bool)), dict(lens=lens.cpu()), dict(bt=bt[:1].expand(3, 4)),
                   dict(status=z(1)), dict(lens_out=z(3, t=torch.int32)), dict(top_out=z(2, t=torch.int32))):
        with pytest.raises(ValueError):
            step_tables(**{**good, **change})
