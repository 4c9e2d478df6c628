"""The block table and the token rows of a step, kept and made on the device (`bx_step_tables`): a decode step that takes pages as its
sequences grow needs no host synchronisation and can be captured into a CUDA graph.

`step_tables` is the operator; `DevicePages` holds the state of a pool (lengths, table, stack of free pages) and steps it in place.
`decode.Session(..., pages=n, on_device=True)` serves from one."""

from typing import NamedTuple

import torch

from . import _native as nv

TOO_LONG, NO_PAGES, TOO_MANY_ROWS, INVALID = 1, 2, 4, 8
MAX_REQUESTS = 8192


class StepTables(NamedTuple):
    seq: torch.Tensor           # int64 [rows]: request of every new token, in order
    pos: torch.Tensor           # int64 [rows]
    slot: torch.Tensor          # int64 [rows]: cache slot; the places behind the last token are (0, 0, -1)
    last: torch.Tensor          # int64 [B]: row of a request's last new token, -1 where it has none
    lens: torch.Tensor          # int64 [B]: the lengths behind the step
    top: torch.Tensor           # int32 [1]: free pages behind the step
    status: torch.Tensor        # int32 [1]: 0, or why nothing was done


def _whole(t, shape, dtype=torch.int64):
    return t.dtype == dtype and t.shape == shape and t.is_contiguous()


def step_tables(lens, counts, bt, free, top, page, rows, drop=None, lens_out=None, top_out=None, status=None):
    """lens, counts int64 [B]: tokens in the cache and new ones; bt int32 [B, blocks] (extended in place); free int32 [pool], top
    int32 [1]: the stack of free pages, of which the first `top` are there (its end is written in place); rows: token rows that the
    step has room for; drop bool [B] or None: requests that are over give their pages back first, and begin anew if they have new tokens.

    lens_out, top_out: where the state behind the step goes (may be lens and top; default: new tensors, so that the same call again
    gives the same rows; with drop the pages of one that is over and begins anew have changed by then). status: an int32 [1] to which this call's bits are added (default: a new one). Bits: TOO_LONG, NO_PAGES,
    TOO_MANY_ROWS, INVALID; with any of them no page changes hands and all rows are padding."""
    shape, i32 = lens.shape, torch.int32
    if lens.dim() != 1 or not (_whole(lens, shape) and _whole(counts, shape)) or lens_out is not None and not _whole(lens_out, shape):
        raise ValueError("step_tables: lens and counts int64 [B], contiguous")
    B, (stride, unit) = shape[0], bt.stride() if bt.dim() == 2 else (0, 0)
    if bt.dtype != i32 or bt.dim() != 2 or bt.shape[0] != B or bt.shape[1] < 1 or bt.shape[1] > 1 and unit != 1 or B > 1 and stride < bt.shape[1]:
        raise ValueError("step_tables: bt int32 [B, blocks], rows contiguous")
    if free.dtype != i32 or free.dim() != 1 or not free.is_contiguous():
        raise ValueError("step_tables: free int32 [pool], contiguous")
    if top.dtype != i32 or top.numel() != 1 or any(t is not None and (t.dtype != i32 or t.numel() != 1) for t in (top_out, status)):
        raise ValueError("step_tables: top and status int32 [1]")
    if drop is not None and not _whole(drop, shape, torch.bool):
        raise ValueError("step_tables: drop bool [B], contiguous")
    if page < 1 or rows < 0 or B > MAX_REQUESTS:
        raise ValueError(f"step_tables: pages of at least one token, at most {MAX_REQUESTS} requests")
    nv.here(lens, counts, bt, free, top, drop, lens_out, top_out, status)
    sticky = status is not None
    # the outputs are parts of two buffers: an allocation each costs more than the kernel
    seq, pos, slot, last, out = torch.empty(3 * rows + 2 * B, dtype=torch.int64, device=lens.device).split_with_sizes((rows, rows, rows, B, B))
    lens_out = out if lens_out is None else lens_out
    if top_out is None or status is None:
        a, b = torch.empty(2, dtype=i32, device=lens.device).split_with_sizes((1, 1))
        top_out, status = a if top_out is None else top_out, b if status is None else status
    rc = nv.lib().bx_step_tables(lens.data_ptr(), counts.data_ptr(), nv.ptr(drop), bt.data_ptr(), stride if B > 1 else bt.shape[1],
                                 bt.shape[1], page, free.data_ptr(), free.shape[0], top.data_ptr(), B, rows, seq.data_ptr(), pos.data_ptr(),
                                 slot.data_ptr(), last.data_ptr(), lens_out.data_ptr(), top_out.data_ptr(), status.data_ptr(), int(sticky),
                                 nv.stream())
    nv.check(rc, "bx_step_tables")
    return StepTables(seq, pos, slot, last, lens_out, top_out, status)


class DevicePages:
    """A pool of `pages` pages (numbers from 1 on, in the order of `order` when given) for B requests of up to `blocks` pages each."""

    def __init__(self, B, blocks, pages, page, dev, order=None):
        self.page = page
        self.lens = torch.zeros(B, dtype=torch.int64, device=dev)
        self.bt = torch.zeros(B, blocks, dtype=torch.int32, device=dev)
        order = torch.arange(1, pages + 1) if order is None else order
        self.free = order.flip(0).to(torch.int32).to(dev)
        self.top = torch.full((1,), pages, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)

    def step(self, counts, rows, drop=None):
        """One step in place: counts int64 [B] new tokens on at most `rows` rows. -> StepTables."""
        return step_tables(self.lens, counts, self.bt, self.free, self.top, self.page, rows, drop, self.lens, self.top, self.status)

    def take(self, counts, rows):
        """As `step`, but the lengths and the stack stay as they are until `commit`: pages for a call that may still fail. Raises at once
        what this call alone found (synchronises). -> StepTables."""
        t = step_tables(self.lens, counts, self.bt, self.free, self.top, self.page, rows)
        _told(int(t.status))
        return t

    def commit(self, t):
        """The state behind `take`."""
        self.lens.copy_(t.lens)
        self.top.copy_(t.top)

    def check(self):
        """Raises what a step found since the last check (synchronises)."""
        bits = int(self.status)
        self.status.zero_()
        _told(bits)


def _told(bits):
    """Raises what the bits of a status say."""
    if bits & NO_PAGES:
        raise MemoryError("the session has no free pages")
    if bits & TOO_LONG:
        raise ValueError("a sequence has more tokens than its row of the block table holds (max_len)")
    if bits:
        raise ValueError("a step had more new tokens than rows" if bits & TOO_MANY_ROWS else "a step's lengths or pages are not valid")
