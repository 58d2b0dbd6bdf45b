"""Serving: a paged K/V cache, the tables of a step, and attention over them.

A cache is two tensors of pages, K and V, ``[num_pages, page_size, Hkv, 128]``
(any strides of the outer three: a ``[num_pages, Hkv, page_size, 128]`` pool is
passed as ``pool.transpose(1, 2)``).  One step of a serving loop is

    t = build_tables(lens, new, table, free, count, page_size=ps, num_tokens=T)
    q = append(k, v, k_pages, v_pages, t.slots, q=q, positions=t.positions, rotary=rotary)
    o = op(q, k_pages, v_pages, table, t.kv_lens, t.cu_q, max_q=longest)

or, the last two together, ``op.step(...)``.  ``t.kv_lens`` and ``t.free_left``
are the next step's lengths and free count.  Nothing synchronizes, and lengths
stay on the device, so a step can be captured into a CUDA graph; the operator and
the rotary must live as long as it.
"""

from __future__ import annotations

import threading
from dataclasses import dataclass

import torch

from . import calls, lib
from .ops import HEAD_DIM, _window
from .rotary import Rotary, differentiated, indexed

_first_use = threading.Lock()  # of an operator on a device


@dataclass
class StepTables:
    """What ``build_tables`` writes; pass it back as ``out`` to reuse its memory."""
    slots: torch.Tensor      # int64 [num_tokens], -1 behind the last token
    positions: torch.Tensor  # int32 [num_tokens]
    cu_q: torch.Tensor       # int32 [R + 1]
    kv_lens: torch.Tensor    # int32 [R]
    free_left: torch.Tensor  # int32 [1]
    status: torch.Tensor     # int32 [1]; None: taken to be 0

    @staticmethod
    def empty(requests: int, num_tokens: int, device) -> "StepTables":
        tables = StepTables(*calls.load().empty_tables(requests, num_tokens, torch.device(device)))
        tables.status.zero_()
        return tables

    def tensors(self) -> tuple:
        return (self.slots, self.positions, self.cu_q, self.kv_lens, self.free_left, self.status)


def build_tables(ctx_lens, new_lens, block_table, free_pages, free_count, *, page_size: int, num_tokens: int,
                 out: StepTables | None = None) -> StepTables:
    """The tables of a step in which request r, holding ctx_lens[r] tokens,
    adds new_lens[r] (int32 [R], on the GPU).

    The pages it needs beyond those it holds are taken from the end of the
    free list (int32 free_pages, of which the first free_count[0] are free), in
    request order, and entered into block_table (int32 [R, width]).
    num_tokens is the size of the step's token buffers; places behind the last
    token get slot -1 and position 0.

    ``status`` (on the GPU) is 0, or 1: too few free pages, 2: a request
    outgrows its row of block_table or 2^31 - 1 tokens, 3: more new tokens than
    num_tokens; then nothing is handed out, every slot is -1, kv_lens are
    ctx_lens (cu_q still counts the new tokens; ``PagedOperator.step`` gives
    zeros) and the table is as it was.  The outputs must not overlap the inputs
    or one another: a loop alternates between two ``StepTables``.
    """
    r = calls.load().build_tables(ctx_lens, new_lens, block_table, free_pages, free_count, page_size, num_tokens,
                                  None if out is None else out.tensors())
    return StepTables(*r) if out is None else out


def append(k, v, k_pages, v_pages, slots, *, q=None, positions=None, rotary: Rotary | None = None, q_out=None):
    """Writes a step's K and V ([T, Hkv, dim]) into the cache at ``slots``
    (int64 [T]; a slot outside the cache marks a padded token, which is
    skipped; the others are distinct).  With ``rotary``, K is turned by
    ``positions`` ([T], int32 or int64) on its way, and so is q [T, Hq, dim],
    which is returned (in q_out, which may be q).  One launch.  q, k and v may
    be slices of one projection's output.

    The cache holds values: derivatives of k and v end there.  The returned q
    keeps its graph, or its tangent, when q has one (then a second launch, and
    q_out must be None)."""
    if q is not None and differentiated(q):
        if q_out is not None:
            raise ValueError("q_out cannot be given when q requires a gradient or carries a tangent")
        if (q.ndim != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k_pages.shape[-1] or q.dtype != k_pages.dtype
                or q.device != k_pages.device):
            raise ValueError("q must be [T, heads, dim] of the cache's type and device")
        append(k, v, k_pages, v_pages, slots, positions=positions, rotary=rotary)
        return q.clone(memory_format=torch.contiguous_format) if rotary is None else rotary(q, positions)
    return calls.load().append(k, v, k_pages, v_pages, slots, q, positions if rotary is not None else None,
                               0 if rotary is None else rotary.desc(k_pages.device), q_out)


class PagedOperator:
    """``op(q, k_pages, v_pages, block_table, kv_lens, cu_q, max_q=n) -> O``:
    attention of a step's new tokens over a paged cache, FP16 or BF16.  Forward
    only: O has no graph.

    The operator owns the status words of each device, made by its first call
    there, which cannot be captured.  Everything else lives for one call, so
    calls may overlap: on any streams, in any graphs (which, as ever, must not
    share a memory pool if they are replayed at the same time).  Keep the
    operator as long as a graph that captured a call of it."""

    def __init__(self, *, timeout_us: int = 0):
        self.timeout_us = int(timeout_us)
        self.workspaces = {}  # device -> its status words
        lib.load()

    def workspace(self, device) -> torch.Tensor:
        """The status words on ``device``, which must exist before a capture."""
        ws = self.workspaces.get(device)
        if ws is None:
            device = indexed(device)
            with _first_use:
                ws = self.workspaces.get(device)
                if ws is None:
                    ws = self.workspaces[device] = self._new_workspace(device)
        return ws

    @staticmethod
    def _new_workspace(device) -> torch.Tensor:
        if device.type != "cuda":
            raise ValueError("the paged operator works on CUDA devices")
        with torch.cuda.device(device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first call on a device cannot be captured: call workspace(device) before")
            ws = torch.zeros(lib.WS_HEADER_BYTES, dtype=torch.uint8, device=device)
            torch.cuda.current_stream(device).synchronize()  # calls on other streams find them zeroed
        return ws

    def __call__(self, q, k_pages, v_pages, block_table, kv_lens, cu_q, *, max_q: int, scale: float | None = None,
                 window: int = 0, sinks: int = 0, out: torch.Tensor | None = None, flags: int = 0,
                 tables_status: torch.Tensor | None = None) -> torch.Tensor:
        """q [T, Hq, 128]; block_table int32 [R, width]; kv_lens int32 [R], the
        cached tokens of each request, its new ones included; cu_q int32
        [R + 1], the requests' rows of q.  Row i of request r stands at
        position kv_lens[r] - (its rows) + i and sees keys up to itself, with
        ``window`` > 0 only the last ``window`` of them and the first
        ``sinks`` of the request.  max_q is the longest request's rows as far
        as the host knows: it picks the kernel, a longer one is still right.

        Rows that see no key become zeros; rows of no request (behind
        cu_q[R]) are left as they were in ``out``, and undefined without it.  A page that holds no key
        any row of its work item sees is not read.  Where the table ends early
        or names a page outside the cache, zeros are read and
        ``status(device)`` says so.  A NaN or infinity in V at a key that some
        row of a work item sees can reach all of that item's rows.

        ``tables_status`` (int32 [1] on the GPU): the status of the step's
        ``build_tables``.  Where it is not 0 the new tokens have no place in the
        cache, and all their rows become zeros."""
        window, sinks = _window(window, sinks, True)
        return calls.load().paged(q, k_pages, v_pages, block_table, kv_lens, cu_q, max_q,
                                  HEAD_DIM ** -0.5 if scale is None else scale, window, sinks, out,
                                  self.workspace(q.device), self.timeout_us, flags, tables_status)

    def step(self, q, k, v, k_pages, v_pages, block_table, tables: StepTables, *, max_q: int,
             rotary: Rotary | None = None, scale: float | None = None, window: int = 0, sinks: int = 0,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """The attention of one layer in a step: appends k and v to the cache
        at ``tables``' slots, rotated when ``rotary`` is given, and returns
        the attention of the (rotated) q over it.  After a step that could not
        be met (``tables.status``) the cache is as it was and the rows are zeros."""
        if q.requires_grad:
            q = q.detach()  # the attention has no graph
        turned = append(k, v, k_pages, v_pages, tables.slots, q=q if rotary is not None else None,
                        positions=tables.positions if rotary is not None else None, rotary=rotary)
        return self(q if turned is None else turned, k_pages, v_pages, block_table, tables.kv_lens, tables.cu_q,
                    max_q=max_q, scale=scale, window=window, sinks=sinks, out=out, tables_status=tables.status)

    def status(self, device) -> tuple[int, int, int, int]:
        """Synchronize the device and read the status words {status, site, block, 0}."""
        ws = self.workspace(device)
        torch.cuda.synchronize(ws.device)
        with torch.cuda.device(ws.device):
            return lib.read_status(ws.data_ptr(), torch.cuda.current_stream(ws.device).cuda_stream)

    def reset_status(self, device) -> None:
        ws = self.workspace(device)
        with torch.cuda.device(ws.device):
            lib.reset_status(ws.data_ptr(), torch.cuda.current_stream(ws.device).cuda_stream)
