"""Serving: a paged K/V cache, the tables of a step, and attention over them.

A cache is two tensors of pages, K and V, ``[num_pages, page_size, Hkv, 128]``
(any strides of the outer three: a ``[num_pages, Hkv, page_size, 128]`` pool is
passed as ``pool.transpose(1, 2)``).  One step of a serving loop is

    t = build_tables(lens, new, table, free, count, page_size=ps, num_tokens=T)
    q = append(k, v, k_pages, v_pages, t.slots, q=q, positions=t.positions, rotary=rotary)
    o = op(q, k_pages, v_pages, table, t.kv_lens, t.cu_q, max_q=longest)

or, the last two together, ``op.step(...)``.  ``t.kv_lens`` and ``t.free_left``
are the next step's lengths and free count.  Nothing synchronizes, and lengths
stay on the device, so a step can be captured into a CUDA graph.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import lib
from .ops import HEAD_DIM, _window
from .rotary import DTYPES, Rotary, _position_bits, call


def _int32(name, t, shape, device):
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or (shape is not None and t.shape != shape):
        want = "" if shape is None else f" of shape {tuple(shape)}"
        raise ValueError(f"{name} must be contiguous int32{want} on the same CUDA device")


@dataclass
class StepTables:
    """What ``build_tables`` writes; pass it back as ``out`` to reuse its memory."""
    slots: torch.Tensor      # int64 [num_tokens], -1 behind the last token
    positions: torch.Tensor  # int32 [num_tokens]
    cu_q: torch.Tensor       # int32 [R + 1]
    kv_lens: torch.Tensor    # int32 [R]
    free_left: torch.Tensor  # int32 [1]
    status: torch.Tensor     # int32 [1]

    @staticmethod
    def empty(requests: int, num_tokens: int, device) -> "StepTables":
        ints = torch.empty(2 * requests + 3 + num_tokens, dtype=torch.int32, device=device)
        cu, kv, left, status, pos = ints.split_with_sizes([requests + 1, requests, 1, 1, num_tokens])
        return StepTables(torch.empty(num_tokens, dtype=torch.int64, device=device), pos, cu, kv, left, status)


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
    outgrows its row of block_table, 3: more new tokens than num_tokens; then
    nothing is handed out, every slot is -1, kv_lens are ctx_lens and the table
    is as it was.  The outputs must not overlap the inputs: a loop alternates
    between two ``StepTables``.
    """
    dev = ctx_lens.device
    if dev.type != "cuda" or ctx_lens.ndim != 1 or block_table.ndim != 2:
        raise ValueError("ctx_lens must be [R] and block_table [R, width] on a CUDA device")
    R = ctx_lens.shape[0]
    _int32("ctx_lens", ctx_lens, (R,), dev)
    _int32("new_lens", new_lens, (R,), dev)
    _int32("free_pages", free_pages, (free_pages.numel(),), dev)
    _int32("free_count", free_count, (1,), dev)
    if (block_table.dtype != torch.int32 or block_table.device != dev or block_table.shape[0] != R
            or block_table.stride(1) != 1):
        raise ValueError("block_table must be int32 [R, width] with contiguous rows on the same CUDA device")
    if num_tokens < 0:
        raise ValueError("num_tokens must be at least 0")
    if out is None:
        out = StepTables.empty(R, num_tokens, dev)
    else:
        if out.slots.dtype != torch.int64 or out.slots.shape != (num_tokens,) or out.slots.device != dev:
            raise ValueError("out.slots must be int64 [num_tokens] on the same CUDA device")
        for name, shape in (("positions", (num_tokens,)), ("cu_q", (R + 1,)), ("kv_lens", (R,)), ("free_left", (1,)),
                            ("status", (1,))):
            _int32("out." + name, getattr(out, name), shape, dev)
        for t in (out.slots, out.positions, out.cu_q, out.kv_lens, out.free_left, out.status):
            for u in (ctx_lens, new_lens, free_pages, free_count):
                a, b = t.data_ptr(), u.data_ptr()
                if a < b + u.numel() * 4 and b < a + t.numel() * t.element_size():
                    raise ValueError("an output overlaps an input: alternate between two StepTables")
    call(dev, "b200fa_build_tables", ctx_lens.data_ptr(), new_lens.data_ptr(), R, block_table.data_ptr(),
         block_table.stride(0), block_table.shape[1], free_pages.data_ptr(), free_pages.numel(), free_count.data_ptr(),
         page_size, out.slots.data_ptr(), out.positions.data_ptr(), num_tokens, out.cu_q.data_ptr(),
         out.kv_lens.data_ptr(), out.free_left.data_ptr(), out.status.data_ptr())
    return out


def _pages(k_pages, v_pages, dim=None):
    """Checked (num_pages, page_size, Hkv, dim) of a cache."""
    if k_pages.ndim != 4 or v_pages.shape != k_pages.shape or (dim is not None and k_pages.shape[3] != dim):
        raise ValueError(f"k_pages and v_pages must be [num_pages, page_size, Hkv, {dim or 'dim'}]")
    if (k_pages.device.type != "cuda" or v_pages.device != k_pages.device or v_pages.dtype != k_pages.dtype
            or k_pages.dtype not in (torch.float16, torch.bfloat16)):
        raise ValueError("the cache must be FP16 or BF16, K and V alike, on one CUDA device")
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        raise ValueError("the head dimension of the cache must be contiguous")
    return k_pages.shape


def _rows(name, t, shape, like):
    if t.ndim != 3 or (t.shape[0] != shape[0] or t.shape[2] != shape[2] or shape[1] not in (None, t.shape[1])):
        raise ValueError(f"{name} must be [{shape[0]}, {shape[1] or 'heads'}, {shape[2]}]")
    if t.dtype != like.dtype or t.device != like.device or t.stride(2) != 1:
        raise ValueError(f"{name} must have the cache's type and device and a contiguous last dimension")


def append(k, v, k_pages, v_pages, slots, *, q=None, positions=None, rotary: Rotary | None = None, q_out=None):
    """Writes a step's K and V ([T, Hkv, dim]) into the cache at ``slots``
    (int64 [T]; a slot outside the cache marks a padded token, which is
    skipped; the others are distinct).  With ``rotary``, K is turned by
    ``positions`` ([T], int32 or int64) on its way, and so is q [T, Hq, dim],
    which is returned (in q_out, which may be q).  One launch.  q, k and v may
    be slices of one projection's output."""
    pages, ps, hkv, dim = _pages(k_pages, v_pages)
    if k.ndim != 3:
        raise ValueError("k must be [T, Hkv, dim]")
    T = k.shape[0]
    _rows("k", k, (T, hkv, dim), k_pages)
    _rows("v", v, (T, hkv, dim), k_pages)
    dev = k_pages.device
    if slots.dtype != torch.int64 or slots.shape != (T,) or slots.device != dev or not slots.is_contiguous():
        raise ValueError("slots must be contiguous int64 [T] on the same CUDA device")
    bits, desc, pos_ptr = 32, None, None
    if rotary is not None:
        if positions is None or positions.shape != (T,):
            raise ValueError("rotary needs positions [T]")
        if rotary.dim != dim:
            raise ValueError(f"the rotary's dim is {rotary.dim}, the cache's {dim}")
        bits, pos_ptr = _position_bits(positions, dev), positions.data_ptr()
        desc = rotary.desc(dev)
    if q is not None:
        _rows("q", q, (T, None, dim), k_pages)
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif q_out.shape != q.shape:
            raise ValueError("q_out must be shaped like q")
        _rows("q_out", q_out, (T, None, dim), k_pages)
        qa = (q.data_ptr(), lib.strides(*q.stride()[:2]), q_out.data_ptr(), lib.strides(*q_out.stride()[:2]))
    else:
        qa = (None, None, None, None)
    call(dev, "b200fa_append", *qa, k.data_ptr(), lib.strides(*k.stride()[:2]), v.data_ptr(),
         lib.strides(*v.stride()[:2]), k_pages.data_ptr(), lib.strides(*k_pages.stride()[:3]), v_pages.data_ptr(),
         lib.strides(*v_pages.stride()[:3]), T, 0 if q is None else q.shape[1], hkv, dim, pages, ps, slots.data_ptr(),
         pos_ptr, bits, desc, DTYPES[k_pages.dtype])
    return q_out


class PagedOperator:
    """``op(q, k_pages, v_pages, block_table, kv_lens, cu_q, max_q=n) -> O``:
    attention of a step's new tokens over a paged cache, FP16 or BF16.

    The operator owns a workspace per device; its calls must not overlap on
    the GPU (one operator per stream, and per graph of graphs that may run at
    the same time).  The first call on a device allocates it and cannot be
    captured."""

    def __init__(self, *, timeout_us: int = 0):
        self.timeout_us = int(timeout_us)
        self.workspaces = {}  # device -> uint8 tensor
        lib.load()

    def workspace(self, device) -> torch.Tensor:
        ws = self.workspaces.get(device)
        if ws is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first call on a device cannot be captured: call workspace(device) before")
            with torch.cuda.device(device):
                n = int(lib.load().b200fa_paged_workspace_size())
                lib.check(n if n < 0 else 0, "b200fa_paged_workspace_size")
                ws = torch.zeros(n, dtype=torch.uint8, device=device)
                torch.cuda.current_stream(device).synchronize()  # calls on other streams find it zeroed
            self.workspaces[device] = ws
        return ws

    def __call__(self, q, k_pages, v_pages, block_table, kv_lens, cu_q, *, max_q: int, scale: float | None = None,
                 window: int = 0, sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
        """q [T, Hq, 128]; block_table int32 [R, width]; kv_lens int32 [R], the
        cached tokens of each request, its new ones included; cu_q int32
        [R + 1], the requests' rows of q.  Row i of request r stands at
        position kv_lens[r] - (its rows) + i and sees keys up to itself, with
        ``window`` > 0 only the last ``window`` of them and the first
        ``sinks`` of the request.  max_q is the longest request's rows as far
        as the host knows: it picks the kernel, a longer one is still right.

        Rows that see no key become zeros; rows of no request (behind
        cu_q[R]) are left as they were in ``out``.  A page that holds no key
        any row of its work item sees is not read.  Where the table ends early
        or names a page outside the cache, zeros are read and
        ``status(device)`` says so.  A NaN or infinity in V at a key that some
        row of a work item sees can reach all of that item's rows."""
        pages, ps, hkv, _ = _pages(k_pages, v_pages, HEAD_DIM)
        if q.ndim != 3:
            raise ValueError(f"q must be [T, Hq, {HEAD_DIM}]")
        T, hq, _ = q.shape
        _rows("q", q, (T, None, HEAD_DIM), k_pages)
        if hq % hkv:
            raise ValueError("the query heads must be a multiple of the cache's heads")
        dev = q.device
        if kv_lens.ndim != 1:
            raise ValueError("kv_lens must be [R]")
        R = kv_lens.shape[0]
        _int32("kv_lens", kv_lens, (R,), dev)
        _int32("cu_q", cu_q, (R + 1,), dev)
        if (block_table.ndim != 2 or block_table.dtype != torch.int32 or block_table.device != dev
                or block_table.shape[0] != R or block_table.stride(1) != 1):
            raise ValueError("block_table must be int32 [R, width] with contiguous rows on the same CUDA device")
        window, sinks = _window(window, sinks, True)
        if out is None:
            out = torch.empty((T, hq, HEAD_DIM), dtype=q.dtype, device=dev)
        elif out.shape != q.shape:
            raise ValueError("out must be shaped like q")
        else:
            _rows("out", out, (T, None, HEAD_DIM), k_pages)
        ws = self.workspace(dev)
        qs, os = q.stride(), out.stride()
        ks, vs = k_pages.stride(), v_pages.stride()
        args = lib.paged_args.pack(
            lib.paged_args.size, DTYPES[q.dtype], q.data_ptr(), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            qs[0], qs[1], os[0], os[1], *ks[:3], *vs[:3], block_table.data_ptr(), block_table.stride(0),
            kv_lens.data_ptr(), cu_q.data_ptr(), T, pages, R, block_table.shape[1], ps, hq, hkv,
            max(0, min(int(max_q), 2**31 - 1)), HEAD_DIM ** -0.5 if scale is None else scale, window, sinks,
            self.timeout_us, ws.data_ptr(), ws.numel())
        call(dev, "b200fa_paged_fwd", args)
        return out

    def step(self, q, k, v, k_pages, v_pages, block_table, tables: StepTables, *, max_q: int,
             rotary: Rotary | None = None, scale: float | None = None, window: int = 0, sinks: int = 0,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """The attention of one layer in a step: appends k and v to the cache
        at ``tables``' slots, rotated when ``rotary`` is given, and returns
        the attention of the (rotated) q over it."""
        turned = append(k, v, k_pages, v_pages, tables.slots, q=q if rotary is not None else None,
                        positions=tables.positions if rotary is not None else None, rotary=rotary)
        return self(q if turned is None else turned, k_pages, v_pages, block_table, tables.kv_lens, tables.cu_q,
                    max_q=max_q, scale=scale, window=window, sinks=sinks, out=out)

    def status(self, device) -> tuple[int, int, int, int]:
        """Synchronize and read the device status header {status, site, block, 0}."""
        ws = self.workspace(_indexed(device))
        with torch.cuda.device(ws.device):
            return lib.read_status(ws.data_ptr(), torch.cuda.current_stream(ws.device).cuda_stream)

    def reset_status(self, device) -> None:
        ws = self.workspace(_indexed(device))
        with torch.cuda.device(ws.device):
            lib.reset_status(ws.data_ptr(), torch.cuda.current_stream(ws.device).cuda_stream)


def _indexed(device) -> torch.device:
    device = torch.device(device)
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device
