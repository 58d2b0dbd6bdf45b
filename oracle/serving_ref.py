"""Float64 restatements of the serving operators, from their formulas: masked
attention rows, attention over a paged cache, rotary positions, and the page
tables of a step.  Test infrastructure only; plain loops, no framework code.
"""

from __future__ import annotations

import math

import torch


def visible(pos: torch.Tensor, nk: int, window: int = 0, sinks: int = 0, causal: bool = True) -> torch.Tensor:
    """[rows, nk] mask: key j is seen from position p when j <= p and, with a
    window, j > p - window or j < sinks."""
    p, j = pos.view(-1, 1), torch.arange(nk, device=pos.device).view(1, -1)
    see = (j <= p) if causal else torch.ones((p.shape[0], nk), dtype=torch.bool, device=pos.device)
    if window:
        see = see & ((j > p - window) | (j < sinks))
    return see


def attend(q, k, v, see, scale):
    """Rows q [m, D] over k, v [n, D]: (O, A) in float64 with O = sum_j w_j v_j
    and A = sum_j w_j |v_j|, the scale of O's rounding errors.  A row that sees
    nothing is zero; values at places a row does not see do not matter."""
    q, k, v = q.double(), k.double(), v.double()
    seen = see.any(0)
    k = torch.where(seen[:, None], k, torch.zeros((), dtype=k.dtype, device=k.device))
    v = torch.where(seen[:, None], v, torch.zeros((), dtype=v.dtype, device=v.device))
    s = (q @ k.T * scale).masked_fill(~see, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[1] else s.new_zeros((s.shape[0], 1))
    w = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    w = w.masked_fill(~see, 0.0)
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total.clamp(min=1e-300), torch.zeros_like(w))
    return w @ v, w @ v.abs()


def window_attention(q, k, v, window, sinks, scale=None):
    """[B,Hq,Nq,D] causal (top-left) attention with a window and sinks: (O, A)."""
    B, Hq, Nq, D = q.shape
    G = Hq // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    see = visible(torch.arange(Nq, device=q.device), k.shape[2], window, sinks)
    pairs = [attend(q[b, h], k[b, h // G], v[b, h // G], see, scale) for b in range(B) for h in range(Hq)]
    return tuple(torch.stack(x).view(B, Hq, Nq, D) for x in zip(*pairs))


def paged_attention(q, k_pages, v_pages, block_table, kv_lens, cu_q, window=0, sinks=0, scale=None):
    """[T,Hq,D] over pages [P, page, Hkv, D]; row i of request r stands at
    position kv_lens[r] - (its new tokens) + i.  Rows of no request are NaN."""
    T, Hq, D = q.shape
    ps, G = k_pages.shape[1], Hq // k_pages.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64, device=q.device)
    mag = out.clone()
    cu, kv = cu_q.tolist(), kv_lens.tolist()
    for r, n in enumerate(kv):
        a, b = cu[r], cu[r + 1]
        pages = block_table[r, : -(-n // ps)].long()
        k = k_pages[pages].flatten(0, 1)[:n]
        v = v_pages[pages].flatten(0, 1)[:n]
        see = visible(torch.arange(n - (b - a), n, device=q.device), n, window, sinks)
        for h in range(Hq):
            out[a:b, h], mag[a:b, h] = attend(q[a:b, h], k[:, h // G], v[:, h // G], see, scale)
    return out, mag


def frequencies(rot, base=10000.0, scaling=None, factor=1.0, original_length=0, low=1.0, high=4.0):
    """Angle per position of each of the rot / 2 pairs."""
    out = []
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        elif scaling == "banded":
            turns = original_length * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            f = f * keep + f / factor * (1.0 - keep)
        out.append(f)
    return torch.tensor(out, dtype=torch.float64)


def rotate(x, pos, freq, layout, inverse=False, magnitude=1.0):
    """Float64 rotation of x [..., n, D] by the angles pos [n] * freq."""
    rot, y = 2 * freq.numel(), x.double().clone()
    a = pos.double()[:, None] * freq.to(x.device)
    c, s = magnitude * torch.cos(a), magnitude * torch.sin(a) * (-1 if inverse else 1)
    i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    u, v = x.double()[..., i], x.double()[..., j]
    y[..., i], y[..., j] = u * c - v * s, v * c + u * s
    return y


def page_tables(ctx, new, table, free, count, page_size, num_tokens):
    """One step's tables with plain loops: (table, slots, positions, cu_q,
    kv_lens, free_left, status); status 0 done, 1 too few free pages, 2 a
    request outgrows its row, 3 more new tokens than num_tokens."""
    ctx, new, free = ctx.tolist(), new.tolist(), free.tolist()
    table = [list(row) for row in table.tolist()]
    width = len(table[0]) if table else 0
    pages = lambda n: -(-n // page_size)  # noqa: E731
    need = [pages(c + n) - pages(c) for c, n in zip(ctx, new)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    status = 0
    if sum(need) > count:
        status = 1
    if any(pages(c + n) > width for c, n in zip(ctx, new)):
        status = 2
    if cu[-1] > num_tokens:
        status = 3
    slots, positions = [-1] * num_tokens, [0] * num_tokens
    left = count
    for r, (c, n) in enumerate(zip(ctx, new)):
        if status == 0:
            for i in range(need[r]):
                left -= 1
                table[r][pages(c) + i] = free[left]
        for i in range(n):
            t = cu[r] + i
            if t >= num_tokens:
                break
            positions[t] = c + i
            if status == 0 and table[r][(c + i) // page_size] >= 0:
                slots[t] = table[r][(c + i) // page_size] * page_size + (c + i) % page_size
    kv = [c + n for c, n in zip(ctx, new)] if status == 0 else ctx
    return table, slots, positions, cu, kv, left, status
