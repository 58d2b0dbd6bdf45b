"""The serving operators: page tables, rotary positions and the cache append,
attention over a paged cache, and a loop of all of them.

Tolerances count roundings of half a step (``finfo.eps / 2`` relative).
Rotary: u cos - v sin in FP32 from FP32 sines.  A sine is off by the angle's
32-bit remainder (2^-25 turns < 2e-7 rad) and two roundings of its own, a
product and the sum by three more: under 6e-7 (|u| + |v|) |magnitude|, plus the
output's rounding.  Attention, with w the weights, A = sum w |v|, O the float64
result: P is rounded to the cache's type, scores are FP32 sums of 128 products
that stay below 2^5 in all (128 * 2^-24 * 2^5 < 3e-4 absolute in the exponent),
exponentials and FP32 sums are good to 2^-16; O is rounded to the cache's type.
"""

import itertools
import random

import pytest
import torch

from oracle import serving_ref as ref

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16, torch.float32)}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
gpu = pytest.mark.gpu


def _within(got, O, A, extra=0.0):
    h = HALF[got.dtype]
    bound = A * (h + 3e-4 + 2.0 ** -16) + O.abs() * h + 2.0 ** -24 + extra
    over = (got.double() - O).abs() - bound
    assert torch.isfinite(got).all()
    assert bool((over <= 0).all()), float(over.max())


# ------------------------------------------------------------------- tables
def _tables_case(R, max_ctx, max_new, ps, seed, spare=3, width=None):
    rng = random.Random(seed)
    ctx = [rng.randint(0, max_ctx) for _ in range(R)]
    new = [rng.randint(0, max_new) for _ in range(R)]
    pages = lambda n: -(-n // ps)  # noqa: E731
    width = width or max(1, max(pages(c + n) for c, n in zip(ctx, new)))
    need = sum(pages(c + n) - pages(c) for c, n in zip(ctx, new))
    ids = list(range(sum(map(pages, ctx)) + need + spare))
    rng.shuffle(ids)
    table, at = [], 0
    for c in ctx:
        table.append((ids[at:at + pages(c)] + [-1] * width)[:width])
        at += pages(c)
    free = ids[at:]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return i32(ctx), i32(new), i32(table), i32(free), len(free), sum(new)


def _check_tables(ctx, new, table, free, count, ps, T):
    from fa_b200.paged import build_tables

    want = ref.page_tables(ctx, new, table, free, count, ps, T)
    dev = "cuda"
    t = table.to(dev)
    got = build_tables(ctx.to(dev), new.to(dev), t, free.to(dev), torch.tensor([count], dtype=torch.int32, device=dev),
                       page_size=ps, num_tokens=T)
    assert got.status.tolist() == [want[6]]
    assert t.tolist() == want[0]
    assert got.slots.tolist() == want[1] and got.positions.tolist() == want[2]
    assert got.cu_q.tolist() == want[3] and got.kv_lens.tolist() == want[4] and got.free_left.tolist() == [want[5]]
    return want[6]


@gpu
@pytest.mark.parametrize("R,max_ctx,max_new,ps", [
    (1, 0, 1, 16), (1, 16, 1, 16), (8, 100, 1, 16), (3, 0, 40, 8), (37, 500, 90, 64), (256, 300, 7, 32),
    (257, 60, 60, 128), (1000, 40, 3, 8), (4096, 9, 2, 8)])
def test_tables(R, max_ctx, max_new, ps):
    ctx, new, table, free, count, total = _tables_case(R, max_ctx, max_new, ps, R + ps)
    assert _check_tables(ctx, new, table, free, count, ps, total + 5) == 0
    assert _check_tables(ctx, new, table, free, count, ps, total) == 0


@gpu
def test_tables_that_cannot_be_met_hand_nothing_out():
    ctx, new, table, free, count, total = _tables_case(9, 200, 50, 16, 4, spare=0)
    assert _check_tables(ctx, new, table, free, count, 16, total) == 0       # to the last page
    assert _check_tables(ctx, new, table, free, count - 1, 16, total) == 1
    assert _check_tables(ctx, new, table, free, count, 16, total - 1) == 3
    ctx, new, table, free, count, total = _tables_case(9, 200, 50, 16, 4, spare=40, width=13)
    assert _check_tables(ctx, new, table[:, :12].contiguous(), free, count, 16, total) == 2


@gpu
def test_tables_with_a_count_beyond_the_list_and_negative_lengths():
    from fa_b200.paged import build_tables

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table = i32([[-1, -1], [7, -1]])
    r = build_tables(i32([-5, 3]), i32([17, -2]), table, i32([4, 5]), i32([1000]), page_size=16, num_tokens=20)
    assert r.status.tolist() == [0] and r.kv_lens.tolist() == [17, 3] and r.free_left.tolist() == [0]
    assert table.tolist() == [[5, 4], [7, -1]]
    assert r.slots.tolist() == [5 * 16 + i for i in range(16)] + [64] + [-1] * 3


# ------------------------------------------------------------------- rotary
SCALINGS = [{}, {"scaling": "linear", "factor": 4.0},
            {"scaling": "banded", "factor": 8.0, "original_length": 4096, "low": 1.0, "high": 4.0, "magnitude": 1.2}]


def _rotary(dim, rot, layout, scaling):
    from fa_b200.rotary import Rotary

    freq = ref.frequencies(rot, **{k: v for k, v in scaling.items() if k != "magnitude"})
    return Rotary(dim, rotary_dim=rot, layout=layout, **scaling), freq, scaling.get("magnitude", 1.0)


def _check_rotation(got, x, pos, freq, layout, inverse, mag):
    want = ref.rotate(x, pos, freq, layout, inverse, mag)
    rot = 2 * freq.numel()
    size = ref.rotate(x.double().abs(), torch.zeros_like(pos), freq, layout, False, 0.0)  # only the copied part
    u = x.double().abs()
    i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    size[..., i] = size[..., j] = (u[..., i] + u[..., j]) * mag
    size[..., rot:] = 0
    tol = 6e-7 * size + HALF[x.dtype] * want.abs() * (1 + 6e-7) + 2.0 ** -25
    tol[..., rot:] = 0
    over = (got.double() - want).abs() - tol
    assert bool((over <= 0).all()), float(over.max())


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 32), (64, 64), (96, 48), (16, 16), (256, 128)])
def test_rotary(dim, rot, layout, dtype):
    g = torch.Generator(device="cuda").manual_seed(dim + rot)
    for k, (scaling, inverse) in enumerate(itertools.product(SCALINGS, (False, True))):
        rotary, freq, mag = _rotary(dim, rot, layout, scaling)
        B, H, N = (1, 3, 1) if k == 0 else (2, 5, 37 * k)
        x = torch.randn((B, H, N, dim), generator=g, device="cuda").to(dtype)
        pos = torch.randint(0, 1 << 20, (N,), generator=g, device="cuda", dtype=torch.int64 if k % 2 else torch.int32)
        _check_rotation(rotary(x, pos, inverse=inverse), x, pos, freq, layout, inverse, mag)


@gpu
def test_rotary_of_far_positions_per_batch_strides_and_in_place():
    rotary, freq, _ = _rotary(128, 128, "half", {})
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((2, 300, 4, 128), generator=g, device="cuda").half().transpose(1, 2)  # [B,H,N,D], token-major
    pos = torch.randint(0, 1 << 26, (2, 300), generator=g, device="cuda")
    y = rotary(x, pos)
    for b in range(2):  # float64 angles are good to 2^26 * 2^-52 here
        _check_rotation(y[b], x[b], pos[b], freq, "half", False, 1.0)
    back = rotary(y.float(), pos, inverse=True)
    assert float((back - y.float()).abs().max()) > 0.1
    z = x.clone(memory_format=torch.preserve_format)
    assert rotary(z, pos, out=z) is z and torch.equal(z, y)
    t = rotary(x[0].transpose(0, 1), pos[0])  # [N,H,D]
    assert torch.equal(t.transpose(0, 1), y[0])
    n = rotary(x[:, :, :7])  # positions 0 .. 6
    _check_rotation(n, x[:, :, :7], torch.arange(7, device="cuda"), freq, "half", False, 1.0)
    assert rotary(x[:, :, :0]).shape == (2, 4, 0, 128)


@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_inverse_is_the_gradient(layout):
    """y = R x is linear: the gradient of sum(g * y) is R^T g, against the
    formula's autograd in float64 and against differences of the kernel."""
    rotary, freq, mag = _rotary(64, 32, layout, SCALINGS[2])
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((1, 2, 9, 64), generator=gen, device="cuda")
    gy = torch.randn_like(x)
    pos = torch.arange(9, device="cuda") * 1001
    grad = rotary(gy, pos, inverse=True)
    xd = x.double().requires_grad_()
    rot = 32
    a = pos.double()[:, None] * freq.cuda()
    c, s = mag * a.cos(), mag * a.sin()
    i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    u, v = xd[..., i], xd[..., j]
    loss = ((u * c - v * s) * gy.double()[..., i] + (v * c + u * s) * gy.double()[..., j]).sum()
    loss = loss + (xd[..., rot:] * gy.double()[..., rot:]).sum()
    loss.backward()
    assert float((grad.double() - xd.grad).abs().max()) <= 6e-7 * 2 * 1.2 * float(gy.abs().max()) + 2.0 ** -20
    step = 2.0 ** -3
    for e in (0, 5, 31, 40):
        d = torch.zeros_like(x)
        d[..., e] = step
        diff = ((rotary(x + d, pos) - rotary(x - d, pos)).double() * gy.double()).sum(-1) / (2 * step)
        # y is off by at most 6e-7 * 2 * |x| at each side, summed over the pair
        assert float((diff - grad[..., e].double()).abs().max()) <= 4 * 6e-7 * 2 * 1.2 * 5 * 5 / (2 * step) + 1e-6


@gpu
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_under_autograd(inverse):
    rotary, freq, _ = _rotary(32, 32, "half", SCALINGS[2])
    x = torch.randn((2, 3, 7, 32), device="cuda", requires_grad=True)
    pos = torch.arange(7, device="cuda") * 37
    for grad in (torch.randn_like(x), torch.ones((1,), device="cuda").expand(2, 3, 7, 32)):
        y = rotary(x, pos, inverse=inverse)
        assert torch.equal(y.detach(), rotary(x.detach(), pos, inverse=inverse))
        (got,) = torch.autograd.grad(y, x, grad)
        assert torch.equal(got, rotary(grad.contiguous(), pos, inverse=not inverse))
        xx = x.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
        rotary(xx).sum().backward()
        assert torch.equal(xx.grad, rotary(torch.ones_like(x).detach(), inverse=True))
    with pytest.raises(ValueError):
        rotary(x, pos, out=torch.empty_like(x))
    with torch.no_grad():
        rotary(x, pos, out=torch.empty_like(x))


@gpu
def test_written_tensors_must_not_be_expanded():
    from fa_b200 import lib
    from fa_b200.paged import append

    rotary, _, _ = _rotary(128, 128, "half", {})
    x = torch.randn((2, 3, 4, 128), device="cuda").half()
    with pytest.raises(lib.B200FAError):
        rotary(x, out=torch.empty((1, 3, 4, 128), dtype=F16, device="cuda").expand(2, -1, -1, -1))
    assert torch.equal(rotary(x[:1].expand(2, -1, -1, -1)), rotary(x[:1].repeat(2, 1, 1, 1)))
    k = torch.randn((4, 2, 128), device="cuda").half()
    pages = torch.zeros((1, 8, 2, 128), dtype=F16, device="cuda").expand(3, -1, -1, -1)
    with pytest.raises(lib.B200FAError):
        append(k, k, pages, pages, torch.arange(4, device="cuda"))


@gpu
def test_rotary_inside_the_dense_operator():
    from fa_b200.ops import Operator

    rotary, freq, _ = _rotary(128, 128, "half", {})
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn((1, h, 333, 128), generator=g, device="cuda").half() for h in (4, 2, 2))
    op = Operator("fp32")
    pos = torch.arange(333, device="cuda") + 70
    assert torch.equal(op(q, k, v, causal=True, rotary=rotary, positions=pos),
                       op(rotary(q, pos), rotary(k, pos), v, causal=True))
    assert torch.equal(op(q, k, v, rotary=rotary), op(rotary(q), rotary(k), v))
    with pytest.raises(ValueError):
        op(q, k[:, :, :300].contiguous(), v[:, :, :300].contiguous(), rotary=rotary, positions=pos)
    with pytest.raises(ValueError):
        op(q, k, v, positions=pos)


# ------------------------------------------------------------------- append
@gpu
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("layout,rot", [("half", 128), ("interleaved", 64), (None, 0)])
@pytest.mark.parametrize("T,hq,hkv,ps,heads_first", [(1, 4, 1, 8, False), (5, 2, 2, 16, True), (300, 12, 1, 64, False),
                                                     (2111, 32, 8, 16, True)])
def test_append(T, hq, hkv, ps, heads_first, layout, rot, dtype):
    from fa_b200.paged import append

    g = torch.Generator(device="cuda").manual_seed(T + rot)
    qkv = torch.randn((T, hq + 2 * hkv, 128), generator=g, device="cuda").to(dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    pages = -(-T // ps) + 2
    shape = (pages, hkv, ps, 128) if heads_first else (pages, ps, hkv, 128)
    kp, vp = (torch.full(shape, 3.0, dtype=dtype, device="cuda") for _ in range(2))
    if heads_first:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    slots = torch.randperm(pages * ps, generator=g, device="cuda")[:T]
    slots[::7] = -1
    slots[3::7] = pages * ps + slots[3::7]  # outside: skipped as well
    pos = torch.randint(0, 100000, (T,), generator=g, device="cuda", dtype=torch.int32)
    rotary = freq = None
    if layout:
        rotary, freq, _ = _rotary(128, rot, layout, SCALINGS[1])
    out = append(k, v, kp, vp, slots, q=q, positions=pos if layout else None, rotary=rotary)
    real = (slots >= 0) & (slots < pages * ps)
    at = slots[real]
    gk, gv = kp[at // ps, at % ps], vp[at // ps, at % ps]
    assert torch.equal(gv, v[real])
    if layout:
        _check_rotation(gk.transpose(0, 1), k[real].transpose(0, 1), pos[real], freq, layout, False, 1.0)
        _check_rotation(out.transpose(0, 1), q.transpose(0, 1), pos, freq, layout, False, 1.0)
    else:
        assert torch.equal(gk, k[real]) and torch.equal(out, q)
    left = torch.ones(pages * ps, dtype=torch.bool, device="cuda")
    left[at] = False
    for t in (kp, vp):
        assert bool((t.reshape(pages * ps, hkv, 128)[left] == 3.0).all())


@gpu
def test_append_without_q_in_place_q_and_no_tokens():
    from fa_b200.paged import append

    rotary, _, _ = _rotary(128, 128, "half", {})
    k = torch.randn((6, 2, 128), device="cuda").half()
    v, q = torch.randn_like(k), torch.randn((6, 4, 128), device="cuda").half()
    kp, vp = (torch.zeros((3, 8, 2, 128), dtype=F16, device="cuda") for _ in range(2))
    slots, pos = torch.arange(6, device="cuda") + 9, torch.arange(6, device="cuda")
    assert append(k, v, kp, vp, slots, positions=pos, rotary=rotary) is None
    assert torch.equal(kp.view(24, 2, 128)[9:15], rotary(k, pos))
    want = rotary(q, pos)
    assert torch.equal(append(k, v, kp, vp, slots, positions=pos, rotary=rotary, q=q), want)
    assert append(k, v, kp, vp, slots, positions=pos, rotary=rotary, q=q, q_out=q) is q and torch.equal(q, want)
    assert append(k[:0], v[:0], kp, vp, slots[:0]) is None


# -------------------------------------------------------------------- paged
def _paged_case(lens, hq, hkv, ps, dtype, seed, heads_first=False, spare_rows=0, extra_pages=3):
    """lens: (new tokens, cached tokens) per request.  Everything no row may
    read is NaN: unused pages, and offsets behind a request's last key."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    R, width = len(lens), max(1, max(-(-kv // ps) for _, kv in lens)) + 1
    T = sum(n for n, _ in lens)
    q = torch.randn((T + spare_rows, hq, 128), generator=g, device="cuda").to(dtype)
    used = [-(-kv // ps) for _, kv in lens]
    pages = sum(used) + extra_pages
    ids = torch.randperm(pages, generator=g, device="cuda").tolist()
    shape = (pages, hkv, ps, 128) if heads_first else (pages, ps, hkv, 128)
    kp, vp = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    if heads_first:
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    table = torch.full((R, width), -1, dtype=torch.int32)
    at = 0
    for r, (_, kv) in enumerate(lens):
        table[r, :used[r]] = torch.tensor(ids[at:at + used[r]], dtype=torch.int32)
        at += used[r]
        i = torch.arange(kv, device="cuda")
        pg = table[r].cuda().long()[i // ps]
        kp[pg, i % ps] = torch.randn((kv, hkv, 128), generator=g, device="cuda").to(dtype)
        vp[pg, i % ps] = torch.randn((kv, hkv, 128), generator=g, device="cuda").to(dtype)
    cu = [0]
    for n, _ in lens:
        cu.append(cu[-1] + n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return q, kp, vp, table.cuda(), i32([kv for _, kv in lens]), i32(cu), max(n for n, _ in lens)


def _check_paged(case, window=0, sinks=0, op=None, max_q=None, scale=None):
    from fa_b200.paged import PagedOperator

    q, kp, vp, table, kv, cu, longest = case
    op = op or PagedOperator()
    out = torch.full_like(q, 7.0)
    got = op(q, kp, vp, table, kv, cu, max_q=max_q or longest, window=window, sinks=sinks, out=out, scale=scale)
    assert got is out
    torch.cuda.synchronize()
    assert op.status(q.device)[0] == 0, op.status(q.device)
    O, A = ref.paged_attention(q, kp, vp, table, kv, cu, window, sinks, scale)
    n = int(cu[-1])
    _within(out[:n], O[:n], A[:n])
    assert bool((out[n:] == 7.0).all())
    blank = A[:n].amax(-1) == 0
    assert bool((out[:n][blank] == 0).all())
    return out


LENGTHS = {
    "one": [(1, 1)],
    "one_long": [(1, 5000)],
    "block_edges": [(1, 127), (1, 128), (1, 129), (1, 256), (1, 8)],
    "ragged": [(1, 33), (1, 2000), (1, 1), (1, 700), (1, 64)],
    "empty_requests": [(0, 10), (1, 5), (0, 0), (2, 300), (0, 7)],
    "short": [(5, 400), (1, 90), (3, 3), (7, 1000)],
    "chunks": [(130, 130), (70, 900), (1, 500), (33, 2000)],
    "chunk_long": [(600, 3300)],
    "rows_before_the_cache": [(9, 4), (3, 0), (2, 50)],
    "many": [(1 + i % 3, 10 + 37 * i) for i in range(40)],
}


@gpu
@pytest.mark.parametrize("lens,hq,hkv,ps,window", [
    ([(1, 1 + 7 * i % 400) for i in range(1500)], 4, 4, 16, 0),           # more requests than threads of a block
    ([(2 if i % 3 else 0, 3 + i % 90) for i in range(900)], 6, 1, 8, 50),
    ([(3, 700), (1, 40), (9, 2000)], 128, 1, 32, 0),                      # one token per tile and CTA
    ([(3, 700), (1, 40), (9, 2000)], 100, 1, 16, 129),
    ([(5, 600), (200, 900)], 65, 65, 64, 0)])
def test_paged_many_requests_and_wide_groups(lens, hq, hkv, ps, window):
    _check_paged(_paged_case(lens, hq, hkv, ps, F16, 31, spare_rows=1), window, 3 if window else 0)


@gpu
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv,ps", [(12, 1, 16), (32, 8, 32), (2, 2, 64), (6, 2, 8), (40, 1, 128), (16, 4, 256)])
@pytest.mark.parametrize("name", list(LENGTHS))
def test_paged(name, hq, hkv, ps, dtype):
    case = _paged_case(LENGTHS[name], hq, hkv, ps, dtype, seed=hq + ps, heads_first=hkv == 8, spare_rows=3)
    _check_paged(case)


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 4), (128, 0), (129, 130), (500, 16), (10000, 5), (37, 100000)])
@pytest.mark.parametrize("hq,hkv,ps,dtype", [(12, 1, 16, F16), (8, 8, 64, BF16), (32, 8, 32, BF16)])
def test_paged_window(window, sinks, hq, hkv, ps, dtype):
    for name in ("ragged", "short", "chunks", "rows_before_the_cache", "chunk_long"):
        _check_paged(_paged_case(LENGTHS[name], hq, hkv, ps, dtype, seed=window + hq), window, sinks)


@gpu
@pytest.mark.parametrize("max_q", [1, 8, 4096])
def test_paged_any_max_q_is_right(max_q):
    for name in ("short", "chunks", "ragged"):
        _check_paged(_paged_case(LENGTHS[name], 12, 1, 16, F16, 5), max_q=max_q, scale=0.2)


@gpu
@pytest.mark.parametrize("lens", [[(1, 3000), (4, 1500)], [(300, 3000), (1, 900)]], ids=["short", "chunk"])
def test_pages_behind_the_window_may_be_gone(lens):
    from fa_b200.paged import PagedOperator

    op, ps, window, sinks = PagedOperator(), 16, 200, 20
    case = _paged_case(lens, 12, 1, ps, F16, 6)
    want = _check_paged(case, window, sinks, op)
    q, kp, vp, table, kv, cu, longest = case
    for r, (n, total) in enumerate(lens):
        # Every page between the sinks and the first row's window.
        table[r, -(-sinks // ps):(total - n + 1 - window) // ps] = -1
    out = torch.full_like(want, 7.0)
    op(q, kp, vp, table, kv, cu, max_q=longest, window=window, sinks=sinks, out=out)
    assert op.status(q.device)[0] == 0
    assert torch.equal(out, want)


@gpu
@pytest.mark.parametrize("lens", [[(1, 600)], [(200, 600)]], ids=["short", "chunk"])
def test_bad_pages_read_as_zeros_and_are_reported(lens):
    from fa_b200 import lib
    from fa_b200.paged import PagedOperator

    op = PagedOperator()
    case = _paged_case(lens, 4, 2, 32, F16, 8)
    q, kp, vp, table, kv, cu, longest = case
    good = table.clone()
    for bad in (-1, kp.shape[0], 2**31 - 1):
        table.copy_(good)
        table[0, 3] = bad
        out = op(q, kp, vp, table, kv, cu, max_q=longest)
        assert op.status(q.device)[0] == lib.DEV_PAGE
        op.reset_status(q.device)
        k2, v2 = kp.clone(), vp.clone()
        k2[good[0, 3].long()] = 0
        v2[good[0, 3].long()] = 0
        O, A = ref.paged_attention(q, k2, v2, good, kv, cu)
        _within(out, O, A)
    # A length beyond the table's width is cut to it; its last entry is no page.
    table.copy_(good)
    op(q, kp, vp, table, torch.tensor([2**31 - 1], dtype=torch.int32, device="cuda"), cu, max_q=longest)
    assert op.status(q.device)[0] == lib.DEV_PAGE
    op.reset_status(q.device)
    # Row bounds outside q are cut to it.
    out = torch.full_like(q, 7.0)
    op(q[:1], kp, vp, good, kv, torch.tensor([-3, 2**31 - 1], dtype=torch.int32, device="cuda"), max_q=1, out=out[:1])
    torch.cuda.synchronize()
    assert bool((out[1:] == 7.0).all())


@gpu
def test_paged_strides_and_slices():
    q, kp, vp, table, kv, cu, longest = _paged_case(LENGTHS["chunks"], 6, 2, 16, BF16, 9)
    want = _check_paged((q, kp, vp, table, kv, cu, longest))
    from fa_b200.paged import PagedOperator

    op = PagedOperator()
    wide = torch.zeros((q.shape[0], 10, 128), dtype=BF16, device="cuda")
    wide[:, 2:8] = q
    pool = torch.zeros((kp.shape[0], 2, 16, 2, 128), dtype=BF16, device="cuda")  # K and V of a page beside each other
    pool[:, 0], pool[:, 1] = kp, vp
    big = torch.full((table.shape[0], table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    big[:, :table.shape[1]] = table
    out = torch.zeros((6, q.shape[0], 128), dtype=BF16, device="cuda")
    op(wide[:, 2:8], pool[:, 0], pool[:, 1], big[:, :table.shape[1]], kv, cu, max_q=longest, out=out.transpose(0, 1))
    assert torch.equal(out.transpose(0, 1), want)


@gpu
@pytest.mark.parametrize("name", ["ragged", "chunk_long"])
def test_paged_runs_give_the_same_bits_and_can_be_captured(name):
    from fa_b200.paged import PagedOperator

    q, kp, vp, table, kv, cu, longest = _paged_case(LENGTHS[name], 12, 1, 16, F16, 11)
    op = PagedOperator()
    want = op(q, kp, vp, table, kv, cu, max_q=longest)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(q, kp, vp, table, kv, cu, max_q=longest, out=out)
    for _ in range(3):
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # The lengths are the device's: a replay follows them.
    kv.sub_(longest)
    want = op(q, kp, vp, table, kv, cu, max_q=longest)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        side = PagedOperator()(q, kp, vp, table, kv, cu, max_q=longest)
    here = op(q, kp, vp, table, kv, cu, max_q=longest)
    torch.cuda.synchronize()
    assert torch.equal(side, want) and torch.equal(here, want)


@gpu
def test_dimensions_of_one_element_may_have_any_stride():
    from fa_b200.paged import PagedOperator, append, build_tables

    rotary, _, _ = _rotary(128, 128, "half", {})
    buf = torch.randn(1 + 12 * 128 + 3, device="cuda").half()
    x = buf[:12 * 128].as_strided((1, 12, 128), (1537, 128, 1))
    pos = torch.tensor([5], device="cuda")
    assert torch.equal(rotary(x, pos), rotary(x.clone(memory_format=torch.contiguous_format), pos))
    kp, vp = (torch.zeros((1, 8, 1, 128), dtype=F16, device="cuda").as_strided((1, 8, 1, 128), (7, 128, 3, 1)) for _ in range(2))
    k = torch.randn((1, 1, 128), device="cuda").half().as_strided((1, 1, 128), (13, 9, 1))
    assert torch.equal(append(k, k, kp, vp, torch.tensor([2], device="cuda"), q=x, positions=pos, rotary=rotary), rotary(x, pos))
    assert torch.equal(vp[0, 2], k[0])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = i32([0, -1]).as_strided((1, 2), (1, 1))
    t = build_tables(i32([2]), i32([1]), table, i32([]), i32([0]), page_size=8, num_tokens=1)
    assert t.slots.tolist() == [2]
    out = PagedOperator()(x, kp, vp, table, t.kv_lens, t.cu_q, max_q=1)
    O, A = ref.paged_attention(x, kp, vp, table, t.kv_lens, t.cu_q)
    _within(out, O, A)


@gpu
@pytest.mark.parametrize("name", ["ragged", "chunk_long"])
def test_a_wait_that_runs_out_is_reported_and_nothing_hangs(name):
    """No block of V is loaded (a test flag): every role gives up after its
    bound, the status says so, and the same operator is right afterwards."""
    from fa_b200 import lib
    from fa_b200.paged import PagedOperator

    case = _paged_case(LENGTHS[name], 12, 1, 16, F16, 13)
    q, kp, vp, table, kv, cu, longest = case
    op = PagedOperator(timeout_us=20000)
    _check_paged(case, op=op)
    op(q, kp, vp, table, kv, cu, max_q=longest, flags=lib.PAGED_TEST_WITHHOLD_V)
    assert op.status(q.device)[0] == lib.DEV_TIMEOUT
    op.reset_status(q.device)
    assert op.status(q.device)[0] == lib.DEV_OK
    _check_paged(case, op=op)


@gpu
def test_paged_first_use_in_a_capture_is_refused():
    from fa_b200.paged import PagedOperator
    from fa_b200.rotary import Rotary

    q, kp, vp, table, kv, cu, longest = _paged_case(LENGTHS["one"], 2, 1, 16, F16, 12)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError):
            PagedOperator()(q, kp, vp, table, kv, cu, max_q=1)
        with pytest.raises(RuntimeError):
            Rotary()(q)
        q.add_(0)


@gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 5)])
@pytest.mark.parametrize("dtype,hq,hkv,ps", [(F16, 12, 1, 16), (BF16, 8, 2, 32)])
def test_a_serving_loop(dtype, hq, hkv, ps, window, sinks):
    """Prompts in chunks, then single tokens, through tables, append and
    attention, against rotated dense attention of everything seen so far."""
    from fa_b200.paged import PagedOperator, StepTables, build_tables

    dev, g = "cuda", torch.Generator(device="cuda").manual_seed(21)
    rotary, freq, _ = _rotary(128, 64, "interleaved", SCALINGS[1])
    steps = [[40, 3, 0, 17], [100, 1, 5, 1], [1, 1, 1, 0], [1, 1, 1, 1], [0, 2, 150, 1]]
    R, width, T = 4, 12, 256
    pages = R * width
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table, free = torch.full((R, width), -1, dtype=torch.int32, device=dev), torch.randperm(pages, device=dev).int()
    kp, vp = (torch.full((pages, ps, hkv, 128), float("nan"), dtype=dtype, device=dev) for _ in range(2))
    lens, count = i32([0] * R), i32([pages])
    buffers = [StepTables.empty(R, T, dev) for _ in range(2)]
    op = PagedOperator()
    seen_k, seen_v = ([torch.zeros((0, hkv, 128), dtype=dtype, device=dev) for _ in range(R)] for _ in range(2))
    for n, new in enumerate(steps):
        q, k, v = (torch.randn((T, h, 128), generator=g, device=dev).to(dtype) for h in (hq, hkv, hkv))
        t = build_tables(lens, i32(new), table, free, count, page_size=ps, num_tokens=T, out=buffers[n % 2])
        out = op.step(q, k, v, kp, vp, table, t, max_q=max(new), rotary=rotary, window=window, sinks=sinks)
        torch.cuda.synchronize()
        assert int(t.status) == 0 and op.status(dev)[0] == 0
        at = 0
        for r, m in enumerate(new):  # the cache holds the rotated keys and the values of every token so far
            seen_k[r], seen_v[r] = torch.cat([seen_k[r], k[at:at + m]]), torch.cat([seen_v[r], v[at:at + m]])
            pos = torch.arange(seen_k[r].shape[0], device=dev)
            pg = table[r].long()[pos // ps]
            _check_rotation(kp[pg, pos % ps].transpose(0, 1), seen_k[r].transpose(0, 1), pos, freq, "interleaved", False, 1.0)
            assert torch.equal(vp[pg, pos % ps], seen_v[r])
            at += m
        O, A = ref.paged_attention(rotary(q, t.positions), kp, vp, table, t.kv_lens, t.cu_q, window, sinks)
        _within(out[:at], O[:at], A[:at])
        lens, count = t.kv_lens, t.free_left
    assert int(count) == pages - sum(-(-sum(s[r] for s in steps) // ps) for r in range(R))


@gpu
def test_a_captured_generation_step_follows_the_device():
    """One step -- tables, append with rotary, attention, and the lengths' and
    the count's update -- as a graph, replayed with other new lengths."""
    from fa_b200.paged import PagedOperator, StepTables, append, build_tables

    dev, g, R, ps, width, T = "cuda", torch.Generator(device="cuda").manual_seed(2), 5, 16, 40, 24
    rotary, _, _ = _rotary(128, 128, "half", {})
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    lens, new, count = i32([100, 0, 33, 250, 16]), i32([1, 1, 1, 1, 1]), i32([R * width])
    table, free = torch.full((R, width), -1, dtype=torch.int32, device=dev), torch.randperm(R * width, device=dev).int()
    kp, vp = (torch.full((R * width, ps, 2, 128), float("nan"), dtype=BF16, device=dev) for _ in range(2))
    q, k, v = (torch.zeros((T, h, 128), dtype=BF16, device=dev) for h in (8, 2, 2))
    # What is cached already, written as a step of its own.
    t0 = build_tables(torch.zeros_like(lens), lens, table, free, count, page_size=ps, num_tokens=399)
    append(torch.randn((399, 2, 128), generator=g, device=dev).to(BF16), torch.randn((399, 2, 128), generator=g, device=dev).to(BF16),
           kp, vp, t0.slots)
    count.copy_(t0.free_left)
    op, t, out = PagedOperator(), StepTables.empty(R, T, dev), torch.zeros_like(q)
    op.workspace(q.device)
    rotary.table(q.device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        build_tables(lens, new, table, free, count, page_size=ps, num_tokens=T, out=t)
        op.step(q, k, v, kp, vp, table, t, max_q=4, rotary=rotary, out=out)
        lens.copy_(t.kv_lens)
        count.copy_(t.free_left)
    for step in ([1, 1, 1, 1, 1], [1, 3, 0, 1, 16], [0, 1, 1, 4, 1], [1, 1, 1, 1, 1]):
        new.copy_(i32(step))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=dev))
        had = lens.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert int(t.status) == 0 and op.status(dev)[0] == 0
        assert lens.tolist() == [a + b for a, b in zip(had.tolist(), step)]
        n = sum(step)
        O, A = ref.paged_attention(rotary(q, t.positions), kp, vp, table, t.kv_lens, t.cu_q)
        _within(out[:n], O[:n], A[:n])


# ----------------------------------------------------------------- refusals
def test_rotary_refusals():
    from fa_b200.rotary import Rotary

    for kw in ({"dim": 24}, {"dim": 8}, {"rotary_dim": 256}, {"rotary_dim": 8}, {"layout": "odd"}, {"scaling": "x"},
               {"base": 0.0}, {"scaling": "linear", "factor": 0.0}, {"scaling": "banded"}, {"magnitude": float("inf")}):
        with pytest.raises(ValueError):
            Rotary(**kw)
    with pytest.raises(ValueError):
        Rotary()(torch.zeros(3, 2, 128))  # no CUDA tensor
    with pytest.raises(ValueError):
        Rotary()(torch.zeros(2, 128))


def test_paged_refusals_on_the_host():
    from fa_b200.paged import PagedOperator, append, build_tables

    t = torch.zeros
    with pytest.raises(ValueError):
        build_tables(t(2, dtype=torch.int32), t(2, dtype=torch.int32), t(2, 3, dtype=torch.int32),
                     t(4, dtype=torch.int32), t(1, dtype=torch.int32), page_size=16, num_tokens=4)
    pool = t(2, 16, 1, 128, dtype=F16)
    with pytest.raises(ValueError):
        append(t(1, 1, 128, dtype=F16), t(1, 1, 128, dtype=F16), pool, pool, t(1, dtype=torch.int64))
    with pytest.raises(ValueError):
        PagedOperator()(t(1, 1, 128, dtype=F16), pool, pool, t(1, 1, dtype=torch.int32), t(1, dtype=torch.int32),
                        t(2, dtype=torch.int32), max_q=1)


def _args(**kw):
    import ctypes as C

    from fa_b200 import lib

    a = lib.PagedArgs(C.sizeof(lib.PagedArgs), lib.DTYPE_FP16, 16, 16, 16, 16, (512, 128), (512, 128), (2048, 128, 128),
                      (2048, 128, 128), 16, 4, 16, 16, 5, 8, 2, 4, 16, 4, 1, 1, 0.1, 0, 0, 0, 0, 256, 1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    ({"struct_size": 8}, -11), ({"dtype": 2}, -14), ({"requests": -1}, -3), ({"width": 0}, -3), ({"heads_kv": 3}, -4),
    ({"heads_q": 512}, -4), ({"page_size": 24}, -15), ({"page_size": 4}, -15), ({"tokens": 2**31}, -5),
    ({"requests": 5000}, -5), ({"width": 2**30}, -5), ({"width": 2**27}, -5), ({"window": -1}, -11), ({"sinks": 3}, -11), ({"scale": 0.0}, -10),
    ({"flags": 2}, -11), ({"q": None}, -1), ({"kv_lens": None}, -1), ({"o": 8}, -7), ({"table_stride": 3}, -16), ({"q_strides": (100, 128)}, -16),
    ({"k_strides": (2048, 0, 128)}, -16), ({"workspace": None}, -8), ({"workspace": 128}, -8)])
def test_paged_validation_codes_without_gpu(kw, code):
    import ctypes as C

    from fa_b200 import lib

    a = _args(**{k: (type(getattr(_args(), k))(*v) if isinstance(v, tuple) else v) for k, v in kw.items()})
    assert lib.load().b200fa_paged_fwd(C.byref(a), None) == code
    assert lib.last_error() != ""


def test_paged_nothing_to_do_without_gpu():
    import ctypes as C

    from fa_b200 import lib

    assert lib.load().b200fa_paged_fwd(C.byref(_args(requests=0)), None) == 0
    assert lib.load().b200fa_paged_fwd(C.byref(_args(tokens=0)), None) == 0
    assert lib.load().b200fa_paged_fwd(None, None) == -1


def test_light_kernels_validation_codes_without_gpu():
    import ctypes as C

    from fa_b200 import lib

    so = lib.load()
    tables = [16, 16, 2, 16, 4, 4, 16, 9, 16, 16, 16, 16, 30, 16, 16, 16, 16, None]

    def rc(**kw):
        a = list(tables)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return so.b200fa_build_tables(*a)

    assert rc(_0=None) == -1 and rc(_2=0) == -3 and rc(_5=0) == -3 and rc(_4=3) == -3 and rc(_12=-1) == -3
    assert rc(_2=5000) == -5 and rc(_9=20) == -15
    d = lib.RotaryDesc(C.sizeof(lib.RotaryDesc), 128, 128, 0, 0, 1.0, 16)
    s = lib.Strides3(0, 256, 128)
    rot = lambda desc, n=4, x=16, st=s, dt=0: so.b200fa_rotary(x, 16, 1, n, 2, st, s, None, 32, 0, C.byref(desc), dt, None)  # noqa: E731
    assert rot(d, n=0) == 0 and rot(d, n=-1) == -3 and rot(d, x=None) == -1 and rot(d, x=8) == -7 and rot(d, dt=3) == -14
    assert rot(d, st=lib.Strides3(0, 250, 128)) == -16
    assert rot(lib.RotaryDesc(C.sizeof(lib.RotaryDesc), 128, 144, 0, 0, 1.0, 16)) == -17
    assert rot(lib.RotaryDesc(C.sizeof(lib.RotaryDesc), 20, 16, 0, 0, 1.0, 16)) == -2
    s2 = lib.Strides2(256, 128)

    def app(tokens=0, dim=128, dtype=0, pages=2, ps=16, slots=16, hkv=2):
        return so.b200fa_append(None, None, None, None, 16, s2, 16, s2, 16, s, 16, s, tokens, 0, hkv, dim, pages, ps,
                                slots, None, 32, None, dtype, None)

    assert app() == 0 and app(dtype=2) == -14 and app(dim=20) == -2 and app(pages=0) == -3 and app(ps=12) == -15
    assert app(tokens=3, slots=None) == -1 and app(hkv=0) == -3
