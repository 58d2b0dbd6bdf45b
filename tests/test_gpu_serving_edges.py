"""The serving operators where they went wrong once: first use by two threads,
forward-mode derivatives, values that no row sees, steps that could not be met,
bounds of waits, ends of the number ranges.  Tolerances as in
test_gpu_serving.py; most checks here are for equality."""

import copy
import math
import pickle
import re
import threading
import time
from pathlib import Path

import pytest
import torch

from oracle import serving_ref as ref

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
gpu = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
HALF = {t: torch.finfo(t).eps / 2 for t in (F16, BF16, F32)}
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731


def _in_two_threads(a, b):
    """a() and b() begun together; their results."""
    gate, out, errors = threading.Barrier(2), [None, None], []

    def run(i, f):
        try:
            gate.wait()
            out[i] = f()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i, f)) for i, f in enumerate((a, b))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors, errors
    return out


def _cache(lens, hq, hkv, ps, dtype, seed):
    """A filled cache and a step's tables; lens: (new, cached) tokens per request."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    used = [-(-kv // ps) for _, kv in lens]
    width = max(used)
    ids = torch.randperm(sum(used), generator=g, device="cuda").int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(used):
        table[r, :n] = ids[at:at + n]
        at += n
    kp, vp = (torch.randn((sum(used), ps, hkv, 128), generator=g, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn((sum(n for n, _ in lens), hq, 128), generator=g, device="cuda").to(dtype)
    cu = [0]
    for n, _ in lens:
        cu.append(cu[-1] + n)
    return q, kp, vp, table, i32([kv for _, kv in lens]), i32(cu)


# ------------------------------------------------------------- bounds of the waits
@gpu
@pytest.mark.parametrize("lens", [[(1, 900), (2, 3000)], [(400, 2000)]], ids=["short", "chunk"])
def test_the_bound_of_a_wait_is_the_one_asked_for(lens):
    """V is withheld: every role gives up, the first after the bound and the
    others with it, not one bound after another."""
    from fa_b200 import lib
    from fa_b200.paged import PagedOperator

    q, kp, vp, table, kv, cu = _cache(lens, 4, 2, 16, F16, 9)
    op, n = PagedOperator(timeout_us=300000), max(a for a, _ in lens)
    want = op(q, kp, vp, table, kv, cu, max_q=n)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    torch.cuda.synchronize()
    begin.record()
    op(q, kp, vp, table, kv, cu, max_q=n, flags=lib.PAGED_TEST_WITHHOLD_V)
    end.record()
    assert op.status("cuda")[0] == lib.DEV_TIMEOUT
    # The last copies in flight are given up to 100 ms more.
    assert 290.0 <= begin.elapsed_time(end) <= 500.0, begin.elapsed_time(end)
    op.reset_status("cuda")
    assert torch.equal(op(q, kp, vp, table, kv, cu, max_q=n), want) and op.status("cuda")[0] == 0


# ------------------------------------------------------------ calls that overlap
@gpu
def test_calls_of_one_operator_may_overlap():
    """Single tokens on one stream, a chunk on another, both split over many
    workers: eagerly, and as two graphs replayed at the same time."""
    from fa_b200.paged import PagedOperator

    op = PagedOperator()
    cases = [_cache([(1, 30000), (1, 777)], 12, 1, 16, F16, 20), _cache([(300, 9000)], 12, 1, 64, F16, 21)]
    longest = [1, 300]
    wants = [op(*c, max_q=n) for c, n in zip(cases, longest)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[torch.zeros_like(w) for _ in range(20)] for w in wants]
    torch.cuda.synchronize()
    for i in range(20):
        for c, n, s, o in zip(cases, longest, streams, outs):
            with torch.cuda.stream(s):
                op(*c, max_q=n, out=o[i])
    torch.cuda.synchronize()
    assert op.status("cuda")[0] == 0
    for w, o in zip(wants, outs):
        assert all(torch.equal(x, w) for x in o)
    graphs = [torch.cuda.CUDAGraph() for _ in cases]
    for graph, c, n, o in zip(graphs, cases, longest, outs):
        with torch.cuda.graph(graph):
            for x in o:
                op(*c, max_q=n, out=x)
    for o in outs:
        for x in o:
            x.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert op.status("cuda")[0] == 0
    for w, o in zip(wants, outs):
        assert all(torch.equal(x, w) for x in o)


@gpu
def test_an_operator_first_used_by_two_threads_has_one_status(monkeypatch):
    from fa_b200.paged import PagedOperator

    zeros = torch.zeros

    def slowly(*args, **kw):
        time.sleep(0.02)
        return zeros(*args, **kw)

    monkeypatch.setattr(torch, "zeros", slowly)
    dev = torch.device("cuda", 0)
    for _ in range(3):
        op = PagedOperator()
        a, b = _in_two_threads(lambda: op.workspace(dev), lambda: op.workspace(dev))
        assert a is b is op.workspace(dev)


def test_a_paged_call_without_the_status_pointer_is_still_accepted():
    import ctypes as C

    from fa_b200 import lib

    a = lib.PagedArgs(lib.PagedArgs.status.offset, lib.DTYPE_FP16)
    a.width = a.num_pages = a.heads_q = a.heads_kv = 1
    a.page_size, a.scale, a.workspace = 16, 1.0, 256
    assert lib.load().b200fa_paged_fwd(C.byref(a), None) == 0  # no requests
    a.struct_size = C.sizeof(lib.PagedArgs)
    assert lib.load().b200fa_paged_fwd(C.byref(a), None) == 0
    a.status = 2
    assert lib.load().b200fa_paged_fwd(C.byref(a), None) == -7
    a.struct_size += 8
    assert lib.load().b200fa_paged_fwd(C.byref(a), None) == -11


# ------------------------------------------------- first use by two threads
@pytest.mark.parametrize("directions", [(False, True), (False, False)], ids=["both_directions", "one_direction"])
def test_a_rotary_first_used_by_two_threads_has_one_table(directions, monkeypatch):
    """A stand-in takes the place of the copy to the device and lets the other
    thread run, as the copy does."""
    from fa_b200 import rotary as module

    def to(self, *args, **kw):
        time.sleep(0.02)
        return self.clone()

    monkeypatch.setattr(torch.Tensor, "to", to)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    dev = torch.device("cuda", 0)
    for _ in range(5):
        r = module.Rotary(64)
        got = _in_two_threads(*[lambda inv=inv: r.desc(dev, inv) for inv in directions])
        assert got == [r.desc(dev, inv) for inv in directions]  # neither was replaced behind its reader's back
        for inv in directions:
            d = module.lib.RotaryDesc.from_address(r.desc(dev, inv))
            assert d.freq == r.table(dev).data_ptr()


# ------------------------------------------------------------- devices and copies
@gpu
def test_preparing_a_capture_with_the_device_without_its_number():
    from fa_b200.paged import PagedOperator
    from fa_b200.rotary import Rotary

    q, kp, vp, table, kv, cu = _cache([(1, 40)], 4, 2, 16, F16, 12)
    for device in ("cuda", torch.device("cuda"), "cuda:0"):
        op, rotary = PagedOperator(), Rotary(128)
        op.workspace(device)
        rotary.table(device)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = op(rotary(q, torch.zeros(1, dtype=torch.int64, device="cuda")), kp, vp, table, kv, cu, max_q=1)
        graph.replay()
        assert torch.equal(out, op(q, kp, vp, table, kv, cu, max_q=1))


@gpu
def test_a_used_rotary_can_be_copied_and_pickled():
    from fa_b200.rotary import Rotary

    rotary = Rotary(64, layout="interleaved", base=500.0)
    x, pos = torch.randn((3, 2, 64), device="cuda"), torch.tensor([4, 9, 1], device="cuda")
    want = rotary(x, pos)
    for other in (copy.deepcopy(rotary), pickle.loads(pickle.dumps(rotary))):
        assert torch.equal(other(x, pos), want)


# ------------------------------------------------------ derivatives of a rotary
@gpu
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_carries_forward_mode_derivatives(inverse):
    import torch.autograd.forward_ad as fwd

    from fa_b200.rotary import Rotary

    rotary = Rotary(32, scaling="linear", factor=2.0, magnitude=1.5)
    x, dx = torch.randn((2, 3, 7, 32), device="cuda"), torch.randn((2, 3, 7, 32), device="cuda")
    pos = torch.arange(7, device="cuda") * 31
    with fwd.dual_level():
        y = fwd.unpack_dual(rotary(fwd.make_dual(x, dx), pos, inverse=inverse))
        assert torch.equal(y.primal, rotary(x, pos, inverse=inverse))
        assert y.tangent is not None and torch.equal(y.tangent, rotary(dx, pos, inverse=inverse))
        plain = rotary(x, pos, inverse=inverse)  # no tangent in, none out
        assert fwd.unpack_dual(plain).tangent is None
        z = x.clone().requires_grad_()  # both modes at once
        both = fwd.unpack_dual(rotary(fwd.make_dual(z, dx), pos, inverse=inverse))
        assert torch.equal(both.tangent, rotary(dx, pos, inverse=inverse))
        (grad,) = torch.autograd.grad(both.primal.sum(), z)
        assert torch.equal(grad, rotary(torch.ones_like(x), pos, inverse=not inverse))
        with pytest.raises(ValueError):
            rotary(fwd.make_dual(x, dx), pos, out=torch.empty_like(x))


@gpu
def test_the_rotated_q_of_an_append_keeps_its_graph():
    """q's derivatives pass through append as through the rotary itself; the
    cache holds values only."""
    import torch.autograd.forward_ad as fwd

    from fa_b200.paged import append
    from fa_b200.rotary import Rotary

    rotary = Rotary(128)
    T, pos = 5, torch.arange(5, device="cuda") + 3
    q, g = (torch.randn((T, 4, 128), device="cuda").half() for _ in range(2))
    k, v = (torch.randn((T, 2, 128), device="cuda").half().requires_grad_() for _ in range(2))
    kp, vp = (torch.zeros((1, 8, 2, 128), dtype=F16, device="cuda") for _ in range(2))
    slots = torch.arange(T, device="cuda")
    want = append(k.detach(), v.detach(), kp, vp, slots, q=q, positions=pos, rotary=rotary)
    keys = kp.clone()
    for turned in (rotary, None):
        x = q.clone().requires_grad_()
        kp.zero_(), vp.zero_()
        y = append(k, v, kp, vp, slots, q=x, positions=pos, rotary=turned)
        (grad,) = torch.autograd.grad(y, x, g)
        assert torch.equal(grad, rotary(g, pos, inverse=True) if turned else g)
        if turned:
            assert torch.equal(y.detach(), want) and torch.equal(kp, keys) and torch.equal(vp[0, :T], v.detach())
        assert not kp.requires_grad and not vp.requires_grad
    with pytest.raises(ValueError):
        append(k, v, kp, vp, slots, q=q.clone().requires_grad_(), positions=pos, rotary=rotary, q_out=torch.empty_like(q))
    with torch.no_grad():
        append(k, v, kp, vp, slots, q=q.clone().requires_grad_(), positions=pos, rotary=rotary, q_out=torch.empty_like(q))
    for bad in (q[:4], q.float(), q[..., :64], q[0]):
        with pytest.raises(ValueError):
            append(k, v, kp, vp, slots, q=bad.clone().requires_grad_())
    with fwd.dual_level():
        y = fwd.unpack_dual(append(k, v, kp, vp, slots, q=fwd.make_dual(q, g), positions=pos, rotary=rotary))
        assert torch.equal(y.primal, want) and torch.equal(y.tangent, rotary(g, pos))


# ---------------------------------------------------------- in-place writes count
@gpu
def test_written_tensors_change_their_version():
    """A tensor saved for a backward pass and written by an operator makes that
    pass raise, as after torch's own in-place operations."""
    from fa_b200.paged import PagedOperator, append, build_tables
    from fa_b200.rotary import Rotary

    rotary = Rotary(128)
    q, kp, vp, table, kv, cu = _cache([(2, 40)], 4, 2, 16, F16, 7)
    k, slots, pos = torch.randn((2, 2, 128), device="cuda").half(), torch.arange(2, device="cuda"), torch.arange(2, device="cuda")
    q_out, x, out = torch.zeros_like(q), q.clone(), torch.zeros_like(q)

    def bumped(call, *tensors):
        before = [t._version for t in tensors]
        call()
        return all(t._version > b for t, b in zip(tensors, before))

    assert bumped(lambda: append(k, k, kp, vp, slots, q=q, q_out=q_out, positions=pos, rotary=rotary), kp, vp, q_out)
    assert bumped(lambda: rotary(x, pos, out=x), x)
    assert bumped(lambda: PagedOperator()(q, kp, vp, table, kv, cu, max_q=2, out=out), out)
    t = build_tables(kv, i32([1]), table, i32([]), i32([0]), page_size=16, num_tokens=2)
    assert bumped(lambda: build_tables(kv, i32([1]), table, i32([]), i32([0]), page_size=16, num_tokens=2, out=t), table, *t.tensors())
    w = torch.ones((), device="cuda", dtype=F16, requires_grad=True)
    loss = (w * kp).sum()
    append(k, k, kp, vp, slots)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        y = q.clone()
        rotary(y, pos, out=y)
    unchanged = q._version
    rotary(q, pos)
    assert q._version == unchanged


@gpu
def test_a_table_of_one_column_may_have_any_stride():
    from fa_b200.paged import PagedOperator, build_tables

    q, kp, vp, table, kv, cu = _cache([(1, 5), (1, 9), (1, 2)], 4, 2, 16, F16, 11)
    column = table.view(1, 3).t()  # [3, 1], strides (1, 3)
    assert column.stride() == (1, 3)
    want = PagedOperator()(q, kp, vp, table, kv, cu, max_q=1)
    assert torch.equal(PagedOperator()(q, kp, vp, column, kv, cu, max_q=1), want)
    t = build_tables(kv, i32([1, 1, 1]), column, i32([]), i32([0]), page_size=16, num_tokens=3)
    assert t.status.tolist() == [0] and t.slots.tolist() == [int(p) * 16 + n for p, n in zip(table.view(-1).tolist(), (5, 9, 2))]


# ------------------------------------------------------------------- overlaps
@gpu
def test_outputs_that_overlap_inputs_partly_are_refused():
    from fa_b200.paged import PagedOperator, StepTables, append, build_tables
    from fa_b200.rotary import Rotary

    rotary, pos = Rotary(128), torch.arange(6, device="cuda")
    buf = torch.randn((8, 4, 128), device="cuda").half()
    with pytest.raises(ValueError):
        rotary(buf[:6], pos, out=buf[1:7])
    rotary(buf[:4], pos[:4], out=buf[4:])  # side by side in one buffer
    square = torch.randn((6, 6, 128), device="cuda").half()
    with pytest.raises(ValueError):
        rotary(square, pos, out=square.transpose(0, 1))
    k = torch.randn((6, 2, 128), device="cuda").half()
    kp, vp = (torch.zeros((2, 8, 2, 128), dtype=F16, device="cuda") for _ in range(2))
    slots = torch.arange(6, device="cuda")
    with pytest.raises(ValueError):
        append(k, k, kp, vp, slots, q=buf[:6], positions=pos, rotary=rotary, q_out=buf[1:7])
    with pytest.raises(ValueError):
        append(kp.view(16, 2, 128)[:6], k, kp, vp, slots + 2)  # moves within the cache
    with pytest.raises(ValueError):
        append(k, k, kp, kp, slots)  # one tensor for both
    q, kp, vp, table, kv, cu = _cache([(2, 30)], 4, 2, 16, F16, 13)
    op, wide = PagedOperator(), torch.zeros((3, 4, 128), dtype=F16, device="cuda")
    wide[:2] = q
    want = op(q, kp, vp, table, kv, cu, max_q=2)
    with pytest.raises(ValueError):
        op(wide[:2], kp, vp, table, kv, cu, max_q=2, out=wide[1:])
    assert torch.equal(op(wide[:2], kp, vp, table, kv, cu, max_q=2, out=wide[:2]), want)  # the whole of q is fine
    ints = torch.zeros(64, dtype=torch.int32, device="cuda")
    args = dict(page_size=16, num_tokens=4)
    t = StepTables.empty(1, 4, "cuda")
    for out in (StepTables(t.slots, ints[:4], t.cu_q, t.kv_lens, t.free_left, t.status),       # on the table
                StepTables(t.slots, t.positions, t.cu_q, t.kv_lens, t.status, t.status),       # two outputs in one
                StepTables(t.slots, t.positions, ints[32:34], t.kv_lens, t.free_left, t.status)):  # on the free list
        with pytest.raises(ValueError):
            build_tables(i32([3]), i32([1]), ints[:8].view(1, 8), ints[32:40], i32([8]), out=out, **args)
    with pytest.raises(ValueError):
        build_tables(i32([3]), i32([1]), ints[:8].view(1, 8), ints[4:12], i32([8]), **args)  # the table on the free list


@gpu
def test_lengths_that_leave_32_bits_are_refused_by_the_tables():
    """A row wide enough for more than 2^31 - 1 tokens: the length would wrap."""
    from fa_b200.paged import build_tables

    top = 2**31 - 1
    table = torch.full((2, 4096), -1, dtype=torch.int32, device="cuda")
    table[0, :2048] = torch.arange(2048, device="cuda").int()
    ctx, free = i32([top - 4, 3]), torch.arange(2048, 2060, device="cuda").int()
    before = table.clone()
    t = build_tables(ctx, i32([5, 1]), table, free, i32([12]), page_size=1 << 20, num_tokens=8)
    assert t.status.tolist() == [2] and t.kv_lens.tolist() == [top - 4, 3] and t.slots.tolist() == [-1] * 8
    assert torch.equal(table, before) and t.free_left.tolist() == [12]
    t = build_tables(ctx, i32([4, 0]), table, free, i32([12]), page_size=1 << 20, num_tokens=8)
    assert t.status.tolist() == [0] and t.kv_lens.tolist() == [top, 3]
    assert t.slots.tolist()[:4] == [top - 4 + i for i in range(4)] and t.positions.tolist()[:4] == [top - 4 + i for i in range(4)]


SLOW = r"""
extern "C" __global__ void slow(unsigned long long ns) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  do {
    __nanosleep(1000);
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  } while (t - t0 < ns);
}
"""


@gpu
def test_time_spent_waiting_for_the_kernel_before_is_no_timeout():
    """A kernel that lets its dependents start early and runs longer than
    timeout_us: what is launched behind it begins its waits after it."""
    from fa_b200.ops import Operator
    from fa_b200.paged import PagedOperator

    slow = torch.cuda._compile_kernel(SLOW, "slow")
    q, k, v = (torch.randn((1, h, 600, 128), device="cuda").half() for h in (4, 2, 2))
    op = Operator("fp16", timeout_us=20000)
    want = op(q, k, v, causal=True, window=100)
    out = torch.zeros_like(want)
    pq, kp, vp, table, kv, cu = _cache([(1, 900), (2, 300)], 4, 2, 16, F16, 8)
    pop = PagedOperator(timeout_us=20000)
    pwant = pop(pq, kp, vp, table, kv, cu, max_q=2)
    pout = torch.zeros_like(pwant)
    torch.cuda.synchronize()
    slow((1, 1, 1), (32, 1, 1), (100_000_000,))
    op(q, k, v, causal=True, window=100, out=out)
    torch.cuda.synchronize()
    assert op.status(q.device)[0] == 0 and torch.equal(out, want)
    slow((1, 1, 1), (32, 1, 1), (100_000_000,))
    pop(pq, kp, vp, table, kv, cu, max_q=2, out=pout)
    torch.cuda.synchronize()
    assert pop.status(q.device)[0] == 0 and torch.equal(pout, pwant)


@gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")], ids=["nan", "inf"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (64, 0), (64, 130), (100, 200), (128, 4), (200, 1), (200, 129), (255, 128), (300, 300),
                                          (513, 20), (700, 0)])
@pytest.mark.parametrize("debug", [False, True], ids=["product", "checking"])
def test_dense_values_outside_every_window_may_be_anything(window, sinks, value, debug):
    """Work items of 256 rows: the ones from row `at` on must not notice what is
    planted at keys that none of their rows sees."""
    from fa_b200.ops import Operator

    B, Hq, Hkv, N = 1, 4, 2, 1300
    g = torch.Generator(device="cuda").manual_seed(window)
    q, k, v = (torch.randn((B, h, N, 128), generator=g, device="cuda").half() for h in (Hq, Hkv, Hkv))
    op = Operator("fp16", debug=debug)
    want = op(q, k, v, causal=True, window=window, sinks=sinks)
    O, A = ref.window_attention(q, k, v, window, sinks)
    over = (want.double() - O).abs() - (A * (HALF[F16] + 7.5e-5 + 2.0 ** -16 + 3e-4) + O.abs() * HALF[F16] + 2.0 ** -24)
    assert bool((over <= 0).all()), float(over.max())
    for at in (256, 512, 1024, 1280):
        k2, v2 = k.clone(), v.clone()
        end = max(sinks, at - window + 1)
        k2[:, :, sinks:end], v2[:, :, sinks:end] = float("nan"), value
        got = op(q, k2, v2, causal=True, window=window, sinks=sinks)
        torch.cuda.synchronize()
        assert op.status(q.device)[0] == 0
        assert torch.equal(got[:, :, at:], want[:, :, at:])


@gpu
@pytest.mark.parametrize("nq,nk,window,sinks", [(130, 2000, 50, 10), (1, 300, 1, 0), (300, 301, 1000, 0), (257, 700, 20, 600)])
def test_dense_values_behind_the_last_row_may_be_anything(nq, nk, window, sinks):
    from fa_b200.ops import Operator

    q, k, v = (torch.randn((1, h, n, 128), device="cuda").half() for h, n in ((4, nq), (2, nk), (2, nk)))
    op = Operator("fp32")
    want = op(q, k, v, causal=True, window=window, sinks=sinks)
    k[:, :, nq:], v[:, :, nq:] = float("nan"), float("nan")
    assert torch.equal(op(q, k, v, causal=True, window=window, sinks=sinks), want)


# --------------------------------------- values at keys that no row of an item sees
def _plant(pages, table, r, keys, value):
    ps = pages.shape[1]
    pages[table[r].long()[keys // ps], keys % ps] = value


@gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")], ids=["nan", "inf"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (64, 0), (64, 130), (128, 4), (200, 1), (200, 129), (300, 20), (513, 300)])
@pytest.mark.parametrize("hq,hkv,ps,dtype", [(12, 1, 16, F16), (8, 2, 64, BF16), (4, 4, 8, F16), (16, 1, 256, BF16)])
@pytest.mark.parametrize("lens", [[(1, 1500), (1, 333), (3, 900), (1, 130)], [(300, 1500), (1, 700), (90, 640)]], ids=["short", "chunk"])
def test_paged_values_outside_every_window_may_be_anything(lens, hq, hkv, ps, dtype, window, sinks, value):
    from fa_b200.paged import PagedOperator

    q, kp, vp, table, kv, cu = _cache(lens, hq, hkv, ps, dtype, 3)
    op, longest = PagedOperator(), max(n for n, _ in lens)
    want = op(q, kp, vp, table, kv, cu, max_q=longest, window=window, sinks=sinks)
    for r, (n, total) in enumerate(lens):
        hidden = torch.arange(sinks, max(sinks, total - n + 1 - window), device="cuda")
        _plant(vp, table, r, hidden, value)
        _plant(kp, table, r, hidden, float("nan"))
    got = op(q, kp, vp, table, kv, cu, max_q=longest, window=window, sinks=sinks)
    assert op.status("cuda")[0] == 0
    assert torch.isfinite(want).all() and torch.equal(got, want)


@gpu
@pytest.mark.parametrize("hq,hkv", [(12, 1), (6, 6)])
def test_a_value_leaves_the_rows_behind_its_window_alone(hq, hkv):
    """A key that an earlier tile of the same chunk sees, and later ones do not."""
    from fa_b200.paged import PagedOperator

    window, sinks, n = 70, 3, 1200
    q, kp, vp, table, kv, cu = _cache([(n, n + 40)], hq, hkv, 16, F16, 4)
    op = PagedOperator()
    want = op(q, kp, vp, table, kv, cu, max_q=n, window=window, sinks=sinks)
    for key in (17, 128, 255, 300, 511):
        _plant(vp, table, 0, torch.tensor([key], device="cuda"), float("nan"))
        got = op(q, kp, vp, table, kv, cu, max_q=n, window=window, sinks=sinks)
        clean = key - 40 + window + 256  # a tile of 256 rows further on
        assert torch.equal(got[max(0, clean):], want[max(0, clean):])
        if key > 40:
            assert torch.isnan(got[key - 40]).all()  # the row at the key itself does see it


# ------------------------------------------------- a step that could not be met
@gpu
@pytest.mark.parametrize("R,new,width,T,status", [(2, [5, 90], 8, 256, 1), (2, [5, 300], 8, 512, 2), (2, [5, 90], 8, 64, 3)])
@pytest.mark.parametrize("max_q", [1, 90])
def test_a_step_without_pages_gives_zeros_and_leaves_the_cache(R, new, width, T, status, max_q):
    """Nothing was handed out, so the new tokens have no place: their rows must
    not look like an answer, and the next step that can be met is right."""
    from fa_b200.paged import PagedOperator, build_tables

    ps, hq, hkv = 16, 4, 2
    lens, free = i32([20, 30]), torch.arange(4, 8, device="cuda").int()
    table = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    table[0, :2], table[1, :2] = i32([0, 1]), i32([2, 3])
    kp, vp = (torch.randn((8, ps, hkv, 128), device="cuda").half() for _ in range(2))
    kc, vc = kp.clone(), vp.clone()
    q, k, v = (torch.randn((T, h, 128), device="cuda").half() for h in (hq, hkv, hkv))
    op = PagedOperator()
    t = build_tables(lens, i32(new), table, free, i32([4]), page_size=ps, num_tokens=T)
    assert t.status.tolist() == [status]
    out = torch.full_like(q, 7.0)
    op.step(q, k, v, kp, vp, table, t, max_q=max_q, out=out)
    n = min(sum(new), T)
    assert bool((out[:n] == 0).all()) and bool((out[n:] == 7.0).all())
    assert op.status("cuda")[0] == 0 and torch.equal(kp, kc) and torch.equal(vp, vc)
    t = build_tables(t.kv_lens, i32([5, 20]), table, free, t.free_left, page_size=ps, num_tokens=T)
    assert t.status.tolist() == [0]
    out = op.step(q, k, v, kp, vp, table, t, max_q=max_q)
    O, A = ref.paged_attention(q, kp, vp, table, t.kv_lens, t.cu_q)
    bound = A[:25] * (HALF[F16] + 3e-4 + 2.0 ** -16) + O[:25].abs() * HALF[F16] + 2.0 ** -24
    assert bool(((out[:25].double() - O[:25]).abs() <= bound).all())


@gpu
def test_tables_filled_by_hand_need_no_status():
    from fa_b200.paged import PagedOperator, StepTables

    q, kp, vp, table, kv, cu = _cache([(2, 40), (1, 7)], 4, 2, 16, F16, 5)
    op = PagedOperator()
    want = op(q, kp, vp, table, kv, cu, max_q=2)
    k, v = (torch.zeros((3, 2, 128), dtype=F16, device="cuda") for _ in range(2))
    t = StepTables.empty(2, 3, "cuda")
    t.slots.fill_(-1), t.positions.zero_(), t.cu_q.copy_(cu), t.kv_lens.copy_(kv)
    assert torch.equal(op.step(q, k, v, kp, vp, table, t, max_q=2), want)
    t.status = None
    assert torch.equal(op.step(q, k, v, kp, vp, table, t, max_q=2), want)


# ------------------------------------------------------------------ the README
@gpu
def test_the_readme_serving_loop_keeps_its_layers_apart():
    """The loop as printed, for two layers and three steps, against attention of
    each layer's own keys."""
    text = (ROOT / "README.md").read_text()
    block = next(b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "build_tables" in b)
    g = torch.Generator(device="cuda").manual_seed(6)
    results = []

    class Layer:
        def __init__(self, number):
            self.number, self.rows = number, []

        def qkv(self):
            x = [torch.randn((scope["T"], h, 128), generator=g, device="cuda").half() for h in (12, 1, 1)]
            self.rows.append(x)
            return x

        def take(self, o):
            results.append((self.number, len(self.rows) - 1, o.clone()))

    made = [Layer(0), Layer(1)]
    steps = [i32([9, 3]), i32([1, 40]), i32([1, 1])]
    scope = {"torch": torch, "R": 2, "layers": made, "steps": steps, "longest": 40}
    exec(compile(block, "README.md", "exec"), scope)
    assert len(results) == 6
    from fa_b200.rotary import Rotary

    rotary, counts = Rotary(128), [s.tolist() for s in steps]
    for number, step, o in results:
        layer = made[number]
        for r in range(2):
            ks, vs, had = [], [], 0
            for s in range(step + 1):
                a = sum(counts[s][:r])
                ks.append(layer.rows[s][1][a:a + counts[s][r]])
                vs.append(layer.rows[s][2][a:a + counts[s][r]])
                had += counts[s][r]
            n, a = counts[step][r], sum(counts[step][:r])
            k = rotary(torch.cat(ks).contiguous(), torch.arange(had, device="cuda"))
            q = rotary(layer.rows[step][0][a:a + n].contiguous(), torch.arange(had - n, had, device="cuda"))
            see = ref.visible(torch.arange(had - n, had, device="cuda"), had)
            for h in range(12):
                O, A = ref.attend(q[:, h], k[:, 0], torch.cat(vs)[:, 0], see, 128 ** -0.5)
                bound = A * (HALF[F16] + 3e-4 + 2.0 ** -16) + O.abs() * HALF[F16] + 2.0 ** -24
                assert bool(((o[a:a + n, h].double() - O).abs() <= bound).all())


# --------------------------------------------------------- ends of the number ranges
@gpu
@pytest.mark.parametrize("kw", [{}, {"scaling": "linear", "factor": 3.0}, {"base": 500000.0, "scaling": "banded", "factor": 8.0,
                                                                       "original_length": 8192}], ids=["plain", "linear", "banded"])
def test_angles_of_very_far_positions(kw):
    """Against 60-digit arithmetic.  The angle of position p is off by at most
    p * 2^-65 turns (the frequency's rounding) and 2^-25 turns (its 32-bit sine)."""
    from decimal import Decimal, localcontext

    from fa_b200.rotary import Rotary

    rot = 64
    x = torch.zeros((1, 1, 1, rot), device="cuda")
    x[..., : rot // 2] = 1.0  # y = (cos, sin) of each pair
    rotary = Rotary(rot, **kw)
    for p in (3, 2**20 + 1, 2**31 - 1, 2**40 + 12345, 2**50 + 7):
        y = rotary(x, torch.tensor([p], device="cuda"))[0, 0, 0].double().cpu()
        with localcontext() as ctx:
            ctx.prec = 60
            pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
            base, factor = Decimal(kw.get("base", 10000.0)), Decimal(kw.get("factor", 1.0))
            for i in range(rot // 2):
                f = (base.ln() * Decimal(-2 * i) / rot).exp()
                if kw.get("scaling") == "linear":
                    f /= factor
                elif kw.get("scaling") == "banded":
                    turns = kw["original_length"] * f / (2 * pi)
                    keep = min(Decimal(1), max(Decimal(0), (turns - 1) / 3))
                    f = f * keep + f / factor * (1 - keep)
                turn = p * f / (2 * pi) % 1
                a = float(turn * 2 * pi)
                tol = 6e-7 * 2 + 2 * math.pi * p * 2.0 ** -65
                assert abs(float(y[i]) - math.cos(a)) <= tol and abs(float(y[i + rot // 2]) - math.sin(a)) <= tol, (p, i)


@gpu
@pytest.mark.parametrize("hq,hkv,tokens", [(12, 1, 1), (5, 1, 3), (3, 1, 5), (7, 7, 16), (9, 1, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 0), (260, 131)])
def test_many_tiles_of_few_tokens_are_placed_right(hq, hkv, tokens, window, sinks):
    """max_q = 1 for long requests: tiles of 1, 3, 5 or 16 tokens, hundreds of a request."""
    from fa_b200.paged import PagedOperator

    assert 16 // (hq // hkv) == tokens
    q, kp, vp, table, kv, cu = _cache([(700, 900), (1, 40), (333, 1000), (129, 129)], hq, hkv, 16, F16, 14)
    out = PagedOperator()(q, kp, vp, table, kv, cu, max_q=1, window=window, sinks=sinks)
    O, A = ref.paged_attention(q, kp, vp, table, kv, cu, window, sinks)
    bound = A * (HALF[F16] + 3e-4 + 2.0 ** -16) + O.abs() * HALF[F16] + 2.0 ** -24
    assert bool(((out.double() - O).abs() <= bound).all())


@gpu
def test_a_rotary_and_its_gradient_in_a_graph():
    from fa_b200.rotary import Rotary

    rotary, pos = Rotary(64), torch.arange(9, device="cuda") * 5
    x, g = torch.randn((2, 3, 9, 64), device="cuda").requires_grad_(), torch.randn((2, 3, 9, 64), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(rotary(x, pos), x, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rotary(x, pos)
        (grad,) = torch.autograd.grad(y, x, g)
    for _ in range(2):
        with torch.no_grad():
            x.add_(1.0), g.mul_(0.5)
        graph.replay()
        assert torch.equal(y.detach(), rotary(x.detach(), pos)) and torch.equal(grad, rotary(g, pos, inverse=True))


@gpu
def test_steps_of_two_threads_on_streams_of_their_own():
    from fa_b200.paged import PagedOperator
    from fa_b200.rotary import Rotary

    op, rotary = PagedOperator(), Rotary(128)
    cases = [_cache([(1, 9000), (2, 500)], 12, 1, 16, F16, 30), _cache([(200, 4000)], 8, 2, 64, F16, 31)]
    longest = [2, 200]
    wants = [op(rotary(c[0], torch.zeros(c[0].shape[0], dtype=torch.int64, device="cuda")), *c[1:], max_q=n)
             for c, n in zip(cases, longest)]
    torch.cuda.synchronize()

    def work(c, n):
        with torch.cuda.stream(torch.cuda.Stream()):
            zero = torch.zeros(c[0].shape[0], dtype=torch.int64, device="cuda")
            out = [op(rotary(c[0], zero), *c[1:], max_q=n) for _ in range(30)]
            torch.cuda.current_stream().synchronize()
            return out

    for want, got in zip(wants, _in_two_threads(*[lambda c=c, n=n: work(c, n) for c, n in zip(cases, longest)])):
        assert all(torch.equal(o, want) for o in got)
