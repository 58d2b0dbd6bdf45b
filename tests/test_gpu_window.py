"""Sliding window with sinks (``Operator(...)(q, k, v, causal=True, window=W,
sinks=S)``): key j is seen from row i when j <= i and (j > i - W or j < S).

Tolerance, per output element, with w the softmax weights, A = sum w |v| and
O the float64 result.  P is rounded to FP16 (half a step, 2^-11 relative) and
its exponentials are good to 7.5e-5 (the polynomial; the others 2^-22); the
normalizer's relative error adds to O: FP32 sums 2^-16 at most here.  (The
causal kernel of the FP16 variant: FP16 partial sums, 9 roundings, 7 adds of a
chain of 8 and two folds.)
Scores are FP32 sums of 128 products below 2^5 in all: 128 * 2^-24 * 2^5 <
3e-4 absolute before the exponential.  O itself is rounded to FP16.
"""

import pytest
import torch

from oracle import serving_ref as ref

HALF = 2.0 ** -11

SHAPES = [
    # (B, Hq, Hkv, Nq, Nk, window, sinks)
    (1, 2, 1, 1, 1, 1, 0),
    (1, 2, 1, 300, 300, 1, 0),          # a row sees itself only
    (1, 2, 2, 257, 257, 64, 1),
    (1, 4, 2, 700, 700, 128, 4),
    (1, 2, 1, 1000, 1000, 127, 129),    # sinks end inside a second block
    (1, 2, 1, 900, 900, 255, 300),      # sinks and window overlap at first
    (2, 8, 2, 1111, 777, 200, 5),       # rows behind the keys see the sinks only
    (1, 2, 1, 1200, 130, 100, 0),       # rows that see nothing
    (1, 2, 1, 130, 2000, 50, 10),       # keys that no row reaches
    (1, 12, 1, 2500, 2500, 513, 4),     # several items per pair
    (1, 2, 1, 500, 500, 5000, 0),       # a window wider than the sequence: causal
    (1, 2, 1, 600, 600, 32, 2**31),     # every key a sink: causal
]


def _inputs(B, Hq, Hkv, Nq, Nk, seed, device):
    g = torch.Generator(device="cpu").manual_seed(seed)
    q = torch.randn((B, Hq, Nq, 128), generator=g)
    k = torch.randn((B, Hkv, Nk, 128), generator=g)
    v = torch.randn((B, Hkv, Nk, 128), generator=g)
    return [t.half().to(device) for t in (q, k, v)]


def _bound(O, A, variant):
    sums = 9 * HALF if variant == "fp16" else 2.0 ** -16
    return A * (HALF + 7.5e-5 + sums + 3e-4) + O.abs() * HALF + 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("debug", [False, True], ids=["product", "checking"])
@pytest.mark.parametrize("variant", ["fp16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_window_against_the_formula(shape, variant, debug):
    from fa_b200.ops import Operator

    *dims, window, sinks = shape
    q, k, v = _inputs(*dims, seed=sum(dims) + window, device="cuda")
    op = Operator(variant, debug=debug)
    out = op(q, k, v, causal=True, window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert op.status(q.device)[0] == 0
    O, A = ref.window_attention(q, k, v, window, sinks)
    over = (out.double() - O).abs() - _bound(O, A, "fp32")
    assert bool((over <= 0).all()), float(over.max())
    assert torch.equal(out[A == 0], torch.zeros_like(out[A == 0]))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["fp16", "fp32"])
def test_a_window_over_everything_is_the_causal_mask(variant):
    from fa_b200.ops import Operator

    q, k, v = _inputs(1, 12, 1, 1500, 1500, 3, "cuda")
    op = Operator(variant)
    a = op(q, k, v, causal=True)
    b = op(q, k, v, causal=True, window=1500)
    torch.cuda.synchronize()
    # The causal kernels evaluate part of the exponentials on the FMA pipe and
    # (fp16) sum in FP16; the window kernel does neither, so the two agree to
    # the sum of their bounds against the formula, not bit for bit.
    O, A = ref.window_attention(q, k, v, 1500, 0)
    over = (a.double() - b.double()).abs() - _bound(O, A, variant) - _bound(O, A, "fp32")
    assert bool((over <= 0).all()), float(over.max())


@pytest.mark.gpu
def test_window_shards_equal_the_whole_range_and_out_of_window_keys_are_not_used():
    from fa_b200 import shard
    from fa_b200.ops import Operator

    q, k, v = _inputs(1, 12, 1, 2048, 2048, 5, "cuda")
    op = Operator("fp32")
    whole = op(q, k, v, causal=True, window=300, sinks=4)
    parts = torch.full_like(q, float("nan"))
    units = shard.num_units(1, 12, 2048)
    for rank in range(3):
        op(q, k, v, causal=True, window=300, sinks=4, out=parts, unit_range=shard.partition(units, 3, rank))
    assert torch.equal(parts, whole)
    # Blocks between the sinks and the last units' window: not read by them.
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 128:1152], v2[:, :, 128:1152] = float("nan"), float("inf")
    tail = torch.full_like(q, 7.0)
    for h in range(12):
        op(q, k2, v2, causal=True, window=300, sinks=4, out=tail, unit_range=(h * 16 + 12, h * 16 + 16))
    torch.cuda.synchronize()
    assert torch.equal(tail[:, :, 1536:], whole[:, :, 1536:])
    assert bool((tail[:, :, :1536] == 7.0).all())


@pytest.mark.gpu
def test_window_through_host_buffers_and_a_graph():
    from fa_b200.ops import Operator

    q, k, v = _inputs(1, 4, 2, 1000, 1000, 9, "cuda")
    op = Operator("fp16")
    want = op(q, k, v, causal=True, window=200, sinks=3)
    host = [t.cpu().pin_memory() for t in (q, k, v)]
    got = torch.empty_like(host[0]).pin_memory()
    dev = [torch.empty_like(t) for t in (q, k, v, q)]
    op.forward_host(*host, got, q_dev=dev[0], k_dev=dev[1], v_dev=dev[2], o_dev=dev[3], causal=True, window=200, sinks=3)
    torch.cuda.synchronize()
    assert torch.equal(got, want.cpu())
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(q, k, v, causal=True, window=200, sinks=3, out=out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_a_withheld_hand_over_ends_the_window_kernel_with_a_status():
    """Every role of the window kernel, the storing warp among them, leaves when
    a bounded wait runs out (the flag withholds one arrival)."""
    from fa_b200 import lib
    from fa_b200.ops import Operator

    q, k, v = _inputs(1, 2, 1, 600, 600, 2, "cuda")
    op = Operator("fp32", timeout_us=20000)
    want = op(q, k, v, causal=True, window=300)
    op(q, k, v, causal=True, window=300, flags=lib.FLAG_TEST_WITHHOLD_P)
    assert op.status(q.device)[0] == lib.DEV_TIMEOUT
    op.reset_status(q.device)
    assert torch.equal(op(q, k, v, causal=True, window=300), want)
    assert op.status(q.device)[0] == lib.DEV_OK


def test_window_refusals():
    from fa_b200 import lib
    from fa_b200.ops import _window

    for args in ((-1, 0, True), (5, -1, True), (5, 0, False), (0, 4, True), (None, 0, True)):
        with pytest.raises(ValueError):
            _window(*args)
    assert _window(2**40, 2**40, True) == (2**31 - 1, 2**31 - 1)
    import ctypes as C

    def rc(flags, window, sinks):
        opts = lib.Options(C.sizeof(lib.Options), flags, 0, 0, None, 0, window, sinks)
        return lib.load().b200fa_fwd_ex(16, 16, 16, 16, 1, 2, 1, 300, 1000, 128, 0.088, 0, 2, 2,
                                        256, 1 << 20, None, C.byref(opts))

    both = lib.FLAG_CAUSAL | lib.FLAG_WINDOW
    assert rc(both, 7, 0) == 0  # empty range: nothing launched
    assert rc(lib.FLAG_WINDOW, 7, 0) == -11
    assert rc(both, 0, 0) == -11 and rc(both, 7, -1) == -11
    opts = lib.Options(32, 0, 0, 0, None, 0)  # the layout without the window fields
    assert lib.load().b200fa_fwd_ex(16, 16, 16, 16, 1, 2, 1, 300, 1000, 128, 0.088, 0, 2, 2,
                                    256, 1 << 20, None, C.byref(opts)) == 0
