"""The serving operators where they went wrong once: first use by two threads,
forward-mode derivatives, values that no row sees, steps that could not be met,
bounds of waits, ends of the number ranges.  Tolerances as in
test_gpu_serving.py; most checks here are for equality."""

import pytest
import torch

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
gpu = pytest.mark.gpu
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731


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
