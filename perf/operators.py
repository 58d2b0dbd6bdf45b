"""The measured cases of the serving operators: page tables, rotary positions
with the cache append, attention over a paged cache, and attention with a
sliding window and sinks.

``run`` computes a case in plain torch operations, or, with ``own``, through
the framework's entry points.  Head layouts (12 query heads on 1 key/value
head, 32 on 8) and lengths follow the repository's attention cases.
"""

import functools
import math

import torch

own = False

DIM = 128
DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ----------------------------------------------------------------- the cases
def listed():
    return [
        # One generation step of a few requests: one new token each; latency is all.
        {"name": "tables_decode", "op": "tables", "requests": 8, "max_new": 1, "max_ctx": 2048, "page": 16},
        # A large admission step: many requests with ragged prompts on top of what they hold.
        {"name": "tables_prompts", "op": "tables", "requests": 250, "max_new": 700, "max_ctx": 8192, "page": 64},
        # Rotation and cache write of one generation step.
        {"name": "append_decode", "op": "append", "tokens": 8, "hq": 12, "hkv": 1, "page": 16, "rot": 128,
         "layout": "half", "scaling": "none", "max_pos": 32768, "dtype": "fp16"},
        # A prompt of grouped heads, only part of each head rotated, adjacent pairs.
        {"name": "append_prompt", "op": "append", "tokens": 16000, "hq": 32, "hkv": 8, "page": 16, "rot": 64,
         "layout": "interleaved", "scaling": "banded", "max_pos": 131072, "dtype": "bf16"},
        # The gradient direction (rotation by the negative angle) on the dense [B,H,N,D] layout.
        {"name": "rotary_inverse", "op": "rotary", "batch": 2, "heads": 12, "n": 32768, "rot": 128,
         "layout": "half", "scaling": "linear", "inverse": True, "max_pos": 131072, "dtype": "fp16"},
        # One request, one token: the shortest chain a user waits for.
        {"name": "paged_decode_one", "op": "paged", "requests": 1, "max_q": 1, "max_kv": 2048, "hq": 12, "hkv": 1,
         "page": 16, "window": 0, "sinks": 0, "dtype": "fp16"},
        # A batch in generation: bound by reading the cache.
        {"name": "paged_decode_batch", "op": "paged", "requests": 32, "max_q": 1, "max_kv": 16384, "hq": 32, "hkv": 8,
         "page": 16, "window": 0, "sinks": 0, "dtype": "bf16"},
        # Long prompts fed in chunks over what is cached already: bound by the products.
        {"name": "paged_chunk", "op": "paged", "requests": 2, "max_q": 4096, "max_kv": 32768, "hq": 12, "hkv": 1,
         "page": 64, "window": 0, "sinks": 0, "dtype": "fp16"},
        # A mixed step (short chunks beside single tokens) with a window and sinks.
        {"name": "paged_window_mixed", "op": "paged", "requests": 16, "max_q": 130, "max_kv": 16384, "hq": 32,
         "hkv": 8, "page": 32, "window": 4096, "sinks": 4, "dtype": "bf16"},
        # A short prompt without a cache.
        {"name": "window_small", "op": "window", "batch": 1, "hq": 12, "hkv": 1, "nq": 2048, "nk": 2048,
         "window": 256, "sinks": 4, "variant": "fp16"},
        # The grouped-head configuration with a narrow window.
        {"name": "window_grouped", "op": "window", "batch": 4, "hq": 32, "hkv": 8, "nq": 8192, "nk": 8192,
         "window": 1024, "sinks": 4, "variant": "fp16"},
        # A long sequence, odd length, wide window, softmax sums in 32 bits.
        {"name": "window_long", "op": "window", "batch": 1, "hq": 12, "hkv": 1, "nq": 32700, "nk": 32700,
         "window": 4096, "sinks": 128, "variant": "fp32"},
    ]


def draw(rng):
    def log_int(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    hq, hkv = rng.choice([(12, 1), (32, 8), (8, 8), (16, 2), (6, 2)])
    op = rng.choice(["tables", "append", "rotary", "paged", "paged", "paged", "window", "window"])
    if op == "tables":
        return {"op": op, "requests": log_int(1, 250), "max_new": log_int(1, 700), "max_ctx": log_int(16, 8192),
                "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        return {"op": op, "tokens": log_int(1, 12000), "hq": hq, "hkv": hkv, "page": rng.choice([16, 32, 64, 128]),
                "rot": rng.choice([32, 64, 128]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "banded"]), "max_pos": log_int(2048, 131072),
                "dtype": rng.choice(["fp16", "bf16"])}
    if op == "rotary":
        return {"op": op, "batch": rng.choice([1, 2]), "heads": hq, "n": log_int(1, 24000),
                "rot": rng.choice([32, 64, 128]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "banded"]), "inverse": rng.random() < 0.5,
                "max_pos": log_int(32768, 131072), "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if op == "paged":
        window = rng.choice([0, 0, log_int(64, 4096)])
        kind = rng.choice(["decode", "chunk", "short"])
        if kind == "decode":
            requests, max_q, max_kv = log_int(1, 40), 1, log_int(100, 16384)
        elif kind == "short":
            requests, max_q, max_kv = log_int(1, 16), log_int(2, 130), log_int(200, 12000)
        else:
            requests, max_q, max_kv = rng.choice([1, 2]), log_int(130, 2000), log_int(2000, 24000)
        return {"op": op, "requests": requests, "max_q": max_q, "max_kv": max_kv, "hq": hq, "hkv": hkv,
                "page": rng.choice([16, 32, 64, 128]), "window": window,
                "sinks": rng.choice([0, 4, log_int(1, 200)]) if window else 0, "dtype": rng.choice(["fp16", "bf16"])}
    n = log_int(300, 16000)
    return {"op": op, "batch": rng.choice([1, 2]), "hq": hq, "hkv": hkv, "nq": n,
            "nk": rng.choice([n, n, log_int(300, 16000)]), "window": log_int(64, 2048),
            "sinks": rng.choice([0, 4, log_int(1, 200)]), "variant": rng.choice(["fp16", "fp32"])}


# ------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _lengths(g, count, most, least=1):
    """`count` lengths of [least, most], the first one the longest."""
    x = torch.randint(least, most + 1, (count,), generator=g, device=DEV, dtype=torch.int32)
    x[0] = most
    return x


def _spread(case):
    """The new and cached lengths of a batch's requests, each from longest to
    shortest: chunks fall off with the square (a few long ones beside single
    tokens), contexts evenly to a quarter.  A seed only permutes them, so
    that every input of a case has as many tokens."""
    R, mq, mk = case["requests"], case["max_q"], case["max_kv"]
    q = [1 + (mq - 1) * (R - i) ** 2 // (R * R) for i in range(R)]
    kv = [max(mk - (mk - mk // 4) * i // R, q[i], 1) for i in range(R)]
    return q, kv


def _scaling(case):
    """The keyword arguments that describe a case's frequency scaling."""
    if case["scaling"] == "linear":
        return {"scaling": "linear", "factor": 4.0}
    if case["scaling"] == "banded":
        return {"scaling": "banded", "factor": 8.0, "original_length": 8192, "low": 1.0, "high": 4.0,
                "magnitude": 1.0 + 0.1 * math.log(8.0)}
    return {}


def _frequencies(case):
    """Angle per position of each rotated pair (64 bits), and the magnitude:
    base^(-2i/rot); "linear" divides all by the factor; "banded" leaves the
    pairs that turn more than `high` times in the original length, divides
    those that turn less than `low` times, and blends between."""
    rot = case["rot"]
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    s = _scaling(case)
    if case["scaling"] == "linear":
        return f / s["factor"], 1.0
    if case["scaling"] == "banded":
        turns = s["original_length"] * f / (2 * math.pi)
        keep = ((turns - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        return f * keep + f / s["factor"] * (1 - keep), s["magnitude"]
    return f, 1.0


def prepare(case, seed):
    g = _generator(seed)
    op, s = case["op"], {"case": dict(case)}
    if op == "tables":
        R, ps = case["requests"], case["page"]
        ctx = _lengths(g, R, case["max_ctx"], 0)
        new = _lengths(g, R, case["max_new"])
        width = -(-(case["max_ctx"] + case["max_new"]) // ps)
        held = (ctx + ps - 1) // ps
        order = torch.randperm(R * (width + 1), generator=g, device=DEV).to(torch.int32)
        col = torch.arange(width, device=DEV)[None]
        table = torch.where(col < held[:, None], order[: R * width].view(R, width), -1).to(torch.int32)
        mask = (col >= held[:, None]).view(-1)
        free = torch.cat([order[: R * width][mask], order[R * width:]])
        s.update(ctx=ctx, new=new, table=table.contiguous(), free=free.contiguous(),
                 count=torch.tensor([free.numel()], dtype=torch.int32, device=DEV),
                 tokens=R * case["max_new"])  # the step's token buffer, as a serving loop sizes it
        return s
    if op in ("append", "rotary"):
        dt = TYPES[case["dtype"]]
        if op == "rotary":
            shape = (case["batch"], case["heads"], case["n"], DIM)
            s["x"] = torch.randn(shape, generator=g, device=DEV).to(dt)
            s["pos"] = torch.randint(0, case["max_pos"], (case["n"],), generator=g, device=DEV, dtype=torch.int32)
            return s
        T, hq, hkv, ps = case["tokens"], case["hq"], case["hkv"], case["page"]
        # q, k and v are slices of one projection's output
        s["qkv"] = torch.randn((T, hq + 2 * hkv, DIM), generator=g, device=DEV).to(dt)
        pages = -(-T // ps) + 4
        s["kp"] = torch.randn((pages, ps, hkv, DIM), generator=g, device=DEV).to(dt)
        s["vp"] = torch.randn((pages, ps, hkv, DIM), generator=g, device=DEV).to(dt)
        slots = torch.randperm(pages * ps, generator=g, device=DEV)[:T]
        slots[torch.rand(T, generator=g, device=DEV) < 0.02] = -1  # padded tokens
        s["slots"] = slots
        s["pos"] = torch.randint(0, case["max_pos"], (T,), generator=g, device=DEV, dtype=torch.int32)
        return s
    if op == "paged":
        dt = TYPES[case["dtype"]]
        R, ps, hq, hkv = case["requests"], case["page"], case["hq"], case["hkv"]
        order = torch.randperm(R, generator=g, device=DEV)
        qlen, kv = (torch.tensor(x, dtype=torch.int32, device=DEV)[order] for x in _spread(case))
        cu = torch.zeros(R + 1, dtype=torch.int32, device=DEV)
        cu[1:] = qlen.cumsum(0)
        T = sum(_spread(case)[0])
        width = -(-max(case["max_kv"], case["max_q"]) // ps)
        pages = R * width
        s["q"] = torch.randn((T, hq, DIM), generator=g, device=DEV).to(dt)
        s["kp"] = torch.empty((pages, ps, hkv, DIM), dtype=dt, device=DEV).normal_(generator=g)
        s["vp"] = torch.empty((pages, ps, hkv, DIM), dtype=dt, device=DEV).normal_(generator=g)
        s["table"] = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(R, width)
        s.update(kv=kv, cu=cu, T=T)
        return s
    shape = lambda h, n: (case["batch"], h, n, DIM)  # noqa: E731
    s["q"] = torch.randn(shape(case["hq"], case["nq"]), generator=g, device=DEV).half()
    s["k"] = torch.randn(shape(case["hkv"], case["nk"]), generator=g, device=DEV).half()
    s["v"] = torch.randn(shape(case["hkv"], case["nk"]), generator=g, device=DEV).half()
    return s


# -------------------------------------------------------------- plain forms
def _plain_tables(s):
    c = s["case"]
    ps, R, T = c["page"], c["requests"], s["tokens"]
    ctx, new = s["ctx"].long(), s["new"].long()
    held = (ctx + ps - 1) // ps
    need = (ctx + new + ps - 1) // ps - held
    cu = torch.zeros(R + 1, dtype=torch.int64, device=DEV)
    cu[1:] = new.cumsum(0)
    before = need.cumsum(0) - need
    count = s["count"].long()
    col = torch.arange(s["table"].shape[1], device=DEV)[None]
    nth = before[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    taken = s["free"].long()[(count - 1 - nth).clamp(0, s["free"].numel() - 1)]
    table = torch.where(fresh, taken, s["table"].long())
    t = torch.arange(T, device=DEV)
    req = (torch.searchsorted(cu, t, right=True) - 1).clamp(0, R - 1)
    real = t < cu[R]
    pos = torch.where(real, ctx[req] + t - cu[req], 0)
    page = table[req, (pos // ps).clamp(0, table.shape[1] - 1)]
    slots = torch.where(real, page * ps + pos % ps, -1)
    return {"table": table.int(), "slots": slots, "positions": pos.int(), "cu_q": cu.int(),
            "kv_lens": (ctx + new).int(), "free_left": (count - need.sum()).int()}


def _turn(case, x, pos, sign, dt=torch.float32):
    """Rotation of x [..., n, DIM] by the angles of pos [n]."""
    f, mag = _frequencies(case)
    a = pos.double()[:, None] * f
    cos, sin = (mag * torch.cos(a)).to(dt), (sign * mag * torch.sin(a)).to(dt)
    rot, x = case["rot"], x.to(dt)
    body, rest = x[..., :rot], x[..., rot:]
    if case["layout"] == "half":
        u, v = body[..., : rot // 2], body[..., rot // 2:]
        body = torch.cat([u * cos - v * sin, v * cos + u * sin], -1)
    else:
        u, v = body[..., 0::2], body[..., 1::2]
        body = torch.stack([u * cos - v * sin, v * cos + u * sin], -1).flatten(-2)
    return torch.cat([body, rest], -1)


def _split(s):
    hq, hkv = s["case"]["hq"], s["case"]["hkv"]
    return s["qkv"][:, :hq], s["qkv"][:, hq:hq + hkv], s["qkv"][:, hq + hkv:]


def _plain_append(s):
    q, k, v = _split(s)
    dt = q.dtype
    out = _turn(s["case"], q.transpose(0, 1), s["pos"], 1.0).transpose(0, 1).to(dt).contiguous()
    kr = _turn(s["case"], k.transpose(0, 1), s["pos"], 1.0).transpose(0, 1).to(dt)
    kp, vp = s["kp"].view(-1, *k.shape[1:]), s["vp"].view(-1, *k.shape[1:])
    real = (s["slots"] >= 0)[:, None, None]
    at = s["slots"].clamp(min=0)
    # a padded token rewrites slot 0 with what that slot is to hold: its own row where a token has it
    owner = torch.where(s["slots"] == 0, torch.arange(at.numel(), device=DEV), -1).amax()
    keep_k = torch.where(owner >= 0, kr[owner.clamp(min=0)], kp[0])
    keep_v = torch.where(owner >= 0, v[owner.clamp(min=0)], vp[0])
    kp[at] = torch.where(real, kr, keep_k[None])
    vp[at] = torch.where(real, v, keep_v[None])
    return {"q": out, "k_pages": s["kp"], "v_pages": s["vp"]}


def _plain_paged(s):
    c = s["case"]
    hq, hkv, ps, T = c["hq"], c["hkv"], c["page"], s["T"]
    R, G, mq = c["requests"], c["hq"] // c["hkv"], c["max_q"]
    mk = max(c["max_kv"], mq)
    cu, kv = s["cu"].long(), s["kv"].long()
    qlen = cu[1:] - cu[:-1]
    i, j = torch.arange(mq, device=DEV), torch.arange(mk, device=DEV)
    real = i[None] < qlen[:, None]
    token = torch.where(real, cu[:-1, None] + i[None], T)
    q = s["q"][token.clamp(max=T - 1)].float().view(R, mq, hkv, G, DIM).permute(0, 2, 3, 1, 4).reshape(R, hkv, G * mq, DIM)
    page = s["table"].long()[:, j // ps]
    off = (j % ps)[None].expand(R, mk)
    held = (j[None] < kv[:, None])[:, :, None, None]
    k = torch.where(held, s["kp"][page, off].float(), 0.0).permute(0, 2, 3, 1)
    v = torch.where(held, s["vp"][page, off].float(), 0.0).permute(0, 2, 1, 3)
    p = (kv - qlen)[:, None] + i[None]
    see = (j <= p[..., None]) & (j < kv[:, None, None])
    if c["window"]:
        see &= (j > p[..., None] - c["window"]) | (j < c["sinks"])
    a = (q @ k).mul_(DIM ** -0.5).view(R, hkv, G, mq, mk)
    a.masked_fill_(~see[:, None, None], -math.inf)
    a.sub_(a.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = a.sum(-1, keepdim=True)
    o = (a.view(R, hkv, G * mq, mk) @ v).view(R, hkv, G, mq, DIM)
    o = torch.where(total > 0, o / total, 0.0)
    out = torch.zeros((T + 1, hq, DIM), dtype=s["q"].dtype, device=DEV)
    out[token.view(-1)] = o.permute(0, 3, 1, 2, 4).reshape(R * mq, hq, DIM).to(out.dtype)
    return out[:T]


def _plain_window(s):
    c = s["case"]
    B, hq, hkv, nq, nk, W = c["batch"], c["hq"], c["hkv"], c["nq"], c["nk"], c["window"]
    sinks, G, C = min(c["sinks"], nk), c["hq"] // c["hkv"], 512
    nb = -(-nq // C)
    q = torch.nn.functional.pad(s["q"].float(), (0, 0, 0, nb * C - nq)).view(B, hkv, G, nb, C, DIM)
    q = q.permute(0, 1, 3, 2, 4, 5).reshape(B, hkv, nb, G * C, DIM)
    row = torch.arange(nb * C, device=DEV).view(nb, C, 1)
    key = torch.arange(nb, device=DEV)[:, None] * C + torch.arange(1 - W, C, device=DEV)[None]
    at = key.clamp(0, nk - 1)
    k = torch.cat([s["k"].float()[:, :, at], s["k"].float()[:, :, None, :sinks].expand(-1, -1, nb, -1, -1)], 3)
    v = torch.cat([s["v"].float()[:, :, at], s["v"].float()[:, :, None, :sinks].expand(-1, -1, nb, -1, -1)], 3)
    kk = key[:, None]
    see = (kk >= sinks) & (kk < nk) & (kk <= row) & (kk > row - W)
    see = torch.cat([see, (torch.arange(sinks, device=DEV) <= row)], -1)
    a = (q @ k.transpose(-1, -2)).mul_(DIM ** -0.5).view(B, hkv, nb, G, C, -1)
    a.masked_fill_(~see[:, None], -math.inf)
    a.sub_(a.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = a.sum(-1, keepdim=True)
    o = (a.view(B, hkv, nb, G * C, -1) @ v).view(B, hkv, nb, G, C, DIM)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 1, 3, 2, 4, 5).reshape(B, hq, nb * C, DIM)[:, :, :nq].half()


# ------------------------------------------------------------ the framework
@functools.lru_cache(maxsize=None)
def _operator(variant):
    from fa_b200.ops import Operator

    return Operator(variant)


@functools.lru_cache(maxsize=None)
def _paged_operator():
    from fa_b200.paged import PagedOperator

    return PagedOperator()


@functools.lru_cache(maxsize=None)
def _rotary(rot, layout, scaling):
    from fa_b200.rotary import Rotary

    return Rotary(DIM, rotary_dim=rot, layout=layout, **_scaling({"scaling": scaling}))


def _own(s):
    c = s["case"]
    if c["op"] == "tables":
        from fa_b200.paged import build_tables

        r = build_tables(s["ctx"], s["new"], s["table"], s["free"], s["count"], page_size=c["page"],
                         num_tokens=s["tokens"])
        return {"table": s["table"], "slots": r.slots, "positions": r.positions, "cu_q": r.cu_q,
                "kv_lens": r.kv_lens, "free_left": r.free_left}
    if c["op"] == "append":
        from fa_b200.paged import append

        q, k, v = _split(s)
        out = append(k, v, s["kp"], s["vp"], s["slots"], q=q, positions=s["pos"],
                     rotary=_rotary(c["rot"], c["layout"], c["scaling"]))
        return {"q": out, "k_pages": s["kp"], "v_pages": s["vp"]}
    if c["op"] == "rotary":
        return _rotary(c["rot"], c["layout"], c["scaling"])(s["x"], s["pos"], inverse=c["inverse"])
    if c["op"] == "paged":
        return _paged_operator()(s["q"], s["kp"], s["vp"], s["table"], s["kv"], s["cu"], max_q=c["max_q"],
                                 window=c["window"], sinks=c["sinks"])
    return _operator(c["variant"])(s["q"], s["k"], s["v"], causal=True, window=c["window"], sinks=c["sinks"])


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    if c["op"] == "tables":
        return _plain_tables(state)
    if c["op"] == "append":
        return _plain_append(state)
    if c["op"] == "rotary":
        return _turn(c, state["x"], state["pos"], -1.0 if c["inverse"] else 1.0).to(state["x"].dtype)
    if c["op"] == "paged":
        return _plain_paged(state)
    return _plain_window(state)


# --------------------------------------------------------------------- work
def _seen(first, count, window, sinks, nk):
    """Keys seen by the rows at positions first .. first+count-1 of nk keys."""
    n = 0
    for p in range(first, first + count):
        hi = min(p, nk - 1) + 1
        lo = max(0, p - window + 1) if window else 0
        n += max(0, hi - lo) + (max(0, min(sinks, hi, lo)) if window else 0)
    return n


def _expected(most, least):
    return (most + least) / 2


def work(case):
    op = case["op"]
    if op == "tables":
        R, ps = case["requests"], case["page"]
        new, ctx = _expected(case["max_new"], 1), _expected(case["max_ctx"], 0)
        tokens = R * case["max_new"]
        pages = R * (new / ps + 0.5)
        return {"bytes": R * 4 * 4 + pages * 8 + R * 4 + tokens * 12, "flops": 0}
    if op == "append":
        size = TYPES[case["dtype"]].itemsize
        T, rows = case["tokens"], case["hq"] + 2 * case["hkv"]
        return {"bytes": 2 * T * rows * DIM * size + T * 12, "flops": T * (case["hq"] + case["hkv"]) * case["rot"] * 3}
    if op == "rotary":
        rows = case["batch"] * case["heads"] * case["n"]
        return {"bytes": 2 * rows * DIM * TYPES[case["dtype"]].itemsize + case["n"] * 4, "flops": rows * case["rot"] * 3}
    if op == "paged":
        R, W, S = case["requests"], case["window"], case["sinks"]
        pairs = keys = toks = 0
        for n, kv in zip(*_spread(case)):
            lo = max(0, kv - n - W + 1) if W else 0
            keys += kv - lo + min(S, lo)
            pairs += _seen(kv - n, n, W, S, kv)
            toks += n
        size = 2
        return {"bytes": 2 * keys * case["hkv"] * DIM * size + 2 * toks * case["hq"] * DIM * size
                + R * 8 + keys // case["page"] * 4, "flops": 4 * DIM * case["hq"] * pairs}
    pairs = _seen(0, case["nq"], case["window"], case["sinks"], case["nk"])
    rows_q, rows_k = case["batch"] * case["hq"] * case["nq"], case["batch"] * case["hkv"] * case["nk"]
    return {"bytes": 4 * DIM * (rows_q + rows_k), "flops": 4 * DIM * case["batch"] * case["hq"] * pairs}


# -------------------------------------------------------------------- exact
def _softmax_rows(q, k, v, see):
    """q [m, D], k and v [n, D] in 64 bits, see [m, n]; rows that see nothing give zeros."""
    a = q @ k.T / math.sqrt(DIM)
    a = torch.where(see, a, torch.full_like(a, -math.inf))
    w = torch.softmax(a, -1)
    return torch.nan_to_num(w, nan=0.0) @ v


def _exact_rotation(case, x, pos, inverse):
    """Complex multiplication of the pairs by mag * e^(+-i angle)."""
    f, mag = _frequencies(case)
    turn = torch.polar(torch.full((pos.numel(), f.numel()), mag, dtype=torch.float64, device=DEV),
                       pos.double()[:, None] * f[None] * (-1 if inverse else 1))
    rot, y = case["rot"], x.double().clone()
    if case["layout"] == "half":
        z = torch.complex(y[..., : rot // 2].contiguous(), y[..., rot // 2: rot].contiguous()) * turn
        y[..., : rot // 2], y[..., rot // 2: rot] = z.real, z.imag
    else:
        z = torch.view_as_complex(y[..., :rot].reshape(*y.shape[:-1], rot // 2, 2).contiguous()) * turn
        y[..., :rot] = torch.view_as_real(z).flatten(-2)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "tables":
        return None
    if op == "rotary":
        return _exact_rotation(case, s["x"], s["pos"], case["inverse"])
    if op == "append":
        q, k, v = _split(s)
        out = {"q": _exact_rotation(case, q.transpose(0, 1), s["pos"], False).transpose(0, 1),
               "k_pages": s["kp"].double(), "v_pages": s["vp"].double()}
        kr = _exact_rotation(case, k.transpose(0, 1), s["pos"], False).transpose(0, 1)
        t = torch.nonzero(s["slots"] >= 0).view(-1)
        at = s["slots"][t]
        out["k_pages"][at // case["page"], at % case["page"]] = kr[t]
        out["v_pages"][at // case["page"], at % case["page"]] = v[t].double()
        return out
    W, S, G = case["window"], case["sinks"], case["hq"] // case["hkv"]
    if op == "paged":
        out = torch.zeros((s["T"], case["hq"], DIM), dtype=torch.float64, device=DEV)
        cu, kv = s["cu"].tolist(), s["kv"].tolist()
        for r in range(case["requests"]):
            n, m = cu[r + 1] - cu[r], kv[r]
            pages = s["table"][r, : -(-m // case["page"])].long()
            k = s["kp"][pages].flatten(0, 1)[:m].double()
            v = s["vp"][pages].flatten(0, 1)[:m].double()
            p = torch.arange(m - n, m, device=DEV)[:, None]
            j = torch.arange(m, device=DEV)[None]
            see = j <= p
            if W:
                see &= (j > p - W) | (j < S)
            for h in range(case["hq"]):
                out[cu[r]:cu[r + 1], h] = _softmax_rows(s["q"][cu[r]:cu[r + 1], h].double(), k[:, h // G], v[:, h // G], see)
        return out
    nq, nk = case["nq"], case["nk"]
    out = torch.zeros((case["batch"], case["hq"], nq, DIM), dtype=torch.float64, device=DEV)
    j = torch.arange(nk, device=DEV)[None]
    for r0 in range(0, nq, 2048):
        r1 = min(nq, r0 + 2048)
        p = torch.arange(r0, r1, device=DEV)[:, None]
        pick = torch.nonzero(((j <= p) & ((j > p - W) | (j < S))).any(0)).view(-1)
        see = (pick[None] <= p) & ((pick[None] > p - W) | (pick[None] < S))
        for b in range(case["batch"]):
            for h in range(case["hq"]):
                out[b, h, r0:r1] = _softmax_rows(s["q"][b, h, r0:r1].double(), s["k"][b, h // G, pick].double(),
                                                 s["v"][b, h // G, pick].double(), see)
    return out
