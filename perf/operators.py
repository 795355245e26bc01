"""Operators of a hybrid decoder layer, measured one by one: a selective state space scan, what makes its inputs, and a router that
chooses experts by groups.

    selective_scan      dt = softplus(raw + bias);  h[c, n] <- exp(-dt e^log_rate[c, n]) h[c, n] + dt x[c] B[n]
                        y[c] = (sum_n C[n] h[c, n] + skip[c] x[c]) silu(z[c])              h float32, one matrix a request
    selective_inputs    rows [T, rank + 2 states] -> the step's part in the run's dtype and B | C in float32, each RMS-normed
    moe_route_groups    scores; every group's sum of its best; the best groups; the best experts of those; their weights

`run` computes them in plain form where `own` is false, and calls the framework's kernels where it is true.  A case is a dict of
numbers and texts; how its tokens fall on its requests follows from the case alone, inputs from the seed.
"""
from __future__ import annotations

import math
import random
import types

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
MOST_WORK = 2048 * 7168 * 16        # tokens x channels x state numbers of the largest scan
_handle = []


def listed():
    scan = {"kind": "scan", "states": 16, "dtype": "bfloat16", "step": "float32", "gate": True, "skip": True}
    route = {"kind": "route", "score": "sigmoid", "correction": True, "normalized": True, "best": 2}
    return [
        # one chat's next token through a layer of the 7B shape's width (inner size twice 3,584): launch and latency
        {**scan, "name": "scan_one_token", "channels": 7168, "requests": 1, "tokens": 1},
        # a decode batch: every request's state is read and written once
        {**scan, "name": "scan_decode", "channels": 7168, "requests": 64, "tokens": 64},
        # one long prompt portion of the same layer, the largest call
        {**scan, "name": "scan_prompt", "channels": 7168, "requests": 1, "tokens": 2048},
        # a mixed step: prompts of uneven lengths beside each other, an inner size that is no power of two
        {**scan, "name": "scan_mixed", "channels": 5120, "requests": 6, "tokens": 1531},
        # a small model's long prompt, few channels: the axis of time is the long one
        {**scan, "name": "scan_narrow", "channels": 1024, "requests": 1, "tokens": 4000, "step": "bfloat16"},
        # the 32-bit run, whose bits must not depend on how prompts are cut; a larger state, no gate
        {**scan, "name": "scan_float32", "channels": 2048, "requests": 3, "tokens": 700, "states": 32, "dtype": "float32", "gate": False},
        # what stands in front of a decode batch's scan, and of a prompt portion's, normed and plain
        {"name": "inputs_decode", "kind": "inputs", "rank": 224, "states": 16, "tokens": 64, "dtype": "bfloat16", "norms": True},
        {"name": "inputs_prompt", "kind": "inputs", "rank": 160, "states": 16, "tokens": 8191, "dtype": "bfloat16", "norms": True},
        # 256 experts in eight groups, four of which a token may use, eight experts a token: a decode batch and prompt portions
        {**route, "name": "route_decode", "experts": 256, "groups": 8, "kept": 4, "top": 8, "tokens": 24},
        {**route, "name": "route_prompt", "experts": 256, "groups": 8, "kept": 4, "top": 8, "tokens": 8192},
        # softmax scores, groups ranked by their best expert, weights as they are; sizes that are no powers of two
        {**route, "name": "route_softmax", "experts": 160, "groups": 8, "kept": 3, "top": 6, "tokens": 2047, "score": "softmax",
         "correction": False, "normalized": False, "best": 1},
    ]


def draw(rng):
    """One more case of the listed ones' ranges."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["tokens", "spans", "spans", "spans", "inputs", "route", "route"])
    if kind == "inputs":
        return {"kind": kind, "rank": rng.randint(16, 256), "states": rng.choice([8, 16, 16, 32, rng.randint(1, 64)]), "tokens": log_int(1, 8191),
                "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]), "norms": rng.random() < 0.7}
    if kind == "route":
        groups, size = rng.choice([1, 2, 4, 8, 8, 16]), rng.randint(3, 32)
        kept = rng.randint(1, groups)
        return {"kind": kind, "experts": groups * size, "groups": groups, "kept": kept, "top": rng.randint(1, min(16, kept * size)),
                "tokens": log_int(1, 8192), "score": rng.choice(["sigmoid", "sigmoid", "softmax"]), "correction": rng.random() < 0.7,
                "normalized": rng.random() < 0.6, "best": rng.randint(1, min(3, size))}
    states = rng.choice([16, 16, 16, 8, 32, rng.randint(1, 64)])
    channels = 64 * rng.randint(8, 112) if rng.random() < 0.75 else log_int(100, 7168)
    case = {"kind": "scan", "channels": channels, "states": states, "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]),
            "step": rng.choice(["float32", "float32", "bfloat16"]), "gate": rng.random() < 0.8, "skip": rng.random() < 0.8}
    if kind == "tokens":
        n = log_int(1, 64)
        return {**case, "requests": n, "tokens": n}
    n = rng.randint(1, 8)
    return {**case, "requests": n, "tokens": max(n, log_int(16, max(17, min(4000, MOST_WORK // (channels * states)))))}


# ------------------------------------------------------------------------------- what a case consists of
def _spans(case):
    """New tokens of every request: uneven shares, the same for every seed."""
    n, total = case["requests"], case["tokens"]
    r = random.Random(1000003 * n + total)
    weights = [r.uniform(0.05, 1.95) for _ in range(n)]
    extra = [int((total - n) * w / sum(weights)) for w in weights]
    extra[-1] += total - n - sum(extra)
    return [1 + e for e in extra]


def _step(case):
    """A step's arrays: where every request's tokens lie, and which slot its state is in."""
    spans = _spans(case)
    n = len(spans)
    cu = [sum(spans[:i]) for i in range(n + 1)]
    slots = random.Random(n).sample(range(n + 2), n)
    return types.SimpleNamespace(
        cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV), req_slot=torch.tensor(slots, dtype=torch.int32, device=DEV),
        token_req=torch.tensor([i for i, s in enumerate(spans) for _ in range(s)], dtype=torch.int32, device=DEV),
        spans=[(0, s) for s in spans], num_requests=n, num_tokens=cu[-1], max_span=max(spans), dtype=DTYPES[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    s = types.SimpleNamespace(case=dict(case))
    if case["kind"] == "route":
        s.z = 1.5 * randn(case["tokens"], case["experts"])
        s.correction = 0.1 * randn(case["experts"]) if case["correction"] else None
        return s
    dtype, T, N = DTYPES[case["dtype"]], case["tokens"], case["states"]
    if case["kind"] == "inputs":
        R = case["rank"]
        s.rows = randn(T, R + 2 * N)
        s.norms = tuple(1 + 0.1 * randn(n) for n in (R, N, N)) if case["norms"] else None
        return s
    C = case["channels"]
    s.plan = _step(case)
    # activated convolution output; the gate lies beside it in the wider rows of the input projection
    x = randn(T, C)
    s.x = (x * torch.sigmoid(x)).to(dtype)
    s.z = randn(T, 2 * C).to(dtype)[:, C:] if case["gate"] else None
    s.dt = (0.7 * randn(T, C)).to(DTYPES[case["step"]])
    s.bc = randn(T, 2 * N)
    # steps of 0.001 to 0.1 and rates of 1 to N: memories from a token to a thousand
    s.log_rate = torch.log(torch.arange(1, N + 1, device=DEV).float()).repeat(C, 1) + 0.05 * randn(C, N)
    s.bias = torch.log(torch.expm1(torch.exp(rand(C) * math.log(100.0) + math.log(0.001))))
    s.skip = 1 + 0.2 * randn(C) if case["skip"] else None
    s.state = 0.3 * randn(s.plan.num_requests + 2, C * N)
    return s


# ------------------------------------------------------------------------------- one pass
def _kernels():
    """The program's kernel table, made once."""
    if not _handle:
        from inferflux_b200.csrc import CudaKernels
        _handle.append(CudaKernels(DEV))
    return _handle[0]


def run(s):
    kind = s.case["kind"]
    if own:
        return {"scan": _own_scan, "inputs": _own_inputs, "route": _own_route}[kind](s)
    return {"scan": _plain_scan, "inputs": _plain_inputs, "route": _plain_route}[kind](s)


def _own_scan(s):
    y = _kernels().selective_scan(s.x, s.dt, s.bc, s.log_rate, s.state, s.plan, z=s.z, bias=s.bias, skip=s.skip, out_dtype=s.plan.dtype)
    return {"y": y, "state": s.state}


def _own_inputs(s):
    low, bc = _kernels().selective_inputs(s.rows, s.case["rank"], s.case["states"], out_dtype=DTYPES[s.case["dtype"]], norms=s.norms, eps=EPS)
    return {"low": low, "bc": bc}


def _own_route(s):
    c = s.case
    ids, weights = _kernels().moe_route_groups(s.z, s.correction, c["top"], c["groups"], c["kept"], best=c["best"], score=c["score"],
                                               normalized=c["normalized"], floor=1e-20, scale=2.5)
    return {"ids": ids, "weights": weights}


def _plain_scan(s):
    """The recurrence h <- a h + b of all tokens at once: after the round of distance d, b holds what the last 2 d tokens wrote and a how
    much of what was there before is left.  A span's first token takes the request's state, and keeps nothing of the span before it."""
    x, N, starts = s.x.float(), s.case["states"], s.plan.cu_seqlens[:-1].long()
    raw = s.dt.float() + s.bias
    dt = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    a = torch.exp(-dt[:, :, None] * torch.exp(s.log_rate))
    h = (dt * x)[:, :, None] * s.bc[:, None, :N]
    slots = s.plan.req_slot.long()
    h[starts] += a[starts] * s.state[slots].view(-1, *s.log_rate.shape)
    a[starts] = 0
    d = 1
    while d < s.plan.max_span:
        h[d:] += a[d:] * h[:-d]
        a[d:] *= a[:-d].clone()
        d *= 2
    s.state[slots] = h[s.plan.cu_seqlens[1:].long() - 1].flatten(1)
    y = (h * s.bc[:, None, N:]).sum(-1)
    if s.skip is not None:
        y = y + s.skip * x
    if s.z is not None:
        z = s.z.float()
        y = y * (z / (1 + torch.exp(-z)))
    return {"y": y.to(s.plan.dtype), "state": s.state}


def _plain_inputs(s):
    R, N = s.case["rank"], s.case["states"]
    parts = list(s.rows.split([R, N, N], 1))
    if s.norms is not None:
        parts = [p * torch.rsqrt(p.square().mean(1, keepdim=True) + EPS) * w for p, w in zip(parts, s.norms)]
    return {"low": parts[0].to(DTYPES[s.case["dtype"]], copy=True).contiguous(), "bc": torch.cat(parts[1:], 1)}


def _plain_route(s):
    """In 64 bits: which of two near scores is the larger must not depend on how the exponential is rounded."""
    c, z = s.case, s.z.double()
    if c["score"] == "sigmoid":
        scores = 1 / (1 + torch.exp(-z))
    else:
        e = torch.exp(z - z.amax(1, keepdim=True))
        scores = e / e.sum(1, keepdim=True)
    v = scores if s.correction is None else scores + s.correction.double()
    by_group = v.view(z.shape[0], c["groups"], -1)
    rank = by_group.sort(dim=2, descending=True).values[:, :, :c["best"]].sum(2)
    kept = torch.zeros_like(rank, dtype=torch.bool).scatter_(1, rank.sort(dim=1, descending=True, stable=True).indices[:, :c["kept"]], True)
    v = torch.where(kept[:, :, None], by_group, -math.inf).view_as(z)
    ids = v.sort(dim=1, descending=True, stable=True).indices[:, :c["top"]]
    w = scores.gather(1, ids)
    if c["normalized"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return {"ids": ids.int(), "weights": (2.5 * w).float()}


def work(case):
    T = case["tokens"]
    if case["kind"] == "route":
        n, top = case["experts"], case["top"]
        return {"bytes": 4 * T * n + 8 * T * top + (4 * n if case["correction"] else 0), "flops": T * n * (6 + top)}
    N, size = case["states"], DTYPES[case["dtype"]].itemsize
    if case["kind"] == "inputs":
        R = case["rank"]
        return {"bytes": T * (4 * (R + 2 * N) + size * R + 8 * N) + (4 * (R + 2 * N) if case["norms"] else 0), "flops": 4 * T * (R + 2 * N)}
    C = case["channels"]
    row = size * (3 if case["gate"] else 2) + DTYPES[case["step"]].itemsize       # x, gate, output; step
    vectors = 4 * C * (N + 1 + int(case["skip"]))
    return {"bytes": T * (C * row + 8 * N) + vectors + 8 * case["requests"] * C * N, "flops": T * C * (7 * N + 12)}


# ------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"scan": _exact_scan, "inputs": _exact_inputs, "route": _exact_route}[case["kind"]](s)


def _exact_scan(s):
    """Token after token, all requests side by side."""
    (C, N), spans = s.log_rate.shape, _spans(s.case)
    rate, state = s.log_rate.double().exp(), s.state.double()
    y = torch.empty(s.x.shape, dtype=torch.float64, device=DEV)
    slots, first = s.plan.req_slot.long(), s.plan.cu_seqlens.long()[:-1]
    length = torch.tensor(spans, device=DEV)
    h = state[slots].view(-1, C, N)
    order = sorted(set(spans))
    done = 0
    for until in order:                              # between two lengths the same requests are under way
        on = (length >= until).nonzero()[:, 0]
        at, mine = first[on], h[on]
        for t in range(done, until):
            rows = at + t
            step = torch.logaddexp(s.dt[rows].double() + s.bias.double(), torch.zeros((), dtype=torch.float64, device=DEV))
            x, b, c = s.x[rows].double(), s.bc[rows, :N].double(), s.bc[rows, N:].double()
            mine = mine * torch.exp(step.unsqueeze(2) * -rate) + (step * x).unsqueeze(2) * b.unsqueeze(1)
            out = torch.einsum("rcn,rn->rc", mine, c)
            if s.skip is not None:
                out = out + x * s.skip.double()
            if s.z is not None:
                gate = s.z[rows].double()
                out = out * gate * torch.sigmoid(gate)
            y[rows] = out
        h[on] = mine
        done = until
    state[slots] = h.flatten(1)
    return {"y": y, "state": state}


def _exact_inputs(s):
    R, N = s.case["rank"], s.case["states"]
    rows = s.rows.double()
    if s.norms is not None:
        at = 0
        for w in s.norms:
            part = rows[:, at:at + len(w)]
            part.mul_(w.double() / (part.pow(2).sum(1, keepdim=True) / len(w) + EPS).sqrt())
            at += len(w)
    return {"low": rows[:, :R], "bc": rows[:, R:]}


def _exact_route(s):
    """By counting: an expert's place is the number of experts that stand before it."""
    c, n, size = s.case, s.case["experts"], s.case["experts"] // s.case["groups"]

    def place(v):
        i = torch.arange(v.shape[-1], device=DEV)
        before = (v.unsqueeze(-2) > v.unsqueeze(-1)) | ((v.unsqueeze(-2) == v.unsqueeze(-1)) & (i < i.unsqueeze(1)))
        return before.sum(-1)

    ids, weights = [], []
    for z in s.z.double().split(512):
        score = torch.sigmoid(z) if c["score"] == "sigmoid" else torch.softmax(z, 1)
        v = score if s.correction is None else score + s.correction.double()
        grouped = v.unflatten(1, (c["groups"], size))
        strength = torch.where(place(grouped) < c["best"], grouped, 0.0).sum(2)
        kept = (place(strength) < c["kept"]).repeat_interleave(size, 1)
        at = place(torch.where(kept, v, -math.inf))
        chosen = torch.zeros(len(z), n, dtype=torch.long, device=DEV).scatter_(1, at, torch.arange(n, device=DEV).expand(len(z), n))[:, :c["top"]]
        w = score.gather(1, chosen)
        ids.append(chosen.int())
        weights.append(2.5 * (w / (w.sum(1, keepdim=True) + 1e-20) if c["normalized"] else w))
    return {"ids": torch.cat(ids), "weights": torch.cat(weights)}
