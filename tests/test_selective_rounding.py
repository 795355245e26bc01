"""Models of selective state space layers and experts by groups in bfloat16, every row held: with all experts chosen nothing is decided by a margin,
so what a correct run is off by is rounding alone, and the same run on the plain kernels says how much that is."""
import copy

import numpy as np
import pytest
import torch

import helpers
import selective_models as sm
from plain.plain_kernels import PlainKernels

LENS = [40, 3, 97, 1, 400, 290]                 # (spans of 256 and more go by stretches)
BF16 = torch.bfloat16
_plan = sm.plan


def _every_expert(which):
    """The plan, with every group kept and every expert chosen: what their scores are is in the weights alone."""
    plan = copy.deepcopy(_plan(which))
    for layer in plan.layers:
        p = layer.ffn.params
        p["top"], p["groups"]["kept"] = p["num_experts"], p["groups"]["count"]
    return plan


def _requests():
    return {f"r{i}": helpers.random_tokens(sm.V, n, 900 + i) for i, n in enumerate(LENS)}


def _runner(model, kernels):
    from inferflux_b200.engine import ModelRunner
    return ModelRunner(model, kernels, page_size=sm.PAGE, num_pages=1024 // sm.PAGE, max_seqs=8, max_seq_len=512)


def _rows(model, kernels, steps):
    return helpers.collect(steps, helpers.run_steps_in_process(_runner(model, kernels), steps), sm.V)


def _yard(which, requests):
    """(exact logits of the rounded weights, how far the plain kernels' bfloat16 run is off: a request's rows, each by its worst logit)."""
    model, W = sm.made(which, BF16, "cpu")
    want = {r: sm.logits(which, W, t).numpy() for r, t in requests.items()}
    got = _rows(model, PlainKernels(wide=True), helpers.trace_whole(requests))
    return want, {r: np.abs(got[r] - want[r]).max(axis=1) for r in want}


def _held(got, want, yard):
    """Two correct runs round at about the same stages and differ in which of two neighbours a number near the middle goes to, and in the order of sums:
    each is off by about as much as the other.  Every row within three times the yard's worst row, and on average within twice the yard's, as the other
    designs' bfloat16 models are held, without a row left out."""
    off = {r: np.abs(got[r] - want[r]).max(axis=1) for r in want}
    worst = max(float(y.max()) for y in yard.values())
    for r, o in off.items():
        assert bool(np.isfinite(got[r]).all()) and float(o.max()) <= 3.0 * worst, (r, int(o.argmax()), float(o.max()), worst)
    mean, yard_mean = (float(np.concatenate(list(d.values())).mean()) for d in (off, yard))
    assert mean <= 2.0 * yard_mean, (mean, yard_mean)


@pytest.fixture()
def every_expert(monkeypatch):
    monkeypatch.setattr(sm, "plan", _every_expert)


class _Forgetful(PlainKernels):
    """What a run would give whose spans of 256 tokens and more forget their first 256 tokens' state."""

    def selective_scan(self, x, dt, bc, log_rate, state, ctx, z=None, **kw):
        y = super().selective_scan(x, dt, bc, log_rate, state, ctx, z=z, **kw)
        cu = ctx.cu_seqlens.tolist()
        for r in range(ctx.num_requests):
            if cu[r + 1] - cu[r] >= 256:
                rest, one, slot = slice(cu[r] + 256, cu[r + 1]), copy.copy(ctx), int(ctx.req_slot[r])
                one.cu_seqlens, one.req_slot, one.num_requests = torch.tensor([0, rest.stop - rest.start], dtype=torch.int32), ctx.req_slot[r:r + 1], 1
                state[slot] = 0
                y[rest] = super().selective_scan(x[rest], dt[rest], bc[rest], log_rate, state, one, z=z[rest], **kw)
        return y


@pytest.mark.parametrize("which", ["groups", "softmax"])
def test_the_bound_sees_a_lost_state(every_expert, which):
    """On the plain kernels (no GPU): the bounds hold for a run cut otherwise, and not where spans forget what was in front of them."""
    reqs = _requests()
    want, yard = _yard(which, reqs)
    model, _ = sm.made(which, BF16, "cpu")
    _held(_rows(model, PlainKernels(), helpers.trace_portions(reqs)), want, yard)
    with pytest.raises(AssertionError):
        _held(_rows(model, _Forgetful(wide=True), helpers.trace_whole(reqs)), want, yard)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["groups", "softmax"])
def test_every_row_of_every_cutting(cuda_kernels, every_expert, which):
    reqs = _requests()
    want, yard = _yard(which, reqs)
    model, _ = sm.made(which, BF16, "cuda:0")
    inner, states = (96, 5) if which == "softmax" else (128, 16)
    assert cuda_kernels.lib.ifx_selective_scan_scratch(1, max(LENS), inner, states) > 0     # whole prompts go by stretches
    for make in (helpers.trace_whole, helpers.trace_tail, helpers.trace_portions, lambda r: helpers.trace_mixed(r, 1024)):
        steps = make(reqs)
        _held(_rows(model, cuda_kernels, steps), want, yard)
