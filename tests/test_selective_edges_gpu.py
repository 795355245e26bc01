"""The selective state space scan at the ends of its range: rates beyond float32's, whatever a span's length and however it is cut."""
import math
from types import SimpleNamespace

import pytest
import torch

from test_selective_gpu import BF16, DEV, F32, _ctx, _data, _oracle

pytestmark = pytest.mark.gpu
FAST = [89.0, 200.0, math.inf]         # of log_rate: e^88.7 is float32's largest number


def _with_fast_rates(lens, C, N, dtype, seed=0):
    """Operands of which two thirds of the channels have rates beyond float32 at every state number, at some, or at the last one."""
    d = _data(sum(lens), C, N, len(lens), dtype, seed=seed)
    for c in range(C):
        if c % 6 in (0, 1, 2):
            d.log_rate[c] = FAST[c % 3]
        elif c % 6 == 3:
            d.log_rate[c, N - 1] = FAST[c // 6 % 3]
    return d


def _want(d, ctx):
    """The steps here are above e^-10, so that every decay e^(-step e^60) is 0 in 64 bits as it is with the rates themselves: with those as they are,
    the oracle's own bound would have zero times infinity."""
    near = SimpleNamespace(**vars(d))
    near.log_rate, near.state = d.log_rate.clamp(max=60.0), d.state.clone()
    assert float(torch.nn.functional.softplus(d.dt.double() + d.bias.double()).min()) > math.exp(-10)
    return _oracle(near, ctx, d.z, d.bias, d.skip)


def _scan(k, d, ctx):
    return k.selective_scan(d.x, d.dt, d.bc, d.log_rate, d.state, ctx, z=d.z, bias=d.bias, skip=d.skip)


def _holds(y, state, want):
    y64, state64, off, s_off = want
    assert bool(torch.isfinite(state).all())
    assert bool(((y.double() - y64).abs() <= off + (y64.abs() + off) * torch.finfo(y.dtype).eps / 2 + 1e-38).all())
    assert bool(((state.double() - state64).abs() <= s_off * 1.001 + 1e-38).all())


@pytest.mark.parametrize("lens", [(1,), (2,), (3,), (33,), (257,), (1, 1, 1), (5, 0, 31, 4), (257, 3, 300)])
@pytest.mark.parametrize("C,N", [(48, 16), (24, 4), (37, 5), (30, 40)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rates_beyond_float32(cuda_kernels, lens, C, N, dtype):
    """A decay of 0, in tokens that are there; those that fill up a pair or a group of four change nothing.  bfloat16: spans of 257 and more go by
    stretches, and whole."""
    ctx, d = _ctx(lens, dtype=dtype), _with_fast_rates(lens, C, N, dtype)
    want, state = _want(d, ctx), d.state.clone()
    _holds(_scan(cuda_kernels, d, ctx), d.state, want)
    if dtype == BF16 and max(lens) > 256:
        assert cuda_kernels.lib.ifx_selective_scan_scratch(len(lens), max(lens), C, N) > 0
        d.state.copy_(state)
        cuda_kernels.chunk_scans = False
        try:
            _holds(_scan(cuda_kernels, d, ctx), d.state, want)
        finally:
            cuda_kernels.chunk_scans = True


@pytest.mark.parametrize("C,N", [(48, 16), (37, 5)])
def test_cuts_with_rates_beyond_float32(cuda_kernels, C, N):
    """float32 bits do not depend on the cut there either."""
    T = 101
    one = _with_fast_rates((T,), C, N, F32, seed=2)
    cut = SimpleNamespace(**vars(one))
    cut.state = one.state.clone()
    y, at = _scan(cuda_kernels, one, _ctx((T,))), 0
    for n in (1, 3, 33, 2, 1, 31, 30):
        s = slice(at, at + n)
        got = cuda_kernels.selective_scan(cut.x[s], cut.dt[s], cut.bc[s], cut.log_rate, cut.state, _ctx((n,)), z=cut.z[s], bias=cut.bias, skip=cut.skip)
        assert torch.equal(got, y[s])
        at += n
    assert at == T and torch.equal(cut.state, one.state)


@pytest.mark.parametrize("lens", [(1,), (3,), (4,), (257,)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_rate_that_is_no_number(cuda_kernels, lens, dtype):
    """It makes its own state no number and its own channel's output, and nothing else."""
    d, ctx = _data(sum(lens), 40, 16, 1, dtype), _ctx(lens, dtype=dtype)
    d.log_rate[7, 3] = math.nan
    rest = SimpleNamespace(**vars(d))
    rest.log_rate, rest.state = torch.where(d.log_rate.isnan(), 0.0, d.log_rate), d.state.clone()
    want_y, want_state = _scan(cuda_kernels, rest, ctx), rest.state
    y = _scan(cuda_kernels, d, ctx)
    others = torch.arange(40, device=DEV) != 7
    assert bool(y[:, 7].isnan().all()) and torch.equal(y[:, others], want_y[:, others])
    bad = d.state.view(40, 16).isnan()
    assert bool(bad[7, 3]) and int(bad.sum()) == 1
    assert torch.equal(d.state.view(40, 16)[~bad], want_state.view(40, 16)[~bad])


def _few(k, v, z=None, dtype=F32):
    """The steps of v [T, C] (times their gates) as the scan gives them: a state of one number from 0, with x, B and C of 1, is the step, in the
    single-token kernel and in the other one (which a longest span of two tokens stands for)."""
    T, C = v.shape
    one, bc, rate = torch.ones(T, C, device=DEV, dtype=dtype), torch.ones(T, 2, device=DEV), torch.full((C, 1), math.inf, device=DEV)
    ctx, got = _ctx((1,) * T), []
    for ctx.max_span in (1, 2):
        got.append(k.selective_scan(one, v, bc, rate, torch.zeros(T, C, device=DEV), ctx, z=z, out_dtype=F32))
    assert torch.equal(got[0].isnan(), got[1].isnan()) and torch.equal(got[0].nan_to_num(), got[1].nan_to_num())
    return got[0]


@pytest.mark.parametrize("lo,hi", [(-85, -20), (-20, -9), (-9, 2), (2, 40)])
def test_steps_and_gates_to_a_few_float32_steps(cuda_kernels, lo, hi):
    """In halves of a float32 step: the exponential unit 4, what its argument's rounding left out 1; s = e / (2 + e) 1 + 2 + 1 more; the polynomial
    1, its coefficients 1, what s does to it 1; the last multiply-add 1: 13 at most for a step.  A gate: 5 for the exponential, 1 + 2 for the quotient,
    2 for products, and 1 for the output's: 11."""
    v = (lo + (hi - lo) * torch.rand(40, 1000, generator=torch.Generator().manual_seed(hi))).to(DEV)
    step = _few(cuda_kernels, v)
    want = torch.logaddexp(v.double(), torch.zeros((), dtype=torch.float64, device=DEV))
    assert float((step.double() / want - 1).abs().max()) <= 13 * 2.0 ** -24
    ones = torch.zeros_like(v)
    gated, plain = _few(cuda_kernels, ones, z=v), _few(cuda_kernels, ones)
    want = plain.double() * v.double() * torch.sigmoid(v.double())
    assert float((gated.double() - want).abs().div(want.abs()).max()) <= 11 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps_and_gates_far_out(cuda_kernels, dtype):
    """No step below e^-88, the argument itself above; gates of 0 and of z; what is no number stays none."""
    v = torch.tensor([-math.inf, -1000.0, -104.5, 50.0, 1e30, math.nan], device=DEV)[None].repeat(4, 1)
    step = _few(cuda_kernels, v)
    assert bool((step[:, :3] == 0).all()) and torch.equal(step[:, 3:5], v[:, 3:5]) and bool(step[:, 5].isnan().all())
    z = torch.tensor([-3e38, -1000.0, -104.5, 0.0, 50.0, 1e30, math.nan], device=DEV)[None].repeat(4, 1).to(dtype)
    ones = torch.zeros(4, 7, device=DEV)
    plain, gated = _few(cuda_kernels, ones, dtype=dtype), _few(cuda_kernels, ones, z=z, dtype=dtype)
    assert bool((gated[:, :4] == 0).all()) and torch.equal(gated[:, 4:6], (plain * z.float())[:, 4:6]) and bool(gated[:, 6].isnan().all())
