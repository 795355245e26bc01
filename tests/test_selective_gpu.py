"""The selective state space scan and its inputs against their statement in 64 bits, with bounds that are carried along the recurrence."""
import math
from types import SimpleNamespace

import pytest
import torch

from plain.plain_kernels import PlainKernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64
U = 2.0 ** -24                      # half a step of float32, relative


def _ctx(lens, slots=None, dtype=F32):
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    slots = list(range(len(lens))) if slots is None else slots
    return SimpleNamespace(cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV), req_slot=torch.tensor(slots, dtype=torch.int32, device=DEV),
                           spans=[(0, n) for n in lens], num_requests=len(lens), num_tokens=cu[-1], max_span=max(lens, default=0), dtype=dtype,
                           token_req=torch.tensor([r for r, n in enumerate(lens) for _ in range(n)], dtype=torch.int32, device=DEV))


def _data(T, C, N, slots, dtype=F32, step=F32, seed=0, off=0, pad=0):
    """Operands as columns of wider rows (`off` the first one), a state whose rows are `pad` floats longer than they need be."""
    g = torch.Generator().manual_seed(seed + 131 * T + 17 * C + N)
    wide = torch.randn(T, 2 * C + off, generator=g).to(dtype).to(DEV)
    d = SimpleNamespace(
        x=wide[:, off:off + C], z=wide[:, off + C:], dt=(0.7 * torch.randn(T, C + off, generator=g)).to(step).to(DEV)[:, off:],
        bc=torch.randn(T, 2 * N + off, generator=g).to(DEV)[:, off:],
        log_rate=(torch.rand(C, N, generator=g) * math.log(16.0)).to(DEV), bias=(torch.rand(C, generator=g) * 5 - 6.5).to(DEV),
        skip=(1 + 0.2 * torch.randn(C, generator=g)).to(DEV), state=0.5 * torch.randn(slots, C * N + pad, generator=g).to(DEV))
    return d


def _oracle(d, ctx, z, bias, skip):
    """(y, state, how far y and the state may be off) in 64 bits.

    Relative errors of a step, in halves of a float32 step U: the argument v of softplus is rounded once and its exponential's argument and
    result a few times (|v| + 8) 4; the rate (an exponential of a log_rate up to 3, times log2 e) 16; a product of the two, 2; the exponential of the
    decay 4 (two steps) and its argument's error times |argument|; h's multiply-add and the two products of what is written, 3 and the step's own."""
    C, N = d.log_rate.shape
    x, state = d.x.double(), d.state.double()
    v = d.dt.double() + (0 if bias is None else bias.double())
    step = torch.logaddexp(v, torch.zeros_like(v))
    e_step = 4 * (v.abs() + 8) * U
    rate = d.log_rate.double().exp()
    y, off = torch.zeros(*x.shape, dtype=F64, device=DEV), torch.zeros(*x.shape, dtype=F64, device=DEV)
    s_off = torch.zeros_like(state)
    cu, slots = ctx.cu_seqlens.tolist(), ctx.req_slot.tolist()
    for r in range(ctx.num_requests):
        h = state[slots[r], :C * N].view(C, N).clone()
        e = torch.zeros_like(h)
        for t in range(cu[r], cu[r + 1]):
            arg = step[t][:, None] * rate
            a = torch.exp(-arg)
            w = (step[t] * x[t])[:, None] * d.bc[t, :N].double()
            e = a * e + a * h.abs() * (arg * (e_step[t][:, None] + 18 * U) + 4 * U) + w.abs() * (e_step[t][:, None] + 3 * U)
            h = a * h + w
            e = e + 2 * U * h.abs()
            terms = h * d.bc[t, N:].double()
            y[t] = terms.sum(1)
            off[t] = (e * d.bc[t, N:].double().abs()).sum(1) + terms.abs().sum(1) * (math.ceil(math.log2(N + 1)) + 2) * U
        state[slots[r], :C * N] = h.flatten()
        s_off[slots[r], :C * N] = e.flatten()
    if skip is not None:
        y = y + skip.double() * x
        off = off + 2 * U * (y.abs() + (skip.double() * x).abs())
    if z is not None:
        gate = z.double() * torch.sigmoid(z.double())
        off = off * gate.abs() + (y * gate).abs() * 4 * (z.double().abs() + 8) * U
        y = y * gate
    return y, state, off, s_off


def _check(k, d, ctx, z=True, bias=True, skip=True, out_dtype=None):
    z, bias, skip = (d.z if z else None), (d.bias if bias else None), (d.skip if skip else None)
    want, want_state, off, s_off = _oracle(d, ctx, z, bias, skip)
    n = int(ctx.cu_seqlens[-1])
    got = k.selective_scan(d.x, d.dt, d.bc, d.log_rate, d.state, ctx, z=z, bias=bias, skip=skip, out_dtype=out_dtype)
    out_dtype = out_dtype or d.x.dtype
    assert got.dtype == out_dtype and got.shape == d.x.shape
    bound = off[:n] + (want[:n].abs() + off[:n]) * torch.finfo(out_dtype).eps / 2 + 1e-38
    assert bool(((got[:n].double() - want[:n]).abs() <= bound).all()), float(((got[:n].double() - want[:n]).abs() / bound).max())
    s_bound = s_off * 1.001 + 1e-38
    assert bool(((d.state.double() - want_state).abs() <= s_bound).all()), float(((d.state.double() - want_state).abs() / s_bound).max())
    return got


LENS = [(1,), (1, 1, 1, 1, 1), (3, 0, 1, 5), (33, 1, 64, 65), (0, 0), (130,), (31, 32, 2)]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("C,N", [(1, 1), (5, 3), (33, 16), (200, 16), (96, 64), (129, 5), (40, 128), (64, 100)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan(cuda_kernels, lens, C, N, dtype):
    ctx = _ctx(lens, slots=[(3 * i + 1) % (len(lens) + 3) for i in range(len(lens))] if len(lens) != 3 else None, dtype=dtype)
    slots = len(lens) + 3
    assert len(set(ctx.req_slot.tolist())) == len(lens)
    d = _data(sum(lens), C, N, slots, dtype, pad=7 if C % 2 else 0)
    _check(cuda_kernels, d, ctx)


@pytest.mark.parametrize("dtype,step,out", [(BF16, BF16, BF16), (BF16, F32, F32), (F32, BF16, F32), (F32, F32, BF16), (BF16, BF16, F32)])
@pytest.mark.parametrize("off", [0, 1, 4, 8])
@pytest.mark.parametrize("z,bias,skip", [(True, True, True), (False, True, True), (True, False, False), (False, False, False)])
def test_scan_types_strides_options(cuda_kernels, dtype, step, out, off, z, bias, skip):
    for C, N, lens in ((48, 16, (70, 1, 3)), (130, 8, (1, 1)), (64, 32, (200,))):
        _check(cuda_kernels, _data(sum(lens), C, N, len(lens), dtype, step, off=off), _ctx(lens, dtype=dtype), z=z, bias=bias, skip=skip, out_dtype=out)


def test_scan_many_requests_and_wide_rows(cuda_kernels):
    lens = [1 + (i * 7) % 5 for i in range(300)]
    _check(cuda_kernels, _data(sum(lens), 64, 16, 300, BF16), _ctx(lens, slots=list(reversed(range(300))), dtype=BF16))
    _check(cuda_kernels, _data(3, 7168, 16, 3, BF16), _ctx((1, 1, 1), dtype=BF16))
    _check(cuda_kernels, _data(90, 5120, 16, 2, BF16), _ctx((40, 50), dtype=BF16))


def test_scan_long_and_few_channels(cuda_kernels):
    """What a bfloat16 run's long spans of few channels do, and a float32 run's."""
    for dtype, lens in ((BF16, (1100,)), (F32, (1100,)), (BF16, (700, 1, 300, 128, 129))):
        _check(cuda_kernels, _data(sum(lens), 48, 16, len(lens), dtype), _ctx(lens, dtype=dtype))


def test_rows_behind_the_last_request(cuda_kernels):
    """Rows that no request has are not read into any state."""
    lens = (5, 0, 9)
    d, ctx = _data(30, 40, 16, 4), _ctx(lens, slots=[3, 0, 1])
    d.x[14:] = math.nan
    d.dt[14:] = math.inf
    d.bc[14:] = math.nan
    before = d.state.clone()
    _check(cuda_kernels, d, ctx)
    assert torch.equal(d.state[0], before[0]) and torch.equal(d.state[2], before[2])


@pytest.mark.parametrize("C,N", [(72, 16), (30, 5), (16, 64)])
def test_float32_bits_do_not_depend_on_the_cut(cuda_kernels, C, N):
    T = 333
    one = _data(T, C, N, 2)
    cut = SimpleNamespace(**vars(one))
    cut.state = one.state.clone()
    y = cuda_kernels.selective_scan(one.x, one.dt, one.bc, one.log_rate, one.state, _ctx((T,)), z=one.z, bias=one.bias, skip=one.skip)
    at, parts = 0, []
    for n in (1, 64, 1, 1, 130, 33, 100, 3):
        s = slice(at, at + n)
        parts.append(cuda_kernels.selective_scan(cut.x[s], cut.dt[s], cut.bc[s], cut.log_rate, cut.state, _ctx((n,)), z=cut.z[s], bias=cut.bias,
                                                 skip=cut.skip))
        at += n
    assert at == T and torch.equal(torch.cat(parts), y) and torch.equal(cut.state, one.state)
    beside = _data(T, C, N, 2)                             # the same request beside another one
    both = SimpleNamespace(**{n: torch.cat([getattr(beside, n)[:50], getattr(beside, n)]) for n in ("x", "z", "dt", "bc")})
    got = cuda_kernels.selective_scan(both.x, both.dt, both.bc, beside.log_rate, beside.state, _ctx((50, T), slots=[1, 0]), z=both.z, bias=beside.bias,
                                      skip=beside.skip)
    assert torch.equal(got[50:], y) and torch.equal(beside.state[0], one.state[0])


def test_scan_extreme_values(cuda_kernels):
    """Steps from nothing to a state's end, gates far out, rates of zero and beyond: as the formula has it, and nothing spreads to others."""
    lens = (6, 40)
    d, ctx = _data(46, 35, 6, 2), _ctx(lens)
    d.dt[:, 0], d.dt[:, 1], d.dt[:, 2] = -200.0, 90.0, -20.0
    d.log_rate[3], d.log_rate[4] = -math.inf, 40.0
    d.z[:, 5], d.z[:, 6] = -300.0, 300.0
    d.z[:, 7] = -math.inf                                   # silu's limit there is 0, its formula's value -inf * 0
    d.x[:, 8], d.x[2, 9], d.dt[3, 10] = 0.0, math.inf, math.nan
    state = d.state.clone()
    want, _, off, _ = _oracle(d, ctx, d.z, d.bias, d.skip)
    y = cuda_kernels.selective_scan(d.x, d.dt, d.bc, d.log_rate, d.state, ctx, z=d.z, bias=d.bias, skip=d.skip)
    plain = [c for c in range(35) if c not in (7, 9, 10, 1, 4)]
    err = (y.double() - want).abs()[:, plain]
    assert bool((err <= off[:, plain] + want[:, plain].abs() * U + 1e-38).all())
    assert bool(torch.isfinite(y[:, [1, 4]]).all())
    near = (y.double() - want).abs()[:, [1, 4]] <= 1e-4 * want[:, [1, 4]].abs() + 1e-6      # arguments of thousands: what is left is 0 either way
    assert bool(near.all())
    assert bool((~torch.isfinite(y[2:6, 9])).all()) and bool(torch.isfinite(y[6:, 9]).all())
    assert bool(y[3:6, 10].isnan().all()) and bool(torch.isfinite(y[6:, 10]).all())
    assert torch.equal(d.state.view(2, 35, 6)[:, 0], state.view(2, 35, 6)[:, 0])       # no step, no change


def test_an_infinity_does_not_become_another(cuda_kernels):
    """States that are there only to fill a lane up add nothing, not even to an infinity."""
    d, ctx = _data(3, 4, 5, 1), _ctx((3,))
    d.x[:] = math.inf
    d.bc[:] = 1.0
    y = cuda_kernels.selective_scan(d.x, d.dt, d.bc, d.log_rate, d.state, ctx)
    assert bool((y == math.inf).all())


def test_two_streams_and_a_captured_graph(cuda_kernels):
    lens = (140, 1, 20)
    a, b = _data(161, 64, 16, 3, BF16, seed=1), _data(161, 64, 16, 3, BF16, seed=2)
    ctx = _ctx(lens, dtype=BF16)

    def scan(d, state):
        return cuda_kernels.selective_scan(d.x, d.dt, d.bc, d.log_rate, state, ctx, z=d.z, bias=d.bias, skip=d.skip)
    sa, sb = a.state.clone(), b.state.clone()
    want = scan(a, sa), scan(b, sb)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    ta, tb = a.state.clone(), b.state.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gb = scan(b, tb)
    ga = scan(a, ta)
    torch.cuda.synchronize()
    assert torch.equal(ga, want[0]) and torch.equal(gb, want[1]) and torch.equal(ta, sa) and torch.equal(tb, sb)
    graphs, outs, states = [], [], [a.state.clone(), b.state.clone()]
    for d, st in zip((a, b), states):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(scan(d, st))
        graphs.append(g)
    for _ in range(2):                                      # replayed twice, one behind the other
        for st, d in zip(states, (a, b)):
            st.copy_(d.state)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(states[0], sa) and torch.equal(states[1], sb)


@pytest.mark.parametrize("T,rank,N", [(1, 1, 1), (3, 224, 16), (65, 160, 16), (300, 48, 8), (2, 8192, 128), (7, 33, 5), (1000, 64, 64), (130, 100, 3)])
@pytest.mark.parametrize("dtype,out", [(F32, BF16), (F32, F32), (BF16, BF16)])
@pytest.mark.parametrize("which", [(1, 1, 1), (0, 0, 0), (1, 0, 1), None])
def test_inputs(cuda_kernels, T, rank, N, dtype, out, which):
    g = torch.Generator().manual_seed(T + rank)
    wide = (2 * torch.randn(T, rank + 2 * N + 3, generator=g)).to(dtype)
    norms = None if which is None else tuple((1 + 0.3 * torch.randn(n, generator=g)) if w else None for w, n in zip(which, (rank, N, N)))
    on = None if norms is None else tuple(None if w is None else w.to(DEV) for w in norms)
    for rows in (wide[:, :rank + 2 * N].contiguous(), wide[:, 1:1 + rank + 2 * N], wide):
        want = PlainKernels(wide=True)
        want.acc = F64
        low, bc = want.selective_inputs(rows, rank, N, F64, norms, 1e-6)
        placed = wide.to(DEV)[:, 1:1 + rank + 2 * N] if rows.storage_offset() else rows.to(DEV)
        got_low, got_bc = cuda_kernels.selective_inputs(placed, rank, N, out, on, 1e-6)
        assert got_low.dtype == out and got_bc.dtype == F32
        # a sum of n squares by 32 lanes and a tree, its root, two products; then the result's own rounding
        for got, ref, n, normed in ((got_low, low, rank, which and which[0]), (got_bc[:, :N], bc[:, :N], N, which and which[1]),
                                    (got_bc[:, N:], bc[:, N:], N, which and which[2])):
            rel = ((n / 32 + 8) / 2 + 6) * U if normed else 0.0
            tol = ref.abs().double() * (rel + torch.finfo(got.dtype).eps / 2 * (1 + rel)) + (U * ref.abs().double() if got is not got_low else 0)
            assert bool(((got.double().cpu() - ref.double()).abs() <= tol + 1e-38).all())


def test_inputs_from_slices(cuda_kernels):
    """K slices of a product are added in their order first."""
    from inferflux_b200.csrc.ops import PartialSum
    g = torch.Generator().manual_seed(5)
    parts = torch.randn(3, 40, 96, generator=g).to(DEV)
    total = parts[0] + parts[1] + parts[2]
    norms = tuple(1 + 0.1 * torch.randn(n, generator=g).to(DEV) for n in (64, 16, 16))
    for got, want in zip(cuda_kernels.selective_inputs(PartialSum(parts, BF16), 64, 16, BF16, norms, 1e-5),
                         cuda_kernels.selective_inputs(total, 64, 16, BF16, norms, 1e-5)):
        assert torch.equal(got, want)


def test_nothing_to_do(cuda_kernels):
    d = _data(0, 16, 4, 2)
    before = d.state.clone()
    assert cuda_kernels.selective_scan(d.x, d.dt, d.bc, d.log_rate, d.state, _ctx(())).shape == (0, 16)
    assert cuda_kernels.selective_scan(d.x, d.dt, d.bc, d.log_rate, d.state, _ctx((0, 0))).shape == (0, 16)
    low, bc = cuda_kernels.selective_inputs(torch.empty(0, 24, device=DEV), 16, 4, F32)
    assert low.shape == (0, 16) and bc.shape == (0, 8) and torch.equal(d.state, before)


def test_stretches_on_two_streams_and_in_two_graphs(cuda_kernels):
    """Long spans of few channels go through scratch of their own in every call, captured or not."""
    lens = (900, 1, 300)
    ctx = _ctx(lens, dtype=BF16)
    data = [_data(sum(lens), 64, 16, 3, BF16, seed=s) for s in (5, 6)]
    assert cuda_kernels.lib.ifx_selective_scan_scratch(3, 900, 64, 16) > 0

    def scan(d, state):
        return cuda_kernels.selective_scan(d.x, d.dt, d.bc, d.log_rate, state, ctx, z=d.z, bias=d.bias, skip=d.skip)
    states = [d.state.clone() for d in data]
    want = [scan(d, s) for d, s in zip(data, states)]
    torch.cuda.synchronize()
    again, got, streams = [d.state.clone() for d in data], [None, None], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        streams[i].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i]):
            got[i] = scan(data[i], again[i])
    torch.cuda.synchronize()
    graphs, outs, held = [], [], [d.state.clone() for d in data]
    for d, s in zip(data, held):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(scan(d, s))
        graphs.append(g)
    for d, s in zip(data, held):
        s.copy_(d.state)
    torch.cuda.synchronize()
    for i in range(2):                                      # at the same time
        with torch.cuda.stream(streams[i]):
            graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i], want[i]) and torch.equal(again[i], states[i])
        assert torch.equal(outs[i], want[i]) and torch.equal(held[i], states[i])


def test_stretches_meet_the_walk(cuda_kernels):
    """A span by stretches and the same one walked whole (its scratch left out by the switch): as near as both are to 64 bits."""
    for lens, C, N in (((1500,), 72, 16), ((257,), 130, 8), ((640, 2, 256, 31), 33, 5), ((1024, 512), 16, 64)):
        ctx, d = _ctx(lens, dtype=BF16), _data(sum(lens), C, N, len(lens), BF16)
        assert cuda_kernels.lib.ifx_selective_scan_scratch(len(lens), max(lens), C, N) > 0
        state = d.state.clone()
        _check(cuda_kernels, d, ctx, out_dtype=BF16)
        d.state.copy_(state)
        cuda_kernels.chunk_scans = False
        try:
            _check(cuda_kernels, d, ctx, out_dtype=BF16)
        finally:
            cuda_kernels.chunk_scans = True
