"""The selective scan's single-token kernel as decode batches run it (two requests a thread from 12 on), and state sizes of every number of lanes."""
from types import SimpleNamespace

import pytest
import torch

from test_selective_gpu import BF16, F32, _check, _ctx, _data

pytestmark = pytest.mark.gpu
EVERY_OTHER = (1, 0) * 9 + (1,)


def _spread(n):
    """Slots in another order than the requests, with some left free."""
    return [(5 * i + 3) % (n + 4) for i in range(n)] if (n + 4) % 5 else [(3 * i + 1) % (n + 4) for i in range(n)]


def _idle_slots_stay(before, state, ctx, lens):
    idle = set(range(len(before))) - {s for s, n in zip(ctx.req_slot.tolist(), lens) if n}
    assert all(torch.equal(before[i], state[i]) for i in idle)


@pytest.mark.parametrize("lens", [(1,) * 12, (1,) * 13, (1,) * 65, EVERY_OTHER, (0, 0) * 5 + (1, 0, 0, 1), (0,) * 12 + (1,), (1, 0, 1)])
@pytest.mark.parametrize("C,N", [(70, 4), (33, 5), (64, 8), (50, 12), (72, 16), (41, 32), (20, 40), (12, 64), (9, 100), (5, 128)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_single_tokens(cuda_kernels, lens, C, N, dtype):
    """An odd last request, requests without a token inside a pair, channels that do not fill a block, slots in any order; the slots of those
    that have no token, and of none, stay as they are."""
    slots = _spread(len(lens))
    assert len(set(slots)) == len(lens)
    ctx, d = _ctx(lens, slots=slots, dtype=dtype), _data(sum(lens), C, N, len(lens) + 4, dtype, pad=5 if C % 2 else 0)
    assert ctx.max_span == 1
    before = d.state.clone()
    _check(cuda_kernels, d, ctx)
    _idle_slots_stay(before, d.state, ctx, lens)


@pytest.mark.parametrize("dtype,step,out", [(BF16, F32, BF16), (BF16, BF16, F32), (F32, BF16, BF16)])
@pytest.mark.parametrize("off", [0, 1, 4])
@pytest.mark.parametrize("z,bias,skip", [(True, True, True), (False, True, False), (True, False, True), (False, False, False)])
def test_single_tokens_types_strides_options(cuda_kernels, dtype, step, out, off, z, bias, skip):
    for C, N, R in ((136, 16, 24), (35, 8, 13), (130, 4, 12)):
        _check(cuda_kernels, _data(R, C, N, R, dtype, step, off=off), _ctx((1,) * R, slots=list(reversed(range(R))), dtype=dtype), z=z, bias=bias,
               skip=skip, out_dtype=out)


def test_single_tokens_of_a_wide_layer(cuda_kernels):
    for R in (12, 64):
        _check(cuda_kernels, _data(R, 7168, 16, R, BF16), _ctx((1,) * R, slots=list(reversed(range(R))), dtype=BF16))


@pytest.mark.parametrize("R", [2, 12, 13])
@pytest.mark.parametrize("C,N", [(72, 16), (30, 5), (70, 4)])
def test_float32_bits_do_not_depend_on_the_kernel(cuda_kernels, R, C, N):
    """A token beside others, alone, and in the kernel that spans of several tokens take."""
    d = _data(R + 3, C, N, R + 1)
    state, args = d.state, dict(bias=d.bias, skip=d.skip)

    def scan(rows, lens, slots, st):
        return cuda_kernels.selective_scan(d.x[rows], d.dt[rows], d.bc[rows], d.log_rate, st, _ctx(lens, slots=slots), z=d.z[rows], **args)
    beside, alone, mixed = state.clone(), state.clone(), state.clone()
    y = scan(slice(0, R), (1,) * R, list(range(R)), beside)
    for r in range(R):
        assert torch.equal(scan(slice(r, r + 1), (1,), [r], alone), y[r:r + 1])
    got = scan(slice(0, R + 3), (1,) * R + (3,), list(range(R + 1)), mixed)
    assert torch.equal(got[:R], y) and torch.equal(alone, beside) and torch.equal(mixed[:R], beside[:R])


@pytest.mark.parametrize("lens", [(1, 40), (33, 64, 1, 5)])
@pytest.mark.parametrize("C,N", [(70, 4), (33, 12), (20, 20), (41, 40), (24, 33), (130, 2)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_spans_of_every_number_of_lanes(cuda_kernels, lens, C, N, dtype):
    """States that fill one lane, and that leave places empty in the last of four, eight and sixteen."""
    _check(cuda_kernels, _data(sum(lens), C, N, len(lens), dtype), _ctx(lens, dtype=dtype))


def test_a_replayed_decode_batch_of_changing_requests(cuda_kernels):
    """What a captured step reads of its requests is read at every replay: other slots, other tokens, fewer requests."""
    R, C, N = 16, 96, 16
    d = _data(R, C, N, R + 2, BF16)
    ctx = _ctx((1,) * R, dtype=BF16)

    def scan(ctx, st):
        return cuda_kernels.selective_scan(d.x, d.dt, d.bc, d.log_rate, st, ctx, z=d.z, bias=d.bias, skip=d.skip)
    held = d.state.clone()
    scan(ctx, held.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = scan(ctx, held)
    for lens, slots in (((1,) * R, list(range(R))), ((1,) * 11 + (0,) * 5, list(reversed(range(2, R + 2)))), (EVERY_OTHER[:R], list(range(R)))):
        new = _ctx(lens, slots=slots, dtype=BF16)
        ctx.cu_seqlens.copy_(new.cu_seqlens)
        ctx.req_slot.copy_(new.req_slot)
        held.copy_(d.state)
        graph.replay()
        want = d.state.clone()
        y = scan(SimpleNamespace(**{**vars(new), "max_span": 1}), want)
        torch.cuda.synchronize()
        n = sum(lens)
        assert torch.equal(out[:n], y[:n]) and torch.equal(held, want)
