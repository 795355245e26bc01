"""What the selective scan, its inputs and the router by groups refuse (no GPU: before anything is launched)."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from inferflux_b200.csrc import CudaKernels
from inferflux_b200.csrc.build import load_library
from inferflux_b200.csrc.ops import KernelError

F32, BF16 = torch.float32, torch.bfloat16


class _NoLibrary:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture()
def kernels():
    k = CudaKernels.__new__(CudaKernels)
    k.lib, k.launches = _NoLibrary(), 0
    return k


def _scan(**changes):
    T, C, N = 6, 8, 4
    a = dict(x=torch.zeros(T, C), dt=torch.zeros(T, C), bc=torch.zeros(T, 2 * N), log_rate=torch.zeros(C, N), state=torch.zeros(3, C * N),
             ctx=SimpleNamespace(num_requests=2, max_span=4, cu_seqlens=torch.tensor([0, 4, 6], dtype=torch.int32),
                                 req_slot=torch.tensor([0, 2], dtype=torch.int32)), z=torch.zeros(T, C), bias=torch.zeros(C), skip=torch.zeros(C))
    a.update(changes)
    return a


@pytest.mark.parametrize("changes,words", [
    ({}, "not the current CUDA device"),                                    # all is well but where it lies
    ({"x": torch.zeros(6, 8, dtype=torch.float16)}, "x must be"), ({"x": torch.zeros(6)}, "rows"), ({"dt": torch.zeros(6, 7)}, "dt must be"),
    ({"dt": torch.zeros(5, 8)}, "dt must be"), ({"x": torch.zeros(8, 6).t()}, "x must be"), ({"z": torch.zeros(6, 8, dtype=BF16)}, "gate"),
    ({"z": torch.zeros(6, 9)}, "z must be"), ({"x": torch.zeros(8).expand(6, 8)}, "overlap"), ({"bc": torch.zeros(6, 8, dtype=BF16)}, "B and C"),
    ({"bc": torch.zeros(6, 7)}, "B | C"), ({"log_rate": torch.zeros(8, 129), "bc": torch.zeros(6, 258)}, "129 states"),
    ({"log_rate": torch.zeros(4, 8).t(), "bc": torch.zeros(6, 8)}, "rates"), ({"log_rate": torch.zeros(8, 4, dtype=torch.float64)}, "rates"),
    ({"bias": torch.zeros(7)}, "bias and skip"), ({"skip": torch.zeros(8, dtype=BF16)}, "bias and skip"), ({"state": torch.zeros(3, 31)}, "state"),
    ({"state": None}, "state"), ({"state": torch.zeros(3, 32, dtype=BF16)}, "state"), ({"state": torch.zeros(32).expand(3, 32)}, "state"),
    ({"out_dtype": torch.float16}, "y in float32 or bfloat16"),
    ({"ctx": SimpleNamespace(num_requests=2, max_span=4, cu_seqlens=torch.tensor([0, 6]).int(), req_slot=torch.tensor([0, 1]).int())}, "spans"),
    ({"ctx": SimpleNamespace(num_requests=1, max_span=6, cu_seqlens=torch.tensor([0, 6]), req_slot=torch.tensor([0]).int())}, "spans")])
def test_scan_refuses(kernels, changes, words):
    with pytest.raises(KernelError, match=words.replace("|", r"\|")):
        kernels.selective_scan(**_scan(**changes))


@pytest.mark.parametrize("rows,rank,states,norms,words", [
    (torch.zeros(3, 24), 16, 4, None, "not the current CUDA device"), (torch.zeros(3, 23), 16, 4, None, "rows of 23"),
    (torch.zeros(3, 24, dtype=torch.float16), 16, 4, None, "float32 or bfloat16"), (torch.zeros(24, 3).t(), 16, 4, None, "unit column stride"),
    (torch.zeros(3, 24), 0, 4, None, "rank of 0"), (torch.zeros(3, 300), 16, 129, None, "129 states"), (torch.zeros(3, 9000), 8193, 4, None, "rank of 8193"),
    (torch.zeros(3, 24), 16, 4, (torch.ones(15), None, None), "norm weights"), (torch.zeros(3, 24), 16, 4, (None, torch.ones(4).bfloat16(), None), "norm weights")])
def test_inputs_refuse(kernels, rows, rank, states, norms, words):
    with pytest.raises(KernelError, match=words):
        kernels.selective_inputs(rows, rank, states, F32, norms)


@pytest.mark.parametrize("changes,words", [
    ({}, "not the current CUDA device"), ({"score": "tanh"}, "unknown score"), ({"z": torch.zeros(3, 64, dtype=BF16)}, "float32 logits"),
    ({"z": torch.zeros(64, 3).t()}, "float32 logits"), ({"correction": torch.zeros(63)}, "float32 logits"), ({"groups": 5}, "64 experts in 5 groups"),
    ({"groups": 0}, "in 0 groups"), ({"groups": 64, "kept": 1, "best": 1, "top": 1}, "64 groups"), ({"kept": 9}, "9 kept"), ({"kept": 0}, "0 kept"),
    ({"best": 9}, "best 9"), ({"best": 0}, "best 0"), ({"top": 17, "kept": 2}, "17 chosen"), ({"top": 33}, "33 chosen"), ({"top": 0}, "0 chosen"),
    ({"z": torch.zeros(3, 2048), "correction": None}, "2048 experts")])
def test_router_refuses(kernels, changes, words):
    a = dict(z=torch.zeros(3, 64), correction=torch.zeros(64), top=8, groups=8, kept=4)
    a.update(changes)
    with pytest.raises(KernelError, match=words):
        kernels.moe_route_groups(**a)


def test_entry_points_refuse():
    """The C entry points by themselves: sizes and types are looked at before anything is launched."""
    lib, p, n = load_library(), ctypes.c_void_p(16), ctypes.c_void_p(0)
    ll, f = ctypes.c_longlong, ctypes.c_float

    def scan(x_dtype=0, dt_dtype=0, out_dtype=0, R=1, T=2, span=2, C=8, N=4, ld=8, ld_bc=8, slot=32, x=p, out=p):
        return lib.ifx_selective_scan(x, ll(ld), x_dtype, p, ll(8), dt_dtype, p, ll(ld_bc), n, ll(0), p, n, n, p, ll(slot), p, p, out, out_dtype, R, T, span,
                                      C, N, n, ll(0), n)
    assert scan(C=0) == scan(N=0) == scan(R=-1) == scan(T=-1) == scan(ld=7) == scan(ld_bc=7) == scan(slot=31) == scan(x=n) == scan(out=n) == -1
    assert scan(x_dtype=2) == scan(dt_dtype=7) == scan(out_dtype=-1) == -2
    assert scan(N=129, ld_bc=300, slot=9999) == scan(R=65536) == -4
    assert scan(R=0) == scan(T=0) == scan(span=0) == 0

    def inputs(ld=24, dtype=0, splits=1, low_dtype=0, T=3, rank=16, states=4, rows=p):
        return lib.ifx_selective_inputs(rows, ll(ld), dtype, splits, n, n, n, f(0), p, low_dtype, p, T, rank, states, n)
    assert inputs(ld=23) == inputs(splits=0) == inputs(T=-1) == inputs(rank=0) == inputs(states=0) == inputs(rows=n) == -1
    assert inputs(dtype=3) == inputs(low_dtype=5) == inputs(dtype=1, splits=2) == -2
    assert inputs(rank=8193, ld=9999) == -4 and inputs(T=0) == 0

    def route(splits=1, T=3, n_=64, groups=8, kept=4, best=2, top=8, z=p):
        return lib.ifx_moe_route_groups(z, splits, n, p, p, T, n_, groups, kept, best, top, 0, 1, f(0), f(1), n)
    assert route(splits=0) == route(T=-1) == route(groups=5) == route(kept=0) == route(kept=9) == route(best=9) == route(top=0) == route(z=n) == -1
    assert route(top=33, kept=8) == route(n_=2048) == route(groups=64, kept=8, best=1) == -4 and route(T=0) == 0


# ------------------------------------------------------------------------- a model of such layers, on the plain kernels
LENS = [40, 33, 3, 61, 97, 1]


@pytest.mark.parametrize("which", ["groups", "softmax"])
@pytest.mark.parametrize("cutting", ["whole", "tail", "portions", "mixed"])
def test_layers_through_the_step_function(which, cutting):
    """The selective mixer and experts by groups in a model of their own, cut into steps in every way: the host's side of both parts."""
    import helpers
    import selective_models as sm
    from inferflux_b200.engine import ModelRunner
    from plain.plain_kernels import PlainKernels
    model, W = sm.made(which, F32, "cpu")
    reqs = {f"r{i}": helpers.random_tokens(sm.V, n, 400 + i) for i, n in enumerate(LENS)}
    want = {r: sm.logits(which, W, toks).numpy() for r, toks in reqs.items()}
    steps = {"whole": helpers.trace_whole, "tail": helpers.trace_tail, "portions": helpers.trace_portions,
             "mixed": lambda r: helpers.trace_mixed(r, 256)}[cutting](reqs)
    runner = ModelRunner(model, PlainKernels(wide=True), page_size=sm.PAGE, num_pages=256 // sm.PAGE, max_seqs=4, max_seq_len=512)
    got = helpers.collect(steps, helpers.run_steps_in_process(runner, steps), sm.V)
    bad = helpers.first_bad(got, want, 2e-4)
    assert bad is None, f"first wrong row (request, position, diff): {bad}"


@pytest.mark.parametrize("changes,words", [
    ({"groups": {"count": 3, "kept": 1, "best": 1}}, "16 experts in 3 groups"), ({"groups": {"count": 4, "kept": 5, "best": 1}}, "5 kept"),
    ({"groups": {"count": 4, "kept": 1, "best": 5}}, "best 5"), ({"groups": {"count": 4, "kept": 1, "best": 2}, "top": 5}, "top 5"),
    ({"routing": "softmax_of_chosen", "groups": {"count": 4, "kept": 2, "best": 2}}, "chosen alone"), ({"routing": "other"}, "unknown routing")])
def test_parts_refuse(changes, words):
    from inferflux_b200.config import PartSpec
    from inferflux_b200.parts import build_part
    p = {"hidden_size": 8, "expert_size": 4, "num_experts": 16, "top": 4, "routing": "sigmoid_normalized", **changes}
    with pytest.raises(ValueError, match=words):
        build_part("ffn", PartSpec("moe", p))


@pytest.mark.parametrize("changes", [{"state_dim": 129}, {"state_dim": 0}, {"conv_taps": 17}, {"step_rank": 9000}, {"inner_size": -1}])
def test_mixer_refuses(changes):
    from inferflux_b200.config import PartSpec
    from inferflux_b200.parts import build_part
    with pytest.raises(ValueError, match="selective_state_space"):
        build_part("mixer", PartSpec("selective_state_space", {"hidden_size": 8, "inner_size": 16, "state_dim": 4, "step_rank": 2, "conv_taps": 4, **changes}))
