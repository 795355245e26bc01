"""What the selective scan's and its inputs' entry points hand to the kernels, without a GPU: nothing is launched."""
import ctypes

import pytest
import torch

from inferflux_b200.csrc import CudaKernels, ops
from inferflux_b200.csrc.build import load_library
from inferflux_b200.csrc.ops import PartialSum

F32 = torch.float32


class _Recorder:
    """A library whose functions keep their arguments and answer 0."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture()
def kernels(monkeypatch):
    monkeypatch.setattr(ops, "_device_of", lambda what, first, *more: first.device)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    k = CudaKernels.__new__(CudaKernels)
    k.lib, k.launches = _Recorder(), 0
    return k


@pytest.mark.parametrize("splits,T", [(1, 1), (3, 1), (2, 5)])
def test_slices_of_a_single_row(kernels, splits, T):
    """The stride of an axis with one entry may be anything, in a tensor that counts as contiguous too; slices lie T rows of their width apart."""
    rank, states = 16, 4
    width = rank + 2 * states
    whole = torch.zeros(T, splits, width) if T == 1 else torch.zeros(splits, T, width)
    parts = whole.transpose(0, 1) if T == 1 else whole
    assert parts.shape == (splits, T, width) and parts.is_contiguous()
    assert T > 1 or splits == 1 or parts.stride(1) == splits * width
    low, bc = kernels.selective_inputs(PartialSum(parts, F32), rank, states, F32)
    (name, args), = kernels.lib.calls
    assert name == "ifx_selective_inputs" and args[0] is parts and args[3] == splits
    assert T * args[1] == width * T          # what the kernel takes for the distance between slices
    assert low.shape == (T, rank) and bc.shape == (T, 2 * states)


def test_stretches_without_their_scratch():
    """The C entry point: room that is said to be there, and no address for it, is refused before anything is launched."""
    lib, p, n = load_library(), ctypes.c_void_p(16), ctypes.c_void_p(0)
    ll = ctypes.c_longlong
    T, C, N = 300, 64, 16
    lib.ifx_selective_scan_scratch.restype = ctypes.c_longlong
    room = lib.ifx_selective_scan_scratch(1, T, C, N)
    assert room > 0

    def scan(scratch, floats):
        return lib.ifx_selective_scan(p, ll(C), 0, p, ll(C), 0, p, ll(2 * N), n, ll(0), p, n, n, p, ll(C * N), p, p, p, 0, 1, T, T, C, N, scratch,
                                      ll(floats), n)
    assert scan(n, room) == -1
    assert scan(p, room - 1) == -1
