"""Routing by groups: the choice is that of the formula in 64 bits, whatever float32 makes of an exponential."""
import math

import pytest
import torch

from plain.plain_kernels import PlainKernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _same(k, z, correction, **kw):
    on = None if correction is None else correction.to(DEV)
    ids, w = k.moe_route_groups(z.to(DEV), on, **kw)
    want_ids, want_w = PlainKernels().moe_route_groups(z, correction, **kw)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(ids.cpu(), want_ids)
    # 64-bit numbers rounded once, by both sides
    assert torch.equal(w.isnan().cpu(), want_w.isnan())
    assert bool(((w.cpu() - want_w).abs() <= want_w.abs() * 2.0 ** -23).logical_or(want_w.isnan()).all())
    return ids, w


@pytest.mark.parametrize("T,n,groups,kept,best,top", [
    (24, 256, 8, 4, 2, 8), (1, 64, 8, 3, 2, 6), (333, 160, 8, 3, 1, 6), (5, 60, 4, 2, 3, 4), (70, 1024, 32, 5, 2, 32), (4, 7, 1, 1, 1, 7),
    (9, 32, 32, 4, 1, 4), (3, 1, 1, 1, 1, 1), (17, 96, 2, 1, 48, 32), (2000, 30, 1, 1, 4, 5), (13, 72, 8, 8, 9, 8), (100, 384, 1, 1, 1, 8), (6, 1023, 3, 2, 2, 9)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("normalized,with_correction,scale", [(True, True, 2.5), (False, False, 1.0), (True, False, 16.0)])
def test_choice(cuda_kernels, T, n, groups, kept, best, top, score, normalized, with_correction, scale):
    g = torch.Generator().manual_seed(T + n)
    z, c = 2 * torch.randn(T, n, generator=g), 0.2 * torch.randn(n, generator=g)
    _same(cuda_kernels, z, c if with_correction else None, top=top, groups=groups, kept=kept, best=best, score=score, normalized=normalized,
          floor=1e-20, scale=scale)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_neighbours_and_ties(cuda_kernels, score):
    """Logits a float32 step apart are told apart, equal ones go by their index; corrections that all but make up for the difference too."""
    g = torch.Generator().manual_seed(3)
    base = torch.randn(400, 1, generator=g)
    steps = torch.randint(0, 3, (400, 64), generator=g)
    z = base.expand(400, 64).contiguous()
    for _ in range(2):
        z = torch.where(steps > 0, torch.nextafter(z, torch.tensor(10.0)), z)
        steps = steps - 1
    _same(cuda_kernels, z, None, top=8, groups=8, kept=3, best=2, score=score)
    # scores whose sum with the correction is the same but for what float32 cannot see
    z = torch.randn(300, 64, generator=g)
    z[150:] = z[0]
    s = torch.sigmoid(z.double()) if score == "sigmoid" else torch.softmax(z.double(), 1)
    c = (1.0 - s[200]).float()
    _same(cuda_kernels, z, c, top=8, groups=4, kept=2, best=2, score=score)
    _same(cuda_kernels, torch.zeros(5, 48), None, top=8, groups=6, kept=2, best=2, score=score)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("normalized", [True, False])
def test_rows_that_leave_nothing(cuda_kernels, score, normalized):
    z = torch.randn(12, 40, generator=torch.Generator().manual_seed(1))
    z[0] = -math.inf                                       # all masked
    z[1, :38] = -math.inf                                  # two left, in one group
    z[2, 5], z[3] = math.nan, math.nan
    z[4, 7] = math.inf
    z[5] = torch.finfo(torch.float32).min                  # masked by the type's lowest value
    z[6, ::2] = torch.finfo(torch.float32).min
    z[7, 30:] = math.nan
    for kept, top in ((2, 8), (5, 8), (1, 8), (5, 32)):
        ids, w = _same(cuda_kernels, z, None, top=top, groups=5, kept=kept, best=2, score=score, normalized=normalized, floor=1e-20)
        assert bool((ids >= 0).all()) and bool((ids < 40).all())
        assert all(len(set(row)) == top for row in ids.tolist())
        assert not bool(w[[0, 1, 5, 6]].isnan().any())
    c = torch.zeros(40)
    c[3], c[12], c[20] = math.inf, -math.inf, math.nan
    _same(cuda_kernels, z[8:], c, top=8, groups=5, kept=3, best=2, score=score, normalized=normalized)


def test_slices_and_graph(cuda_kernels):
    from inferflux_b200.csrc.ops import PartialSum
    g = torch.Generator().manual_seed(9)
    parts = torch.randn(4, 33, 256, generator=g).to(DEV)
    total = ((parts[0] + parts[1]) + parts[2]) + parts[3]
    c = 0.1 * torch.randn(256, generator=g).to(DEV)
    kw = dict(top=8, groups=8, kept=4, floor=1e-20, scale=2.5)
    want = cuda_kernels.moe_route_groups(total, c, **kw)
    got = cuda_kernels.moe_route_groups(PartialSum(parts, torch.float32), c, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert cuda_kernels.moe_route_groups(total[:0], c, **kw)[0].shape == (0, 8)
    graph = torch.cuda.CUDAGraph()
    static = total.clone()
    with torch.cuda.graph(graph):
        out = cuda_kernels.moe_route_groups(static, c, **kw)
    static.copy_(total.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0].flip(0)) and torch.equal(out[1], want[1].flip(0))


def test_one_group_is_the_flat_router(cuda_kernels):
    """With one group, the choice of `moe_route` (where no two scores are near) and its weights but for float32's rounding."""
    z = 2 * torch.randn(200, 64, generator=torch.Generator().manual_seed(2)).to(DEV)
    c = 0.1 * torch.randn(64, generator=torch.Generator().manual_seed(4)).to(DEV)
    ids, w = cuda_kernels.moe_route_groups(z, c, 6, 1, 1, score="sigmoid", normalized=True, floor=1e-6)
    flat_ids, flat_w = cuda_kernels.moe_route(z, c, 6, kind="sigmoid_normalized", floor=1e-6)
    assert torch.equal(ids, flat_ids) and torch.allclose(w, flat_w, rtol=2e-6, atol=0)


def test_numbers_of_all_sizes(cuda_kernels):
    """Corrections that dwarf the scores, of both signs in one group, scores at both ends, and many near ones a row: as in 64 bits."""
    g = torch.Generator().manual_seed(12)
    z = torch.randn(300, 96, generator=g)
    big = torch.where(torch.rand(96, generator=g) < 0.5, 1000.0, -1000.0) + 1e-4 * torch.randn(96, generator=g)
    for score in ("sigmoid", "softmax"):
        for best in (1, 2, 3, 4, 5):
            _same(cuda_kernels, z, big, top=8, groups=12, kept=5, best=best, score=score)
            _same(cuda_kernels, z, 1e-6 * torch.randn(96, generator=g), top=12, groups=12, kept=5, best=best, score=score)
            _same(cuda_kernels, 1e-6 * z, None, top=16, groups=6, kept=2, best=best, score=score, normalized=False)
    wide = 25 * torch.randn(400, 512, generator=g)
    _same(cuda_kernels, wide, None, top=16, groups=8, kept=4, best=2, score="softmax", floor=1e-20)
    _same(cuda_kernels, wide.clamp(-30, 30), 0.1 * torch.randn(512, generator=g), top=16, groups=8, kept=4, best=2, score="sigmoid")
    _same(cuda_kernels, torch.randn(64, 1024, generator=g), None, top=32, groups=32, kept=32, best=2, score="sigmoid")


def _near(k, z, correction, top, groups, kept, best, score):
    """As in 64 bits, where 64 bits can tell.  Of logits some float32 steps d apart, two pairs' sums differ by as little as s'' d^2 = 0.06 (6e-8)^2 =
    2e-16, and each side's terms are off by up to a step of 64 bits, 2^-53 for scores below one: two of a strength and one for its sum, on both sides,
    so strengths within 2^-50 may be taken either way.  Then the choice has to be right for the groups that were taken."""
    ids, w = k.moe_route_groups(z.to(DEV), None if correction is None else correction.to(DEV), top=top, groups=groups, kept=kept, best=best, score=score)
    want, _ = PlainKernels().moe_route_groups(z, correction, top=top, groups=groups, kept=kept, best=best, score=score)
    ids, size = ids.cpu().long(), z.shape[1] // groups
    s = torch.sigmoid(z.double()) if score == "sigmoid" else torch.softmax(z.double(), 1)
    v = s if correction is None else s + correction.double()
    strength = v.view(len(z), groups, size).sort(dim=2, descending=True).values[:, :, :best].sum(2)
    line = strength.sort(dim=1, descending=True).values[:, kept - 1:kept]
    slack = 2.0 ** -50
    for t in (ids != want.long()).any(1).nonzero()[:, 0].tolist():
        taken = set((ids[t] // size).tolist())
        assert len(taken) <= kept and all(float(strength[t, g]) >= float(line[t]) - slack for g in taken), t
        # groups without a chosen expert may be among the kept ones too: those that must be, and of the near ones none that need be
        allowed = taken | {g for g in range(groups) if float(strength[t, g]) > float(line[t]) + slack}
        assert len(allowed) <= kept, t
        order = [i for i in v[t].sort(descending=True, stable=True).indices.tolist() if i // size in allowed]
        assert ids[t].tolist() == order[:top], t
    return ids, w


@pytest.mark.parametrize("n,groups,kept,best,top", [(256, 8, 4, 2, 8), (64, 8, 3, 2, 8), (32, 4, 2, 1, 5), (512, 16, 5, 2, 12), (30, 1, 1, 1, 9), (160, 8, 3, 1, 6)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("spread", [1e-7, 1e-6, 1e-5])
def test_groups_and_experts_all_near(cuda_kernels, n, groups, kept, best, top, score, spread):
    """Scores within some float32 steps of one another, in one lane's experts, in other lanes', and in whole groups; half of the experts a little
    further off; corrections that move them by as little."""
    g = torch.Generator().manual_seed(n + top)
    z = 0.5 + spread * torch.randn(500, n, generator=g)
    z[:, ::2] -= 0.01
    _near(cuda_kernels, z, None, top=top, groups=groups, kept=kept, best=best, score=score)
    _near(cuda_kernels, z, spread * torch.randn(n, generator=g), top=top, groups=groups, kept=kept, best=best, score=score)
    rows = 2 * torch.randn(500, n, generator=g)                # rows as they are, but two groups alike but for a step, and two experts
    size = n // groups
    if groups > 1:
        rows[:, size:2 * size] = torch.nextafter(rows[:, :size].flip(1), torch.tensor(9.0))
    rows[:, n - 1] = torch.nextafter(rows[:, 0], torch.tensor(-9.0))
    rows[:, n // 2] = rows[:, 1]
    _near(cuda_kernels, rows, None, top=top, groups=groups, kept=kept, best=best, score=score)


@pytest.mark.parametrize("n,groups,kept,best,top", [(8, 8, 3, 1, 3), (24, 8, 5, 2, 9), (12, 4, 2, 3, 6), (950, 19, 4, 2, 12), (1020, 17, 3, 4, 20), (1008, 24, 7, 1, 32),
                                                    (45, 5, 2, 2, 8), (930, 31, 6, 2, 8), (992, 31, 6, 2, 8), (1024, 1, 1, 1, 32), (1022, 2, 1, 2, 5)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_groups_of_every_size(cuda_kernels, n, groups, kept, best, top, score):
    """Fewer experts in a group than lanes, lanes with none, and up to sixty of a lane; rows as they are, near ones, and some that are no numbers."""
    g = torch.Generator().manual_seed(n + groups)
    z, c = 2 * torch.randn(90, n, generator=g), 0.1 * torch.randn(n, generator=g)
    z[3, 0], z[4], z[5, n - 1], z[6, : n // 2] = math.nan, -math.inf, -math.inf, -math.inf
    _same(cuda_kernels, z, c, top=top, groups=groups, kept=kept, best=best, score=score)
    best = min(best, 2)                                      # (what `_near` allows for is of two terms)
    near = 0.5 + 1e-6 * torch.randn(90, n, generator=g)
    _near(cuda_kernels, near, None, top=top, groups=groups, kept=kept, best=best, score=score)
    _near(cuda_kernels, near, 1e-6 * torch.randn(n, generator=g), top=top, groups=groups, kept=kept, best=best, score=score)
