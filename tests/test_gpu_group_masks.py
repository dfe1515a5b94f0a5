"""GPU: `group_topk` with experts masked by large finite biases, and values closer than fp32 resolves at sixteen values a lane: picks are those of 64 bits."""
import itertools

import pytest
import torch

from .test_gpu_group_router import route64, scores64

pytestmark = pytest.mark.gpu
DEV = "cuda"
LOWEST = torch.finfo(torch.float32).min


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def check(pkg, z, k, b, groups, opened, scoring, by):
    idx, w, counts = pkg.group_topk(z, k, b, groups, opened, scoring, by, return_counts=True)
    ri, rw = route64(z, k, b, groups, opened, scoring, by)
    assert torch.equal(idx, ri), (scoring, by, groups, (idx != ri).any(1).nonzero().flatten().tolist()[:5])
    assert torch.equal(counts.long(), torch.bincount(ri.reshape(-1), minlength=z.shape[1]))
    # roundings as in test_gpu_group_router: 2^-18 of a weight
    assert ((w - rw).abs() <= 2.0 ** -18 * rw).all()


@pytest.mark.parametrize("E,k,groups,opened", [(24, 4, 4, 2), (64, 6, 1, 1), (64, 6, 8, 3), (255, 8, 17, 5), (256, 8, 8, 4), (256, 8, 1, 1)])
@pytest.mark.parametrize("scoring,by", list(itertools.product(("sigmoid", "softmax"), ("top2", "max"))))
def test_masks_of_large_biases(pkg, E, k, groups, opened, scoring, by):
    g = gen(E)
    z = torch.randn(500, E, generator=g, device=DEV)
    base = (torch.randn(E, generator=g, device=DEV) * 20).round() * 1e-3
    masked = torch.rand(E, generator=g, device=DEV) < 0.6
    masked[:: E // k] = False                                     # k live ones at least
    for size in (-1e4, -1e9, LOWEST, 1e4):
        check(pkg, z, k, torch.where(masked, size, base), groups, opened, scoring, by)
    sizes = torch.tensor([-1e4, -1e9, -3e38, LOWEST], device=DEV)[torch.randint(0, 4, (E,), generator=g, device=DEV)]
    check(pkg, z, k, torch.where(masked, sizes, base), groups, opened, scoring, by)
    few = torch.full((E,), -1e4, device=DEV)                      # fewer live experts than picks: the masked ones are told apart too
    few[: k // 2] = base[: k // 2]
    check(pkg, z, k, few, groups, opened, scoring, by)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_groups_of_nothing_but_large_biases(pkg, scoring):
    """The sum of a group's two best values is past fp32's range; it orders the groups all the same."""
    z = torch.randn(100, 16, generator=gen(0), device=DEV)
    b = torch.zeros(16, device=DEV)
    b[8:12], b[12:] = -3.2e38, -3.0e38                            # the later group is the better one
    check(pkg, z, 10, b, 4, 3, scoring, "top2")
    b[:4], b[4:8] = 2.9e38, 3.1e38
    check(pkg, z, 4, b, 4, 1, scoring, "top2")
    b[8], b[9], b[10:12] = 1e9, -1e9, -2e9                        # large values that cancel: off by the size of each, not of their sum
    b[12:] = 0.0
    b[13] = 1e-3
    b[:8] = -LOWEST
    z[:, 8:10] = 0.25
    check(pkg, z, 3, b, 4, 3, scoring, "top2")


@pytest.mark.parametrize("groups,opened", [(17, 17), (17, 5), (1, 1)])
@pytest.mark.parametrize("by", ["top2", "max"])
def test_near_ties_at_sixteen_values_a_lane(pkg, groups, opened, by):
    """As test_values_that_fp32_does_not_tell_apart: 17 groups of 15 experts put 15 values in a lane, whose softmax sums have the most additions."""
    T, E, k = 2048, 255, 8
    g = gen(5)
    for scoring in ("sigmoid", "softmax"):
        z = torch.randn(1, E, generator=g, device=DEV).clamp(-3, 3)
        s = scores64(z, scoring)[0]
        b = torch.zeros(E, device=DEV)
        b[1::2] = (s[0:-1:2] - s[1::2]).float()
        z = z.expand(T, E).contiguous()
        z[1:, 2:] += torch.randn(T - 1, E - 2, generator=g, device=DEV) * 1e-6
        check(pkg, z, k, b, groups, opened, scoring, by)


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_groups_of_one_expert(pkg, scoring):
    """Without a bias the logits decide, also where the scores are equal in 64 bits: a group of one expert is worth its best one."""
    z = torch.arange(60.0, 68.0, device=DEV).repeat(5, 1)
    z[1] = z[1].flip(0)
    z[2] = -torch.arange(8, device=DEV) * 900.0
    z[3] = -z[2]
    z[4] = 3.0
    for by in ("top2", "max"):
        for opened in (3, 8):
            idx, _ = pkg.group_topk(z, 3, None, 8, opened, scoring, by)
            assert idx.tolist() == [[7, 6, 5], [0, 1, 2], [0, 1, 2], [7, 6, 5], [0, 1, 2]], (by, opened)
