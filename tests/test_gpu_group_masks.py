"""GPU: `group_topk` with experts masked by large finite biases: picks are those of 64 bits."""
import pytest
import torch

from .test_gpu_group_router import route64

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
