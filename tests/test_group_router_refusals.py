"""CPU: what the group-limited top-k and the router losses refuse, before anything is launched."""
import pytest
import torch

from tests.conftest import load_pkg

P = 1 << 20      # an address that is never read


def test_group_topk_refusals():
    lib = load_pkg().lib()

    def call(logits=P, kind=0, E=64, k=6, groups=8, opened=4, scoring=0, idx=P, w=P, T=4):
        return lib.b200moe_group_topk_fwd(logits, kind, None, T, E, k, groups, opened, scoring, 1, 1, 1.0, idx, w, None, None)

    assert call(logits=None) == -6 and call(idx=None) == -6 and call(w=None) == -6
    assert call(kind=2) == -3 and call(kind=7) == -3 and call(scoring=2) == -3
    assert call(E=257, groups=1) == -3 and call(E=0, groups=1) == -3
    assert call(groups=7) == -1 and call(groups=0) == -1 and call(E=256, groups=64) == -1
    assert call(opened=0) == -1 and call(opened=9) == -1
    assert call(k=0) == -1 and call(k=33) == -1 and call(k=9, opened=1) == -1 and call(T=-1) == -1
    bwd = lambda kind=0, E=64, k=6, scoring=0: lib.b200moe_group_topk_bwd(P, kind, P, P, 4, E, k, scoring, 1, 1.0, P, None)    # noqa: E731
    assert bwd(kind=2) == -3 and bwd(E=300) == -3 and bwd(k=65) == -1 and bwd(scoring=5) == -3


def test_router_losses_refusals():
    lib = load_pkg().lib()

    def call(kind=0, S=4, segs=2, E=64, k=6, scoring=1, ws=P, logits=P):
        return lib.b200moe_router_losses_fwd(logits, kind, P, None, S, segs, E, k, scoring, ws, P, P, P, None, None)

    assert call(ws=None) == -6 and call(logits=None) == -6
    assert call(kind=2) == -3 and call(E=257) == -3 and call(scoring=3) == -3
    assert call(segs=0) == -1 and call(segs=65536) == -1 and call(S=-1) == -1 and call(k=0) == -1 and call(k=33) == -1
    assert lib.b200moe_router_losses_ws_bytes(100, 2, 64) >= 2 * (16 + 8 * 64) + 48
    assert lib.b200moe_router_losses_bwd(P, 0, None, None, None, None, 4, 1, 64, 1, P, None) == -6
    assert lib.b200moe_router_losses_bwd(P, 2, None, P, None, None, 4, 1, 64, 1, P, None) == -3


def test_python_refusals():
    pkg = load_pkg()
    z, idx = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.group_topk(z, 2)
    with pytest.raises(ValueError, match="scoring"):
        pkg.group_topk(z, 2, scoring="relu")
    with pytest.raises(ValueError, match="group_score"):
        pkg.group_topk(z, 2, group_score="mean")
    with pytest.raises(ValueError, match=r"\(N,E\)"):
        pkg.group_topk(z[0], 2)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.router_losses(z, idx)
    with pytest.raises(ValueError, match="scoring"):
        pkg.router_losses(z, idx, scoring="none")
    with pytest.raises(ValueError, match="num_experts"):
        pkg.fused_group_router(z, torch.zeros(8, 8), None, 2, 16)
