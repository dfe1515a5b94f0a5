"""CPU: what the low-rank adapters refuse, before anything is launched."""
import pytest
import torch

from tests.conftest import load_pkg

P = 1 << 20      # an address that is never read


def test_c_entry_points():
    lib = load_pkg().lib()

    def fwd(x=P, ldx=64, a=P, b=P, i=P, ib=8, bs=P, ldb=64, T=4, K=64, N=64, R=8, L=2, ws=P, out=P, st=P):
        return lib.b200moe_lora_forward(x, ldx, a, b, i, ib, None, 1.0, bs, ldb, T, K, N, R, L, 0, ws, out, st, None)

    assert fwd(T=0) == 0
    for name in ("x", "a", "b", "ws", "out", "st"):
        assert fwd(**{name: None}) == -6, name
    for name in ("x", "a", "b", "ws", "out", "bs"):
        assert fwd(**{name: P + 8}) == -2, name
    assert fwd(i=P + 4) == -2 and fwd(ib=2) == -3 and fwd(R=12) == -3 and fwd(R=136) == -3 and fwd(R=0) == -3
    assert fwd(K=60) == -1 and fwd(N=0) == -1 and fwd(T=-1) == -1 and fwd(T=1 << 31) == -1 and fwd(L=0) == -1 and fwd(L=65537) == -1
    assert fwd(ldx=56) == -1 and fwd(ldx=68) == -1 and fwd(ldb=56) == -1 and fwd(ldb=66) == -1 and fwd(L=65536, N=1 << 20) == -1

    def bwd(g=P, x=P, ldx=64, a=P, T=4, K=64, N=64, R=8, L=2, fw=P, ws=P, gx=P, ga=P):
        return lib.b200moe_lora_backward(g, x, ldx, a, P, 1, None, 1.0, T, K, N, R, L, fw, ws, gx, ga, P, 0, P, None)

    for name in ("g", "x", "a", "fw", "ws"):
        assert bwd(**{name: None}) == -6, name
    assert bwd(gx=P + 4) == -2 and bwd(ga=P + 8) == -2 and bwd(T=0) == -1 and bwd(ldx=60) == -1 and bwd(R=20) == -3
    assert lib.b200moe_lora_fwd_ws_bytes(0, 8, 1, 1) == 0 and lib.b200moe_lora_fwd_ws_bytes(300, 8, 5, 1) >= 300 * 32 + 300 * 4 + 3 * 5
    assert b"adapter" in lib.b200moe_status_string(9)


def test_python_callable():
    pkg = load_pkg()
    x, a, b = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((4, 64), (1, 8, 64), (1, 64, 8)))
    with pytest.raises(ValueError, match="CUDA"):
        pkg.lora_linear(x, a, b)


def test_an_index_off_its_type():
    lib = load_pkg().lib()
    for bytes_, off in ((4, 2), (8, 4)):
        assert lib.b200moe_lora_forward(P, 64, P, P, P + off, bytes_, None, 1.0, P, 64, 4, 64, 64, 8, 2, 0, P, P, P, None) == -2
