"""CPU: what the block-scaled 8-bit products refuse, before anything is launched."""
import pytest
import torch

from tests.conftest import load_pkg

P = 1 << 20      # an address that is never read


def test_c_entry_points():
    lib = load_pkg().lib()
    q = lambda x=P, rows=4, K=128, ldq=128, pitch=4: lib.b200moe_fp8_block_quant(x, rows, K, P, ldq, P, pitch, None)     # noqa: E731
    assert q(x=None) == -6 and q(K=12) == -1 and q(K=0) == -1 and q(ldq=64) == -1 and q(pitch=3) == -1 and q(x=P + 2) == -2 and q(rows=-1) == -1
    assert lib.b200moe_fp8_block_quant_weight(None, 1, 8, 8, P, P, None) == -6
    assert lib.b200moe_fp8_block_quant_weight(P, 1, 8, 12, P, P, None) == -1 and lib.b200moe_fp8_block_quant_weight(P, 0, 8, 8, P, P, None) == -1
    lin = lambda x=P, w=P, M=4, N=64, K=128, out=P: lib.b200moe_fp8_block_linear(x, w, P, M, N, K, 0, P, out, None, None)     # noqa: E731
    assert lin(x=None) == -6 and lin(N=12) == -1 and lin(K=24) == -1 and lin(M=-1) == -1 and lin(w=P + 8) == -2 and lin(out=P + 2) == -2
    assert lin(M=0) == 0
    assert lib.b200moe_fp8_block_linear_ws_bytes(5, 130) >= 5 * 144 + 128 * 2 * 4

    def moe(x=P, T=4, H=128, I=128, E=4, k=2, gu=P):
        return lib.b200moe_moe_fp8_block_forward(x, P, P, gu, P, P, P, T, H, I, E, k, P, P, P, None)

    assert moe(x=None) == -6 and moe(H=192) == -1 and moe(I=64) == -1 and moe(E=257) == -3 and moe(k=0) == -1 and moe(k=33) == -1
    assert moe(gu=P + 4) == -2 and moe(T=0) == 0 and moe(T=1 << 30, k=8) == -1


def test_python_callables():
    pkg = load_pkg()
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    w, s = torch.zeros(64, 128).to(torch.float8_e4m3fn), torch.ones(1, 1)
    for call in (lambda: pkg.fp8_block_linear(x, w, s), lambda: pkg.fp8_block_quantize(x), lambda: pkg.fp8_block_quantize_weight(x),
                 lambda: pkg.moe_fp8_block(x, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2), w, s, w, s)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
