"""CPU: what the root-mean-square norm and the products of codes refuse, before anything is launched."""
import pytest
import torch

from tests.conftest import load_pkg

P = 1 << 20      # an address that is never read


def test_c_entry_points():
    lib = load_pkg().lib()

    def fwd(x=P, ldx=64, r=P, ldr=64, t=0, w=P, wt=0, rows=4, K=64, eps=1e-6, y=P, h=P, q=P, s=P, pitch=128, st=P):
        return lib.b200moe_rms_norm_fwd(x, ldx, r, ldr, t, w, wt, rows, K, eps, y, h, q, s, pitch, st, None)

    assert fwd(rows=0) == 0
    assert fwd(x=None) == -6 and fwd(w=None) == -6 and fwd(s=None) == -6 and fwd(y=None, h=None, q=None) == -6 and fwd(r=None) == -6
    assert fwd(t=2) == -3 and fwd(wt=3) == -3 and fwd(t=1, wt=0) == -3 and fwd(rows=-1) == -1 and fwd(rows=1 << 31) == -1
    assert fwd(K=0) == -1 and fwd(K=16385, ldx=1 << 20, ldr=1 << 20) == -1 and fwd(ldx=63) == -1 and fwd(ldr=8) == -1
    assert fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1 and fwd(K=60) == -1 and fwd(pitch=3) == -1 and fwd(q=P + 4) == -2

    def bwd(gy=P, gh=P, h=P, ldh=64, t=0, w=P, wt=0, rows=4, K=64, ws=P, gx=P, gw=P, st=P):
        return lib.b200moe_rms_norm_bwd(gy, gh, h, ldh, t, w, wt, rows, K, 1e-6, ws, gx, gw, st, None)

    assert bwd(rows=0, gw=None) == 0
    assert fwd(st=None) == -6 and bwd(st=None) == -6 and bwd(ws=P + 8) == -2
    assert bwd(gy=None) == -6 and bwd(h=None) == -6 and bwd(w=None) == -6 and bwd(gx=None, gw=None) == -6 and bwd(ws=None) == -6
    assert bwd(t=7) == -3 and bwd(ldh=60) == -1 and bwd(K=0) == -1 and bwd(rows=-2) == -1
    assert lib.b200moe_rms_norm_bwd_ws_bytes(0, 64) == 0 and lib.b200moe_rms_norm_bwd_ws_bytes(4, 1 << 20) == 0

    def rows(q=P, qs=P, pitch=128, w=P, M=4, N=64, K=128, out=P):
        return lib.b200moe_fp8_block_linear_rows(q, qs, pitch, w, P, M, N, K, out, None, None)

    assert rows(M=0) == 0 and rows(q=None) == -6 and rows(pitch=4) == -1 and rows(pitch=130) == -1 and rows(M=129) == -1 and rows(N=12) == -1
    assert rows(K=24) == -1 and rows(q=P + 8) == -2 and rows(qs=P + 4) == -2 and rows(out=P + 2) == -2


def test_python_callables():
    pkg = load_pkg()
    x, w = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(128, dtype=torch.bfloat16)
    q, s = x.to(torch.float8_e4m3fn), torch.ones(4, 1)
    for call in (lambda: pkg.rms_norm(x, w), lambda: pkg.rms_norm_fp8_block(x, w),
                 lambda: pkg.fp8_block_linear(x, q[:64], s, quantized=(q, s))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_an_infinite_eps():
    lib = load_pkg().lib()
    for eps in (float("inf"), 1e39):      # the second is one in fp32
        assert lib.b200moe_rms_norm_fwd(P, 64, None, 64, 0, P, 0, 4, 64, eps, P, None, None, None, 0, P, None) == -1
        assert lib.b200moe_rms_norm_bwd(P, None, P, 64, 0, P, 0, 4, 64, eps, P, P, P, P, None) == -1
