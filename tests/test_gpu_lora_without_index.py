"""GPU: the C entry points of the adapters without an index and with several adapters: every row has adapter 0, and the others have no row.

Bounds as in tests/test_gpu_lora.py."""
import importlib

import pytest
import torch

from .test_gpu_lora import BF, DEV, F32, close, gen, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad_type", [BF, F32])
@pytest.mark.parametrize("T,K,N,R,n", [(5, 264, 136, 24, 2), (40, 64, 72, 8, 3), (1000, 520, 264, 64, 3), (3000, 1040, 680, 16, 5), (3000, 136, 2816, 128, 2)])
def test_all_rows_have_the_first_adapter(pkg, T, K, N, R, n, grad_type):
    x, a, b, s, bs, _ = make(T, K, N, R, n, seed=7)
    go = torch.randn(T, N, generator=gen(8), device=DEV).to(BF)
    lib, L = pkg.lib(), importlib.import_module(pkg.__name__ + "._lib")
    ref = reference(x, a, b, s, bs, torch.zeros(T, dtype=torch.int64, device=DEV), go)
    status, stream = L.status_word(x.device).data_ptr(), L.stream_of(x)
    for keep in (0, 1):
        ws = L.workspace(lib.b200moe_lora_fwd_ws_bytes(T, R, n, keep), x.device)
        out = torch.empty_like(bs)
        L.check(lib.b200moe_lora_forward(x.data_ptr(), K, a.data_ptr(), b.data_ptr(), None, 0, s.data_ptr(), 1.0, bs.data_ptr(), N, T, K, N, R, n, keep, ws.data_ptr(),
                                         out.data_ptr(), status, stream))
        close(out, ref["y"], max(K, R))
    for asked in ((1, 1, 1), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        tmp = L.workspace(lib.b200moe_lora_bwd_ws_bytes(T, K, N, R, n), x.device)
        grads = [torch.full_like(t, float("nan"), dtype=dt) if want else None for t, dt, want in zip((x, a, b), (BF, grad_type, grad_type), asked)]
        L.check(lib.b200moe_lora_backward(go.data_ptr(), x.data_ptr(), K, a.data_ptr(), b.data_ptr(), 0, s.data_ptr(), 1.0, T, K, N, R, n, ws.data_ptr(), tmp.data_ptr(),
                                          *(L.ptr(t) for t in grads), int(grad_type == F32), status, stream))
        for got, name, terms in zip(grads, ("gx", "ga", "gb"), (max(N, R), max(N, T), max(K, T))):
            if got is None:
                continue
            assert name == "gx" or (got[1:] == 0).all(), name
            close(got, ref[name], terms)
    pkg.check_status()
