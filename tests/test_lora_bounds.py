"""CPU: how many adapters a call may have."""
import pytest

from tests.conftest import load_pkg

P = 1 << 20      # an address that is never read


@pytest.mark.parametrize("K,N,R,L", [(16384, 64, 128, 65536), (64, 16384, 128, 65536), (16384, 16384, 16, 65536), (8072, 8072, 128, 65536), (32768, 64, 64, 65536),
                                     (65536, 65536, 128, 16384), (1 << 20, 64, 8, 16384)])
def test_as_many_adapters_as_documented(K, N, R, L):
    """No rows: what is checked before anything is launched."""
    lib = load_pkg().lib()
    assert lib.b200moe_lora_forward(P, K, P, P, P, 8, None, 1.0, None, N, 0, K, N, R, L, 0, P, P, P, None) == 0
    # the gradient's check of its sizes comes before that of its pointers
    assert lib.b200moe_lora_backward(None, P, K, P, P, 1, None, 1.0, 4, K, N, R, L, P, P, P, P, P, 0, P, None) == -6


def test_stacks_that_no_memory_holds():
    lib = load_pkg().lib()
    for K, N, R, L in ((64, 1 << 20, 8, 65536), (1 << 20, 64, 8, 65536), (32768, 64, 128, 65536)):
        assert lib.b200moe_lora_forward(P, K, P, P, P, 8, None, 1.0, None, N, 0, K, N, R, L, 0, P, P, P, None) == -1
        assert lib.b200moe_lora_backward(None, P, K, P, P, 1, None, 1.0, 4, K, N, R, L, P, P, P, P, P, 0, P, None) == -1
