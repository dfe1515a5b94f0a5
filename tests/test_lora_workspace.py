"""CPU: the workspace of the adapters' gradients."""
import pytest

from tests.conftest import load_pkg


@pytest.mark.parametrize("T,K,N,R,L", [(1000, 2048, 2176, 64, 100), (1000, 2048, 2176, 64, 101), (300, 640, 384, 128, 1001), (2000, 136, 2176, 16, 333)])
def test_one_share_of_many_adapters(T, K, N, R, L):
    """Where the adapters' columns alone are more CTAs than SMs, no gradient is split over shares of the rows, whose sums would be as many times the factors' size: what is left
    is u, two bf16 numbers a row and rank."""
    got = load_pkg().lib().b200moe_lora_bwd_ws_bytes(T, K, N, R, L)
    ranks = 16
    while ranks < R:
        ranks *= 2
    assert 4 * T * ranks <= got <= 4 * T * ranks + 1024
