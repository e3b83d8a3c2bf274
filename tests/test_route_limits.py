"""The router of expert groups without a GPU: the largest token count that the C entries take."""
from mlx_kquant_b200 import _lib


def test_counts_beyond_the_limit_are_refused():
    L, p = _lib.lib(), 256   # p is never followed
    for T in (2 ** 30 + 1, 2 ** 31 - 1, 2 ** 31, -1):
        assert L.kq_moe_router_grouped(p, _lib.KQ_F32, T, 64, 4, 1, 1, 1, b"sigmoid", None, 1, 1.0, p, p, None) == _lib.KQ_ERR_INVALID_ARGUMENT
        assert L.kq_moe_router_grouped_backward(p, _lib.KQ_F32, T, 64, 4, b"sigmoid", 1, 1.0, p, p, p, None) == _lib.KQ_ERR_INVALID_ARGUMENT
