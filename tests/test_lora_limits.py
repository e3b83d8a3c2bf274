"""Low-rank adapters without a GPU: the largest counts that the C entries take (32-bit positions, some steps ahead of the last)."""
from mlx_kquant_b200 import _lib


def test_counts_beyond_the_limit_are_refused():
    L, F16, bad, p = _lib.lib(), _lib.KQ_F16, _lib.KQ_ERR_INVALID_ARGUMENT, 256   # p is never followed
    most = 2 ** 30
    assert L.kq_lora_plan_bytes(most, 4) > 4 * most and L.kq_lora_plan_bytes(most + 1, 4) == 0
    for rows, K, N in ((most + 1, 8, 8), (4, most + 1, 8), (4, 8, most + 1), (2 ** 31 - 100, 8, 8), (4, 2 ** 31 - 1, 8)):
        assert L.kq_lora_update(p, F16, rows, K, K, 1, 0, p, p, F16, 2, N, 2, 1, p, None, None, 1.0, p, N, p, N, None, None, 0, None) == bad
        assert L.kq_lora_backward(p, F16, rows, N, N, p, K, K, 1, 0, p, p, F16, 2, 2, 1, p, None, None, 1.0, p, p, p, p, p, 1 << 40, p, 1 << 40,
                                  None) == bad
    assert L.kq_lora_plan(p, None, most + 1, 1, 4, 1, p, 1 << 40, None) == bad
