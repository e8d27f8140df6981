"""Packed attention where a few queries of each sequence are served by kernels that split the keys, on both sides of every rule that chooses them."""
import pytest

from test_gpu_packed import BF16, F16, F32, _check, _inputs

pytestmark = pytest.mark.gpu

# dtype, queries of a sequence, sequences, keys of one, H, Hk, D
CASES = [
    # up to 16 columns, 17 to 32 with shared heads: many sequences, long ones, neither
    (BF16, 1, 4, 300, 8, 8, 64), (F16, 16, 3, 50, 2, 2, 96), (BF16, 5, 260, 40, 8, 2, 32), (F16, 7, 256, 33, 8, 2, 128), (BF16, 3, 200, 33, 24, 3, 80), (BF16, 6, 2, 1100, 8, 2, 64),
    (F16, 3, 3, 1300, 8, 1, 96), (BF16, 3, 3, 900, 8, 1, 96), (F16, 2, 40, 1024, 32, 2, 32), (BF16, 32, 2, 2000, 1, 1, 128),
    # with heads of their own: long sequences that are few, many, short ones
    (BF16, 31, 2, 1500, 4, 4, 64), (F16, 17, 1, 5000, 8, 8, 32), (BF16, 20, 32, 1024, 4, 4, 128), (F16, 20, 5, 100, 4, 4, 40),
    # in parts: by queries and keys, heads that share a key head, the head dim, sequences
    (BF16, 1, 32, 500, 8, 8, 64), (F16, 8, 34, 300, 8, 8, 64), (BF16, 4, 33, 512, 16, 4, 64), (BF16, 8, 33, 400, 16, 4, 64), (F16, 8, 64, 900, 16, 4, 128), (BF16, 8, 16, 1100, 8, 8, 32), (F16, 20, 16, 1100, 8, 8, 64), (BF16, 24, 17, 10000, 8, 8, 64),
    (BF16, 8, 100, 60, 4, 2, 64), (BF16, 16, 400, 60, 4, 2, 64),
    # fp32: by the rows that are made beside the keys, by sequences, by columns beyond 32
    (F32, 1, 600, 20, 2, 1, 64), (F32, 8, 300, 8, 2, 2, 64), (F32, 9, 300, 9, 2, 2, 64), (F32, 4, 300, 66, 2, 2, 64), (F32, 5, 300, 30, 2, 2, 64), (F32, 1, 5, 100, 8, 2, 32), (F32, 1, 5, 200, 8, 2, 33), (F32, 30, 40, 600, 1, 1, 128), (F32, 12, 2, 2000, 8, 2, 64), (F32, 12, 2, 5000, 8, 2, 64),
    (F32, 16, 20, 700, 8, 2, 96), (F32, 60, 33, 900, 1, 1, 77),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("causal", [True, False])
def test_few_queries(gpu_device, case, causal):
    dtype, q, n, k, H, Hk, D = case
    queries, keys = [q] * n, [k] * n
    if n > 2:      # (of one key fewer and more, and none)
        queries[1], keys[0], keys[1], keys[2] = 0, k - 1, k + 1, 0
    x = _inputs(dtype, queries, keys, H, Hk, D, padding=2)
    out, = _check(*x[:3], None, queries, keys, causal, grad=False)
    assert not out[sum(queries):].any()
