"""Paged attention where values are far apart: weights far below the largest one."""
import pytest
import torch

from test_gpu_attention import DEV, TYPES, _attend64, _cache_case, _close

pytestmark = pytest.mark.gpu


def _one_key_above_the_rest(gap, lengths, heads, kv_heads, dtype, columns=None, page=64):
    """Caches in which each request's key 0 scores `gap` above the others (which are 0.3 apart, as a standard deviation); the
    values are positive and those of token 0 are zero, so that the output is what the far weights make of it."""
    dim = 64
    kc, vc, table, n = _cache_case(lengths, kv_heads, dim, page, TYPES[dtype], columns=columns)
    q = torch.zeros(len(lengths), heads, dim, dtype=TYPES[dtype], device=DEV)
    q[..., 0] = 1.0
    kc.mul_(0.3)
    vc.abs_().mul_(0.1).add_(1.0)
    for r in range(len(lengths)):
        kc[table[r, 0].long(), :, 0, 0] = gap
        vc[table[r, 0].long(), :, 0] = 0.0
    return q, kc, vc, table, n


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("gap", [9.0, 14.0, 17.0, 17.5, 18.0, 22.0])
@pytest.mark.parametrize("lengths,columns", [([131072], None), ([700, 650], None), ([9440] * 40, None)])
def test_small_weights_beside_a_large_one(dtype, gap, lengths, columns):
    import dlr_lock_b200 as D
    q, kc, vc, table, n = _one_key_above_the_rest(gap, lengths, 4, 2, dtype, columns)
    got = D.paged_attention(q, kc, vc, table, n, scale=1.0)
    want, _ = _attend64(q, kc, vc, table, lengths, 1.0)
    # Every term is positive, so bounds are relative to the output: scores of 64 products (one that is not zero) and their scale,
    # difference and exponential are off by some half-steps of fp32 of the gap (2^-24 x 32 x 8 = 2^-16); the two terms of a weight
    # by 2^-16 of it, in fp16 where the weight is above 2^-24 of the largest, else by 2^-40 of the largest at most; sums over n
    # tokens add n / 64 half-steps at most
    for r, length in enumerate(lengths):
        floor = 2.0 ** -40 * length * 1.6 if dtype == "fp16" else 0.0
        _close(got[r], want[r], want[r].abs() * (2.0 ** -15 + (16 + length / 64) * 2.0 ** -24) + floor)
