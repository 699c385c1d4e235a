"""Paged attention where values are far apart: weights far below the largest one, and infinite values that a request holds."""
import pytest
import torch

from test_gpu_attention import DEV, TYPES, _attend64, _cache_case, _close, _gen, _normal

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


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 2, 2), (96, 9, 1), (128, 8, 1), (128, 40, 2), (256, 3, 1), (256, 16, 1)])
@pytest.mark.parametrize("columns", [None, 900])
def test_infinite_values_that_a_request_holds(dtype, dim, heads, kv_heads, columns):
    # weights are positive, so a column of values with +inf gives +inf, with -inf -inf, with both or with NaN NaN, whatever the
    # weights' bits are; the other columns are as they would be without
    import dlr_lock_b200 as D
    lengths = [1, 5, 64, 200, 700, 0, 3000 if columns else 300]
    kc, vc, table, n = _cache_case(lengths, kv_heads, dim, 32, TYPES[dtype], columns=columns)
    q = _normal(_gen(heads), len(lengths), heads, dim, dtype=TYPES[dtype], std=0.7)
    want, extra = _attend64(q, kc, vc, table, lengths, dim ** -0.5)
    inf = float("inf")
    for r, length in enumerate(lengths):
        for t in range(0, length, max(1, length // 7)):
            page, slot = table[r, t // 32].long(), t % 32
            vc[page, :, slot, 3], vc[page, :, slot, dim - 6] = inf, -inf
            vc[page, :, slot, 8] = inf if t else -inf
        for t in range(length // 2, length, 97):
            vc[table[r, t // 32].long(), :, t % 32, 17] = float("nan")
    got = D.paged_attention(q, kc, vc, table, n)
    held = torch.tensor([length > 0 for length in lengths], device=DEV)
    both = torch.tensor([length > 1 for length in lengths], device=DEV)
    assert (got[held][..., 3] == inf).all() and (got[held][..., dim - 6] == -inf).all()
    assert torch.isnan(got[both][..., 8]).all() and (got[0, :, 8] == -inf).all() and torch.isnan(got[held][..., 17]).all()
    assert not got[~held].any()
    rest = [c for c in range(dim) if c not in (3, 8, 17, dim - 6)]
    _close(got[..., rest], want[..., rest], extra)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lengths", [[500], [40000]])
def test_an_infinite_value_of_a_small_weight(dtype, lengths):
    # e^-30 beside the largest weight: 2^-43, which no term of 16 bits holds in fp16.  One such token stands in the same 16 as the
    # largest weight, one in a later step, one far away
    import dlr_lock_b200 as D
    q, kc, vc, table, n = _one_key_above_the_rest(30.0, lengths, 4, 2, dtype)
    for t, column in ((5, 5), (131, 6), (lengths[0] // 3, 7)):
        vc[table[0, t // 64].long(), :, t % 64, column] = float("inf")
    got = D.paged_attention(q, kc, vc, table, n, scale=1.0)
    assert (got[..., 5:8] == float("inf")).all() and torch.isfinite(got[..., :5]).all() and torch.isfinite(got[..., 8:]).all()
