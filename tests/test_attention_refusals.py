"""What the attention operators refuse, on the CPU: wrong types, shapes, sizes and devices by the Python entry points, null
and inconsistent arguments by the C ABI, before anything reaches a GPU."""
import ctypes

import pytest
import torch

import dlr_lock_b200 as D
from dlr_lock_b200 import _lib
from dlr_lock_b200.build import build_library


@pytest.fixture(scope="module")
def lib():
    build_library()
    return _lib.load()


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _plan_args(**changed):
    a = dict(lengths=_i32(3), new_tokens=_i32(3), block_table=_i32(3, 4), free_pages=_i32(8), n_free=_i32(1), page_size=16)
    return {**a, **changed}


@pytest.mark.parametrize("changed,error", [
    (dict(), ValueError),                                                   # CPU tensors
    (dict(lengths=torch.zeros(3)), TypeError),
    (dict(lengths=[1, 2, 3]), TypeError),
    (dict(new_tokens=_i32(2)), ValueError),
    (dict(new_tokens=_i32(6)[::2]), ValueError),
    (dict(block_table=_i32(4, 4)), ValueError),
    (dict(block_table=_i32(4, 3).t()), ValueError),
    (dict(block_table=_i32(1, 4).expand(3, 4)), ValueError),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int64)), TypeError),
    (dict(free_pages=torch.zeros(8, dtype=torch.int64)), TypeError),
    (dict(n_free=_i32(2)), ValueError),
    (dict(page_size=8), ValueError),
    (dict(page_size=48), ValueError),
    (dict(width=0), ValueError),
    (dict(width=None), ValueError),
    (dict(width=2, rows=5), ValueError),
    (dict(finished=torch.zeros(2, dtype=torch.bool)), ValueError),
    (dict(finished=torch.zeros(3)), ValueError),
    (dict(finished=[True, False, True]), TypeError),
    (dict(page_size=2 ** 21), ValueError),
    (dict(width=None, rows=2 ** 30 + 1), ValueError),
    (dict(lengths=_i32(8193), new_tokens=_i32(8193), block_table=_i32(8193, 1)), ValueError),
])
def test_plan_refuses(changed, error):
    with pytest.raises(error):
        D.paged_plan(**_plan_args(**changed))


def _heads_args(**changed):
    bf = dict(dtype=torch.bfloat16)
    a = dict(q=torch.zeros(5, 4, 64, **bf), k=torch.zeros(5, 2, 64, **bf), q_weight=torch.ones(64, **bf), k_weight=torch.ones(64, **bf),
             cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), positions=_i32(5))
    return {**a, **changed}


HEADS = [
    (dict(), ValueError),                                                   # CPU tensors
    (dict(q=torch.zeros(5, 4, 64)), TypeError),
    (dict(k=torch.zeros(5, 2, 64, dtype=torch.float16)), TypeError),
    (dict(k=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k=torch.zeros(5, 2, 32, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(64, dtype=torch.bfloat16), k=torch.zeros(64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(5, 4, 68, dtype=torch.bfloat16), k=torch.zeros(5, 2, 68, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(5, 4, 264, dtype=torch.bfloat16), k=torch.zeros(5, 2, 264, dtype=torch.bfloat16)), ValueError),
    (dict(q_weight=torch.ones(32, dtype=torch.bfloat16)), ValueError),
    (dict(k_weight=1.0), TypeError),
    (dict(q_weight=torch.ones(64, dtype=torch.float16)), TypeError),
    (dict(q_weight=torch.ones(64)), TypeError),                             # one in bf16, one in fp32
    (dict(cos=torch.zeros(9, 40), sin=torch.zeros(9, 40)), ValueError),
    (dict(cos=torch.zeros(9, 30), sin=torch.zeros(9, 30)), ValueError),
    (dict(cos=torch.zeros(8, 32)), ValueError),
    (dict(cos=torch.zeros(9, 32, dtype=torch.bfloat16)), ValueError),
    (dict(cos=torch.zeros(9, 64)[:, ::2]), ValueError),
    (dict(positions=_i32(4)), ValueError),
    (dict(positions=torch.zeros(5)), TypeError),
]


@pytest.mark.parametrize("changed,error", HEADS)
def test_norm_rope_refuses(changed, error):
    with pytest.raises(error):
        D.qk_norm_rope(**_heads_args(**changed))


def _append_args(**changed):
    bf = dict(dtype=torch.bfloat16)
    a = _heads_args(v=torch.zeros(5, 2, 64, **bf), slots=_i32(5), k_cache=torch.zeros(3, 2, 16, 64, **bf), v_cache=torch.zeros(3, 2, 16, 64, **bf))
    return {**a, **changed}


@pytest.mark.parametrize("changed,error", HEADS + [
    (dict(v=torch.zeros(5, 4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(v=torch.zeros(5, 2, 64)), ValueError),
    (dict(slots=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(slots=_i32(4)), ValueError),
    (dict(k_cache=torch.zeros(3, 2, 16, 64)), TypeError),
    (dict(k_cache=torch.zeros(3, 1, 16, 64, dtype=torch.bfloat16), v_cache=torch.zeros(3, 1, 16, 64, dtype=torch.bfloat16)), ValueError),
    (dict(v_cache=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k_cache=torch.zeros(3, 2, 8, 64, dtype=torch.bfloat16), v_cache=torch.zeros(3, 2, 8, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k_cache=torch.zeros(3, 2, 64, 16, dtype=torch.bfloat16).transpose(2, 3)), ValueError),
])
def test_append_refuses(changed, error):
    with torch.no_grad(), pytest.raises(error):
        D.qk_norm_rope_append(**_append_args(**changed))


def test_serving_forms_refuse_gradients():
    args = _append_args()
    args["q"].requires_grad_(True)
    with pytest.raises(RuntimeError):
        D.qk_norm_rope_append(**args)
    args = _attention_args()
    args["q"].requires_grad_(True)
    with pytest.raises(RuntimeError):
        D.paged_attention(**args)


def _attention_args(**changed):
    bf = dict(dtype=torch.bfloat16)
    a = dict(q=torch.zeros(2, 4, 64, **bf), k_cache=torch.zeros(3, 2, 16, 64, **bf), v_cache=torch.zeros(3, 2, 16, 64, **bf),
             block_table=_i32(2, 5), lengths=_i32(2))
    return {**a, **changed}


@pytest.mark.parametrize("changed,error", [
    (dict(), ValueError),                                                   # CPU tensors
    (dict(q=torch.zeros(2, 4, 64)), TypeError),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.float16)), TypeError),
    (dict(q=torch.zeros(4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 0, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 4, 80, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 4, 128, dtype=torch.bfloat16)), ValueError),
    (dict(k_cache=torch.zeros(3, 2, 24, 64, dtype=torch.bfloat16), v_cache=torch.zeros(3, 2, 24, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k_cache=torch.zeros(2, 16, 64, dtype=torch.bfloat16)), ValueError),
    (dict(block_table=_i32(3, 5)), ValueError),
    (dict(block_table=_i32(5, 2).t()), ValueError),
    (dict(block_table=torch.zeros(2, 5)), TypeError),
    (dict(lengths=_i32(3)), ValueError),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), TypeError),
])
def test_attention_refuses(changed, error):
    with pytest.raises(error):
        D.paged_attention(**_attention_args(**changed))


def test_the_c_abi_refuses_before_any_cuda_call(lib):
    ref = ctypes.byref
    word = (ctypes.c_int * 64)()
    at = ctypes.cast(word, ctypes.c_void_p).value & ~63
    assert lib.dlrb200_paged_plan(None, None) == 1
    plan = dict(lengths=at, new_tokens=at, block_table=at, table_stride=4, free_pages=at, n_free=at, slots=at, positions=at, starts=at,
                lengths_out=at, n_free_out=at, requests=2, columns=4, pages=8, page_size=16, width=1, rows=2)
    for changed, code in ((dict(page_size=24), 2), (dict(page_size=8), 2), (dict(requests=8193, rows=8193), 2), (dict(rows=3), 1),
                          (dict(requests=-1), 1), (dict(n_free=None), 1), (dict(slots=None), 1), (dict(pages=1 << 28), 2),
                          (dict(block_table=None), 1)):
        assert lib.dlrb200_paged_plan(ref(_lib.PlanStep(**{**plan, **changed})), None) == code, changed

    assert lib.dlrb200_qk_norm_rope(None, None) == 1
    norm = dict(q=at, k=at, q_token=64, q_head=64, k_token=64, k_head=64, cos=at, sin=at, positions=at, q_out=at, k_out=at, tokens=1,
                q_heads=1, k_heads=1, dim=64, half=32, table_rows=1)
    for changed, code in ((dict(dim=60), 2), (dict(dim=264), 2), (dict(half=36), 2), (dict(half=30), 2), (dict(type=2), 1), (dict(q=None), 1),
                          (dict(q_out=None), 1), (dict(k_out=None), 1), (dict(slots=at), 2), (dict(slots=at, page_size=16), 1), (dict(q_head=63), 3),
                          (dict(q=at + 2), 3), (dict(cos=at + 4), 3), (dict(tokens=-1), 1), (dict(tokens=0, q=None), 0)):
        assert lib.dlrb200_qk_norm_rope(ref(_lib.NormRopeArgs(**{**norm, **changed})), None) == code, changed

    assert lib.dlrb200_qk_norm_rope_backward(None, None) == 1
    grad = dict(q=at, k=at, q_grad=at, k_grad=at, cos=at, sin=at, positions=at, dq=at, dk=at, tokens=1, q_heads=1, k_heads=1, dim=64, half=32,
                table_rows=1)
    for changed, code in ((dict(dim=4), 2), (dict(q_heads=0), 1), (dict(dq=None), 1), (dict(dq_weight=at), 1), (dict(qg_token=2), 3),
                          (dict(q_weight=at), 4), (dict(q_weight=at, q=None), 1)):
        assert lib.dlrb200_qk_norm_rope_backward(ref(_lib.NormRopeGradArgs(**{**grad, **changed})), None) == code, changed

    assert lib.dlrb200_paged_attention(None, None) == 1
    attend = dict(q=at, q_request=64, q_head=64, k_cache=at, v_cache=at, block_table=at, table_stride=1, lengths=at, out=at, requests=1,
                  heads=1, kv_heads=1, dim=64, columns=1, pages=1, page_size=16)
    for changed, code in ((dict(dim=80), 2), (dict(heads=3, kv_heads=2), 2), (dict(kv_heads=0), 2), (dict(page_size=17), 2), (dict(q=None), 1),
                          (dict(k_cache=None), 1), (dict(block_table=None), 1), (dict(kc_slot=60), 3), (dict(q_head=63), 3),
                          (dict(out=at + 8), 3), (dict(), 4), (dict(columns=1 << 27), 2), (dict(requests=-1), 1), (dict(requests=0, q=None), 0)):
        assert lib.dlrb200_paged_attention(ref(_lib.PagedAttentionArgs(**{**attend, **changed})), None) == code, changed
