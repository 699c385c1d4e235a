"""Calls of the attention operators that are refused by name rather than answered wrongly, on the CPU."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import dlr_lock_b200 as D
from test_attention_refusals import _append_args, _attention_args, _heads_args, _plan_args


@pytest.mark.parametrize("call,args,names", [
    (D.qk_norm_rope, _heads_args, ("q", "k", "q_weight", "k_weight", "cos")),
    (D.qk_norm_rope_append, _append_args, ("q", "k", "v", "q_weight", "sin", "k_cache")),
    (D.paged_attention, _attention_args, ("q", "k_cache", "v_cache")),
])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(call, args, names, grad):
    # a tangent would be dropped without a word (torch.no_grad() does not switch forward mode off)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for name in names:
            given = args()
            given[name] = forward_ad.make_dual(given[name], torch.ones_like(given[name]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(**given)
        with pytest.raises(ValueError, match="CUDA"):              # (no tangent: the next check)
            call(**args())


class _NoTruth:
    def __bool__(self):
        raise ValueError("neither true nor false")


@pytest.mark.parametrize("call,args,name", [
    (D.qk_norm_rope, _heads_args, "interleaved"),
    (D.qk_norm_rope_append, _append_args, "interleaved"),
    (D.qk_norm_rope_append, _append_args, "return_keys"),
    (D.paged_plan, _plan_args, "in_place"),
])
def test_a_flag_without_a_truth_value_raises_its_own_error(call, args, name):
    with torch.no_grad(), pytest.raises(ValueError, match="neither true nor false"):
        call(**args(), **{name: _NoTruth()})


@pytest.mark.parametrize("name", ["k_cache", "v_cache"])
@pytest.mark.parametrize("shape", [(1, 2, 16, 64), (3, 1, 16, 64), (3, 2, 1, 64)])
def test_append_refuses_caches_of_which_slots_share_memory(name, shape):
    shared = torch.zeros(shape, dtype=torch.bfloat16).expand(3, 2, 16, 64)
    with torch.no_grad(), pytest.raises(ValueError, match="share memory"):
        D.qk_norm_rope_append(**_append_args(**{name: shared}))


def test_the_c_abi_refuses_tables_whose_rows_overlap():
    import ctypes
    from dlr_lock_b200 import _lib
    from dlr_lock_b200.build import build_library
    build_library()
    lib = _lib.load()
    word = (ctypes.c_int * 64)()
    at = ctypes.cast(word, ctypes.c_void_p).value & ~63
    plan = dict(lengths=at, new_tokens=at, block_table=at, free_pages=at, n_free=at, slots=at, positions=at, starts=at, lengths_out=at,
                n_free_out=at, requests=2, columns=4, pages=8, page_size=16, width=1, rows=2)
    for stride in (0, 3, -4):
        assert lib.dlrb200_paged_plan(ctypes.byref(_lib.PlanStep(**plan, table_stride=stride)), None) == 1


@pytest.mark.parametrize("name", ["cos", "sin"])
def test_append_names_tables_that_want_a_gradient(name):
    given = _append_args()
    given[name].requires_grad_(True)
    with pytest.raises(RuntimeError, match="has no gradient"):
        D.qk_norm_rope_append(**given)


def test_the_c_abi_refuses_integers_off_their_boundaries():
    import ctypes
    from dlr_lock_b200 import _lib
    from dlr_lock_b200.build import build_library
    build_library()
    lib, ref = _lib.load(), ctypes.byref
    word = (ctypes.c_int * 64)()
    at = ctypes.cast(word, ctypes.c_void_p).value & ~63
    plan = dict(lengths=at, new_tokens=at, block_table=at, table_stride=4, free_pages=at, n_free=at, slots=at, positions=at, starts=at,
                lengths_out=at, n_free_out=at, requests=2, columns=4, pages=8, page_size=16, width=1, rows=2)
    for name in [n for n, v in plan.items() if v == at]:
        assert lib.dlrb200_paged_plan(ref(_lib.PlanStep(**{**plan, name: at + 2})), None) == 3, name
    heads = dict(cos=at, sin=at, positions=at, tokens=1, q_heads=1, k_heads=1, dim=64, half=32, table_rows=1)
    norm = dict(heads, q=at, k=at, v=at, q_out=at, k_out=at, slots=at, k_cache=at, v_cache=at, pages=1, page_size=16)
    grad = dict(heads, q=at, k=at, q_grad=at, k_grad=at, dq=at, dk=at)
    for changed in (dict(positions=at + 2), dict(positions=at + 4, positions_64=1), dict(positions_64=1, positions=at + 1)):
        assert lib.dlrb200_qk_norm_rope(ref(_lib.NormRopeArgs(**{**norm, **changed})), None) == 3, changed
        assert lib.dlrb200_qk_norm_rope_backward(ref(_lib.NormRopeGradArgs(**{**grad, **changed})), None) == 3, changed
    assert lib.dlrb200_qk_norm_rope(ref(_lib.NormRopeArgs(**{**norm, "slots": at + 2})), None) == 3
    for changed in (dict(dq_weight=at + 1), dict(dk_weight=at + 1), dict(dk_weight=at + 2, weights_f32=1)):
        weights = dict(q_weight=at, k_weight=at, workspace=at, workspace_bytes=1 << 40)
        assert lib.dlrb200_qk_norm_rope_backward(ref(_lib.NormRopeGradArgs(**{**grad, **weights, **changed})), None) == 3, changed
    attend = dict(q=at, q_request=64, q_head=64, k_cache=at, v_cache=at, block_table=at, table_stride=1, lengths=at, out=at, requests=1,
                  heads=1, kv_heads=1, dim=64, columns=1, pages=1, page_size=16)
    for name in ("block_table", "lengths"):
        assert lib.dlrb200_paged_attention(ref(_lib.PagedAttentionArgs(**{**attend, name: at + 2})), None) == 3, name
