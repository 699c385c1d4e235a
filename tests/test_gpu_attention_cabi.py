"""The attention operators through the C ABI alone, as a host without torch's headers binds them: plain structs and addresses
(here torch only owns the memory).  The same bits as the Python entry points give."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_a_step_through_the_c_abi():
    import dlr_lock_b200 as D
    from dlr_lock_b200 import _lib
    lib = _lib.load()
    gen = torch.Generator(device=DEV).manual_seed(0)
    ref = ctypes.byref
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    requests, heads, kv_heads, dim, page, pages, columns, width = 3, 8, 2, 128, 32, 40, 12, 100
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    bf = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(torch.bfloat16)  # noqa: E731
    q, k, v = (bf(requests * width, h, dim) for h in (heads, kv_heads, kv_heads))
    weight = (1 + 0.2 * torch.randn(2, dim, generator=gen, device=DEV)).to(torch.bfloat16)
    cos, sin = D.rope_tables(1e4 ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim), 300)
    new = i32([100, 7, 64])

    def state():
        return {"lengths": i32([0, 0, 0]), "table": torch.full((requests, columns), -1, dtype=torch.int32, device=DEV),
                "free": torch.arange(pages, dtype=torch.int32, device=DEV), "n_free": i32([pages]),
                "k": torch.zeros(pages, kv_heads, page, dim, dtype=torch.bfloat16, device=DEV),
                "v": torch.zeros(pages, kv_heads, page, dim, dtype=torch.bfloat16, device=DEV)}

    s = state()
    plan = D.paged_plan(s["lengths"], new, s["table"], s["free"], s["n_free"], page, width=width)
    turned = D.qk_norm_rope_append(q, k, v, weight[0], weight[1], cos, sin, plan.positions, plan.slots, s["k"], s["v"])
    out = D.paged_attention(turned[::width].contiguous(), s["k"], s["v"], s["table"], plan.lengths)

    c = state()
    slots, positions = (torch.empty(requests * width, dtype=torch.int32, device=DEV) for _ in range(2))
    starts = torch.empty(requests + 1, dtype=torch.int32, device=DEV)
    step = _lib.PlanStep(lengths=c["lengths"].data_ptr(), new_tokens=new.data_ptr(), block_table=c["table"].data_ptr(), table_stride=columns,
                         free_pages=c["free"].data_ptr(), n_free=c["n_free"].data_ptr(), slots=slots.data_ptr(), positions=positions.data_ptr(),
                         starts=starts.data_ptr(), lengths_out=c["lengths"].data_ptr(), n_free_out=c["n_free"].data_ptr(), requests=requests,
                         columns=columns, pages=pages, page_size=page, width=width, rows=requests * width)
    assert lib.dlrb200_paged_plan(ref(step), stream) == 0
    assert torch.equal(slots, plan.slots) and torch.equal(positions, plan.positions) and torch.equal(c["table"], s["table"])
    assert torch.equal(c["lengths"], plan.lengths) and torch.equal(c["n_free"], plan.n_free) and torch.equal(starts, plan.starts)

    q_out = torch.empty_like(q)
    strides = dict(kc_page=kv_heads * page * dim, kc_head=page * dim, kc_slot=dim, vc_page=kv_heads * page * dim, vc_head=page * dim, vc_slot=dim)
    args = _lib.NormRopeArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_token=heads * dim, q_head=dim, k_token=kv_heads * dim, k_head=dim,
                             v_token=kv_heads * dim, v_head=dim, q_weight=weight[0].data_ptr(), k_weight=weight[1].data_ptr(),
                             cos=cos.data_ptr(), sin=sin.data_ptr(), positions=positions.data_ptr(), q_out=q_out.data_ptr(), slots=slots.data_ptr(),
                             k_cache=c["k"].data_ptr(), v_cache=c["v"].data_ptr(), tokens=requests * width, q_heads=heads, k_heads=kv_heads,
                             dim=dim, half=dim // 2, table_rows=300, pages=pages, page_size=page, eps=1e-6, **strides)
    assert lib.dlrb200_qk_norm_rope(ref(args), stream) == 0
    assert torch.equal(q_out, turned) and torch.equal(c["k"], s["k"]) and torch.equal(c["v"], s["v"])

    need = lib.dlrb200_paged_attention_workspace_bytes(heads, kv_heads, dim)
    assert need > 0
    workspace = torch.empty(need, dtype=torch.uint8, device=DEV)
    got = torch.empty(requests, heads, dim, dtype=torch.bfloat16, device=DEV)
    call = dict(q=q_out.data_ptr(), q_request=width * heads * dim, q_head=dim, k_cache=c["k"].data_ptr(), v_cache=c["v"].data_ptr(),
                block_table=c["table"].data_ptr(), table_stride=columns, lengths=c["lengths"].data_ptr(), out=got.data_ptr(),
                workspace=workspace.data_ptr(), workspace_bytes=need, requests=requests, heads=heads, kv_heads=kv_heads, dim=dim,
                columns=columns, pages=pages, page_size=page, scale=dim ** -0.5, **strides)
    assert lib.dlrb200_paged_attention(ref(_lib.PagedAttentionArgs(**call)), stream) == 0
    assert torch.equal(got, out)
    assert lib.dlrb200_paged_attention(ref(_lib.PagedAttentionArgs(**{**call, "workspace_bytes": need - 1})), stream) == 4
    assert lib.dlrb200_paged_attention(ref(_lib.PagedAttentionArgs(**{**call, "workspace": workspace.data_ptr() + 8})), stream) == 3

    # the gradient
    leaves = [t.detach().requires_grad_(True) for t in (q, k, weight[0], weight[1])]
    grads = [bf(*t.shape) for t in (q, k)]
    want = torch.autograd.grad(D.qk_norm_rope(*leaves, cos, sin, positions), leaves, grads)
    mine = [torch.empty_like(t) for t in (q, k, weight[0], weight[1])]
    need = lib.dlrb200_qk_norm_rope_backward_workspace_bytes(dim)
    workspace = torch.empty(need, dtype=torch.uint8, device=DEV)
    args = _lib.NormRopeGradArgs(q=q.data_ptr(), k=k.data_ptr(), q_grad=grads[0].data_ptr(), k_grad=grads[1].data_ptr(), q_token=heads * dim,
                                 q_head=dim, k_token=kv_heads * dim, k_head=dim, qg_token=heads * dim, qg_head=dim, kg_token=kv_heads * dim,
                                 kg_head=dim, q_weight=weight[0].data_ptr(), k_weight=weight[1].data_ptr(), cos=cos.data_ptr(), sin=sin.data_ptr(),
                                 positions=positions.data_ptr(), dq=mine[0].data_ptr(), dk=mine[1].data_ptr(), dq_weight=mine[2].data_ptr(),
                                 dk_weight=mine[3].data_ptr(), workspace=workspace.data_ptr(), workspace_bytes=need, tokens=requests * width,
                                 q_heads=heads, k_heads=kv_heads, dim=dim, half=dim // 2, table_rows=300, eps=1e-6)
    assert lib.dlrb200_qk_norm_rope_backward(ref(args), stream) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(mine, want))
