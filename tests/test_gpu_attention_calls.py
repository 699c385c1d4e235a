"""Calls of the attention operators as programs make them around the edges: forward-mode tensors, odd gradients, other layouts."""
import pytest
import torch

from test_gpu_attention import DEV, _cache_case, _gen, _norm_rope_case, _normal

pytestmark = pytest.mark.gpu


def test_forward_mode_derivatives_are_refused():
    import dlr_lock_b200 as D
    import torch.autograd.forward_ad as forward_ad
    q, k, v, qw, kw, cos, sin, positions = _norm_rope_case(9, 4, 2, 64, 32, torch.bfloat16, False, True)
    kc, vc, table, n = _cache_case([40], 2, 64, 32, torch.bfloat16)
    with forward_ad.dual_level(), torch.no_grad():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for args in ((dual(q), k, qw, kw, cos, sin), (q, dual(k), qw, kw, cos, sin), (q, k, qw, dual(kw), cos, sin), (q, k, qw, kw, dual(cos), sin)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                D.qk_norm_rope(*args, positions)
        slots = torch.arange(9, dtype=torch.int32, device=DEV)
        for values, cache in ((dual(v), vc), (v, dual(vc))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                D.qk_norm_rope_append(q, k, values, qw, kw, cos, sin, positions, slots, kc, cache)
        row = _normal(_gen(0), 1, 4, 64, dtype=torch.bfloat16)
        for args in ((dual(row), kc, vc), (row, dual(kc), vc), (row, kc, dual(vc))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                D.paged_attention(*args, table, n)
        D.qk_norm_rope(q, k, qw, kw, cos, sin, positions)          # (without a tangent all is as ever)
        D.paged_attention(row, kc, vc, table, n)


def test_gradients_that_are_negated_lazily():
    # (the imaginary part of a conjugate is such a tensor)
    import dlr_lock_b200 as D
    q, k, _, qw, kw, cos, sin, positions = _norm_rope_case(40, 4, 2, 64, 32, torch.float16, False, True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, qw, kw)]
    out = D.qk_norm_rope(*leaves, cos, sin, positions)
    grads = [_normal(_gen(i), *o.shape, dtype=o.dtype) for i, o in enumerate(out)]
    want = torch.autograd.grad(out, leaves, [-g for g in grads], retain_graph=True)
    got = torch.autograd.grad(out, leaves, [torch._neg_view(g) for g in grads])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tensors_saved_through_hooks():
    import dlr_lock_b200 as D
    q, k, _, qw, kw, cos, sin, positions = _norm_rope_case(40, 4, 2, 64, 32, torch.bfloat16, False, True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, qw, kw)]
    grads = [_normal(_gen(i), *t.shape, dtype=t.dtype) for i, t in enumerate((q, k))]

    def gradient(pack, unpack):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = D.qk_norm_rope(*leaves, cos, sin, positions)
        return torch.autograd.grad(out, leaves, grads)

    want = gradient(lambda t: t, lambda t: t)

    def other_layout(t):
        return torch.stack([t, t], -1)[..., 0] if t.dim() < 3 else t.transpose(0, 1).contiguous().transpose(0, 1)

    def off_boundary(t):
        wide = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        wide[1:] = t.flatten()
        return wide[1:].view(t.shape)

    for pack, unpack in ((lambda t: t.cpu(), lambda t: t.to(DEV)), (lambda t: t, other_layout), (lambda t: t, off_boundary),
                         (lambda t: -t, lambda t: torch._neg_view(t))):
        assert all(torch.equal(a, b) for a, b in zip(gradient(pack, unpack), want))
    # what comes back as something else is refused by the host
    for unpack in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[:1], lambda t: t[None]):
        for index in range(7):
            seen = []

            def once(t):
                seen.append(t)
                return unpack(t) if len(seen) == index + 1 else t

            with pytest.raises(RuntimeError):
                gradient(lambda t: t, once)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_positions_of_one_row_for_a_batch_are_taken_as_they_are(kind):
    # what the host framework gives its layers: one row, expanded; taken by the native side, not checked and copied in Python first
    import dlr_lock_b200 as D
    from dlr_lock_b200 import attention
    q, k, v, qw, kw, cos, sin, _ = _norm_rope_case(3 * 50, 4, 2, 64, 32, torch.bfloat16, False, True)
    q, k, v = (t.unflatten(0, (3, 50)) for t in (q, k, v))
    row = torch.arange(7, 57, device=DEV, dtype=kind)[None]
    want = D.qk_norm_rope(q, k, qw, kw, cos, sin, row.repeat(3, 1))
    native = attention._native()
    got = native.qk_norm_rope(q, k, qw, kw, cos, sin, row.expand(3, 50), 1e-6, False)
    assert type(got) is tuple and all(torch.equal(a, b) for a, b in zip(got, want))
    slots = torch.arange(150, device=DEV, dtype=torch.int32).view(3, 50)
    kc, vc = torch.zeros(2, 10, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    got = native.qk_norm_rope_append(q, k, qw, kw, cos, sin, row.expand(3, 50), v, slots, kc, vc, 1e-6, False, False)
    assert torch.equal(got, want[0]) and torch.equal(kc.transpose(1, 2).flatten(0, 1)[:150], want[1].flatten(0, 1))
    leaves = [t.detach().requires_grad_(True) for t in (q, k)]
    grads = [_normal(_gen(i), *t.shape, dtype=t.dtype) for i, t in enumerate(leaves)]
    both = [torch.autograd.grad(D.qk_norm_rope(*leaves, qw, kw, cos, sin, p), leaves, grads) for p in (row.expand(3, 50), row.repeat(3, 1))]
    assert all(torch.equal(a, b) for a, b in zip(*both))


def test_plans_of_many_requests_from_two_threads():
    # through the C ABI, which a host calls without Python's lock
    import ctypes
    import threading
    from dlr_lock_b200 import _lib
    lib = _lib.load()
    refused = {}

    def plans(requests):
        def zeros(*shape):
            return torch.zeros(*shape, dtype=torch.int32, device=DEV)

        t = dict(lengths=zeros(requests), new_tokens=zeros(requests), block_table=zeros(requests, 1), free_pages=zeros(8), n_free=zeros(1),
                 slots=zeros(requests), positions=zeros(requests), starts=zeros(requests + 1), lengths_out=zeros(requests), n_free_out=zeros(1))
        step = _lib.PlanStep(**{n: x.data_ptr() for n, x in t.items()}, table_stride=1, requests=requests, columns=1, pages=8, page_size=16,
                             width=1, rows=requests)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        refused[requests] = sum(lib.dlrb200_paged_plan(ctypes.byref(step), ctypes.c_void_p(stream.cuda_stream)) != 0 for _ in range(4000))
        stream.synchronize()
        assert t["starts"].tolist() == list(range(requests + 1))

    threads = [threading.Thread(target=plans, args=(n,)) for n in (8192, 2600, 700)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert refused == {8192: 0, 2600: 0, 700: 0}


def test_append_refuses_caches_of_which_slots_share_memory():
    import dlr_lock_b200 as D
    q, k, v, qw, kw, cos, sin, positions = _norm_rope_case(9, 4, 2, 64, 32, torch.bfloat16, False, True)
    slots = torch.arange(9, dtype=torch.int32, device=DEV)
    whole = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    for shape in ((1, 2, 16, 64), (3, 1, 16, 64), (3, 2, 1, 64)):
        shared = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        for caches in ((shared.expand(3, 2, 16, 64), whole), (whole, shared.expand(3, 2, 16, 64))):
            with pytest.raises(ValueError, match="share memory"):
                D.qk_norm_rope_append(q, k, v, qw, kw, cos, sin, positions, slots, *caches)
        assert not shared.any()
    assert not whole.any()


@pytest.mark.parametrize("kind", ["expanded", "transposed", "strided", "as they are"])
def test_incoming_gradients_of_any_layout(kind):
    # four dimensions, no query norm, int32 positions; an expanded gradient has stride 0, others are read where they lie or copied
    import dlr_lock_b200 as D
    q, k, _, qw, kw, cos, sin, positions = _norm_rope_case(300, 16, 8, 128, 64, torch.bfloat16, False, True)
    leaves = [q.view(3, 100, 16, 128).detach().requires_grad_(True), k.view(3, 100, 8, 128).detach().requires_grad_(True),
              kw.detach().requires_grad_(True)]
    where = positions.view(3, 100).int()
    out = D.qk_norm_rope(leaves[0], leaves[1], None, leaves[2], cos, sin, where)
    grads = [_normal(_gen(i), *o.shape, dtype=o.dtype) for i, o in enumerate(out)]
    if kind == "expanded":
        grads = [torch.ones((), dtype=g.dtype, device=DEV).expand(g.shape) for g in grads]
    elif kind == "transposed":
        grads = [g.transpose(1, 2).contiguous().transpose(1, 2) for g in grads]
    elif kind == "strided":
        grads = [torch.stack([g, g], 3)[:, :, :, 0] for g in grads]
    got = torch.autograd.grad(out, leaves, grads)
    # 64 bits
    exact = [t.detach().double().requires_grad_(True) for t in leaves]
    c, s = cos[where.long()][:, :, None].double(), sin[where.long()][:, :, None].double()
    x = exact[1] * (exact[1].square().mean(-1, keepdim=True) + 1e-6).rsqrt() * exact[2]
    turned = []
    for t in (exact[0], x):
        a, b = t.chunk(2, -1)
        turned.append(torch.cat([a * c - b * s, b * c + a * s], -1))
    want = torch.autograd.grad(turned, exact, [g.double() for g in grads])
    for mine, its in zip(got, want):
        # rounded once; fp32 before: 128 products in each sum of a head, 2400 heads in that of the weight, half-steps of 2^-24 of the
        # sizes summed, which are below 16 times (a head) and 2400 x 16 (the weight) a gradient of 1 to 5
        sums = 2400 * 16 * 5 if its.dim() == 1 else 128 * 16 * 5
        bound = torch.finfo(mine.dtype).eps / 2 * its.abs() + sums * 2.0 ** -24
        assert ((mine.double() - its).abs() <= bound).all()


def test_inputs_that_are_negated_lazily():
    import dlr_lock_b200 as D
    q, k, v, qw, kw, cos, sin, positions = _norm_rope_case(40, 4, 2, 64, 32, torch.float16, False, True)

    def lazy(t):
        return torch._neg_view(-t)

    want = D.qk_norm_rope(q, k, qw, kw, cos, sin, positions)
    got = D.qk_norm_rope(lazy(q), lazy(k), lazy(qw), lazy(kw), lazy(cos), lazy(sin), lazy(positions))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    slots = torch.arange(40, dtype=torch.int32, device=DEV)
    caches = [torch.zeros(2, 3, 2, 16, 64, dtype=torch.float16, device=DEV) for _ in range(2)]
    D.qk_norm_rope_append(q, k, v, qw, kw, cos, sin, positions, slots, *caches[0])
    D.qk_norm_rope_append(q, k, lazy(v), qw, kw, cos, sin, positions, lazy(slots), *caches[1])
    assert torch.equal(*caches)
    kc, vc, table, n = _cache_case([40], 2, 64, 32, torch.float16)
    row = _normal(_gen(0), 1, 4, 64, dtype=torch.float16)
    want = D.paged_attention(row, kc, vc, table, n)
    assert torch.equal(D.paged_attention(lazy(row), kc, vc, lazy(table), lazy(n)), want)
    # what would be written to is refused
    with pytest.raises(ValueError, match="negated"):
        D.qk_norm_rope_append(q, k, v, qw, kw, cos, sin, positions, slots, torch._neg_view(caches[0][0]), caches[0][1])
    with pytest.raises(ValueError, match="negated"):
        D.paged_attention(row, torch._neg_view(kc), vc, table, n)
    free, count = torch.arange(4, dtype=torch.int32, device=DEV), torch.tensor([4], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="negated"):
        D.paged_plan(n, torch._neg_view(n), table, free, count, 32)
