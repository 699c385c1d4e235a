"""What smoke() checks can fail: its comparison of gradients, on the CPU, with the operator's place taken by torch's own
arithmetic and by broken forms of it."""
import types

import pytest
import torch

import __graft_entry__ as entry
import dlr_lock_b200 as D


class _NormRope(torch.autograd.Function):
    """Norm and rotation in torch, with the gradient of one input replaced by zeros."""

    @staticmethod
    def forward(ctx, broken, q, k, q_weight, k_weight, cos, sin, positions):
        ctx.broken = broken
        with torch.enable_grad():
            ctx.leaves = [t.detach().double().requires_grad_(True) for t in (q, k, q_weight, k_weight)]
            c, s = cos[positions.long()][:, None].double(), sin[positions.long()][:, None].double()
            ctx.outs = []
            for x, w in zip(ctx.leaves[:2], ctx.leaves[2:]):
                a, b = (x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w).chunk(2, -1)
                ctx.outs.append(torch.cat([a * c - b * s, b * c + a * s], -1))
        return tuple(o.detach().to(q.dtype) for o in ctx.outs)

    @staticmethod
    def backward(ctx, *grads):
        got = list(torch.autograd.grad(ctx.outs, ctx.leaves, [g.double() for g in grads]))
        if ctx.broken is not None:
            got[ctx.broken] = torch.zeros_like(got[ctx.broken])
        return (None, *(g.to(torch.bfloat16) for g in got), None, None, None)


@pytest.mark.parametrize("broken", [None, 0, 1, 2, 3])
def test_a_gradient_of_zeros_fails_the_smoke(broken):
    torch.manual_seed(0)
    q, k = (torch.randn(20, h, 64).to(torch.bfloat16) for h in (4, 2))
    cos, sin = D.rope_tables(1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64), 50)
    fake = types.SimpleNamespace(qk_norm_rope=lambda *a: _NormRope.apply(broken, *a))
    positions = torch.randint(0, 50, (20,), dtype=torch.int32)
    if broken is None:
        entry._smoke_gradient(fake, q, k, cos, sin, positions)
    else:
        with pytest.raises(AssertionError):
            entry._smoke_gradient(fake, q, k, cos, sin, positions)
