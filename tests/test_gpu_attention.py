"""The attention block on a paged cache, each operator against its formula in 64 bits.

Tolerances: an output is rounded once to its type, off by at most eps / 2 of its value; what the fp32 arithmetic before adds is
bounded beside each comparison.
"""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
F32 = 2.0 ** -24                                     # half a step of fp32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)


def _close(got, want, extra):
    """|got - want| <= eps / 2 |want| + extra (a tensor or a number); subnormals of the type are rounded to absolute steps."""
    assert torch.isfinite(got.double()).all()
    kind = torch.finfo(got.dtype)
    bound = kind.eps / 2 * want.abs() + extra + kind.smallest_normal * kind.eps
    off = (got.double() - want).abs() - bound
    assert (off <= 0).all(), f"worst excess {off.max().item():.3g}, at want {want.flatten()[off.argmax()].item():.4g}"


# ---- plan -------------------------------------------------------------------------------------------------------------------
def _plan_by_hand(lengths, new, table, free, n_free, page, width, rows, finished):
    """The documented semantics, one request after the other."""
    table, free = [list(r) for r in table], list(free)
    columns = len(table[0]) if table else 0
    pages = lambda n: -(-n // page)  # noqa: E731
    lengths = [min(max(n, 0), columns * page) for n in lengths]
    if finished:
        for r, done in enumerate(finished):
            if done:
                for c in range(pages(lengths[r])):
                    free[n_free] = table[r][c]
                    n_free += 1
                lengths[r] = 0
    slots, positions, starts, after, asked, used, row = [-1] * rows, [0] * rows, [], [], 0, 0, 0
    for r, old in enumerate(lengths):
        n = max(new[r], 0)
        start = r * width if width else row
        row += n
        starts.append(start)
        possible = old + n <= columns * page and (n <= width if width else row <= rows)
        room = old + n <= columns * page and (not width or n <= width)
        need = pages(old + n) - pages(old) if room else 0
        first, asked = asked, asked + need
        if possible and (need == 0 or asked <= n_free):
            for i in range(need):
                table[r][pages(old) + i] = free[n_free - 1 - first - i]
            used = max(used, asked) if need else used
            for j in range(n):
                slots[start + j] = table[r][(old + j) // page] * page + (old + j) % page
                positions[start + j] = old + j
            after.append(old + n)
        else:
            after.append(old)
    starts.append(len(lengths) * width if width else row)
    return slots, positions, starts, after, n_free - used, table, free


def _run_plan(lengths, new, table, free, n_free, page, width=1, rows=None, finished=None, in_place=False):
    import dlr_lock_b200 as D
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    t = {"lengths": i32(lengths), "new": i32(new), "table": i32(table).reshape(len(lengths), -1), "free": i32(free), "n_free": i32([n_free])}
    done = None if finished is None else torch.tensor(finished, dtype=torch.bool, device=DEV)
    got = D.paged_plan(t["lengths"], t["new"], t["table"], t["free"], t["n_free"], page, width=width, rows=rows, finished=done, in_place=in_place)
    want = _plan_by_hand(lengths, new, table, free, n_free, page, width or 0, rows if width is None else width * len(lengths), finished)
    for name, g, w in zip(("slots", "positions", "starts", "lengths", "n_free", "table"),
                          (got.slots, got.positions, got.starts, got.lengths, got.n_free, t["table"]), want):
        assert g.dtype == torch.int32
        assert g.flatten().tolist() == (w if isinstance(w, list) and (not w or not isinstance(w[0], list)) else
                                        [x for row in w for x in row] if isinstance(w, list) else [w]), name
    # the free part of the stack and what lies under it
    assert t["free"].tolist()[:want[4]] == want[6][:want[4]]
    if in_place:
        assert got.lengths.data_ptr() == t["lengths"].data_ptr() and got.n_free.data_ptr() == t["n_free"].data_ptr()
    else:
        assert t["lengths"].tolist() == lengths and t["n_free"].tolist() == [n_free]
    return got


def _random_state(rng, requests, columns, page, spare):
    lengths = [rng.choice([0, 0, 1, page - 1, page, page + 1, rng.randint(0, columns * page)]) for _ in range(requests)]
    lengths = [min(n, columns * page) for n in lengths]
    held = sum(-(-n // page) for n in lengths)
    ids = list(range(held + spare))
    rng.shuffle(ids)
    table, at = [], 0
    for n in lengths:
        h = -(-n // page)
        table.append(ids[at:at + h] + [-1] * (columns - h))
        at += h
    return lengths, table, ids[held:] + [-7] * held, spare


@pytest.mark.parametrize("requests", [1, 2, 31, 512, 513, 1500])
@pytest.mark.parametrize("page,width", [(16, 1), (64, 1), (16, 40), (128, 3), (32, None)])
@pytest.mark.parametrize("finishing", [False, True])
def test_plan(requests, page, width, finishing):
    rng = random.Random(requests * 1000 + page + (width or 0) + finishing)
    columns = rng.choice([1, 3, 9])
    for spare in (0, requests // 2 + 1, 10 * requests):        # refusals for want of pages, some of them, none
        lengths, table, free, n_free = _random_state(rng, requests, columns, page, spare)
        most = width or 50
        new = [rng.choice([0, 1, most, most + 1, rng.randint(0, most), -3]) for _ in range(requests)]
        rows = None if width else max(0, sum(max(n, 0) for n in new) - rng.choice([0, 0, 5]) + rng.choice([0, 7]))
        finished = [rng.random() < 0.4 for _ in range(requests)] if finishing else None
        _run_plan(lengths, new, table, free, n_free, page, width, rows, finished, in_place=rng.random() < 0.5)


@pytest.mark.parametrize("width", [5000, None])
def test_plan_of_long_prompts(width):
    # many rows: the cluster's form; one long prompt among short ones, a finished request whose pages come back first
    lengths, table, free, n_free = _random_state(random.Random(1), 7, 400, 16, 2000)
    new = [4999, 0, 1, 5000, 17, 16, 3000]
    _run_plan(lengths, new, table, free, n_free, 16, width, None if width else sum(new) + 3, [True, False, False, True, False, False, False])
    _run_plan([100000], [1], [list(range(6250)) + [-1]], [6250, 6251], 2, 16)


def test_plan_of_nothing_and_of_broken_lengths():
    import dlr_lock_b200 as D
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    plan = D.paged_plan(none, none, none.view(0, 4), torch.arange(3, dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV), 16)
    assert plan.slots.numel() == 0 and plan.starts.tolist() == [0] and plan.n_free.tolist() == [3]
    plan = D.paged_plan(none, none, none.view(0, 4), none, torch.tensor([0], dtype=torch.int32, device=DEV), 16, width=None, rows=5)
    assert plan.slots.tolist() == [-1] * 5
    # lengths outside 0 .. columns x page, a count of free pages beyond the stack: held to their range
    _run_plan([-5, 64], [3, 0], [[-1, -1], [0, 1]], [5, 6], 2, 16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    plan = D.paged_plan(i32([0]), i32([20]), i32([[-1, -1]]), i32([4, 5]), i32([99]), 16, width=32)
    assert plan.n_free.tolist() == [0] and plan.slots.tolist()[:20] == [5 * 16 + j for j in range(16)] + [4 * 16 + j for j in range(4)]


# ---- norm and rotation ------------------------------------------------------------------------------------------------------
def _tables(far, half, gen):
    angle = torch.rand(far, half, generator=gen, device=DEV, dtype=torch.float64) * 100 - 50
    return angle.cos().float(), angle.sin().float()


def _norm_rope64(x, w, c, s, interleaved, eps):
    """x (tokens, heads, dim) in 64 bits; c, s (tokens, half)."""
    if w is not None:
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
    half = c.shape[1]
    c, s = c[:, None], s[:, None]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    return y


def _norm_rope_case(tokens, heads, kv_heads, dim, half, dtype, interleaved, normed, weights_f32=False, strided=False, seed=0):
    gen = _gen(seed + tokens + heads + dim)
    if strided:                                     # as one product for all three gives them, with a gap behind each row
        qkv = _normal(gen, tokens, (heads + 2 * kv_heads) * dim + 8, dtype=dtype, std=2.0)
        q, k, v, _ = qkv.split([heads * dim, kv_heads * dim, kv_heads * dim, 8], -1)
        q, k, v = (t.unflatten(-1, (-1, dim)) for t in (q, k, v))
    else:
        q, k, v = (_normal(gen, tokens, h, dim, dtype=dtype, std=2.0) for h in (heads, kv_heads, kv_heads))
    wt = torch.float32 if weights_f32 else dtype
    qw, kw = ((1 + 0.3 * _normal(gen, dim)).to(wt) if normed else None for _ in range(2))
    cos, sin = _tables(97, half, gen)
    positions = torch.randint(0, 97, (tokens,), generator=gen, device=DEV)
    return q, k, v, qw, kw, cos, sin, positions


SHAPES = [(1, 1, 1, 64, 32), (7, 16, 8, 128, 64), (33, 12, 4, 96, 24), (3, 5, 1, 256, 128), (130, 9, 3, 64, 16), (2, 3, 2, 8, 4),
          (5, 24, 6, 80, 40), (64, 2, 2, 200, 0), (1000, 32, 8, 128, 64)]


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,half", SHAPES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed", [False, True])
def test_norm_rope_and_gradient(tokens, heads, kv_heads, dim, half, dtype, interleaved, normed):
    import dlr_lock_b200 as D
    strided, weights_f32 = heads % 2 == 1, tokens % 2 == 0
    q, k, _, qw, kw, cos, sin, positions = _norm_rope_case(tokens, heads, kv_heads, dim, half, TYPES[dtype], interleaved, normed, weights_f32, strided)
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, qw, kw)]
    out = D.qk_norm_rope(*leaves, cos, sin, positions, eps=1e-5, interleaved=interleaved)
    gen = _gen(dim)
    grads = [_normal(gen, *o.shape, dtype=o.dtype) for o in out]
    got = torch.autograd.grad(out, [t for t in leaves if t is not None], grads)
    c, s = cos[positions].double(), sin[positions].double()
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        x64 = x.double().requires_grad_(True)
        w64 = w.double().requires_grad_(True) if w is not None else None
        want = _norm_rope64(x64, w64, c, s, interleaved, 1e-5)
        # fp32: the mean of squares over dim / 8 lanes of 8 (16 steps at most), then about eight operations, each half a step
        # of values up to the two partners' sum
        reach = want.detach().abs().amax(-1, keepdim=True) * 2
        _close(out[i].detach(), want.detach(), 32 * F32 * reach)
        dx, *dw = torch.autograd.grad(want, [x64] + ([w64] if w is not None else []), grads[i].double())
        if w is None:
            _close(got[i], dx, 8 * F32 * grads[i].double().abs().amax() * 2)
        else:
            # dx = rstd (g w - u mean(g w u)): each term is at most rstd times the largest g w times (1 + max u mean|u|)
            rstd = torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + 1e-5)
            u = x.double() * rstd
            gw = 2 * grads[i].double().abs().amax(-1, keepdim=True) * w.double().abs().max()
            _close(got[i], dx, 64 * F32 * rstd * gw * (1 + u.abs().amax(-1, keepdim=True)))
            # the weight's gradient: at most tokens x heads terms in chains of fp32 sums
            terms = (2 * grads[i].double().abs().amax(-1, keepdim=True) * u.abs()).sum((0, 1))
            _close(got[2 + i], dw[0], 64 * F32 * terms)


def test_norm_rope_gradient_against_differences():
    import dlr_lock_b200 as D
    q, k, _, qw, kw, cos, sin, positions = _norm_rope_case(9, 4, 2, 64, 16, torch.bfloat16, False, True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, qw, kw)]
    out = D.qk_norm_rope(*leaves, cos, sin, positions)
    gen = _gen(3)
    grads = [_normal(gen, *o.shape, dtype=o.dtype) for o in out]
    got = torch.autograd.grad(out, leaves, grads)
    c, s = cos[positions].double(), sin[positions].double()

    def loss(values):
        return sum((_norm_rope64(x, w, c, s, False, 1e-6) * g.double()).sum() for x, w, g in zip(values[:2], values[2:], grads))

    for i, g in enumerate(got):
        for _ in range(4):
            d = _normal(gen, *g.shape).double()
            step = 1e-4
            up, down = ([v.detach().double() + (sign * step * d if j == i else 0) for j, v in enumerate(leaves)] for sign in (1, -1))
            slope = (loss(up) - loss(down)) / (2 * step)
            # the gradient is rounded to bf16; the quotient is off by about step^2
            assert abs(slope - (g.double() * d).sum()) <= (g.double() * d).abs().sum() * 2.0 ** -8 + 1e-4


def test_gradients_of_part_of_the_outputs_and_repeats():
    import dlr_lock_b200 as D
    q, k, _, qw, kw, cos, sin, positions = _norm_rope_case(300, 16, 8, 128, 64, torch.bfloat16, False, True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, qw, kw)]
    runs = []
    for _ in range(2):
        out = D.qk_norm_rope(*leaves, cos, sin, positions)
        runs.append(torch.autograd.grad(out[0].float().square().sum(), leaves, allow_unused=True))
    assert all(torch.equal(a, b) for a, b in zip(*runs))                      # sums in a fixed order
    assert not runs[0][1].any() and not runs[0][3].any()                      # nothing came in for the keys
    # an expanded gradient (stride 0), an input of more dimensions
    out = D.qk_norm_rope(q.view(3, 100, 16, 128).detach().requires_grad_(True), k.view(3, 100, 8, 128), None, kw, cos, sin, positions.view(3, 100).int())
    out[0].sum().backward()
    assert out[0].shape == (3, 100, 16, 128)


def test_norm_rope_of_no_tokens_of_layouts_that_are_copied_and_twice():
    import dlr_lock_b200 as D
    q, k, v, qw, kw, cos, sin, positions = _norm_rope_case(24, 4, 2, 64, 32, torch.float16, True, True)
    # no tokens: empty outputs, gradients of zero
    leaves = [t.detach().requires_grad_(True) for t in (q[:0], k[:0], qw, kw)]
    out = D.qk_norm_rope(*leaves, cos, sin, positions[:0])
    got = torch.autograd.grad(out, leaves, [torch.zeros_like(o) for o in out])
    assert [tuple(o.shape) for o in out] == [(0, 4, 64), (0, 2, 64)] and not got[2].any() and not got[3].any()
    cache = torch.zeros(1, 2, 16, 64, dtype=torch.float16, device=DEV)
    assert D.qk_norm_rope_append(q[:0], k[:0], v[:0], qw, kw, cos, sin, positions[:0], positions[:0].int(), cache, cache.clone()).shape == (0, 4, 64)
    # what cannot be read where it lies gives the same bits: other orders, a weight and rows off their boundaries
    want = D.qk_norm_rope(q, k, qw, kw, cos, sin, positions, interleaved=True)
    off = torch.empty(65, dtype=torch.float16, device=DEV)[1:].copy_(qw)
    wide = torch.empty(24, 4 * 64 + 1, dtype=torch.float16, device=DEV)
    wide[:, 1:] = q.flatten(1)
    for q2, w2 in ((q.transpose(0, 1).contiguous().transpose(0, 1), qw), (q.transpose(1, 2).contiguous().transpose(1, 2), off),
                   (wide[:, 1:].unflatten(-1, (4, 64)), qw)):
        got = D.qk_norm_rope(q2, k, w2, kw, cos, sin, positions, interleaved=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    batched = q.view(4, 6, 4, 64).transpose(0, 1), k.view(4, 6, 2, 64).transpose(0, 1), positions.view(4, 6).t()      # (6, 4, ...)
    leaf = batched[0].detach().requires_grad_(True)
    got = D.qk_norm_rope(leaf, batched[1], qw, kw, cos, sin, batched[2], interleaved=True)
    assert torch.equal(got[0], want[0].view(4, 6, 4, 64).transpose(0, 1))
    g = torch.autograd.grad(got[0].float().sum(), leaf)[0]
    straight = q.detach().requires_grad_(True)
    assert torch.equal(g, torch.autograd.grad(D.qk_norm_rope(straight, k, qw, kw, cos, sin, positions, interleaved=True)[0].float().sum(),
                                              straight)[0].view(4, 6, 4, 64).transpose(0, 1))
    # a gradient of the gradient is refused, not taken for zero
    leaf = q.detach().requires_grad_(True)
    once = torch.autograd.grad(D.qk_norm_rope(leaf, k, qw, kw, cos, sin, positions)[0].float().square().sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(once.float().sum(), leaf)


@pytest.mark.parametrize("lead", [(2, 0), (0, 2), (2, 0, 3), (0,)])
def test_norm_rope_of_empty_batches(lead):
    import dlr_lock_b200 as D
    q, k, v, qw, kw, cos, sin, positions = _norm_rope_case(1, 4, 2, 64, 32, torch.bfloat16, False, True)
    empty = [t.new_empty(*lead, *t.shape[1:]) for t in (q, k, v)]
    where = torch.empty(lead, dtype=torch.int32, device=DEV)
    leaves = [t.detach().requires_grad_(True) for t in (empty[0], empty[1], qw, kw)]
    out = D.qk_norm_rope(*leaves, cos, sin, where)
    got = torch.autograd.grad(out, leaves, [torch.zeros_like(o) for o in out])
    assert [g.shape for g in got] == [t.shape for t in leaves] and out[0].shape == empty[0].shape and out[1].shape == empty[1].shape
    assert not got[2].any() and not got[3].any()
    cache = torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    assert D.qk_norm_rope_append(*empty, qw, kw, cos, sin, where, where, cache, cache.clone()).shape == empty[0].shape


def test_norm_rope_gradient_captured():
    import dlr_lock_b200 as D
    q, k, _, qw, kw, cos, sin, positions = _norm_rope_case(200, 8, 2, 128, 64, torch.bfloat16, False, True)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, qw, kw)]
    gen = _gen(9)
    grads = [_normal(gen, *t.shape, dtype=t.dtype) for t in (q, k)]

    def step():
        out = D.qk_norm_rope(*leaves, cos, sin, positions)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, grads))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_norm_rope_positions_outside_the_tables_give_nan_rows():
    import dlr_lock_b200 as D
    q, k, v, qw, kw, cos, sin, positions = _norm_rope_case(6, 4, 2, 64, 16, torch.float16, False, True)
    positions[1], positions[4] = -1, cos.shape[0]
    a, b = D.qk_norm_rope(q, k, qw, kw, cos, sin, positions)
    for t in (a, b):
        assert torch.isnan(t[[1, 4]]).all() and torch.isfinite(t[[0, 2, 3, 5]]).all()


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,half", SHAPES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("order", ["heads first", "tokens first"])
def test_append(tokens, heads, kv_heads, dim, half, dtype, order):
    import dlr_lock_b200 as D
    interleaved, normed, page = dim % 64 == 0, heads % 2 == 0, 16 if tokens % 2 else 64
    q, k, v, qw, kw, cos, sin, positions = _norm_rope_case(tokens, heads, kv_heads, dim, half, TYPES[dtype], interleaved, normed, strided=True)
    pages = -(-tokens // page) + 2
    gen = _gen(tokens)
    slots = torch.randperm(pages * page, generator=gen, device=DEV)[:tokens].int()
    if tokens > 2:
        slots[1], slots[2] = -1, pages * page                # rows without a place
    shape = (pages, kv_heads, page, dim) if order == "heads first" else (pages, page, kv_heads, dim)
    caches = [_normal(gen, *shape, dtype=TYPES[dtype]) for _ in range(2)]
    before = [c.clone() for c in caches]
    kc, vc = caches if order == "heads first" else [c.transpose(1, 2) for c in caches]
    got = D.qk_norm_rope_append(q, k, v, qw, kw, cos, sin, positions.int(), slots, kc, vc, eps=1e-5, interleaved=interleaved)
    # the same bits as the form without a cache
    want_q, want_k = D.qk_norm_rope(q, k, qw, kw, cos, sin, positions, eps=1e-5, interleaved=interleaved)
    assert torch.equal(got, want_q)
    at = (slots >= 0) & (slots < pages * page)
    slot = slots[at].long()
    for cache, old, rows in zip((kc, vc), before, (want_k, v)):
        assert torch.equal(cache.transpose(1, 2)[slot // page, slot % page], rows[at])
        changed = (cache.transpose(1, 2) != (old if order == "tokens first" else old.transpose(1, 2))).any(-1).any(-1).flatten()
        changed[slot] = False
        assert not changed.any()                             # everything else as it was
    both = D.qk_norm_rope_append(q, k, v, qw, kw, cos, sin, positions, slots, *(c.clone() for c in (kc, vc)), eps=1e-5,
                                 interleaved=interleaved, return_keys=True)
    assert torch.equal(both[0], want_q) and torch.equal(both[1], want_k)


# ---- attention --------------------------------------------------------------------------------------------------------------
def _cache_case(lengths, kv_heads, dim, page, dtype, seed=0, columns=None, fill=None, order="heads first"):
    """Caches with each request's tokens on shuffled pages; what no request holds is `fill`."""
    gen = _gen(seed)
    have = [-(-n // page) for n in lengths]
    total = sum(have) + 2
    ids = torch.randperm(total, generator=gen, device=DEV).int()
    columns = columns or max(1, max(have, default=1))
    table = torch.full((len(lengths), columns), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    at = 0
    shape = (total, kv_heads, page, dim) if order == "heads first" else (total, page, kv_heads, dim)
    caches = [_normal(gen, *shape, dtype=dtype) for _ in range(2)]
    if order != "heads first":
        caches = [c.transpose(1, 2) for c in caches]
    for r, h in enumerate(have):
        table[r, :h] = ids[at:at + h]
        at += h
    if fill is not None:
        keep = torch.zeros(total, page, dtype=torch.bool, device=DEV)
        for r, n in enumerate(lengths):
            j = torch.arange(n, device=DEV)
            keep[table[r, j // page].long(), j % page] = True
        for c in caches:
            c.transpose(1, 2)[~keep] = fill
    return (*caches, table, torch.tensor(lengths, dtype=torch.int32, device=DEV))


def _attend64(q, kc, vc, table, lengths, scale):
    """Outputs in 64 bits and a bound on what fp32 scores and weights add."""
    out, extra = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    kv_heads, page, dim = kc.shape[1:]
    for r, n in enumerate(lengths):
        if n == 0:
            continue
        pages = table[r, :-(-n // page)].long()
        k, v = (c[pages].transpose(0, 1).flatten(1, 2)[:, :n].double() for c in (kc, vc))
        x = q[r].double().view(kv_heads, -1, dim)
        weight = torch.softmax(torch.einsum("hgd,hnd->hgn", x, k) * scale, -1)
        out[r] = torch.einsum("hgn,hnd->hgd", weight, v).flatten(0, 1)
        # a score is a sum of dim products in fp32 (off by dim half-steps of the sum of their sizes, and some for the scale and
        # the exponential); weights are split in two terms of 16 bits (2^-16); sums over n tokens add n / 64 half-steps at most
        sizes = torch.einsum("hgd,hnd->hgn", x.abs(), k.abs()).amax(-1) * abs(scale)
        extra[r] = ((2 * dim * F32 * sizes + 2.0 ** -16 + (16 + n / 64) * F32) * v.abs().amax((1, 2))[:, None]).flatten()
    return out, extra[..., None]


def _check_attention(lengths, heads, kv_heads, dim, page, dtype, scale=None, **kw):
    import dlr_lock_b200 as D
    kc, vc, table, n = _cache_case(lengths, kv_heads, dim, page, TYPES[dtype], **kw)
    q = _normal(_gen(heads), len(lengths), heads, dim, dtype=TYPES[dtype])
    got = D.paged_attention(q, kc, vc, table, n, scale=scale)
    want, extra = _attend64(q, kc, vc, table, lengths, dim ** -0.5 if scale is None else scale)
    _close(got, want, extra)
    assert torch.equal(got, D.paged_attention(q, kc, vc, table, n, scale=scale))          # bit for bit
    for r, length in enumerate(lengths):
        assert length or not got[r].any()
    return got


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (16, 8), (12, 12), (5, 1), (32, 4), (27, 3), (16, 1), (40, 2), (17, 1)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_heads(dim, heads, kv_heads, dtype):
    # lengths around the step of 16 tokens, the tile of 64 and the page, none among them; a table of short contexts (clusters) and
    # one with room for long ones (runs and their join), which give the same up to the order of sums
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 200, 0]
    _check_attention(lengths, heads, kv_heads, dim, 32, dtype)
    _check_attention(lengths, heads, kv_heads, dim, 32, dtype, columns=1000)
    _check_attention([4000, 0, 700], heads, kv_heads, dim, 32, dtype, columns=1000)


@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("lengths", [[1], [0], [2, 1], [64 * 9 + 5], [3000], [40000], [5000, 1, 0, 77, 12345, 16, 0],
                                     [0] * 7 + [130] + [0] * 200 + [1]])
def test_attention_lengths(page, lengths):
    _check_attention(lengths, 8, 2, 128, page, "bf16", seed=len(lengths) + page)


@pytest.mark.parametrize("columns", [None, 900])
@pytest.mark.parametrize("requests", [129, 300])
def test_attention_many_requests(requests, columns):
    rng = random.Random(requests)
    _check_attention([rng.choice([0, 1, rng.randint(0, 700)]) for _ in range(requests)], 6, 2, 64, 16, "fp16", columns=columns)


def test_attention_long_and_short_requests_of_many_heads():
    # heads of hundreds of parts beside heads of few and of one, several rounds of heads to a CTA of the join
    lengths = [30000, 3, 0, 700, 9000, 1] * 3 + [50] * 30
    _check_attention(lengths, 64, 2, 64, 64, "bf16")
    _check_attention([20000, 0, 40], 32, 1, 128, 16, "fp16")


@pytest.mark.parametrize("columns", [9, 900])
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -65504.0])
def test_attention_never_reads_what_no_request_holds(fill, columns):
    # the rest of a page, pages of nobody, and table entries beyond the length (outside the cache)
    _check_attention([1, 15, 33, 0, 129], 8, 4, 64, 32, "fp16", fill=fill, columns=columns)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 3.0])
def test_attention_scale(scale):
    # 3.0: nearly all weight on one token; scores far apart
    _check_attention([500, 3], 4, 2, 64, 64, "bf16", scale=scale)


def test_attention_orders_and_strides():
    import dlr_lock_b200 as D
    _check_attention([100, 37, 300], 8, 4, 128, 64, "bf16", order="tokens first")
    # both caches of all layers in one tensor, queries from the middle of a wider product, a table with spare columns
    gen = _gen(5)
    both = _normal(gen, 3, 2, 7, 2, 16, 64, dtype=torch.bfloat16)
    kc, vc = both[1, 0], both[1, 1]
    wide = _normal(gen, 4, 6 * 64 + 40, dtype=torch.bfloat16)
    q = wide[:, 8:8 + 6 * 64].unflatten(-1, (6, 64))
    table = torch.randint(0, 7, (4, 10), generator=gen, device=DEV, dtype=torch.int32)[:, 2:7]
    lengths = [80, 3, 0, 41]
    got = D.paged_attention(q, kc, vc, table, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    _close(got, *_attend64(q, kc, vc, table, lengths, 0.125))
    # rows that are not aligned are copied
    q = wide[:, 1:1 + 6 * 64].unflatten(-1, (6, 64))
    got = D.paged_attention(q, kc, vc, table, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    _close(got, *_attend64(q, kc, vc, table, lengths, 0.125))


def test_dimensions_of_one_have_any_stride():
    import dlr_lock_b200 as D
    kc, vc, table, n = _cache_case([30], 1, 64, 32, torch.bfloat16)
    odd = [c[:1].as_strided((1, 1, 32, 64), (7, 3, 64, 1)) for c in (kc, vc)]
    q = _normal(_gen(1), 1, 1, 64, dtype=torch.bfloat16)
    zero = torch.zeros_like(table)
    assert torch.equal(D.paged_attention(q.as_strided((1, 1, 64), (5, 9, 1)), *odd, zero, n), D.paged_attention(q, kc[:1], vc[:1], zero, n))
    cos, sin = D.rope_tables(torch.ones(32, device=DEV), 4)
    at = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = D.qk_norm_rope_append(q.as_strided((1, 1, 64), (5, 9, 1)), q, q, None, None, cos, sin, at, at + 31, *odd)
    assert torch.equal(got, q) and torch.equal(kc[0, 0, 31], q[0, 0]) and torch.equal(vc[0, 0, 31], q[0, 0])


def test_attention_of_no_requests_no_columns_no_pages():
    import dlr_lock_b200 as D
    kc, vc, table, n = _cache_case([70, 5], 2, 64, 32, torch.bfloat16)
    q = _normal(_gen(1), 2, 4, 64, dtype=torch.bfloat16)
    assert D.paged_attention(q[:0], kc, vc, table[:0], n[:0]).shape == (0, 4, 64)
    assert not D.paged_attention(q, kc, vc, table[:, :0], n).any()
    assert not D.paged_attention(q, kc[:0], vc[:0], table, n).any()


def test_attention_with_offsets_beyond_32_bits():
    # keys and values of 2^32 elements each, the values behind the keys
    import dlr_lock_b200 as D
    whole = torch.empty(2, 2 ** 22, 1, 16, 64, dtype=torch.float16, device=DEV)
    kc, vc = whole[0], whole[1]
    gen = _gen(3)
    q = _normal(gen, 1, 2, 64, dtype=torch.float16)
    ids = [2 ** 22 - 1, 0, 2 ** 22 - 2, 2 ** 21 + 1]
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    for i in ids:
        kc[i], vc[i] = (_normal(gen, 1, 16, 64, dtype=torch.float16) for _ in range(2))
    got = D.paged_attention(q, kc, vc, table, torch.tensor([60], dtype=torch.int32, device=DEV))
    _close(got, *_attend64(q, kc, vc, table, [60], 0.125))
    row = _normal(gen, 1, 1, 64, dtype=torch.float16)
    slot = (2 ** 22 - 1) * 16 + 15
    cos, sin = D.rope_tables(torch.ones(32, device=DEV), 4)
    D.qk_norm_rope_append(row, row, row, None, None, cos, sin, torch.zeros(1, dtype=torch.int32, device=DEV),
                          torch.tensor([slot], dtype=torch.int32, device=DEV), kc, vc)
    assert torch.equal(kc[2 ** 22 - 1, 0, 15], row[0, 0]) and torch.equal(vc[2 ** 22 - 1, 0, 15], row[0, 0])
    del whole, kc, vc
    torch.cuda.empty_cache()


def test_attention_far_scores_and_hidden_tokens():
    # keys of the type's lowest and highest values: weights of exactly 0 and 1, nothing overflows
    import dlr_lock_b200 as D
    kc, vc, table, n = _cache_case([100], 1, 64, 32, torch.bfloat16)
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    kc.fill_(torch.finfo(torch.bfloat16).min / 128)
    page, slot = table[0, 37 // 32].item(), 37 % 32
    kc[page, 0, slot] = 1.0
    got = D.paged_attention(q, kc, vc, table, n)
    assert torch.equal(got, vc[page, 0, slot].expand(1, 2, 64))
    kc.fill_(torch.finfo(torch.bfloat16).min / 128)          # all alike: the mean
    got = D.paged_attention(q, kc, vc, table, n)
    _close(got, *_attend64(q, kc, vc, table, [100], 0.125 * 0))


def test_attention_table_entries_outside_the_cache_count_as_zeros():
    import dlr_lock_b200 as D
    kc, vc, table, n = _cache_case([70], 2, 64, 32, torch.bfloat16)
    q = _normal(_gen(1), 1, 4, 64, dtype=torch.bfloat16)
    for bad in (-1, kc.shape[0], 2 ** 31 - 1, -2 ** 31):
        broken = table.clone()
        broken[0, 1] = bad
        got = D.paged_attention(q, kc, vc, broken, n)
        zeroed = [c.clone() for c in (kc, vc)]
        for c in zeroed:
            c[table[0, 1].item()] = 0
        assert torch.equal(got, D.paged_attention(q, *zeroed, table, n))
    # lengths beyond the table, and below none
    assert torch.equal(D.paged_attention(q, kc, vc, table, n + 10 ** 6), D.paged_attention(q, kc, vc, table, torch.full_like(n, 96)))
    assert not D.paged_attention(q, kc, vc, table, torch.full_like(n, -3)).any()


# ---- streams, graphs, and all of it together --------------------------------------------------------------------------------
@pytest.mark.parametrize("columns", [None, 500])
def test_attention_on_another_stream_and_replayed_with_other_lengths(columns):
    import dlr_lock_b200 as D
    kc, vc, table, n = _cache_case([900, 40, 2000], 4, 128, 64, torch.bfloat16, columns=columns)
    q = _normal(_gen(2), 3, 16, 128, dtype=torch.bfloat16)
    want = D.paged_attention(q, kc, vc, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = D.paged_attention(q, kc, vc, table, n)
    side.synchronize()
    assert torch.equal(got, want)
    # two captured graphs, replayed at the same time on two streams: no workspace is shared
    pair = []
    for _ in range(2):
        held = n.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = D.paged_attention(q, kc, vc, table, held)
        pair.append((g, held, out, torch.cuda.Stream()))
    other = torch.tensor([77, 0, 1999], dtype=torch.int32, device=DEV)
    want_other = D.paged_attention(q, kc, vc, table, other)
    pair[1][1].copy_(other)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, _, _, stream in pair:
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(pair[0][2], want) and torch.equal(pair[1][2], want_other)


@pytest.mark.parametrize("columns", [8, 1000])
def test_decode_steps_together_captured(columns):
    """Plan, norm and rotation with append, attention: prompts admitted, then steps replayed from one graph, against the same
    attention over everything that a request was given."""
    import dlr_lock_b200 as D
    gen = _gen(11)
    requests, heads, kv_heads, dim, page = 5, 8, 2, 64, 16
    dtype = torch.bfloat16
    kc, vc = (torch.full((30, kv_heads, page, dim), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    table = torch.full((requests, columns), -1, dtype=torch.int32, device=DEV)
    free, n_free = torch.randperm(30, generator=gen, device=DEV).int(), torch.tensor([30], dtype=torch.int32, device=DEV)
    lengths = torch.zeros(requests, dtype=torch.int32, device=DEV)
    qw, kw = (1 + 0.2 * _normal(gen, 2, dim)).to(dtype).unbind(0)
    cos, sin = D.rope_tables(1.0 / 10000.0 ** (torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim), 200)
    history = [[] for _ in range(requests)]          # (normed and turned key, value) rows

    def record(k, v, plan, who):
        want_k = D.qk_norm_rope(k, k, kw, kw, cos, sin, plan.positions)[1]
        for row, r in who:
            history[r].append((want_k[row].double(), v[row].double()))

    prompts = [17, 0, 33, 1, 16]
    new = torch.tensor(prompts, dtype=torch.int32, device=DEV)
    plan = D.paged_plan(lengths, new, table, free, n_free, page, width=40, in_place=True)
    rows = requests * 40
    q, k, v = (_normal(gen, rows, h, dim, dtype=dtype) for h in (heads, kv_heads, kv_heads))
    D.qk_norm_rope_append(q, k, v, qw, kw, cos, sin, plan.positions, plan.slots, kc, vc)
    record(k, v, plan, [(r * 40 + j, r) for r, n in enumerate(prompts) for j in range(n)])

    q, k, v = (_normal(gen, requests, h, dim, dtype=dtype) for h in (heads, kv_heads, kv_heads))
    one = torch.tensor([1, 1, 1, 1, 0], dtype=torch.int32, device=DEV)
    D.paged_attention(q, kc, vc, table, lengths)      # (first calls outside the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = D.paged_plan(lengths, one, table, free, n_free, page, in_place=True)
        turned = D.qk_norm_rope_append(q, k, v, qw, kw, cos, sin, step.positions, step.slots, kc, vc)
        out = D.paged_attention(turned, kc, vc, table, lengths)
    for i in range(40):
        for t in (q, k, v):
            t.copy_(_normal(gen, *t.shape, dtype=dtype))
        graph.replay()
        record(k, v, step, [(r, r) for r in range(4)])
        if i in (0, 1, 15, 39):
            assert lengths.tolist() == [len(h) for h in history]
            want, extra = torch.zeros(requests, heads, dim, dtype=torch.float64, device=DEV), 0.0
            for r, h in enumerate(history):
                keys, values = (torch.stack([x[j] for x in h]) for j in (0, 1))
                x = turned[r].double().view(kv_heads, -1, dim)
                weight = torch.softmax(torch.einsum("hgd,nhd->hgn", x, keys) * 0.125, -1)
                want[r] = torch.einsum("hgn,nhd->hgd", weight, values).flatten(0, 1)
                sizes = torch.einsum("hgd,nhd->hgn", x.abs(), keys.abs()).max() * 0.125
                extra = max(extra, float((2 * dim * F32 * sizes + 2.0 ** -15) * values.abs().max()))
            _close(out, want, extra)
    assert n_free.item() == 30 - sum(-(-len(h) // page) for h in history)
