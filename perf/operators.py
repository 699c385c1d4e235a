"""The attention block of a locked decoder on a paged key-value cache, as a list of timed cases.

A serving process keeps the keys and values of its requests in pages.  Every step it plans where the new tokens go
(``paged_plan``), normalises and rotates the queries and keys of each layer and puts keys and values into their pages
(``qk_norm_rope_append``), and lets each request's new token attend to its pages (``paged_attention``).  Training runs
``qk_norm_rope`` with its gradient.  Head counts are those of the decoders that ``registry.MODEL_CONFIGS`` names (16, 32 and
64 query heads on 8 key-value heads of 128) and generic others.

Lengths of requests are spread evenly up to the longest and dealt out in an order that the seed gives, so that the work of a
case does not depend on the seed.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def _api():
    path = os.path.join(os.getcwd(), "ml-dlr-lock_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from dlr_lock_b200 import attention

    return attention


def _plan(name, requests, longest, page, width, growing):
    return {"name": name, "op": "plan", "requests": requests, "longest": longest, "page": page, "width": width, "growing": growing}


def _append(name, tokens, heads, kv_heads, dim, rotary, page, dtype="bf16", interleaved=False, normed=True, far=2048):
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "page": page, "dtype": dtype, "interleaved": interleaved, "normed": normed, "far": far}


def _train(name, tokens, heads, kv_heads, dim, rotary, dtype="bf16", interleaved=False, normed=True, far=2048):
    return {"name": name, "op": "train", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "dtype": dtype, "interleaved": interleaved, "normed": normed, "far": far}


def _attend(name, requests, longest, ragged, heads, kv_heads, dim, page, dtype="bf16"):
    return {"name": name, "op": "attend", "requests": requests, "longest": longest, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def listed():
    return [
        # The bookkeeping of one decode step of a small batch: the smallest call, once per token.
        _plan("plan decode 8", 8, 768, 64, 1, True),
        # The same for a full batch on small pages.
        _plan("plan decode 512", 512, 8192, 16, 1, True),
        # A batch of ragged prompts is admitted to an empty cache.
        _plan("plan prompts 64x2000", 64, 2000, 64, 2000, False),
        # A layer of a decode step of the small model at batch 8.
        _append("append 8 tokens 16/8", 8, 16, 8, 128, 128, 64),
        # A layer of a ragged prompt batch of the widest model, far into a long context.
        _append("append 5001 tokens 64/8", 5001, 64, 8, 128, 128, 64, far=131072),
        # Another family's layout: interleaved pairs over part of the head, no norm, fp16.
        _append("append 999 tokens fp16", 999, 24, 6, 96, 64, 16, dtype="fp16", interleaved=True, normed=False),
        # Fine-tuning: forward and gradients of a micro-batch of the large model.
        _train("train 4x2048 tokens 32/8", 8192, 32, 8, 128, 128),
        # A short, odd micro-batch in fp16 with heads of 64.
        _train("train 300 tokens fp16", 300, 12, 4, 64, 64, dtype="fp16"),
        # One user, one token, a short context: the smallest attention.
        _attend("attend 1x513 16/8", 1, 513, False, 16, 8, 128, 64),
        # A serving batch of the large model, contexts of every length.
        _attend("attend 64x8000 32/8", 64, 8000, True, 32, 8, 128, 64),
        # One user with a very long context on the widest model: all of it split over the GPU.
        _attend("attend 1x131072 64/8", 1, 131072, False, 64, 8, 128, 64),
        # Many short ragged requests, a head each (no shared heads), fp16, small pages.
        _attend("attend 200x1500 fp16", 200, 1500, True, 12, 12, 64, 16, dtype="fp16"),
    ]


def draw(rng):
    """Steps of any batch, prompts, micro-batches and contexts, over head sizes, shared heads, layouts, types and pages."""
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    most = max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(["attend"] * 5 + ["append"] * 3 + ["train"] * 3 + ["plan"] * 2)
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        page = rng.choice([16, 32, 64, 128])
        kv_heads = rng.choice([1, 2, 4, 6, 8, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        dim = rng.choice([64, 96, 128, 128, 256])
        rotary = rng.choice([dim, dim, dim // 2])
        interleaved = rng.random() < 0.3
        normed = rng.random() < 0.7
        far = rng.choice([2048, 32768, 131072])
        if op == "plan":
            growing = rng.random() < 0.5
            longest = log(1, 32768) if growing else log(1, 4096)
            c = _plan("", log(1, 1024), longest, page, 1 if growing else longest, growing)
            if c["requests"] * longest > 1 << 22:
                continue
        elif op == "append":
            c = _append("", log(1, 8192), heads, kv_heads, dim, rotary, page, dtype, interleaved, normed, far)
        elif op == "train":
            c = _train("", log(1, 8192), heads, kv_heads, dim, rotary, dtype, interleaved, normed, far)
        else:
            c = _attend("", log(1, 256), log(1, 131072), rng.random() < 0.7, heads, kv_heads, dim, page, dtype)
            if c["requests"] * c["longest"] * kv_heads * dim > 1 << 28:        # the plain form gathers this many values, padded
                continue
        if heads > 128 or work(c)["bytes"] > most:
            continue
        del c["name"]
        return c


def _spread(requests, longest, ragged):
    """Lengths from none to the longest, evenly spread (all the longest where they are not ragged)."""
    if not ragged or requests == 1:
        return [longest] * requests
    return [longest * i // (requests - 1) for i in range(requests)]


def _dealt(lengths, gen, device):
    order = torch.randperm(len(lengths), generator=gen, device=device)
    return torch.tensor(lengths, dtype=torch.int32, device=device)[order]


def _tables(far, rotary, device):
    """cos and sin of position x frequency, from angles in 64 bits."""
    inverse = 1.0 / 10000.0 ** (torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary)
    angle = torch.arange(far, dtype=torch.float64, device=device)[:, None] * inverse
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    op = case["op"]
    s = {"op": op}
    if op == "plan":
        page, width, requests = case["page"], case["width"], case["requests"]
        lengths = _spread(requests, case["longest"], True)
        table_pages = -(-(case["longest"] + 1) // page)
        if case["growing"]:
            s["lengths"] = _dealt(lengths, gen, device)
            s["new_tokens"] = torch.ones(requests, dtype=torch.int32, device=device)
            held = [-(-n // page) for n in lengths]
        else:
            s["lengths"] = torch.zeros(requests, dtype=torch.int32, device=device)
            s["new_tokens"] = _dealt(lengths, gen, device)
            held = [0] * requests
        total = requests * table_pages + 7
        pages = torch.randperm(total, generator=gen, device=device).to(torch.int32)
        in_use = sum(held)
        # the pages in use are the first of the shuffled ones, each request's in a row
        have = (s["lengths"].long() + page - 1) // page
        first = torch.cumsum(have, 0) - have
        column = torch.arange(table_pages, device=device)
        at = (first[:, None] + column).clamp(max=total - 1)
        s["block_table"] = torch.where(column < have[:, None], pages[at], torch.full_like(pages[at], -1))
        s["free_pages"] = torch.cat([pages[in_use:], torch.full((in_use,), -1, dtype=torch.int32, device=device)])
        s["n_free"] = torch.tensor([total - in_use], dtype=torch.int32, device=device)
        s["page"], s["width"] = page, width
        return s
    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=device).to(dtype)  # noqa: E731
    if op in ("append", "train"):
        tokens = case["tokens"]
        # what the projections gave, side by side as one product would give them
        qkv = normal(tokens, (heads + 2 * kv_heads) * dim)
        qkv *= 1.5
        q, k, v = qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=-1)
        s["q"], s["k"], s["v"] = (t.unflatten(-1, (-1, dim)) for t in (q, k, v))
        s["q_weight"], s["k_weight"] = ((1.0 + 0.2 * torch.randn(2, dim, generator=gen, device=device)).to(dtype).unbind(0)
                                        if case["normed"] else (None, None))
        s["cos"], s["sin"] = _tables(case["far"], case["rotary"], device)
        s["positions"] = torch.randint(0, case["far"], (tokens,), generator=gen, device=device, dtype=torch.int32)
        s["interleaved"] = case["interleaved"]
    if op == "append":
        page = case["page"]
        pages = -(-tokens // page) + 3
        s["slots"] = torch.randperm(pages * page, generator=gen, device=device)[:tokens].to(torch.int32)
        s["slots"][tokens // 2:tokens // 2 + (tokens > 4)] = -1                  # a padded row of the batch
        s["k_cache"], s["v_cache"] = (torch.zeros(pages, kv_heads, page, dim, dtype=dtype, device=device) for _ in range(2))
    elif op == "train":
        s["leaves"] = [t.clone().detach().requires_grad_(True) for t in (s["q"], s["k"])]
        if case["normed"]:
            s["leaves"] += [s[n].clone().detach().requires_grad_(True) for n in ("q_weight", "k_weight")]
        s["grads"] = [normal(tokens, heads, dim), normal(tokens, kv_heads, dim)]
    elif op == "attend":
        page, requests = case["page"], case["requests"]
        lengths = _spread(requests, case["longest"], case["ragged"])
        s["lengths"] = _dealt(lengths, gen, device)
        have = (s["lengths"].long() + page - 1) // page
        total = sum(-(-n // page) for n in lengths) + 3
        order = torch.randperm(total, generator=gen, device=device).to(torch.int32)
        columns = max(1, -(-case["longest"] // page))
        first = torch.cumsum(have, 0) - have
        column = torch.arange(columns, device=device)
        at = (first[:, None] + column).clamp(max=total - 1)
        s["block_table"] = torch.where(column < have[:, None], order[at], torch.full_like(order[at], -1))
        s["q"] = normal(requests, heads, dim)
        s["k_cache"], s["v_cache"] = normal(total, kv_heads, page, dim), normal(total, kv_heads, page, dim)
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------------
def _plain_plan(s):
    lengths, new, page, width = s["lengths"].long(), s["new_tokens"].long(), s["page"], s["width"]
    table, free, n_free = s["block_table"], s["free_pages"], s["n_free"].long()
    device, requests, columns = table.device, table.shape[0], table.shape[1]
    have = (lengths + page - 1) // page
    fits = (new <= width) & (lengths + new <= columns * page)
    need = torch.where(fits, (lengths + new + page - 1) // page - have, torch.zeros_like(have))
    last = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (last <= n_free))
    first = last - need
    column = torch.arange(columns, device=device)
    nth = column - have[:, None]
    taken = granted[:, None] & (nth >= 0) & (nth < need[:, None])
    at = (n_free - 1 - (first[:, None] + nth)).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(taken, free[at], table))
    added = torch.where(granted, new, torch.zeros_like(new))
    j = torch.arange(width, device=device)
    place = lengths[:, None] + j
    real = j < added[:, None]
    in_page = torch.gather(table.long(), 1, (place // page).clamp(max=columns - 1))
    slots = torch.where(real, in_page * page + place % page, torch.full_like(place, -1)).reshape(-1).int()
    positions = torch.where(real, place, torch.zeros_like(place)).reshape(-1).int()
    starts = (torch.arange(requests + 1, device=device) * width).int()
    used = torch.where(granted, need, torch.zeros_like(need)).sum()
    return {"slots": slots, "positions": positions, "starts": starts, "lengths": (lengths + added).int(),
            "n_free": (n_free - used).int(), "block_table": table}


def _plain_norm_rope(x, weight, cos, sin, interleaved):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([turned, rest], -1)


def _plain_append(s):
    at = s["positions"].long()
    c, n = s["cos"][at], s["sin"][at]
    q = _plain_norm_rope(s["q"], s["q_weight"], c, n, s["interleaved"]).to(s["q"].dtype)
    k = _plain_norm_rope(s["k"], s["k_weight"], c, n, s["interleaved"]).to(s["k"].dtype)
    rows = (s["slots"] >= 0).nonzero()[:, 0]
    slot = s["slots"][rows].long()
    page = s["k_cache"].shape[2]
    s["k_cache"][slot // page, :, slot % page] = k[rows]
    s["v_cache"][slot // page, :, slot % page] = s["v"][rows]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_train(s):
    at = s["positions"].long()
    c, n = s["cos"][at], s["sin"][at]
    leaves = s["leaves"]
    weights = leaves[2:] if len(leaves) > 2 else (None, None)
    q = _plain_norm_rope(leaves[0], weights[0], c, n, s["interleaved"]).to(s["q"].dtype)
    k = _plain_norm_rope(leaves[1], weights[1], c, n, s["interleaved"]).to(s["k"].dtype)
    return [q.detach(), k.detach(), *torch.autograd.grad([q, k], leaves, s["grads"])]


def _plain_attend(s):
    q, lengths = s["q"], s["lengths"].long()
    kv_heads, page, dim = s["k_cache"].shape[1:]
    requests, heads = q.shape[:2]
    pages = s["block_table"].long().clamp(min=0)

    def gathered(cache):
        return cache[pages].transpose(1, 2).reshape(requests, kv_heads, -1, dim).float()

    scores = q.float().view(requests, kv_heads, -1, dim) @ gathered(s["k_cache"]).transpose(-1, -2) / math.sqrt(dim)
    held = (torch.arange(scores.shape[-1], device=q.device) < lengths[:, None])[:, None, None]
    scores = scores.masked_fill(~held, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(held.any(-1, keepdim=True), top, torch.zeros_like(top)))
    total = weight.sum(-1, keepdim=True)
    out = weight @ gathered(s["v_cache"]) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(requests, heads, dim).to(q.dtype)


_PLAIN = {"plan": _plain_plan, "append": _plain_append, "train": _plain_train, "attend": _plain_attend}


# ---- the framework's calls -------------------------------------------------------------------------------------------------
def _own_plan(s):
    plan = _api().paged_plan(s["lengths"], s["new_tokens"], s["block_table"], s["free_pages"], s["n_free"], s["page"], width=s["width"])
    return {"slots": plan.slots, "positions": plan.positions, "starts": plan.starts, "lengths": plan.lengths,
            "n_free": plan.n_free, "block_table": s["block_table"]}


def _own_append(s):
    q = _api().qk_norm_rope_append(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["positions"],
                                   s["slots"], s["k_cache"], s["v_cache"], eps=EPS, interleaved=s["interleaved"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_train(s):
    leaves = s["leaves"]
    weights = leaves[2:] if len(leaves) > 2 else (None, None)
    q, k = _api().qk_norm_rope(leaves[0], leaves[1], weights[0], weights[1], s["cos"], s["sin"], s["positions"], eps=EPS,
                               interleaved=s["interleaved"])
    return [q.detach(), k.detach(), *torch.autograd.grad([q, k], leaves, s["grads"])]


def _own_attend(s):
    return _api().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["lengths"])


_OWN = {"plan": _own_plan, "append": _own_append, "train": _own_train, "attend": _own_attend}


def run(state):
    if own:
        return _OWN[state["op"]](state)
    return _PLAIN[state["op"]](state)


def work(case):
    op = case["op"]
    if op == "plan":
        requests, page = case["requests"], case["page"]
        lengths = _spread(requests, case["longest"], True)
        if case["growing"]:
            taken = sum(n % page == 0 for n in lengths)
        else:
            taken = sum(-(-n // page) for n in lengths)
        rows = requests * case["width"]
        # lengths and new tokens in; pages off the stack into the table; slots, positions, starts and lengths out; the count of free pages
        return {"bytes": 4 * (2 * requests + 2 * taken + 2 * rows + requests + 1 + requests + 2), "flops": 0}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if op == "attend":
        held = sum(_spread(case["requests"], case["longest"], case["ragged"]))
        pages = sum(-(-n // case["page"]) for n in _spread(case["requests"], case["longest"], case["ragged"]))
        return {"bytes": 2 * (2 * held * kv_heads * dim + 2 * case["requests"] * heads * dim) + 4 * (pages + case["requests"]),
                "flops": 4 * held * heads * dim}
    tokens = case["tokens"]
    turned = tokens * (heads + kv_heads) * dim
    tables = 8 * min(tokens, case["far"]) * (case["rotary"] // 2) + 4 * tokens
    if op == "append":
        return {"bytes": 2 * (2 * turned + 2 * tokens * kv_heads * dim) + tables + 4 * tokens, "flops": 8 * turned}
    # forward reads and writes q and k; backward reads q, k and the gradients that come in and writes those that go out
    # (without a norm it needs no q and k)
    return {"bytes": 2 * turned * (5 if case["normed"] else 4) + tables, "flops": 24 * turned}


# ---- 64 bits ---------------------------------------------------------------------------------------------------------------
def _exact_turn(x, cos, sin, interleaved, back=False):
    """The pairs of a head as complex numbers, times the unit number of each angle (its conjugate on the way back)."""
    half = cos.shape[-1]
    unit = torch.complex(cos.double(), -sin.double() if back else sin.double())[:, None]
    x = x.clone()
    low, high = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(x[..., low], x[..., high]) * unit
    x[..., low], x[..., high] = z.real, z.imag
    return x


def _exact_head(x, weight, cos, sin, interleaved):
    x = x.detach().double()
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.detach().double()
    return _exact_turn(x, cos, sin, interleaved)


def _exact_gradient(x, weight, cos, sin, interleaved, grad):
    g = _exact_turn(grad.double(), cos, sin, interleaved, back=True)
    if weight is None:
        return g, None
    x = x.detach().double()
    scale = 1.0 / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    unit = x * scale
    inner = g * weight.detach().double()
    dx = scale * (inner - unit * (inner * unit).sum(-1, keepdim=True) / x.shape[-1])
    return dx, (g * unit).sum((0, 1))


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None                                                              # whole numbers only
    s = prepare(case, seed)
    if op == "attend":
        q, cache = s["q"].double(), (s["k_cache"], s["v_cache"])
        out = torch.zeros_like(q)
        kv_heads, page, dim = cache[0].shape[1:]
        for r, n in enumerate(s["lengths"].tolist()):
            if n == 0:
                continue
            pages = s["block_table"][r, :-(-n // page)].long()
            k, v = (c[pages].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double() for c in cache)
            weight = torch.softmax(torch.einsum("hgd,hnd->hgn", q[r].view(kv_heads, -1, dim), k) * dim ** -0.5, -1)
            out[r] = torch.einsum("hgn,hnd->hgd", weight, v).reshape(-1, dim)
        return out
    cos, sin = s["cos"][s["positions"].long()], s["sin"][s["positions"].long()]
    if op == "append":
        q = _exact_head(s["q"], s["q_weight"], cos, sin, s["interleaved"])
        k = _exact_head(s["k"], s["k_weight"], cos, sin, s["interleaved"])
        page = s["k_cache"].shape[2]
        caches = [c.double() for c in (s["k_cache"], s["v_cache"])]
        keep = s["slots"] >= 0
        slot = s["slots"][keep].long()
        for cache, rows in zip(caches, (k, s["v"].double())):
            cache.transpose(1, 2)[torch.div(slot, page, rounding_mode="floor"), slot % page] = rows[keep]
        return {"q": q, "k_cache": caches[0], "v_cache": caches[1]}
    weights = (s["q_weight"], s["k_weight"])
    out = [_exact_head(s[n], w, cos, sin, s["interleaved"]) for n, w in zip(("q", "k"), weights)]
    both = [_exact_gradient(s[n], w, cos, sin, s["interleaved"], g) for n, w, g in zip(("q", "k"), weights, s["grads"])]
    return out + [b[0] for b in both] + ([b[1] for b in both] if case["normed"] else [])
