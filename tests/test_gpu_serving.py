"""The locked decoder on a paged cache, and its fused attention modules in training, against the host framework's own loop.

An fp32 copy of the same bf16-rounded model is the truth; what runs on the operators may be no further from it than the host
framework's bf16 arithmetic is (a quarter more for the scatter of two roundings of the same size, and 2e-3)."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _model(layers=4, head_dim=128, heads=8, kv_heads=4, seed=0, **more):
    import dlr_lock_b200 as D
    from transformers import AutoConfig

    torch.manual_seed(seed)
    cfg = AutoConfig.for_model("qwen3", vocab_size=1000, hidden_size=512, intermediate_size=1536, num_hidden_layers=layers,
                               num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=head_dim, max_position_embeddings=512,
                               tie_word_embeddings=True, **more)
    model = D.locked_model_from_config(cfg, rank=64, device=DEV, alpha_init=0.3).eval()
    for layer in model.model.layers:                       # norms that do something
        for n in (layer.self_attn.q_norm, layer.self_attn.k_norm):
            n.weight.data.uniform_(0.5, 1.5)
    return model


@torch.no_grad()
def _host_logits(model, prompts, forced):
    """Logits of each request after its prompt and after every forced token, one request at a time."""
    rows = []
    for prompt, tail in zip(prompts, forced):
        ids = torch.cat([prompt, tail])[None]
        rows.append(model(ids).logits[0, len(prompt) - 1:])
    return rows


@pytest.mark.parametrize("head_dim,heads,kv_heads,page", [(128, 8, 4, 64), (64, 8, 1, 16)])
def test_paged_decoder_against_the_host_framework(head_dim, heads, kv_heads, page):
    import dlr_lock_b200 as D
    model = _model(head_dim=head_dim, heads=heads, kv_heads=kv_heads)
    truth = copy.deepcopy(model).float()
    D.set_fast_path(truth, False)
    gen = torch.Generator(device=DEV).manual_seed(1)
    counts = [5, 70, 1, 33]
    steps = 20
    prompts = [torch.randint(0, 1000, (n,), generator=gen, device=DEV) for n in counts]
    forced = [torch.randint(0, 1000, (steps,), generator=gen, device=DEV) for _ in counts]
    want, host = _host_logits(truth, prompts, forced), _host_logits(model, prompts, forced)

    decoder = D.PagedDecoder(model, requests=5, max_tokens=128, page_size=page)
    ids = torch.zeros(5, 70, dtype=torch.long, device=DEV)
    for r, p in enumerate(prompts):
        ids[r, :len(p)] = p
    got = [decoder.admit(ids, torch.tensor(counts + [0], dtype=torch.int32, device=DEV))]
    assert decoder.cache.lengths.tolist() == counts + [0]
    active = torch.tensor([True] * 4 + [False], device=DEV)
    for i in range(steps // 2):
        got.append(decoder.step(torch.stack([f[i] for f in forced] + [forced[0][0] * 0]), active))
    # the rest from a graph: all five rows take part, the last one a request without a prompt
    graph, tokens, logits = decoder.capture()
    assert decoder.cache.lengths.tolist() == [n + steps // 2 for n in counts] + [0]
    for i in range(steps // 2, steps):
        tokens[:4] = torch.stack([f[i] for f in forced])
        graph.replay()
        got.append(logits.clone())
    torch.cuda.synchronize()
    D.ops.check_status()
    assert decoder.cache.lengths.tolist() == [n + steps for n in counts] + [steps // 2]
    assert all(torch.isnan(g[4]).all() for g in got[:1 + steps // 2])
    for r in range(4):
        mine = torch.stack([g[r] for g in got])
        e_mine, e_host = _rel(mine, want[r]), _rel(host[r], want[r])
        assert e_mine <= 1.25 * e_host + 2e-3, (r, e_mine, e_host)


def test_pages_run_out_and_come_back():
    import dlr_lock_b200 as D
    model = _model(layers=2)
    decoder = D.PagedDecoder(model, requests=3, max_tokens=64, pages=5, page_size=16)
    cache = decoder.cache
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    ids = torch.randint(0, 1000, (3, 40), device=DEV)
    out = decoder.admit(ids, i32([40, 30, 16]))              # 3 + 2 pages; the third prompt finds none
    assert cache.lengths.tolist() == [40, 30, 0] and cache.n_free.item() == 0
    assert torch.isfinite(out[:2]).all() and torch.isnan(out[2]).all()
    for _ in range(3):                                       # 31, 32: room in the page; 33: none
        out = decoder.step(ids[:, 0], torch.tensor([False, True, False], device=DEV))
    assert cache.lengths.tolist() == [40, 32, 0] and torch.isnan(out).all()
    cache.release(torch.tensor([True, False, False], device=DEV))
    assert cache.lengths.tolist() == [0, 32, 0] and cache.n_free.item() == 3
    first = decoder.admit(ids, i32([0, 0, 16]))
    again = decoder.admit(ids, i32([0, 0, 16]))              # admitted anew: the same prompt, the same logits
    assert cache.lengths.tolist() == [0, 32, 16] and cache.n_free.item() == 2
    assert torch.equal(first[2], again[2]) and torch.isnan(again[:2]).all()
    with pytest.raises(ValueError):
        decoder.step(ids[0])
    with pytest.raises(ValueError):
        decoder.admit(ids[:2], i32([1, 1, 1]))


def test_ids_behind_a_prompt_and_of_inactive_requests_may_be_anything():
    import dlr_lock_b200 as D
    model = _model(layers=2)
    ids = torch.randint(0, 1000, (3, 20), device=DEV)
    counts = torch.tensor([20, 7, 0], dtype=torch.int32, device=DEV)
    active = torch.tensor([True, False, False], device=DEV)
    runs = []
    for fill in (0, -100, 1 << 40):
        decoder = D.PagedDecoder(model, requests=3, max_tokens=64)
        padded = ids.masked_fill(torch.arange(20, device=DEV) >= counts[:, None], fill)
        first = decoder.admit(padded, counts)
        runs.append((first[:2], decoder.step(ids[:, 0].masked_fill(~active, fill), active)[:1]))
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))
    assert all(torch.isfinite(t).all() for t in runs[0])


def test_a_captured_step_keeps_its_cache():
    import dlr_lock_b200 as D
    model = _model(layers=1)
    ids = torch.randint(0, 1000, (2, 9), device=DEV)

    def start():
        decoder = D.PagedDecoder(model, requests=2, max_tokens=64)
        decoder.admit(ids, torch.tensor([9, 4], dtype=torch.int32, device=DEV))
        return decoder

    def replayed(graph, tokens, logits):
        tokens.copy_(ids[:, 0])
        graph.replay()
        return logits.clone()

    held = start()
    want = replayed(*held.capture())
    captured = start().capture()                             # (nothing else holds this decoder)
    others = [torch.full((1 << 20,), float("nan"), device=DEV) for _ in range(8)]
    assert torch.equal(replayed(*captured), want) and all(torch.isnan(t).all() for t in others)


def test_what_the_decoder_refuses():
    import dlr_lock_b200 as D
    model = _model(layers=1)
    with pytest.raises(ValueError):
        D.PagedDecoder(copy.deepcopy(model).float(), 1, 64)
    with pytest.raises(ValueError):
        D.PagedDecoder(_model(layers=1, head_dim=80), 1, 64)
    other = copy.deepcopy(model)
    other.model.layers[0].mlp = other.model.layers[0].mlp.dlrnet
    with pytest.raises(ValueError):
        D.PagedDecoder(other, 1, 64)
    with pytest.raises(ValueError):
        D.PagedCache(1, 1, 64, 1, 64, page_size=24)
    with pytest.raises(TypeError):
        D.PagedCache(1, 1, 64, 1, 64, dtype=torch.float32)


@pytest.mark.parametrize("padded", [False, True])
def test_fused_attention_modules_in_training(padded):
    import dlr_lock_b200 as D
    model = _model(layers=2, seed=3)
    truth = copy.deepcopy(model).float()
    D.set_fast_path(truth, False)
    ids = torch.randint(0, 1000, (3, 50), device=DEV)
    mask = torch.ones_like(ids)
    if padded:
        mask[1, :20] = 0
    labels = ids.masked_fill(mask == 0, -100)

    def gradients(m):
        m.zero_grad()
        out = m(input_ids=ids, attention_mask=mask, labels=labels)
        out.loss.backward()
        picked = {n: p.grad for n, p in m.named_parameters() if "self_attn" in n}
        return out.logits.detach()[mask == 1], picked

    want = gradients(truth)
    assert D.fuse_decoder_layers(model, True) == 2
    host = gradients(model)
    assert D.fuse_decoder_layers(model, True, attention=True) == 2
    mine = gradients(model)
    assert _rel(mine[0], want[0]) <= 1.25 * _rel(host[0], want[0]) + 2e-3
    assert len(mine[1]) == 2 * 6
    for n, g in mine[1].items():
        assert _rel(g, want[1][n]) <= 1.25 * _rel(host[1][n], want[1][n]) + 2e-3, n
    # and back: the host framework's own modules
    assert D.fuse_decoder_layers(model, True) == 2
    assert torch.equal(gradients(model)[0], host[0])


def test_fused_attention_modules_decode_on_the_host_caches():
    import dlr_lock_b200 as D
    from transformers import StaticCache

    model = _model(layers=2, seed=4)
    ids = torch.randint(0, 1000, (2, 30), device=DEV)
    with torch.no_grad():
        D.fuse_decoder_layers(model, True)
        host = model(ids).logits
        D.fuse_decoder_layers(model, True, attention=True)
        for cache in (None, StaticCache(config=model.config, max_cache_len=40)):
            rows = []
            for i in range(30):
                out = model(ids[:, i:i + 1], past_key_values=cache, use_cache=True)
                cache = out.past_key_values
                rows.append(out.logits)
            assert _rel(torch.cat(rows, 1), host) <= 3e-2
        ppl = D.evaluate_ppl(model, D.synthetic_token_stream(1000, 64, 2, seed=1), n_steps=2, device=DEV)
        D.fuse_decoder_layers(model, True)
        want = D.evaluate_ppl(model, D.synthetic_token_stream(1000, 64, 2, seed=1), n_steps=2, device=DEV)
    assert abs(ppl / want - 1) <= 1e-2


def test_fused_attention_modules_first_used_in_inference_mode_or_in_a_capture():
    import dlr_lock_b200 as D
    model = _model(layers=2)
    ids = torch.randint(0, 1000, (2, 24), device=DEV)
    with torch.no_grad():
        D.fuse_decoder_layers(model, True, attention=True)
        want = model(ids).logits                             # (and everything else that a first call makes)

    D.fuse_decoder_layers(model, True, attention=True)       # the tables anew
    with torch.inference_mode():
        assert torch.equal(model(ids).logits, want)
    model.train()
    out = model(ids).logits
    out.float().square().mean().backward()
    grads = [layer.self_attn.q_norm.weight.grad for layer in model.model.layers]
    assert all(g is not None and torch.isfinite(g).all() for g in grads)
    model.eval()

    q, k = (torch.randn(2, 24, n, 128, device=DEV).to(torch.bfloat16) for n in (8, 4))
    positions = torch.arange(24, device=DEV).expand(2, 24)
    tables = model.model.layers[0].self_attn._rotary_tables
    truth = D.qk_norm_rope(q, k, None, None, *tables.on(q.device), positions)
    fresh = type(tables)(model)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = D.qk_norm_rope(q, k, None, None, *fresh.on(q.device), positions)
    eager = D.qk_norm_rope(q, k, None, None, *fresh.on(q.device), positions)      # before any replay
    graph.replay()
    assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(eager, truth, captured))
