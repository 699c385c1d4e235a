"""The rotation's tables of the fused attention modules: who makes them, and when others may read them."""
import threading

import pytest
import torch

from test_gpu_serving import DEV, _model

pytestmark = pytest.mark.gpu


def test_a_capture_of_the_first_step_makes_no_tables(monkeypatch):
    import dlr_lock_b200 as D
    from dlr_lock_b200 import attention
    model = _model(layers=3)
    ids = torch.randint(0, 1000, (2, 16), device=DEV)
    D.fuse_decoder_layers(model, True)
    with torch.no_grad():
        model(ids)                                           # (what the nets make on their first call)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model(ids)
        torch.cuda.current_stream().wait_stream(side)
        D.fuse_decoder_layers(model, True, attention=True)
        made, real = [], attention.rope_tables
        monkeypatch.setattr(attention, "rope_tables", lambda *a: made.append(1) or real(*a))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = model(ids).logits
        graph.replay()
        assert not made
        assert torch.equal(model(ids).logits, out) and not made


def test_tables_made_on_one_stream_are_there_for_another():
    model = _model(layers=1)
    from dlr_lock_b200.model import RotaryTables
    want = [t.clone() for t in RotaryTables(model, 1 << 15).on(DEV)]
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device=DEV)
    for threaded in (False, True):
        first, second = torch.cuda.Stream(), torch.cuda.Stream()
        tables, got = RotaryTables(model, 1 << 15), []
        with torch.cuda.stream(first):
            # (memory that held something else, and work before the tables' own)
            del_me = [torch.full_like(t, float("nan")) for t in want for _ in range(4)]
            del del_me
            for _ in range(30):
                busy = busy @ busy * 1e-4
            tables.on(DEV)

        def use():
            with torch.cuda.device(0), torch.cuda.stream(second):
                got.extend(t.clone() for t in tables.on(DEV))

        if threaded:
            t = threading.Thread(target=use)
            t.start()
            t.join()
        else:
            use()
        second.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        first.synchronize()


def test_a_captured_graph_outlives_the_switch_of_its_modules():
    import copy
    import dlr_lock_b200 as D
    model = _model(layers=2)
    ids = torch.randint(0, 1000, (2, 16), device=DEV)
    with torch.no_grad():
        D.fuse_decoder_layers(model, True, attention=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = model(ids).logits
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = model(ids).logits
        tables = model.model.layers[0].self_attn._rotary_tables
        D.fuse_decoder_layers(model, True)
        D.fuse_decoder_layers(model, True, attention=True)
        assert model.model.layers[0].self_attn._rotary_tables is tables
        D.fuse_decoder_layers(model, True)
        del tables
        others = [torch.full((1 << 14,), float("nan"), device=DEV) for _ in range(64)]
        graph.replay()
        assert torch.equal(out, want) and all(torch.isnan(t).all() for t in others)
        # a copy has tables of its own, and so have other frequencies
        D.fuse_decoder_layers(model, True, attention=True)
        twin = copy.deepcopy(model)
        assert twin.model.layers[0].self_attn._rotary_tables is not model.model.layers[0].self_attn._rotary_tables
        assert torch.equal(twin(ids).logits, want)
        twin.model.rotary_emb.inv_freq.mul_(0.5)
        D.fuse_decoder_layers(twin, True, attention=True)
        other = twin(ids).logits
        fresh = copy.deepcopy(model)
        del fresh.model.rotary_emb.__dict__["_dlr_tables"]
        fresh.model.rotary_emb.inv_freq.mul_(0.5)
        D.fuse_decoder_layers(fresh, True, attention=True)
        assert torch.equal(other, fresh(ids).logits) and not torch.equal(other, want)
        graph.replay()
        assert torch.equal(out, want)
