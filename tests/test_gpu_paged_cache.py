"""A paged cache and its decoder, made in one mode of torch and used in another."""
import pytest
import torch

from test_gpu_serving import DEV, _model

pytestmark = pytest.mark.gpu


def test_a_decoder_made_in_inference_mode_is_captured_outside_of_it():
    import dlr_lock_b200 as D
    model = _model(layers=2)
    ids = torch.randint(0, 1000, (2, 9), device=DEV)
    counts = torch.tensor([9, 4], dtype=torch.int32, device=DEV)
    results = []
    for made, used in ((False, False), (True, False), (False, True), (True, True)):
        with torch.inference_mode(made):
            decoder = D.PagedDecoder(model, requests=2, max_tokens=64)
            first = decoder.admit(ids, counts)
        with torch.inference_mode(used):
            graph, tokens, logits = decoder.capture()
            tokens.copy_(ids[:, 0])
            graph.replay()
            again = decoder.step(ids[:, 1])
            decoder.cache.release(torch.tensor([True, False], device=DEV))
        results.append([t.clone() for t in (first, logits, again, decoder.cache.lengths, decoder.cache.n_free)])
    assert results[0][3].tolist() == [0, 6]
    for got in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, results[0]))


def test_flags_of_another_shape_are_refused():
    # (a single flag would be broadcast, and every request lose its pages)
    import dlr_lock_b200 as D
    model = _model(layers=1)
    ids = torch.randint(0, 1000, (2, 9), device=DEV)
    counts = torch.tensor([9, 4], dtype=torch.int32, device=DEV)
    decoder = D.PagedDecoder(model, requests=2, max_tokens=64)
    decoder.admit(ids, counts)
    for flags in (torch.tensor([True], device=DEV), torch.tensor(True, device=DEV), torch.tensor([True] * 3, device=DEV)):
        with pytest.raises(ValueError, match="finished"):
            decoder.admit(ids, counts * 0, flags)
        with pytest.raises(ValueError, match="active"):
            decoder.step(ids[:, 0], flags)
    assert decoder.cache.lengths.tolist() == [9, 4]
    # flags of another type count by their truth
    for flags in (torch.tensor([0, 255], dtype=torch.uint8, device=DEV), torch.tensor([0, 7], device=DEV)):
        decoder.step(ids[:, 0], flags)
    decoder.admit(ids, counts * 0, torch.tensor([5, 0], device=DEV))
    assert decoder.cache.lengths.tolist() == [0, 6]
