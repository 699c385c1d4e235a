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
