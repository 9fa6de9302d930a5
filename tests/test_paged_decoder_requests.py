"""Life of the requests of models/paged_decoder.py: what is refused, what stays after an error, pools that are too small for all."""

import pytest
import torch

from test_paged_decoder import _decoder, _texts

gpu = pytest.mark.gpu
DEVICES = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])


def _make(device="cpu", kind="normed", **opts):
    from returnn_b200.models.paged_decoder import PagedDecoder

    model = _decoder(kind, dim=32 if device == "cpu" else 128, device=device)
    return PagedDecoder(model, **{**dict(max_requests=3, max_len=24, page_size=4), **opts})


def _is_empty(paged):
    return not paged.lengths.any() and int(paged.free_range[1] - paged.free_range[0]) == paged.num_pages


def test_labels_outside_the_vocabulary_are_refused():
    """before anything runs (the lookup of such a label would be out of range on the GPU)"""
    paged = _make()
    for bad in (-1, 61, 10**9):
        for call in (lambda: paged.add([0, 1], [[1, 2], [3, bad]]), lambda: paged.score([[5], [bad, 2]]), lambda: paged.generate([[5], [1, bad]], max_new=2, eos=0)):
            with pytest.raises(ValueError, match="vocabulary"):
                call()
            assert _is_empty(paged)
    assert len(paged.score([[60, 0]])[0].log_probs) == 1
