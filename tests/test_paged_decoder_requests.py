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


@DEVICES
def test_a_call_that_fails_leaves_nothing_behind(device, monkeypatch):
    """no row or page is kept, and the next call has the results of a new decoder"""
    paged, other = _make(device, max_requests=2), _make(device, max_requests=2)
    texts = _texts(61, [8, 5, 6, 3], seed=3)
    want = other.generate(texts, max_new=4, eos=0)
    for bad in ([], [1] * 25):  # one that joins late
        with pytest.raises(ValueError):
            paged.generate(texts + [bad], max_new=4, eos=0)
        assert _is_empty(paged)
    inner, calls = type(paged)._step, []

    def fail_in_the_third(self):
        calls.append(0)
        if len(calls) == 3:
            raise KeyError("in the middle")
        return inner(self)

    def fail(self, *args):
        raise KeyError("in a layer")

    with monkeypatch.context() as m:
        m.setattr(type(paged), "_step", fail_in_the_third)
        with pytest.raises(KeyError):
            paged.generate(texts, max_new=4, eos=0, use_graph=False)
        assert len(calls) == 3 and _is_empty(paged)
        m.setattr(type(paged), "_layer", fail)
        for call in (lambda: paged.generate(texts, max_new=4, eos=0), lambda: paged.score(texts), lambda: paged.add([1], texts[:1])):
            with pytest.raises(KeyError):
                call()
            assert _is_empty(paged)
    got = paged.generate(texts, max_new=4, eos=0)
    assert [x.labels for x in got] == [x.labels for x in want]
    for a, b in zip(got, want):
        assert a.log_probs == pytest.approx(b.log_probs, abs=1e-4)


@DEVICES
def test_rows_that_hold_a_request_are_not_taken(device):
    """add() refuses them; score() and generate() work beside them in the other rows and leave them as they are"""
    paged, other = _make(device), _make(device)
    texts = _texts(61, [6, 9, 4, 7], seed=5)
    paged.add([1], texts[:1])
    lengths, table = paged.lengths.tolist(), paged.block_table[1, :2].tolist()
    for rows, err in (([1], "holds"), ([0, 1], "holds"), ([0, 0], "twice"), ([-1, 0], "rows"), ([3, 0], "rows"), ([0], "prompts"), ([], "prompts")):
        with pytest.raises(ValueError, match=err):
            paged.add(rows, [[1, 2]] * (len(rows) if "prompts" not in err else len(rows) + 1))
        assert paged.lengths.tolist() == lengths
    for bad in ([-1], [3], [0, 7]):
        with pytest.raises(ValueError, match="rows"):
            paged.end(bad)
    for a, b in zip(paged.score(texts, num_top=2), other.score(texts, num_top=2)):
        assert torch.allclose(a.log_probs, b.log_probs, atol=1e-4) and torch.equal(a.top_labels, b.top_labels)
    for a, b in zip(paged.generate(texts, max_new=5, eos=0), other.generate(texts, max_new=5, eos=0)):
        assert a.labels == b.labels
    assert paged.lengths.tolist() == lengths and paged.block_table[1, :2].tolist() == table
    paged.add([0, 2], texts[1:3])
    for call in (lambda: paged.score(texts), lambda: paged.generate(texts, max_new=5, eos=0)):
        with pytest.raises(RuntimeError, match="rows"):
            call()
    assert paged.lengths.tolist() == [9, 6, 4]
    paged.end([2, 0, 1])
    assert _is_empty(paged) and paged.add([], []).shape[0] == 0


@DEVICES
def test_prompts_that_wait_do_not_run(device, monkeypatch):
    """whether a prompt has room is known before it goes through the layers"""
    paged = _make(device, max_requests=3, num_pages=8)
    texts = _texts(61, [9, 13, 12, 8, 3], seed=6)  # 3, 4, 3, 2 and 1 of the 8 pages
    want = _make(device).generate(texts, max_new=4, eos=-1)
    ran, inner = [], type(paged).add

    def add(self, rows, prompts):
        ran.extend(prompts)
        return inner(self, rows, prompts)

    monkeypatch.setattr(type(paged), "add", add)
    got = paged.generate(texts, max_new=4, eos=-1)
    assert ran == texts and [x.labels for x in got] == [x.labels for x in want] and _is_empty(paged)
    del ran[:]
    small = _make(device, num_pages=2)
    for call in (lambda: small.generate([texts[4], texts[0]], max_new=2, eos=-1), lambda: small.score([texts[4], texts[0]])):
        with pytest.raises(RuntimeError, match="2 pages"):
            call()
        assert _is_empty(small) and not ran
