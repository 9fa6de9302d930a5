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


def _same(got, want, device):
    """
    The same labels and log probabilities: sums of 32 to 140 products in fp32 through two layers, in another order. On the GPU prompts and steps take other kernels, each within 1e-3 of the
    model's call; two labels may be as good as each other there, and what follows is then another text.
    """
    tol = 1e-4 if device == "cpu" else 2e-3
    for a, b, x, y in zip(got.labels, want.labels, got.log_probs, want.log_probs):
        assert abs(x - y) <= tol * (1 + abs(y))
        if a != b:
            assert device != "cpu"
            return
    assert len(got.labels) == len(want.labels)


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
    for a, b in zip(got, want):
        _same(a, b, device)


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
        tol = 1e-4 if device == "cpu" else 2e-3
        assert torch.allclose(a.log_probs, b.log_probs, atol=tol, rtol=tol) and torch.allclose(a.top_log_probs, b.top_log_probs, atol=tol, rtol=tol)
    for a, b in zip(paged.generate(texts, max_new=5, eos=0), other.generate(texts, max_new=5, eos=0)):
        _same(a, b, device)
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
    assert ran == texts and _is_empty(paged)
    for a, b in zip(got, want):
        _same(a, b, device)
    del ran[:]
    small = _make(device, num_pages=2)
    for call in (lambda: small.generate([texts[4], texts[0]], max_new=2, eos=-1), lambda: small.score([texts[4], texts[0]])):
        with pytest.raises(RuntimeError, match="2 pages"):
            call()
        assert _is_empty(small) and not ran


@DEVICES
@pytest.mark.parametrize("lens,pages,max_new", [([8, 8], 6, 14), ([8, 7, 5], 6, 16), ([4, 4, 4, 4, 4], 6, 20), ([1, 1, 1], 3, 11), ([20, 3, 3], 6, 4)])
def test_requests_that_outgrow_the_pool_together(device, lens, pages, max_new):
    """each fits the pool alone: the one that began last gives its pages up and goes on later, with the results of a run of its own"""
    paged = _make(device, num_pages=pages)
    texts = _texts(61, lens, seed=7)
    got = paged.generate(texts, max_new=max_new, eos=-1)
    assert _is_empty(paged)
    for text, res in zip(texts, got):
        (alone,) = _make(device).generate([text], max_new=max_new, eos=-1)
        assert len(res.labels) == len(alone.labels) == max_new
        _same(res, alone, device)


@DEVICES
def test_a_request_that_outgrows_the_pool_alone(device):
    paged = _make(device, num_pages=2)
    with pytest.raises(RuntimeError, match="2 pages"):
        paged.generate(_texts(61, [3, 5], seed=8), max_new=10, eos=-1)
    assert _is_empty(paged)


@DEVICES
def test_the_callers_autocast_changes_nothing(device):
    """the types are those of the decoder: the same bits"""
    paged = _make(device)
    texts = _texts(61, [6, 9, 4], seed=9)
    want, want_texts = paged.score(texts, num_top=2), paged.generate(texts, max_new=3, eos=-1)
    with torch.autocast(device, dtype=torch.bfloat16):
        got, got_texts = paged.score(texts, num_top=2), paged.generate(texts, max_new=3, eos=-1)
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) and x.dtype == y.dtype for x, y in zip(a, b))
    assert got_texts == want_texts


@DEVICES
def test_serving_by_public_calls(device):
    """add, logits, step and end, with requests that join and leave, against generate()"""
    paged = _make(device, kind="rotary")
    texts = _texts(61, [6, 9, 1, 4], seed=10)
    want = _make(device, kind="rotary").generate(texts, max_new=4, eos=-1)
    out, row_of = {}, {}

    def join(i, row):
        x = paged.add([row], [texts[i]])
        label = int(paged.logits(x[-1:])[0].argmax())
        out[i], row_of[i] = [label], row

    join(1, 2)
    join(0, 0)
    waiting = [2, 3]
    while row_of:
        labels, log_probs, rows, granted = paged.step({r: out[i][-1] for i, r in row_of.items()})
        assert rows.tolist()[: len(row_of)] == sorted(row_of.values()) and granted[list(row_of.values())].all()
        by_row = {r: (a, p) for r, a, p in zip(rows.tolist(), labels.tolist(), log_probs.tolist()) if r >= 0}
        for i, r in list(row_of.items()):
            out[i].append(by_row[r][0])
            if len(out[i]) == 4:
                del row_of[i]
                paged.end([r])
        if waiting and len(row_of) < 3:
            join(waiting[0], ({0, 1, 2} - set(row_of.values())).pop())
            del waiting[0]
    assert _is_empty(paged)
    for i, res in enumerate(want):
        assert out[i] == res.labels
    # rows that have ended do not go on; a request can begin with a step
    assert paged.step()[2].tolist() == [-1] * 3 and _is_empty(paged)
    paged.add([1], [texts[0][:-1]])
    labels, _, rows, _ = paged.step({1: texts[0][-1], 0: texts[2][0]})
    assert rows.tolist() == [0, 1, -1] and labels.tolist()[:2] == [want[2].labels[0], want[0].labels[0]] and paged.lengths.tolist() == [1, 6, 0]
    for bad, err in (({3: 1}, "rows"), ({-1: 1}, "rows"), ({0: 61}, "vocabulary"), ({0: -1}, "vocabulary")):
        with pytest.raises(ValueError, match=err):
            paged.step(bad)
    assert paged.lengths.tolist() == [1, 6, 0]


@DEVICES
@pytest.mark.parametrize("kind", ["sinusoidal", "rotary"])
def test_positions_in_the_last_page(device, kind):
    """a page may reach beyond the longest length: positions there are their own, and past the page no token is granted"""
    from test_paged_decoder import _rf_logits

    paged, model = _make(device, kind=kind, max_len=6), _decoder(kind, dim=32 if device == "cpu" else 128, device=device)
    text = _texts(61, [8], seed=11)[0]
    paged.add([1], [text[:6]])
    with torch.no_grad():
        want = torch.log_softmax(_rf_logits(model, text, device).double(), -1)
    for n in (6, 7):
        _, log_probs, rows, granted = paged.step({1: text[n]})
        assert rows.tolist() == [1, -1, -1] and granted.all()
        assert abs(float(log_probs[0]) - float(want[n].max())) <= (1e-4 if device == "cpu" else 1e-3) * (1 + abs(float(want[n].max())))
    _, _, rows, granted = paged.step({1: 5})
    assert granted.tolist() == [True, False, True] and paged.lengths.tolist() == [0, 8, 0]


def test_a_wait_that_ran_out_is_named():
    from returnn_b200.ops import status

    assert "paged cache" in status.describe(status.SLOT_GEMM, 9 << 24 | 1) and "GEMM" not in status.describe(status.SLOT_GEMM, 9 << 24 | 1)
    assert "GEMM" in status.describe(status.SLOT_GEMM, 3 << 24 | 1)


@gpu
def test_a_wait_that_ran_out_is_an_error():
    """what a kernel that gave up leaves on the status board (written here by the host): no labels or scores that are not valid are returned"""
    from returnn_b200.ops import status

    paged = _make("cuda")
    texts = _texts(61, [6, 9], seed=12)
    want = paged.generate(texts, max_new=4, eos=-1)
    word = status.word("cuda", status.SLOT_GEMM)
    for call in (lambda: paged.generate(texts, max_new=4, eos=-1), lambda: paged.score(texts), lambda: [paged.step({}) for _ in range(2)]):
        word.fill_(9 << 24 | 1)
        with pytest.raises(status.KernelWaitTimeout, match="paged cache"):
            call()
        assert _is_empty(paged) and not int(word)
    assert [x.labels for x in paged.generate(texts, max_new=4, eos=-1)] == [x.labels for x in want]


@gpu
def test_bf16_requests_alone_and_together():
    """
    The captured step in bf16 with head dim 64: a request has the log probabilities that it has alone. Batches of another size take other kernels for the products, so that values in bf16 may
    fall to the neighbour, 2^-8 of them: some ten roundings a layer shift logits of a size of up to 10 by about 2^-8 * sqrt(20) * 10 = 0.17, the rounding of the logit itself by 2^-5.
    """
    from returnn_b200.models.paged_decoder import PagedDecoder

    model = _decoder("normed", heads=8, dim=512, vocab=5000, device="cuda")
    opts = dict(max_len=300, page_size=16, dtype=torch.bfloat16)
    together, alone = PagedDecoder(model, max_requests=5, **opts), PagedDecoder(model, max_requests=1, **opts)
    prompts = _texts(5000, [3, 170, 17, 64, 100, 8, 250], seed=1)
    results = together.generate(prompts, max_new=12, eos=0)
    assert _is_empty(together) and len(results) == len(prompts)
    for prompt, got in zip(prompts, results):
        (want,) = alone.generate([prompt], max_new=12, eos=0)
        assert _is_empty(alone)
        for res in (got, want):
            assert 1 <= len(res.labels) <= 12 and len(res.log_probs) == len(res.labels) and 0 not in res.labels[:-1] and (len(res.labels) == 12 or res.labels[-1] == 0)
        for a, b, x, y in zip(got.labels, want.labels, got.log_probs, want.log_probs):
            assert abs(x - y) <= 0.25
            if a != b:  # as good as each other; what follows is another text
                break
        else:
            assert len(got.labels) == len(want.labels)
