"""Serving over a paged cache (models/paged_decoder.py) against the RF decoder on whole sequences, and the RF entry points of its operators."""

import math
import pytest
import torch

gpu = pytest.mark.gpu


def _decoder(kind, *, layers=2, heads=4, dim=32, vocab=61, device="cpu", seed=1):
    import returnn_b200.frontend as rf
    from returnn_b200.tensor import Dim
    from returnn_b200.frontend.decoder.transformer import TransformerDecoder, FeedForwardGated

    rf.select_backend_torch()
    torch.manual_seed(seed)
    opts = dict(num_layers=layers, num_heads=heads, dropout=0.0, att_dropout=0.0)
    if kind != "sinusoidal":
        att = dict(rotary=dict(), normed=dict(qk_norm=True, rope=dict(rotary_dim=dim // heads // 2, interleaved=False, scaling=dict(type="linear", factor=2))),
                   fused=dict(rope={}))[kind]
        opts.update(pos_enc=None, norm=rf.build_dict(rf.RMSNorm), ff=rf.build_dict(FeedForwardGated, ff_dim=dim + 12), input_embedding_scale=1.0,
                    layer_opts=dict(self_att=rf.build_dict(rf.RotaryPosCausalSelfAttention, with_bias=False, **att)))
    model = TransformerDecoder(None, Dim(vocab, name="vocab"), Dim(dim, name="model"), share_embedding=False, **opts)
    for name, p in model.named_parameters():
        t = p.raw_tensor
        with torch.no_grad():
            if "norm" in name:
                t.copy_(torch.randn(t.shape) * 0.2 + (1.0 if "scale" in name else 0.0))
            else:
                t.copy_(torch.randn(t.shape) * (0.6 / math.sqrt(max(t.shape[0], 1)) if t.dim() > 1 else 0.1) * (6.0 if "embedding" in name else 1.0))
    for p in model.parameters():
        p.raw_tensor = torch.nn.Parameter(p.raw_tensor.detach().to(device), requires_grad=True)
    return model


def _rf_logits(model, labels, device="cpu"):
    """[len, vocab] of one text by the RF call"""
    from returnn_b200.tensor import Tensor, Dim

    t = Dim(len(labels), name="time")
    x = Tensor("x", dims=[t], dtype="int64", sparse_dim=model.vocab_dim, raw_tensor=torch.tensor(labels, device=device))
    logits, _ = model(x, spatial_dim=t, state=model.default_initial_state(batch_dims=[]))
    return logits.copy_compatible_to_dims_raw([t, model.vocab_dim])


def _texts(vocab, lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(1, vocab, (n,), generator=g).tolist() for n in lens]


KINDS = ["sinusoidal", "rotary", "normed", "fused"]


def _check_scores(model, paged, texts, device, tol):
    for top in (0, 3):
        for text, got in zip(texts, paged.score(texts, num_top=top)):
            with torch.no_grad():
                lp = torch.log_softmax(_rf_logits(model, text, device).double(), -1)[:-1]
            want = lp.gather(1, torch.tensor(text[1:], device=device)[:, None])[:, 0]
            assert got.log_probs.shape == (len(text) - 1,)
            assert ((got.log_probs.double() - want).abs() <= tol * (1 + want.abs())).all()
            assert ((got.entropy.double() + (lp.exp() * lp).sum(-1)).abs() <= tol * 10).all()
            if top:
                best = lp.topk(3, dim=-1).values
                assert ((got.top_log_probs.double() - best).abs() <= tol * (1 + best.abs())).all()
                assert ((lp.gather(1, got.top_labels.long()) - best).abs() <= 2 * tol * (1 + best.abs())).all()
    assert not paged.lengths.any() and int(paged.free_range[1] - paged.free_range[0]) == paged.num_pages


def _check_generation(model, paged, prompts, device, *, max_new, eos, tol):
    got = paged.generate(prompts, max_new=max_new, eos=eos)
    for prompt, res in zip(prompts, got):
        with torch.no_grad():
            lp = torch.log_softmax(_rf_logits(model, prompt + res.labels, device).double(), -1)
        n = len(res.labels)
        assert 1 <= n <= max_new and eos not in res.labels[:-1] and (res.labels[-1] == eos or n == max_new or len(prompt) + n == paged.max_len)
        for i, (label, p) in enumerate(zip(res.labels, res.log_probs)):
            row = lp[len(prompt) - 1 + i]
            assert abs(float(row[label]) - p) <= tol * (1 + abs(p))
            assert float(row.max() - row[label]) <= 2 * tol * (1 + abs(p))  # the best one, or one as good
    assert not paged.lengths.any() and int(paged.free_range[1] - paged.free_range[0]) == paged.num_pages
    return got


@pytest.mark.parametrize("kind", KINDS)
def test_score_and_generate_cpu(kind):
    from returnn_b200.models.paged_decoder import PagedDecoder

    model = _decoder(kind)
    paged = PagedDecoder(model, max_requests=3, max_len=24, page_size=4)
    # sums of 32 to 44 products in fp32 through two layers
    _check_scores(model, paged, _texts(61, [5, 1, 9, 24, 2]), "cpu", 1e-4)
    _check_generation(model, paged, _texts(61, [3, 7, 1, 20, 4, 23], seed=1), "cpu", max_new=6, eos=0, tol=1e-4)
    # a pool that holds two at a time, on average: requests wait for pages, results are the same
    small = PagedDecoder(model, max_requests=3, max_len=24, page_size=4, num_pages=9)
    a = _check_generation(model, small, _texts(61, [3, 7, 1, 12, 4], seed=2), "cpu", max_new=4, eos=0, tol=1e-4)
    b = paged.generate(_texts(61, [3, 7, 1, 12, 4], seed=2), max_new=4, eos=0)
    assert [x.labels for x in a] == [x.labels for x in b]
    with pytest.raises(RuntimeError):
        PagedDecoder(model, max_requests=1, max_len=24, page_size=4, num_pages=2).generate(_texts(61, [9]), max_new=1, eos=0)
    with pytest.raises(ValueError):
        paged.generate([[]], max_new=1, eos=0)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_score_and_generate(kind):
    """fp32 on the GPU: labels and scores of the RF decoder; with and without the captured step"""
    from returnn_b200.models.paged_decoder import PagedDecoder

    model = _decoder(kind, heads=4, dim=128, vocab=1003, device="cuda")
    with torch.no_grad():
        paged = PagedDecoder(model, max_requests=4, max_len=200, page_size=16)
        _check_scores(model, paged, _texts(1003, [5, 1, 90, 200, 33, 16]), "cuda", 1e-3)
        prompts = _texts(1003, [3, 70, 1, 190, 16, 15], seed=1)
        one = _check_generation(model, paged, prompts, "cuda", max_new=20, eos=0, tol=1e-3)
        two = paged.generate(prompts, max_new=20, eos=0, use_graph=False)
        assert [x.labels for x in one] == [x.labels for x in two]


@gpu
def test_generate_bf16():
    """bf16 with head dim 64: log probabilities within the rounding of two layers, the same requests together and alone"""
    from returnn_b200.models.paged_decoder import PagedDecoder

    model = _decoder("normed", heads=8, dim=512, vocab=5000, device="cuda")
    paged = PagedDecoder(model, max_requests=5, max_len=300, page_size=16, dtype=torch.bfloat16)
    prompts = _texts(5000, [3, 170, 17, 64, 100, 8, 250], seed=1)
    got = paged.generate(prompts, max_new=12, eos=0)
    for prompt, res in zip(prompts, got):
        with torch.no_grad():
            lp = torch.log_softmax(_rf_logits(model, prompt + res.labels, "cuda").double(), -1)
        for i, (label, p) in enumerate(zip(res.labels, res.log_probs)):
            row = lp[len(prompt) - 1 + i]
            # logits of a size of up to 10 through roundings of 2^-9 in two layers and the output product
            assert abs(float(row[label]) - p) <= 0.25 and float(row.max() - row[label]) <= 0.5


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_rf_token_log_probs(device):
    import returnn_b200.frontend as rf
    from returnn_b200.tensor import Tensor, Dim

    rf.select_backend_torch()
    g = torch.Generator().manual_seed(3)
    b, t, v = Dim(3, name="b"), Dim(5, name="t"), Dim(50, name="v")
    raw = torch.randn(3, 50, 5, generator=g).to(device).requires_grad_(True)  # (labels in the middle)
    logits = Tensor("logits", dims=[b, v, t], dtype="float32", raw_tensor=raw)
    target = Tensor("target", dims=[t, b], dtype="int32", sparse_dim=v, raw_tensor=torch.randint(0, 50, (5, 3), generator=g, dtype=torch.int32).to(device))
    r = rf.token_log_probs(logits=logits, target=target, axis=v, entropy=True, num_top=4)
    lp = torch.log_softmax(raw.detach().double(), 1)
    want = lp.gather(1, target.raw_tensor.t().long()[:, None])[:, 0]
    assert r.log_probs.dims == (b, t) and (r.log_probs.raw_tensor.double() - want).abs().max() < 1e-5
    assert (r.entropy.raw_tensor.double() + (lp.exp() * lp).sum(1)).abs().max() < 1e-5
    values, labels = lp.topk(4, dim=1)
    assert r.top_labels.sparse_dim == v and r.top_labels.dims == (b, t, r.top_dim) and torch.equal(r.top_labels.raw_tensor.long(), labels.transpose(1, 2))
    assert (r.top_log_probs.raw_tensor.double() - values.transpose(1, 2)).abs().max() < 1e-5
    (grad,) = torch.autograd.grad(r.log_probs.raw_tensor.sum(), [raw])
    onehot = torch.zeros(3, 50, 5, dtype=torch.float64, device=device).scatter_(1, target.raw_tensor.t().long()[:, None], 1.0)
    assert (grad.double() - (onehot - lp.exp())).abs().max() < 1e-5
    with pytest.raises(ValueError):
        rf.token_log_probs(logits=logits, target=Tensor("x", dims=[t, b], dtype="int32", sparse_dim=b, raw_tensor=target.raw_tensor), axis=v)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_rf_rotary_options(device):
    """rope={} is the rotation of the module without options; whole sequences and steps agree with a norm, a part rotated and scaled frequencies; gradients reach the scales"""
    import returnn_b200.frontend as rf
    from returnn_b200.tensor import Tensor, Dim, single_step_dim

    rf.select_backend_torch()
    torch.manual_seed(0)
    feat, time, batch_dim = Dim(64, name="feat"), Dim(9, name="time"), Dim(3, name="batch")
    base = dict(key_dim_total=feat, value_dim_total=feat, num_heads=2, att_dropout=0.0)
    x = Tensor("x", dims=[batch_dim, time, feat], dtype="float32", feature_dim=feat, raw_tensor=torch.randn(3, 9, 64).to(device))

    def build(cls, **kw):
        m = cls(feat, feat, **base, **kw)
        g = torch.Generator().manual_seed(1)
        for name, p in m.named_parameters():
            t = torch.randn(p.raw_tensor.shape, generator=g) * (0.1 if "norm" in name else 0.2) + (1.0 if "norm" in name else 0.0)
            p.raw_tensor = torch.nn.Parameter(t.to(device))
        return m

    # (the angle of the module without options is a product in fp32, at most 8 radians here)
    plain, fused = build(rf.RotaryPosSelfAttention), build(rf.RotaryPosSelfAttention, rope={})
    assert (plain(x, axis=time).raw_tensor - fused(x, axis=time).raw_tensor).abs().max() < (5e-2 if device == "cuda" else 1e-4)
    m = build(rf.RotaryPosCausalSelfAttention, qk_norm=True, rope=dict(rotary_dim=16, interleaved=False, scaling=dict(type="linear", factor=2.0)))
    assert {n for n, _ in m.named_parameters() if "norm" in n} == {"q_norm.scale", "k_norm.scale"}
    whole, _ = m(x, axis=time)
    state = m.default_initial_state(batch_dims=[batch_dim])
    for t in range(9):
        step = Tensor("s", dims=[batch_dim, feat], dtype="float32", feature_dim=feat, raw_tensor=x.raw_tensor[:, t])
        if device == "cuda":
            for n in ("k_accum", "v_accum"):
                state[n].raw_tensor = state[n].raw_tensor.to(device)
        y, state = m(step, axis=single_step_dim, state=state)
        assert (y.copy_compatible_to_dims_raw([batch_dim, feat]) - whole.copy_compatible_to_dims_raw([batch_dim, time, feat])[:, t]).abs().max() < (5e-2 if device == "cuda" else 1e-4)
    whole.raw_tensor.square().sum().backward()
    for n, p in m.named_parameters():
        assert p.raw_tensor.grad is not None and torch.isfinite(p.raw_tensor.grad).all() and p.raw_tensor.grad.any(), n
    for bad, err in ((dict(rope=dict(other=1)), TypeError), (dict(rope=dict(rotary_dim=34)), ValueError), (dict(rope=dict(rotary_dim=7)), ValueError)):
        with pytest.raises(err):
            build(rf.RotaryPosSelfAttention, **bad)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_demo(device):
    import os
    import subprocess
    import sys

    demos = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "demos")
    res = subprocess.run([sys.executable, "demo-serve-lm.py", "--device", device, "--max-new", "4"], cwd=demos, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.count("log probability") == 12
