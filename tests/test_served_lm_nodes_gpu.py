"""The operators of a served language model through the Python functions (traced programs, installations without the extension) and through the extension: the same bits."""

import pytest
import torch

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("norm", [True, False])
def test_norm_rope(monkeypatch, norm):
    from returnn_b200.ops import nodes
    from returnn_b200.ops.norm_rope import norm_rope, norm_rope_to_cache, rope_frequencies

    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 9, 3, 3 * 64, generator=g).to("cuda", torch.bfloat16)
    q, k, v = (t.detach() for t in x.split(64, -1))
    w = [(torch.randn(64, generator=g) + 1.0).cuda().requires_grad_(True) for _ in range(2)]
    f, pos = rope_frequencies(32, device="cuda")[0], torch.arange(9, device="cuda")
    d = [torch.randn(2, 9, 3, 64, generator=g).to("cuda", torch.bfloat16) for _ in range(2)]
    opts = dict(q_scale=w[0], k_scale=w[1]) if norm else {}

    def run():
        leaves = [q.requires_grad_(True), k.requires_grad_(True)] + (w if norm else [])
        out = norm_rope(q, k, pos, f, **opts)
        res = [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, d))
        caches = torch.zeros(2, 5, 3, 4, 64, dtype=torch.bfloat16, device="cuda").unbind(0)
        with torch.no_grad():
            res.append(norm_rope_to_cache(q.reshape(18, 3, 64), k.reshape(18, 3, 64), v.reshape(18, 3, 64), pos.repeat(2), f, *caches, torch.arange(18, dtype=torch.int32, device="cuda"),
                                          **opts))
            res += list(norm_rope(q, k, pos, f, **opts))
        return res + list(caches)

    assert nodes.active() is not None
    one = run()
    monkeypatch.setattr(nodes, "active", lambda: None)
    two = run()
    assert len(one) == len(two) and all(torch.equal(a, b) and a.dtype == b.dtype and a.shape == b.shape for a, b in zip(one, two))


@gpu
def test_paged(monkeypatch):
    from returnn_b200.ops import nodes
    from returnn_b200.ops.paged import append_tokens, paged_attention, release_pages

    def run():
        g = torch.Generator().manual_seed(0)
        i32 = dict(dtype=torch.int32, device="cuda")
        table, ring = torch.full((4, 8), -1, **i32), torch.arange(40, **i32)
        r = append_tokens(table, torch.zeros(4, **i32), torch.tensor([9, 0, 100, 33], **i32), ring, torch.tensor([35, 75], device="cuda"), page_size=16, max_tokens=150)
        kc, vc = torch.randn(2, 40, 2, 16, 64, generator=g).to("cuda", torch.bfloat16).unbind(0)
        o = paged_attention(torch.randn(4, 4, 64, generator=g).to("cuda", torch.bfloat16), kc, vc, table, r.lengths, scale=0.2)
        back = release_pages(table, r.lengths, torch.tensor([True, True, False, True], device="cuda"), ring, r.free_range, page_size=16)
        return [table, ring, o, *r, *back]

    one = run()
    monkeypatch.setattr(nodes, "active", lambda: None)
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(one, run()))


@gpu
@pytest.mark.parametrize("entropy", [True, False])
@pytest.mark.parametrize("top", [0, 3])
def test_token_log_probs(monkeypatch, entropy, top):
    from returnn_b200.ops import nodes
    from returnn_b200.ops.token_log_probs import token_log_probs

    g = torch.Generator().manual_seed(0)
    x = torch.randn(7, 1003, generator=g).cuda().requires_grad_(True)
    t = torch.randint(-1, 1003, (7,), generator=g).cuda()
    d = [torch.randn(7, generator=g).cuda(), torch.randn(7, generator=g).cuda(), torch.randn(7, 3, generator=g).cuda()]

    def run():
        r = token_log_probs(x, t, entropy=entropy, num_top=top)
        assert (r.entropy is not None) == entropy and (r.top_labels is not None) == bool(top)
        outs = [(o, g) for o, g in zip((r.log_probs, r.entropy, r.top_log_probs), d) if o is not None]
        res = [o.detach() for o, _ in outs] + list(torch.autograd.grad([o for o, _ in outs], [x], [g for _, g in outs], retain_graph=True))
        res += torch.autograd.grad([outs[-1][0]], [x], [outs[-1][1]])  # the others have no gradient
        with torch.no_grad():
            res += [o for o in token_log_probs(x, t, entropy=entropy, num_top=top) if o is not None]
        return res

    one = run()
    monkeypatch.setattr(nodes, "active", lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(one, run()))


def _rope_inputs():
    from returnn_b200.ops.norm_rope import rope_frequencies

    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(5, h, 64, generator=g).cuda() for h in (3, 2))
    w = [(torch.randn(64, generator=g) * 0.3 + 1.0).cuda() for _ in range(2)]
    return q, k, w, rope_frequencies(32, device="cuda")[0], torch.arange(5, device="cuda")


@gpu
@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_function_transforms_are_refused(monkeypatch, python, grad_mode):
    """torch.func and forward mode: an error, not a result without its derivative"""
    from torch.autograd import forward_ad
    from returnn_b200.ops import nodes
    from returnn_b200.ops.norm_rope import norm_rope, norm_rope_to_cache
    from returnn_b200.ops.paged import paged_attention
    from returnn_b200.ops.token_log_probs import token_log_probs

    if python:
        monkeypatch.setattr(nodes, "active", lambda: None)
    q, k, w, f, pos = _rope_inputs()
    kc, vc = torch.zeros(2, 3, 2, 4, 64, device="cuda").unbind(0)
    x, t = torch.randn(5, 40, device="cuda"), torch.arange(5, device="cuda")
    slots, table, lens = (torch.zeros(*s, dtype=torch.int32, device="cuda") for s in ((5,), (5, 2), (5,)))
    calls = [(lambda a: norm_rope(a, k, pos, f)[0], q), (lambda a: norm_rope(q, a, pos, f)[1], k), (lambda a: norm_rope(q, k, pos, f, q_scale=a, k_scale=w[1])[0], w[0]),
             (lambda a: norm_rope(q, k, pos, f, q_scale=w[0], k_scale=a)[1], w[1]), (lambda a: norm_rope(q, k, pos, a)[0], f),
             (lambda a: token_log_probs(a, t).log_probs, x), (lambda a: token_log_probs(a, t, entropy=True, num_top=2).entropy, x),
             (lambda a: norm_rope_to_cache(a, k, k, pos, f, kc, vc, slots), q), (lambda a: norm_rope_to_cache(q, k, a, pos, f, kc, vc, slots), k),
             (lambda a: norm_rope_to_cache(q, k, k, pos, f, a, vc, slots), kc),
             (lambda a: paged_attention(a, kc, vc, table, lens), q[:, :2]), (lambda a: paged_attention(q[:, :2], kc, a, table, lens), vc)]
    with torch.set_grad_enabled(grad_mode):
        for i, (call, arg) in enumerate(calls):
            with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
                call(forward_ad.make_dual(arg, torch.ones_like(arg)))
            with pytest.raises(RuntimeError):
                torch.func.vmap(lambda a: call(a))(arg[None])
            if grad_mode:
                with pytest.raises(RuntimeError):
                    torch.func.grad(lambda a: call(a).sum())(arg)
        with forward_ad.dual_level():  # a level without a tangent on these changes nothing
            norm_rope(q, k, pos, f)
            token_log_probs(x, t)
            norm_rope_to_cache(q, k, k, pos, f, kc, vc, slots)
            paged_attention(q[:, :2], kc, vc, table, lens)


@gpu
@pytest.mark.parametrize("python", [False, True])
def test_second_derivatives_are_refused(monkeypatch, python):
    """an error where a gradient is differentiated through these operators, not a result that leaves them out"""
    from returnn_b200.ops import nodes
    from returnn_b200.ops.norm_rope import norm_rope
    from returnn_b200.ops.token_log_probs import token_log_probs

    if python:
        monkeypatch.setattr(nodes, "active", lambda: None)
    q, k, w, f, pos = _rope_inputs()
    q, w = q.requires_grad_(True), [x.requires_grad_(True) for x in w]
    c = torch.randn(q.shape, device="cuda")
    x = torch.randn(5, 40, device="cuda", requires_grad=True)
    t = torch.arange(5, device="cuda")
    for loss, leaf in (((norm_rope(q, k, pos, f, q_scale=w[0], k_scale=w[1])[0] * c).sum(), q), ((norm_rope(q, k, pos, f, q_scale=w[0], k_scale=w[1])[0] * c).sum(), w[0]),
                       (norm_rope(q, k, pos, f)[0].square().sum(), q), (token_log_probs(x, t).log_probs.sum(), x),
                       (token_log_probs(x, t, entropy=True, num_top=2).top_log_probs.sum(), x)):
        (first,) = torch.autograd.grad(loss, leaf, create_graph=True, retain_graph=True)
        (again,) = torch.autograd.grad(loss, leaf)
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError):
            torch.autograd.grad((first.square().sum() + leaf.square().sum()), leaf)
    # a rotation alone is linear: its gradient does not depend on what was rotated
    (first,) = torch.autograd.grad((norm_rope(q, k, pos, f)[0] * c).sum(), q, create_graph=True)
    (second,) = torch.autograd.grad(first.sum() + q.square().sum(), q)
    assert torch.equal(second, 2 * q)
