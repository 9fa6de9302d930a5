"""Norm per head and rotary positions (ops/norm_rope.py): against 64 bits, gradients against the formula's and against differences, the cache form, refusals."""

import math
import pytest
import torch

gpu = pytest.mark.gpu


def _exact(x, positions, frequencies, scale, eps, interleaved, amplitude):
    """(rotated, before the rotation) in 64 bits, from complex numbers; positions [N]"""
    y = x.double()
    if scale is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * scale.double()
    if frequencies is None:
        return y, y
    f = frequencies.shape[0]
    turn = torch.polar(torch.tensor(amplitude, dtype=torch.float64, device=x.device), positions.double()[:, None] * frequencies.double())[:, None, :]
    order = torch.arange(2 * f, device=x.device)
    order = order.view(f, 2) if interleaved else order.view(2, f).t()
    z = y.clone()
    z[..., order] = torch.view_as_real(torch.complex(y[..., order[:, 0]], y[..., order[:, 1]]) * turn)
    return z, y


def _inputs(n, hq, hk, d, dtype, device, seed=0, fused=True, pos_max=100_000):
    g = torch.Generator(device="cpu").manual_seed(seed)
    if fused:  # slices of one projection
        x = torch.randn(n, (hq + 2 * hk), d, generator=g).to(device, dtype)
        q, k, v = x[:, :hq], x[:, hq: hq + hk], x[:, hq + hk:]
    else:
        q, k, v = (torch.randn(n, h, d, generator=g).to(device, dtype) for h in (hq, hk, hk))
    wq, wk = ((torch.randn(d, generator=g) * 0.3 + 1.0).to(device) for _ in range(2))
    pos = torch.randint(0, pos_max, (n,), generator=g).to(device)
    return q, k, v, wq, wk, pos


def _near(got, want, before, dtype, what):
    # a rounding to the type; in fp32 a sum of up to 256 squares, a root and a division of 2 ulp, two products of a sine of 2 ulp: 2^-19 of the row's largest
    tol = (2.0**-8 if dtype == torch.bfloat16 else 2.0**-23) * want.abs() + 2.0**-19 * before.abs().amax(-1, keepdim=True)
    assert got.dtype == dtype and got.shape == want.shape
    assert ((got.double() - want).abs() <= tol).all(), "%s: %g of the tolerance" % (what, ((got.double() - want).abs() / tol).max())


CASES = [(3, 2, 2, 64, 64), (1, 1, 1, 8, 8), (7, 5, 5, 20, 10), (65, 32, 8, 128, 64), (33, 6, 1, 80, 80), (9, 8, 4, 256, 128), (4, 3, 3, 96, 32), (5, 2, 1, 16, 16), (2, 1, 1, 2, 2),
         (3, 4, 2, 12, 6), (600, 4, 4, 32, 0), (3, 2, 2, 7, 4), (40, 2, 0, 64, 64)]


def test_frequencies():
    from returnn_b200.ops.norm_rope import rope_frequencies

    f, a = rope_frequencies(8)
    assert a == 1.0 and f.dtype == torch.float32 and torch.allclose(f.double(), torch.tensor([1.0, 0.1, 0.01, 0.001]).double())
    assert torch.allclose(rope_frequencies(8, scaling={"type": "linear", "factor": 4})[0], f / 4)
    g, _ = rope_frequencies(64, scaling={"type": "base", "factor": 4})
    f, _ = rope_frequencies(64)
    assert g[0] == 1.0 and math.isclose(float(g[-1] * 4), float(f[-1]), rel_tol=1e-5)
    g, a = rope_frequencies(64, scaling={"type": "by_parts", "factor": 4, "original_length": 2048})
    turns = f.double() * 2048 / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 4)
    assert math.isclose(a, 0.1 * math.log(4) + 1)
    assert ((g <= f) & (g >= f / 4 * (1 - 1e-6))).all()
    for bad in (dict(type="other"), dict(type="linear", factor=2, more=1), dict(type="linear", factor=0), dict(type="by_parts", factor=2, original_length=10, low=3, high=2)):
        with pytest.raises(ValueError):
            rope_frequencies(8, scaling=bad)
    with pytest.raises(ValueError):
        rope_frequencies(7)


def _forward(device, dtype, n, hq, hk, d, rot, interleaved, norm, fused=True):
    from returnn_b200.ops.norm_rope import norm_rope, rope_frequencies

    q, k, _, wq, wk, pos = _inputs(n, hq, hk, d, dtype, device, seed=n + d, fused=fused)
    f = rope_frequencies(rot, device=device)[0] if rot else None
    amp = 1.25 if interleaved else 1.0
    oq, ok = norm_rope(q, k, pos, f, q_scale=wq if norm else None, k_scale=wk if norm else None, eps=1e-5, interleaved=interleaved, amplitude=amp)
    for got, x, w in ((oq, q, wq), (ok, k, wk)):
        want, before = _exact(x, pos, f, w if norm else None, 1e-5, interleaved, amp)
        if before.shape[1]:
            _near(got, want, before * 1.25, dtype, (n, hq, hk, d, rot, interleaved, norm))
        assert got.is_contiguous()


@pytest.mark.parametrize("interleaved", [True, False])
def test_forward_cpu(interleaved):
    for case in CASES:
        for norm in (True, False):
            _forward("cpu", torch.float32, *case, interleaved, norm)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("norm", [True, False])
def test_forward(dtype, interleaved, norm):
    for case in CASES:
        _forward("cuda", dtype, *case, interleaved, norm)
        _forward("cuda", dtype, *case, interleaved, norm, fused=False)


@gpu
def test_rows_and_positions_of_other_layouts():
    """heads before tokens, offsets that are not 16 bytes, features with a stride, positions per token axis and repeated, int32, negative"""
    from returnn_b200.ops.norm_rope import norm_rope, rope_frequencies

    g = torch.Generator().manual_seed(3)
    f = rope_frequencies(64, device="cuda")[0]
    base = torch.randn(2, 4, 9, 64, generator=g).cuda()  # [B, H, T, D]
    views = [base.transpose(1, 2), torch.randn(2, 9, 4, 65, generator=g).cuda()[..., 1:], torch.randn(2, 9, 4, 128, generator=g).cuda()[..., ::2],
             torch.randn(2, 9, 1, 64, generator=g).cuda().expand(2, 9, 4, 64)]
    pos = torch.arange(9, device="cuda", dtype=torch.int32) - 4
    for x in views:
        for dtype in (torch.float32, torch.bfloat16):
            y = x.to(dtype) if x.is_contiguous() else torch.empty_strided(x.shape, x.stride(), dtype=dtype, device="cuda").copy_(x) if 0 not in x.stride() else x.to(dtype)
            oq, ok = norm_rope(y, y, pos, f, interleaved=False)
            full = pos.expand(2, 9).reshape(-1)
            want, before = _exact(y.reshape(18, 4, 64), full, f, None, 0.0, False, 1.0)
            _near(oq.reshape(18, 4, 64), want, before, dtype, x.stride())
            assert torch.equal(oq, ok)
            assert torch.equal(norm_rope(y, y, pos.expand(2, 9).long(), f, interleaved=False)[0], oq)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("norm", [True, False])
def test_gradient(dtype, interleaved, norm):
    from returnn_b200.ops.norm_rope import norm_rope, norm_rope_reference, rope_frequencies

    for n, hq, hk, d, rot in CASES + [(3000, 4, 2, 64, 64), (0, 2, 2, 64, 64)]:
        q, k, _, wq, wk, pos = _inputs(n, hq, hk, d, dtype, "cuda", seed=n + d)
        f = rope_frequencies(rot, device="cuda")[0] if rot else None
        leaves = [q.detach().requires_grad_(True), k.detach().requires_grad_(True)] + ([wq.requires_grad_(True), wk.requires_grad_(True)] if norm else [])
        opts = dict(eps=1e-5, interleaved=interleaved, amplitude=0.75)
        scales = dict(q_scale=wq, k_scale=wk) if norm else {}
        out = norm_rope(leaves[0], leaves[1], pos, f, **scales, **opts)
        g = torch.Generator().manual_seed(n)
        dz = [torch.randn(o.shape, generator=g).cuda().to(dtype) for o in out]
        got = torch.autograd.grad(out, leaves, dz)
        wide = [x.detach().double().requires_grad_(True) for x in leaves]
        again = []
        for i in (0, 1):  # the definition, differentiated in 64 bits
            y = wide[i]
            if norm:
                y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + 1e-5) * wide[2 + i]
            if rot:
                ang = pos.double()[:, None, None] * f.double()
                a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., : rot // 2], y[..., rot // 2: rot])
                a, b = 0.75 * (a * ang.cos() - b * ang.sin()), 0.75 * (a * ang.sin() + b * ang.cos())
                y = torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), y[..., rot:]], -1)
            again.append(y)
        want = torch.autograd.grad(again, wide, [x.double() for x in dz], allow_unused=True)
        for i, (x, y) in enumerate(zip(got, want)):
            y = torch.zeros_like(x, dtype=torch.float64) if y is None else y
            assert x.shape == y.shape and x.dtype == leaves[i].dtype
            # sums of squares and products in fp32 and a rounding to the type; the gradients of scales are sums in fp32 over all rows
            rel = 2.0**-8 if x.dtype == torch.bfloat16 else 2.0**-17
            assert (x.double() - y).norm() <= rel * y.norm() + 1e-12, (n, hq, hk, d, rot, i)
        rerun = torch.autograd.grad(norm_rope(leaves[0], leaves[1], pos, f, **scales, **opts), leaves, dz)
        assert all(torch.equal(a, b) for a, b in zip(got, rerun))
        if dtype == torch.float32 and n == 65:  # the plain form has the same gradients
            ref = torch.autograd.grad(norm_rope_reference(leaves[0], leaves[1], pos, f, **scales, **opts), leaves, dz)
            assert all((a - b).norm() <= 2.0**-16 * b.norm() for a, b in zip(got, ref))


@gpu
def test_gradient_against_differences():
    """along random directions; the step's own error is its square, the rounding of the values divided by the step 2^-23 / 2^-6 of their size"""
    from returnn_b200.ops.norm_rope import norm_rope, rope_frequencies

    for interleaved, d, rot in ((True, 64, 64), (False, 128, 64), (True, 20, 10)):
        q, k, _, wq, wk, pos = _inputs(11, 3, 2, d, torch.float32, "cuda", seed=d)
        leaves = [x.contiguous().requires_grad_(True) for x in (q, k, wq, wk)]
        f = rope_frequencies(rot, device="cuda")[0]
        g = torch.Generator().manual_seed(1)
        c = [torch.randn(x.shape, generator=g).cuda() for x in (q, k)]

        def loss(xs):
            o = norm_rope(xs[0], xs[1], pos, f, q_scale=xs[2], k_scale=xs[3], interleaved=interleaved)
            return sum((a.double() * b.double()).sum() for a, b in zip(o, c))

        grads = torch.autograd.grad(loss(leaves), leaves)
        for i, x in enumerate(leaves):
            v = torch.randn(x.shape, generator=g).cuda()
            h = 2.0**-6
            with torch.no_grad():
                plus, minus = (loss([y + s * h * v if j == i else y for j, y in enumerate(leaves)]) for s in (1, -1))
            want = (plus - minus) / (2 * h)
            size = grads[i].double().norm() * v.double().norm()
            assert (grads[i].double() * v.double()).sum().sub(want).abs() <= 2.0**-9 * size, (interleaved, d, i)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,hq,hk,d,rot,page,layout", [(64, 32, 8, 128, 128, 16, "heads"), (1, 8, 8, 64, 64, 1, "tokens"), (37, 6, 1, 80, 40, 100, "heads"),
                                                       (5, 5, 5, 20, 20, 7, "tokens"), (300, 4, 2, 256, 0, 8, "heads")])
def test_to_cache(dtype, n, hq, hk, d, rot, page, layout):
    from returnn_b200.ops.norm_rope import norm_rope, norm_rope_to_cache, rope_frequencies

    q, k, v, wq, wk, pos = _inputs(n, hq, hk, d, dtype, "cuda", seed=n)
    f = rope_frequencies(rot, device="cuda")[0] if rot else None
    pages = n * 2 // page + 2
    shape = (pages, hk, page, d) if layout == "heads" else (pages, page, hk, d)
    caches = [torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2)]
    kc, vc = (c if layout == "heads" else c.transpose(1, 2) for c in caches)
    g = torch.Generator().manual_seed(n)
    slots = torch.randperm(pages * page, generator=g)[:n].to(torch.int32)
    slots[torch.rand(n, generator=g) < 0.1] = -1
    if n > 3:
        slots[2] = pages * page  # past the end
    slots = slots.cuda()
    opts = dict(q_scale=wq, k_scale=wk, interleaved=False)
    oq = norm_rope_to_cache(q, k, v, pos, f, kc, vc, slots, **opts)
    wantq, wantk = norm_rope(q, k, pos, f, **opts)
    assert torch.equal(oq, wantq)
    kept = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            kept[s // page, s % page] = True
            assert torch.equal(kc[s // page, :, s % page], wantk[t]) and torch.equal(vc[s // page, :, s % page], v[t])
    for c in (kc, vc):  # nothing else is written
        assert c.transpose(1, 2)[~kept].isnan().all() and not c.transpose(1, 2)[kept].isnan().any()


def test_to_cache_cpu():
    from returnn_b200.ops.norm_rope import norm_rope, norm_rope_to_cache, rope_frequencies

    q, k, v, wq, wk, pos = _inputs(5, 4, 2, 8, torch.float32, "cpu")
    f = rope_frequencies(8)[0]
    kc, vc = torch.zeros(2, 2, 2, 3, 8).unbind(0)
    slots = torch.tensor([5, -1, 0, 6, 2], dtype=torch.int32)
    oq = norm_rope_to_cache(q, k, v, pos, f, kc, vc, slots, q_scale=wq, k_scale=wk)
    wq_, wk_ = norm_rope(q, k, pos, f, q_scale=wq, k_scale=wk)
    assert torch.equal(oq, wq_) and torch.equal(kc[1, :, 2], wk_[0]) and torch.equal(vc[0, :, 0], v[2]) and torch.equal(vc[0, :, 2], v[4])
    assert not vc[0, :, 1].any() and not kc[1, :, :2].any()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    from returnn_b200.ops.norm_rope import norm_rope, norm_rope_to_cache, rope_frequencies

    q, k, v, wq, wk, pos = _inputs(6, 4, 2, 16, torch.float32, device)
    f = rope_frequencies(16, device=device)[0]
    for args, kw, err in [((q, k[:5], pos, f), {}, ValueError), ((q, k.double(), pos, f), {}, TypeError), ((q, k, pos.float(), f), {}, TypeError), ((q, k, pos[:5], f), {}, ValueError),
                          ((q, k, pos, f.double()), {}, ValueError), ((q, k, pos, rope_frequencies(18, device=device)[0]), {}, ValueError),
                          ((q, k, pos, f), dict(q_scale=wq), ValueError), ((q, k, pos, f), dict(q_scale=wq, k_scale=wk[:8]), ValueError), ((q[0], k[0], pos, f), {}, ValueError)]:
        with pytest.raises(err):
            norm_rope(*args, **kw)
    kc, vc = torch.zeros(2, 4, 2, 3, 16, device=device).unbind(0)
    slots = torch.zeros(6, dtype=torch.int32, device=device)
    for a in [(q, k, v, pos, f, kc[:, :1], vc[:, :1], slots), (q, k, v, pos, f, kc, vc[:3], slots), (q, k, v, pos, f, kc, vc, slots.long()), (q, k, v, pos, f, kc, vc, slots[:3]),
              (q, k, v[:, :1], pos, f, kc, vc, slots), (q, k, v, pos, f, kc.bfloat16(), vc.bfloat16(), slots)]:
        with pytest.raises(ValueError):
            norm_rope_to_cache(*a)
    with pytest.raises(RuntimeError):
        norm_rope_to_cache(q.detach().requires_grad_(True), k, v, pos, f, kc, vc, slots)
    if device == "cuda":
        with pytest.raises(TypeError):
            norm_rope(q.half(), k.half(), pos, f)
        big = torch.zeros(1, 1, 258, device=device)
        with pytest.raises(ValueError):
            norm_rope(big, big, None, None)


@gpu
@pytest.mark.parametrize("eps", [0.0, 1e-40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_without_epsilon(dtype, eps):
    """places of a tile and groups of lanes without a row add nothing to the gradients of the scales: rows of zeros have no norm there"""
    from returnn_b200.ops.norm_rope import norm_rope, rope_frequencies

    for n, hq, hk, d, rot in [(1, 1, 1, 64, 64), (7, 6, 1, 80, 80), (65, 3, 2, 128, 64), (7, 5, 5, 20, 10), (1, 2, 1, 8, 8), (300, 5, 3, 64, 0), (65, 7, 4, 256, 128)]:
        for interleaved in (True, False):
            q, k, _, wq, wk, pos = _inputs(n, hq, hk, d, dtype, "cuda", seed=n + d)
            f = rope_frequencies(rot, device="cuda")[0] if rot else None
            leaves = [x.detach().requires_grad_(True) for x in (q, k, wq, wk)]
            out = norm_rope(leaves[0], leaves[1], pos, f, q_scale=leaves[2], k_scale=leaves[3], eps=eps, interleaved=interleaved)
            g = torch.Generator().manual_seed(n)
            dz = [torch.randn(o.shape, generator=g).cuda().to(dtype) for o in out]
            got = torch.autograd.grad(out, leaves, dz)
            wide = [x.detach().double().requires_grad_(True) for x in leaves]
            exact = [_exact(wide[i], pos, f, wide[2 + i], eps, interleaved, 1.0)[0] for i in (0, 1)]
            for i, (x, y) in enumerate(zip(got, torch.autograd.grad(exact, wide, [x.double() for x in dz]))):
                rel = 2.0**-8 if x.dtype == torch.bfloat16 else 2.0**-17  # (as with an epsilon)
                assert (x.double() - y).norm() <= rel * y.norm() + 1e-12, (n, hq, hk, d, rot, interleaved, i)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_no_heads_and_several_token_axes(device):
    """results of no elements, and the other operand's as without them"""
    from returnn_b200.ops.norm_rope import norm_rope, rope_frequencies

    f, pos = rope_frequencies(64, device=device)[0], torch.arange(3, device=device)
    w = [torch.ones(64, device=device, requires_grad=True) for _ in range(2)]
    k = torch.randn(2, 3, 4, 64, generator=torch.Generator().manual_seed(1)).to(device).requires_grad_(True)
    q = torch.empty(2, 3, 0, 64, device=device, requires_grad=True)
    for scales in (dict(q_scale=w[0], k_scale=w[1]), {}):
        oq, ok = norm_rope(q, k, pos, f, **scales)
        same, alone = norm_rope(k, k, pos, f, **scales)
        assert oq.shape == q.shape and torch.equal(ok, alone) and torch.equal(same, alone)
        swapped = norm_rope(k, q, pos, f, **scales)
        assert swapped[1].shape == q.shape and torch.equal(swapped[0], alone)
        leaves = [q, k] + (w if scales else [])
        got, want = torch.autograd.grad([oq, ok], leaves, [oq, ok.detach()]), torch.autograd.grad(alone, [k] + w[1:] * bool(scales), ok.detach())
        assert got[0].shape == q.shape and torch.equal(got[1], want[0])
        if scales:
            assert not got[2].any() and torch.allclose(got[3], want[1], rtol=2.0**-20, atol=1e-6)
        with torch.no_grad():
            assert norm_rope(q, k, pos, f, **scales)[0].shape == q.shape


@gpu
def test_gradient_without_tokens():
    """scales of nothing have a gradient of zero, however many heads there are"""
    from returnn_b200.ops.norm_rope import norm_rope, rope_frequencies

    for hq, hk, d in ((5000, 9, 256), (4, 2, 64), (3, 3, 20), (0, 0, 64)):
        q, k = (torch.empty(0, h, d, device="cuda", requires_grad=True) for h in (hq, hk))
        for dtype in (torch.float32, torch.bfloat16):
            w = [torch.ones(d, device="cuda", dtype=dtype, requires_grad=True) for _ in range(2)]
            out = norm_rope(q, k, torch.empty(0, dtype=torch.int32, device="cuda"), rope_frequencies(d, device="cuda")[0], q_scale=w[0], k_scale=w[1])
            got = torch.autograd.grad(out, [q, k] + w, [torch.empty_like(o) for o in out])
            assert got[0].shape == q.shape and got[1].shape == k.shape
            assert all(g.shape == (d,) and g.dtype == dtype and not g.any() for g in got[2:])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_frequencies_have_no_gradient(device):
    from returnn_b200.ops.norm_rope import norm_rope, norm_rope_to_cache, rope_frequencies

    q, k, v, _, _, pos = _inputs(6, 4, 2, 16, torch.float32, device)
    f = rope_frequencies(16, device=device)[0].requires_grad_(True)
    kc, vc = torch.zeros(2, 4, 2, 3, 16, device=device).unbind(0)
    slots = torch.arange(6, dtype=torch.int32, device=device)
    with pytest.raises(RuntimeError, match="frequencies"):
        norm_rope(q, k, pos, f)
    with pytest.raises(RuntimeError):
        norm_rope_to_cache(q, k, v, pos, f, kc, vc, slots)
    with torch.no_grad():
        want = norm_rope(q, k, pos, f.detach())
        assert all(torch.equal(a, b) for a, b in zip(norm_rope(q, k, pos, f), want))
        assert torch.equal(norm_rope_to_cache(q, k, v, pos, f, kc, vc, slots), want[0])


@pytest.mark.parametrize("device,python", [("cpu", False), pytest.param("cuda", False, marks=gpu), pytest.param("cuda", True, marks=gpu)])
def test_caches_written_in_place(monkeypatch, device, python):
    """autograd learns of the write: a cache that a graph still needs is noticed, one that requires a gradient refused"""
    from returnn_b200.ops import nodes
    from returnn_b200.ops.norm_rope import norm_rope_to_cache, rope_frequencies

    if python:
        monkeypatch.setattr(nodes, "active", lambda: None)
    q, k, v, _, _, pos = _inputs(6, 4, 2, 16, torch.float32, device)
    f = rope_frequencies(16, device=device)[0]
    kc, vc = (torch.zeros(4, 2, 3, 16, device=device) for _ in range(2))
    slots = torch.arange(6, dtype=torch.int32, device=device)
    x = torch.ones_like(kc).requires_grad_(True)
    loss = (x * kc).sum() + (x * vc).sum()
    norm_rope_to_cache(q, k, v, pos, f, kc, vc, slots)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    for caches in ((kc.clone().requires_grad_(True), vc), (kc, vc.clone().requires_grad_(True)), (kc, vc * x)):
        with pytest.raises(RuntimeError):
            norm_rope_to_cache(q, k, v, pos, f, *caches, slots)
    with torch.inference_mode():
        inner = torch.zeros(2, 4, 2, 3, 16, device=device)
        norm_rope_to_cache(q, k, v, pos, f, inner[0], inner[1], slots)
    norm_rope_to_cache(q, k, v, pos, f, kc, vc, slots)
    assert torch.equal(inner[0], kc) and torch.equal(inner[1], vc)
