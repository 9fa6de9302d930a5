"""Log probabilities of given tokens with entropy and alternatives (ops/token_log_probs.py): against 64 bits, gradients, ties, masked and broken rows, refusals."""

import math
import pytest
import torch

gpu = pytest.mark.gpu


def _exact(x, t):
    """log probabilities of all labels, of the targets, entropy, in 64 bits"""
    x = x.double()
    lp = torch.log_softmax(x, -1)
    lp[(x == -math.inf).all(-1)] = -math.inf
    given = (t >= 0) & (t < x.shape[1])
    out = torch.where(given, lp.gather(-1, t.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0], 0.0)
    return lp, out, torch.special.entr(lp.exp()).sum(-1)


def _tolerance(lp, v):
    # an exponent rounded to 2^-24 of itself, an exponential of 2 ulp, a sum of v / 256 and 16 terms, a logarithm: of the size of the log probability and absolute
    return 2.0**-21 * lp.abs() + 2.0**-19 + v / 256 * 2.0**-24


def _check(x, t, num_top, entropy=True, got=None):
    from returnn_b200.ops.token_log_probs import token_log_probs

    got = got or token_log_probs(x, t, entropy=entropy, num_top=num_top)
    lp, out, ent = _exact(x, t)
    v = x.shape[1]
    fin = torch.isfinite(out)
    assert torch.equal(got.log_probs.double()[~fin], out[~fin])
    assert ((got.log_probs.double() - out)[fin].abs() <= _tolerance(out, v)[fin]).all()
    if entropy:  # a sum of p z / sum p whose terms have the errors above times their size, up to log v and a few
        assert ((got.entropy.double() - ent).abs() <= 2.0**-17 * (1 + math.log(v))).all()
    if num_top:
        labels = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :num_top]
        assert torch.equal(got.top_labels.long(), labels)
        best = lp.gather(-1, labels)
        fin = torch.isfinite(best)
        assert torch.equal(got.top_log_probs.double()[~fin], best[~fin])
        assert ((got.top_log_probs.double() - best)[fin].abs() <= _tolerance(best, v)[fin]).all()


def _rows(rows, v, dtype, seed=0, scale=2.0, device="cuda"):
    g = torch.Generator().manual_seed(seed + rows + v)
    return (torch.randn(rows, v, generator=g) * scale).to(device, dtype), torch.randint(-1, v, (rows,), generator=g).to(device, torch.int32)


def test_cpu():
    for v, top in ((1, 1), (2, 2), (50, 5)):
        x, t = _rows(9, v, torch.float32, device="cpu")
        x[0] = -math.inf
        x[1, ::2] = -math.inf
        _check(x, t, top)
    x = x.double().requires_grad_(True)
    from returnn_b200.ops.token_log_probs import token_log_probs

    def f(y):
        r = token_log_probs(y, t, entropy=True, num_top=3)
        return r.log_probs[2:], r.entropy, r.top_log_probs[2:]

    y = torch.randn(9, 50, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda y: tuple(f(y)), (y,))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,v,top", [(1, 1, 1), (3, 2, 2), (5, 7, 7), (4, 33, 32), (3, 255, 5), (2, 1001, 8), (7, 4097, 1), (300, 10001, 8), (16, 32000, 5), (1, 128000, 20), (3, 50001, 32),
                                        (1300, 80, 0), (2, 32007, 0)])
@pytest.mark.parametrize("entropy", [True, False])
def test_forward(dtype, rows, v, top, entropy):
    x, t = _rows(rows, v, dtype)
    _check(x, t, top, entropy)
    _check(x, t.long(), top, entropy)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_and_odd_rows(dtype):
    """equal logits, sorted rows, few allowed labels, all large logits in the share of few threads, lowest values, large offsets"""
    v = 20_000
    rows = [torch.zeros(v), torch.arange(v).float(), -torch.arange(v).float(), torch.full((v,), -math.inf), torch.full((v,), torch.finfo(dtype).min),
            (torch.arange(v) % 5).float(), -(torch.arange(v) % 7).float() - 100.0]
    few = torch.full((v,), -math.inf)
    few[[19_999, 3, 700]] = torch.tensor([1.0, 1.0, 0.0])
    rows += [few, torch.where(torch.arange(v) % 2048 < 8, 5.0, -5.0) + torch.arange(v) % 3, torch.where(torch.arange(v) % 2048 < 64, 5.0 + torch.arange(v) * 1e-3, -5.0),
             torch.randn(v, generator=torch.Generator().manual_seed(1)) + 900.0, torch.randn(v, generator=torch.Generator().manual_seed(2)) - 30_000.0]
    mixed = torch.randn(v, generator=torch.Generator().manual_seed(3))
    mixed[100:19_000] = torch.finfo(dtype).min
    zeros = torch.where(torch.arange(v) % 2 == 0, -0.0, 0.0)
    rows += [mixed, zeros]
    x = torch.stack(rows).to(dtype).cuda()
    for top in (1, 8, 32):
        for shift in (0, 1, 3):  # rows that start off a 16-byte boundary
            y = torch.empty(len(rows), v + shift, dtype=dtype, device="cuda")[:, shift:].copy_(x)
            t = torch.arange(len(rows), device="cuda") * 1009
            # (the log probabilities of rows of the lowest values are the difference of such values: their size in the tolerance would say nothing)
            keep = [i for i in range(len(rows)) if i not in (1, 2, 4, 12)]
            from returnn_b200.ops.token_log_probs import token_log_probs

            r = token_log_probs(y, t, entropy=True, num_top=top)
            want = torch.sort(y.float(), dim=-1, descending=True, stable=True)[1][:, :top]
            assert torch.equal(r.top_labels.long(), want)
            assert not r.entropy.isnan().any() and not r.top_log_probs.isnan().any()
            # 2^-24 of an exponent of up to 30000
            lp, out, ent = _exact(y[keep], t[keep])
            assert ((r.entropy[keep].double() - ent).abs() <= 2.0**-17 * (1 + math.log(v))).all()
            best = lp.gather(-1, want[keep])
            fin = torch.isfinite(best)
            assert torch.equal(torch.isfinite(r.top_log_probs[keep]), fin)
            assert ((r.top_log_probs[keep].double() - best)[fin].abs() <= _tolerance(best, v)[fin] + 2.0**-17).all()
    assert math.isclose(float(r.entropy[0]), math.log(v), rel_tol=1e-5) and float(r.entropy[3]) == 0.0
    assert (r.top_log_probs[3] == -math.inf).all() and torch.equal(r.top_labels[3].cpu(), torch.arange(32, dtype=torch.int32))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_broken_rows(dtype):
    """NaN and +inf stay visible, are ranked first, and do not touch other rows; ignored rows have log probability 0"""
    from returnn_b200.ops.token_log_probs import token_log_probs

    v = 5000
    x, _ = _rows(6, v, dtype)
    x[1, 4000] = math.nan
    x[2, 17] = math.inf
    x[3] = math.nan
    x[4, 2:4990] = -math.nan
    t = torch.tensor([5, 5, 5, -1, v, 5], device="cuda")
    for top in (1, 8):
        r = token_log_probs(x, t, entropy=True, num_top=top)
        # (a sort puts NaN of negative sign last)
        want = torch.sort(torch.where(x.isnan(), math.nan, x.float()), dim=-1, descending=True, stable=True)[1][:, :top]
        assert torch.equal(r.top_labels.long(), want)
        assert r.log_probs[1:3].isnan().all() and r.entropy[1:5].isnan().all() and float(r.log_probs[3]) == float(r.log_probs[4]) == 0.0
        for i in (0, 5):
            _check(x[i: i + 1], t[i: i + 1], top)
        assert torch.isfinite(r.log_probs[[0, 5]]).all() and torch.isfinite(r.entropy[[0, 5]]).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,v,top,pad", [(5, 7, 3, 0), (40, 1001, 8, 7), (3, 32000, 0, 0), (2, 10_025, 32, 8), (1, 1, 1, 3), (9, 80, 5, 1)])
def test_gradient(dtype, rows, v, top, pad):
    from returnn_b200.ops.token_log_probs import token_log_probs

    x, t = _rows(rows, v + pad, dtype)
    x = x[:, :v]
    t = t % (v + 1) - 1
    if rows > 3:
        x[1] = -math.inf
        x[2, : v // 2] = -math.inf
    t[0] = int(x[0].float().argmax())  # a target that is among the best
    leaf = x.detach().requires_grad_(True)
    g = torch.Generator().manual_seed(v)
    ds = [torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda(), torch.randn(rows, top, generator=g).cuda()]
    for use in ((0,), (1,), (0, 1), (0, 1, 2), (2,)):
        if 2 in use and not top:
            continue
        r = token_log_probs(leaf, t, entropy=1 in use, num_top=top if 2 in use else 0)
        outs = [r.log_probs, r.entropy, r.top_log_probs]
        (got,) = torch.autograd.grad([outs[i] for i in use], [leaf], [ds[i] for i in use])
        lp, _, ent = _exact(x, t)
        p = lp.exp()
        none = (x == -math.inf).all(-1)
        weight = torch.zeros(rows, dtype=torch.float64, device="cuda")
        own = torch.zeros(rows, v, dtype=torch.float64, device="cuda")
        size = torch.zeros_like(weight)
        if 0 in use:
            d = torch.where(t >= 0, ds[0], 0.0).double()
            own.scatter_add_(1, t.long().clamp(min=0)[:, None], d[:, None])
            weight, size = weight + d, size + d.abs()
        if 2 in use:
            own.scatter_add_(1, r.top_labels.long(), ds[2].double())
            weight, size = weight + ds[2].double().sum(-1), size + ds[2].double().abs().sum(-1)
        want = own - p * weight[:, None]
        scale = own.abs() + p * size[:, None]
        if 1 in use:
            surprise = torch.where(p > 0, lp, 0.0)
            want = want - ds[1].double()[:, None] * p * (surprise + ent[:, None])
            scale = scale + ds[1].double().abs()[:, None] * p * (surprise.abs() + ent[:, None])
        want[none], scale[none] = 0.0, 0.0
        # p to 2^-18 of itself (an exponent of up to 20 in fp32, see above), sums of up to 33 gradients, the rounding to the type
        tol = 2.0**-17 * scale + (2.0**-8 * want.abs() if dtype == torch.bfloat16 else 0.0) + 1e-30
        assert got.dtype == dtype and ((got.double() - want).abs() <= tol).all(), (use, ((got.double() - want).abs() / tol).max())
        # an expanded incoming gradient
        if use == (0,):
            (one,) = torch.autograd.grad(token_log_probs(leaf, t).log_probs.sum(), [leaf])
            (two,) = torch.autograd.grad(token_log_probs(leaf, t).log_probs, [leaf], torch.ones(rows, device="cuda"))
            assert torch.equal(one, two)


@gpu
def test_gradient_against_differences():
    """along random directions; the error of a step of 2^-5 is its square times third derivatives of order one"""
    from returnn_b200.ops.token_log_probs import token_log_probs

    x, t = _rows(6, 500, torch.float32)
    x.requires_grad_(True)
    g = torch.Generator().manual_seed(5)
    c = [torch.randn(6, generator=g).cuda(), torch.randn(6, generator=g).cuda(), torch.randn(6, 4, generator=g).cuda()]

    def loss(y):
        r = token_log_probs(y, t, entropy=True, num_top=4)
        return sum((a.double() * b.double()).sum() for a, b in zip((r.log_probs, r.entropy, r.top_log_probs), c)), r.top_labels

    (grad,) = torch.autograd.grad(loss(x)[0], [x])
    done = 0
    for _ in range(20):
        v = torch.randn(x.shape, generator=g).cuda()
        h = 2.0**-7
        with torch.no_grad():
            (plus, l1), (minus, l2) = loss(x + h * v), loss(x - h * v)
        if not torch.equal(l1, l2):  # the best labels change along the way: not differentiable there
            continue
        done += 1
        want = (plus - minus) / (2 * h)
        assert ((grad.double() * v.double()).sum() - want).abs() <= 2.0**-8 * grad.double().norm() * v.double().norm() / math.sqrt(500) * 8
    assert done


@gpu
def test_another_stream_and_graph():
    from returnn_b200.ops.token_log_probs import token_log_probs

    x, t = _rows(32, 10_001, torch.bfloat16)
    want = token_log_probs(x, t, entropy=True, num_top=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = token_log_probs(x, t, entropy=True, num_top=5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_log_probs(x, t, entropy=True, num_top=5)
    x.copy_(x.flip(0))
    t.copy_(t.flip(0))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, token_log_probs(x, t, entropy=True, num_top=5)))
    assert torch.equal(got.top_labels, want.top_labels.flip(0))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals_and_empty(device):
    from returnn_b200.ops.token_log_probs import token_log_probs

    x, t = _rows(4, 100, torch.float32, device=device)
    for a, kw, err in [((x[0], t), {}, ValueError), ((x, t[:3]), {}, ValueError), ((x, t.float()), {}, TypeError), ((x, t), dict(num_top=33), ValueError),
                       ((x[:, :5], t), dict(num_top=6), ValueError), ((x[:, :0], t), {}, ValueError), ((x, t), dict(num_top=-1), ValueError)]:
        with pytest.raises(err):
            token_log_probs(*a, **kw)
    if device == "cuda":
        with pytest.raises(TypeError):
            token_log_probs(x.half(), t)
    r = token_log_probs(x[:0], t[:0], entropy=True, num_top=3)
    assert r.log_probs.shape == r.entropy.shape == (0,) and r.top_labels.shape == (0, 3)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logits_below_the_normal_numbers_are_zeros(dtype, device):
    """their differences do not show in 32 bits of a log probability: they are equal, the lowest label comes first, on either device"""
    from returnn_b200.ops.token_log_probs import token_log_probs

    for v in (9, 300, 20_000):
        x = (torch.arange(v, dtype=torch.float32) % 100 - 50.0).mul_(2.0**-133).to(dtype)[None].repeat(3, 1)
        x[1, v // 2], x[1, v - 1] = 2.0**-126, -(2.0**-126)  # the smallest that count
        x[2] = -1.0
        x[2, v - 2], x[2, 1] = 2.0**-130, -(2.0**-130)
        r = token_log_probs(x.to(device), torch.zeros(3, dtype=torch.int64, device=device), num_top=5)
        assert r.top_labels.tolist() == [[0, 1, 2, 3, 4], [v // 2] + [i for i in range(6) if i != v // 2][:4], [1, v - 2, 0] + [i for i in range(2, 6) if i != v - 2][:2]]
