"""Paged cache (ops/paged.py): block tables and slots against a loop over the requests, attention of one token against 64 bits, refusals, a life of many steps."""

import math
import pytest
import torch

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------- tables and slots


def _append_loop(table, lens, counts, ring, rng, page, room):
    """the definition, request by request"""
    table, lens, counts, ring, (head, tail) = table.tolist(), lens.tolist(), counts.tolist(), ring.tolist(), rng.tolist()
    blocks = len(table[0]) if table else 0
    left, asked, used = max(0, min(tail - head, len(ring))), 0, 0
    slots, positions, requests, offsets, new_lens, granted = [], [], [], [0], [], []
    for i, (n, add) in enumerate(zip(lens, counts)):
        n0, add = max(n, 0), max(add, 0)
        fits = n0 + add <= blocks * page
        need = -(-(n0 + add) // page) - -(-n0 // page) if fits else 0
        asked += need
        ok = fits and (need == 0 or asked <= left)
        if ok:
            for b in range(need):
                table[i][-(-n0 // page) + b] = ring[(head + used) % len(ring)]
                used += 1
        for t in range(add):
            slots.append(table[i][(n0 + t) // page] * page + (n0 + t) % page if ok else -1)
            positions.append(n0 + t)
            requests.append(i)
        offsets.append(offsets[-1] + add)
        new_lens.append(n0 + add if ok else n)
        granted.append(ok)
    pad = max(0, room - len(slots))
    return table, slots[:room] + [-1] * pad, positions[:room] + [0] * pad, requests[:room] + [-1] * pad, offsets, new_lens, [head + used, tail], granted


def _release_loop(table, lens, done, ring, rng, page):
    table, lens, done, ring, (head, tail) = table.tolist(), lens.tolist(), done.tolist(), ring.tolist(), rng.tolist()
    room = max(0, len(ring) - max(0, tail - head))
    for i, over in enumerate(done):
        if over:
            for b in range(min(-(-max(lens[i], 0) // page), len(table[i]))):
                if room:
                    ring[tail % len(ring)] = table[i][b]
                    tail, room = tail + 1, room - 1
            lens[i] = 0
    return ring, lens, [head, tail]


def _state(n, blocks, page, seed, scarce=False, new=1, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, max(blocks * page - new, 0) + 1, (n,), generator=g, dtype=torch.int32)
    counts = torch.randint(0, new + 1, (n,), generator=g, dtype=torch.int32)
    have = (lens + page - 1) // page
    pages = n * blocks + 3
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((n, blocks), -1, dtype=torch.int32)
    used = 0
    for i, h in enumerate(have.tolist()):
        table[i, :h] = perm[used: used + h]
        used += h
    head = int(torch.randint(0, 4 * pages, (1,), generator=g))
    room = (pages - used) // (8 if scarce else 1)
    ring = torch.full((pages,), -7, dtype=torch.int32)
    for j in range(room):
        ring[(head + j) % pages] = perm[used + j]
    return [x.to(device) for x in (table, lens, counts, ring, torch.tensor([head, head + room]))]


SIZES = [(1, 1, 1, 1), (3, 4, 2, 5), (64, 256, 16, 1), (1000, 5, 16, 40), (1025, 3, 1, 3), (5000, 2, 8, 9), (7, 40, 100, 3000), (2, 3, 7, 0)]


def _append(device, n, blocks, page, new, scarce):
    from returnn_b200.ops.paged import append_tokens

    table, lens, counts, ring, rng = _state(n, blocks, page, seed=n + blocks, scarce=scarce, new=new, device=device)
    if n > 5:
        lens[3] = blocks * page  # full: cannot grow
        counts[3] = 1
        table[3] = torch.arange(blocks)
    for room in (int(counts.sum()), int(counts.sum()) + 5, int(counts.sum()) // 2):
        want = _append_loop(table, lens, counts, ring, rng, page, room)
        before = [x.clone() for x in (lens, counts, ring, rng)]
        t = table.clone()
        for _ in range(2):  # the same call again has the same result
            r = append_tokens(t, lens, counts, ring, rng, page_size=page, max_tokens=room)
            assert [t.tolist(), r.slots.tolist(), r.positions.tolist(), r.requests.tolist(), r.offsets.tolist(), r.lengths.tolist(), r.free_range.tolist(),
                    r.granted.tolist()] == list(want)
        assert all(torch.equal(a, b) for a, b in zip(before, (lens, counts, ring, rng)))


def _release(device, n, blocks, page):
    from returnn_b200.ops.paged import release_pages

    table, lens, _, ring, rng = _state(n, blocks, page, seed=n + blocks, device=device)
    g = torch.Generator().manual_seed(n)
    for share in (0.0, 0.5, 1.0):
        done = (torch.rand(n, generator=g) < share).to(device)
        want = _release_loop(table, lens, done, ring, rng, page)
        mine = ring.clone()
        r = release_pages(table, lens, done, mine, rng, page_size=page)
        assert [mine.tolist(), r.lengths.tolist(), r.free_range.tolist()] == list(want)


@pytest.mark.parametrize("scarce", [False, True])
def test_tables_cpu(scarce):
    for n, blocks, page, new in SIZES[:5] + SIZES[6:]:
        _append("cpu", n, blocks, page, new, scarce)
        _release("cpu", n, blocks, page)


@gpu
@pytest.mark.parametrize("scarce", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_tables(size, scarce):
    n, blocks, page, new = size
    _append("cuda", n, blocks, page, new, scarce)
    _release("cuda", n, blocks, page)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_odd_states(device):
    """no requests, no blocks, negative numbers, a ring whose range is off, a table that is a slice, many tokens"""
    from returnn_b200.ops.paged import append_tokens, release_pages

    i32 = dict(dtype=torch.int32, device=device)
    ring, rng = torch.arange(5, **i32), torch.tensor([3, 8], device=device)
    r = append_tokens(torch.empty(0, 4, **i32), torch.empty(0, **i32), torch.empty(0, **i32), ring, rng, page_size=4, max_tokens=3)
    assert r.slots.tolist() == [-1] * 3 and r.offsets.tolist() == [0] and r.free_range.tolist() == [3, 8]
    r = append_tokens(torch.empty(2, 0, **i32), torch.zeros(2, **i32), torch.tensor([1, 0], **i32), ring, rng, page_size=4, max_tokens=1)
    assert r.slots.tolist() == [-1] and r.granted.tolist() == [False, True] and r.lengths.tolist() == [0, 0]
    for bad_range in ([8, 3], [0, 100], [-7, -2]):
        table = torch.full((4, 3), -1, **i32)
        lens, counts = torch.tensor([-5, 0, 2, 0], **i32), torch.tensor([2, -3, 1, 9], **i32)
        table[2, 0] = 4
        br = torch.tensor(bad_range, device=device)
        want = _append_loop(table, lens, counts, ring, br, 4, 12)
        r = append_tokens(table, lens, counts, ring, br, page_size=4, max_tokens=12)
        assert [table.tolist(), r.slots.tolist(), r.positions.tolist(), r.requests.tolist(), r.offsets.tolist(), r.lengths.tolist(), r.free_range.tolist(),
                r.granted.tolist()] == list(want)
    wide = torch.full((3, 9), -1, **i32)
    table = wide[:, 2:6]
    r = append_tokens(table, torch.zeros(3, **i32), torch.tensor([4, 8, 1], **i32), ring, rng, page_size=4, max_tokens=13)
    assert table[:, :2].tolist() == [[3, -1], [4, 0], [1, -1]] and wide[:, :2].eq(-1).all() and wide[:, 6:].eq(-1).all()
    mine = ring.clone()
    back = release_pages(table, r.lengths, torch.ones(3, dtype=torch.bool, device=device), mine, r.free_range, page_size=4)
    assert back.free_range.tolist() == [7, 12] and back.lengths.tolist() == [0] * 3 and [mine[p % 5].item() for p in range(8, 12)] == [3, 4, 0, 1]
    # no more goes back than the ring has room for
    back = release_pages(table, torch.tensor([4, 8, 1], **i32), torch.ones(3, dtype=torch.bool, device=device), mine, torch.tensor([7, 11], device=device), page_size=4)
    assert back.free_range.tolist() == [7, 12]


# ---------------------------------------------------------------------------------------------------------------- attention


def _exact(q, kc, vc, table, lens, scale):
    """in 64 bits, request by request; and the error that the order and rounding of fp32 may have"""
    n, h, d = q.shape
    pages, hk, page, _ = kc.shape
    out, tol = (torch.zeros(n, h, d, dtype=torch.float64, device=q.device) for _ in range(2))
    for i in range(n):
        toks = [(p, t) for b, p in enumerate(table[i].tolist()) for t in range(page) if b * page + t < int(lens[i]) and 0 <= p < pages]
        if not toks:
            continue
        ps, ts = (torch.tensor(x, device=q.device) for x in zip(*toks))
        k, v = (c[ps, :, ts].double().transpose(0, 1) for c in (kc, vc))  # [hk, T, d]
        qi = q[i].double().view(hk, h // hk, d)
        out[i] = (torch.softmax(torch.einsum("hgd,htd->hgt", qi, k) * scale, -1) @ v).reshape(h, d)
        # scores: sums of d products, each rounding 2^-24 of the sum of their sizes, and of the factor in front; they shift weights by as much, relatively.
        # weights: exponentials of 2 ulp, kept to 2^-16 for the products with the values, sums of up to 2000 terms per lane
        size = torch.einsum("hgd,htd->hgt", qi.abs(), k.abs()).amax(-1) * abs(scale)
        rel = 2 * size * (d + 4) * 2.0**-24 + 2.0**-15 + (len(toks) / 128 + 32) * 2.0**-24
        tol[i] = (rel[..., None] * v.abs().amax(1)[:, None, :]).reshape(h, d)
    return out, tol


def _cache(n, hk, d, page, lens, dtype, seed, layout="heads", junk=float("nan")):
    """pages in no order; what belongs to no token is junk"""
    g = torch.Generator().manual_seed(seed)
    have = [-(-x // page) for x in lens]
    pages = sum(have) + 3
    perm = torch.randperm(pages, generator=g)
    table = torch.full((n, max(have + [1]) + 1), -1, dtype=torch.int32)
    caches = torch.full((2, pages, hk, page, d), junk)
    used = 0
    for i, h in enumerate(have):
        table[i, :h] = perm[used: used + h]
        for b in range(h):
            m = min(page, lens[i] - b * page)
            caches[:, perm[used + b], :, :m] = torch.randn(2, hk, m, d, generator=g)
        used += h
    caches = caches.to(dtype)
    if layout == "tokens":
        caches = caches.transpose(2, 3).contiguous().transpose(2, 3)
    q = torch.randn(n, hk, d, generator=g)
    return caches, table.cuda(), g


def _attend(n, h, hk, d, page, lens, dtype, layout="heads", scale=None, seed=0, q_scale=1.0):
    from returnn_b200.ops.paged import paged_attention

    caches, table, g = _cache(n, hk, d, page, lens, dtype, seed, layout)
    kc, vc = caches.cuda().unbind(0) if layout == "heads" else (c.cuda() for c in caches.unbind(0))
    q = (torch.randn(n, h, d, generator=g) * q_scale).to("cuda", dtype)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = paged_attention(q, kc, vc, table, lens, scale=scale)
    want, tol = _exact(q, kc, vc, table, lens, d ** -0.5 if scale is None else scale)
    if dtype == torch.bfloat16:
        tol = tol + 2.0**-8 * want.abs()
    assert got.dtype == dtype and got.shape == (n, h, d)
    bad = (got.double() - want).abs() > tol
    assert not bad.any() and not got.isnan().any(), "%g of the tolerance" % ((got.double() - want).abs() / (tol + 1e-30)).max()
    again = paged_attention(q, kc, vc, table, lens, scale=scale)
    assert torch.equal(got, again)  # the split and its joining have an order


HEADS = [(8, 8, 64), (4, 4, 32), (1, 1, 8), (32, 8, 128), (16, 2, 128), (6, 1, 80), (20, 1, 128), (40, 1, 64), (40, 8, 96), (8, 4, 256), (24, 1, 256), (12, 1, 16), (33, 1, 40),
         (100, 2, 24)]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("h,hk,d", HEADS)
def test_attention(h, hk, d, dtype):
    for page, lens in ((16, [1, 0, 17, 128, 129, 300, 16]), (1, [5, 131]), (100, [99, 100, 101, 0, 1000]), (64, [1]), (7, [0, 0]), (16, [2000])):
        _attend(len(lens), h, hk, d, page, lens, dtype, seed=page)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_many_and_long(dtype):
    """more requests than threads, units that many CTAs share, one long among short ones"""
    g = torch.Generator().manual_seed(1)
    _attend(400, 4, 2, 64, 8, torch.randint(0, 70, (400,), generator=g).tolist(), dtype)
    _attend(3, 4, 1, 64, 16, [3, 20_000, 500], dtype)
    _attend(2, 8, 8, 128, 64, [5000, 4999], dtype, layout="tokens")
    _attend(5, 8, 2, 64, 16, [64, 700, 5, 0, 129], dtype, scale=1.0)
    _attend(5, 8, 2, 64, 16, [64, 700, 5, 0, 129], dtype, scale=-0.1)
    _attend(5, 8, 2, 64, 16, [64, 700, 5, 0, 129], dtype, scale=0.0)
    _attend(4, 8, 2, 64, 16, [640, 70, 5, 129], dtype, q_scale=30.0)  # one token has nearly all of the weight


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_infinities_and_pages_that_are_none(dtype):
    from returnn_b200.ops.paged import paged_attention, paged_attention_reference

    caches, table, g = _cache(4, 2, 64, 16, [100, 100, 100, 300], dtype, 3)
    kc, vc = caches.cuda().unbind(0)
    q = torch.randn(4, 4, 64, generator=g).to("cuda", dtype)
    lens = torch.tensor([100, 100, 100, 300], dtype=torch.int32, device="cuda")
    table[0, 2] = -1  # its tokens are not there
    table[1, 3] = kc.shape[0]
    table[2, :] = 2**31 - 1
    want, tol = _exact(q, kc, vc, table, lens, 0.125)
    tol = tol + 2.0**-8 * want.abs()
    got = paged_attention(q, kc, vc, table, lens)
    assert ((got.double() - want).abs() <= tol).all() and not got[2].any()
    ref = paged_attention_reference(q, kc, vc, table, lens)
    assert ((ref.double() - want).abs() <= tol).all()
    # lengths past the table end with it; negative ones are none
    long = paged_attention(q, kc, vc, table, torch.tensor([-3, 100, 100, 10_000_000], dtype=torch.int32, device="cuda"))
    full = paged_attention(q, kc, vc, table, torch.tensor([0, 100, 100, table.shape[1] * 16], dtype=torch.int32, device="cuda"))
    assert torch.equal(long.nan_to_num(7.0), full.nan_to_num(7.0)) and not long[0].any()  # (what lies behind the last token is junk)
    # a value that is no number is in the output of its request and heads alone; a key of which the score is infinite takes the row with it
    vc2 = vc.clone()
    vc2[table[3, 5], 1, 3, 7] = math.nan
    got = paged_attention(q, kc, vc2, table, lens)
    assert got[3, 2:, 7].isnan().all() and not got[:3].isnan().any() and not got[3, :2].isnan().any() and not got[3, 2:, :7].isnan().any()
    kc2 = kc.clone()
    kc2[table[3, 0], 0, 0, :] = math.inf
    got = paged_attention(q, kc2, vc, table, lens)
    assert got[3, :2].isnan().all() and not got[3, 2:].isnan().any() and not got[:3].isnan().any()


@gpu
def test_attention_far_in_the_cache():
    """offsets beyond 2^31 elements"""
    from returnn_b200.ops.paged import paged_attention

    pages, hk, page, d = 70_000, 4, 64, 128  # 2.3e9 elements
    kc = torch.zeros(pages, hk, page, d, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[69_999, 0, 69_998], [66_000, 65_999, 3]], dtype=torch.int32, device="cuda")
    for p in table.flatten().tolist():
        kc[p] = torch.randn(hk, page, d, generator=g).cuda()
    q = torch.randn(2, 8, d, generator=g).to("cuda", torch.bfloat16)
    lens = torch.tensor([190, 150], dtype=torch.int32, device="cuda")
    want, tol = _exact(q, kc, kc, table, lens, d ** -0.5)
    assert ((paged_attention(q, kc, kc, table, lens).double() - want).abs() <= tol + 2.0**-8 * want.abs()).all()


def test_attention_cpu():
    from returnn_b200.ops.paged import paged_attention

    g = torch.Generator().manual_seed(0)
    kc, vc = torch.randn(2, 6, 2, 4, 8, generator=g).unbind(0)
    table = torch.tensor([[3, 1, -1], [0, 2, 5], [-1, -1, -1]], dtype=torch.int32)
    lens = torch.tensor([6, 12, 0], dtype=torch.int32)
    q = torch.randn(3, 4, 8, generator=g)
    want, tol = _exact(q, kc, vc, table, lens, 8 ** -0.5)
    assert ((paged_attention(q, kc, vc, table, lens).double() - want).abs() <= tol).all()


@gpu
def test_streams_and_graph():
    """a side stream gives the same; a captured step follows lengths and tables that change in place"""
    from returnn_b200.ops.paged import append_tokens, paged_attention

    lens = [70, 0, 500, 33]
    caches, table, g = _cache(4, 2, 64, 16, [x + 40 for x in lens], torch.bfloat16, 5, junk=0.5)
    kc, vc = caches.cuda().unbind(0)
    q = torch.randn(4, 4, 64, generator=g).to("cuda", torch.bfloat16)
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = paged_attention(q, kc, vc, table, length)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_attention(q, kc, vc, table, length)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    ring, rng, counts = torch.arange(9, dtype=torch.int32, device="cuda"), torch.tensor([0, 9], device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = append_tokens(table, length, counts, ring, rng, page_size=16, max_tokens=4)
        out = paged_attention(q, kc, vc, table, new.lengths)
        length.copy_(new.lengths)
    for step in range(1, 4):
        graph.replay()
        assert length.tolist() == [x + step for x in lens]
        assert torch.equal(out, paged_attention(q, kc, vc, table, length))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    from returnn_b200.ops.paged import append_tokens, paged_attention, release_pages

    i32 = dict(dtype=torch.int32, device=device)
    q, kc = torch.zeros(3, 4, 16, device=device), torch.zeros(5, 2, 4, 16, device=device)
    table, lens = torch.zeros(3, 2, **i32), torch.zeros(3, **i32)
    for a, err in [((q[0], kc, kc, table, lens), ValueError), ((q, kc, kc[:, :, :3], table, lens), ValueError), ((q[..., :8], kc, kc, table, lens), ValueError),
                   ((q.bfloat16(), kc, kc, table, lens), TypeError), ((q[:, :3], kc, kc, table, lens), ValueError), ((q, kc, kc, table.long(), lens), ValueError),
                   ((q, kc, kc, table[:2], lens), ValueError), ((q, kc, kc, table, lens.long()), ValueError), ((q, kc, kc, table.t(), lens[:2]), ValueError)]:
        with pytest.raises(err):
            paged_attention(*a)
    with pytest.raises(RuntimeError):
        paged_attention(q.clone().requires_grad_(True), kc, kc, table, lens)
    if device == "cuda":
        with pytest.raises(TypeError):
            paged_attention(q.half(), kc.half(), kc.half(), table, lens)
        odd = torch.zeros(5, 2, 4, 17, device=device)[..., 1:]
        with pytest.raises(ValueError):
            paged_attention(q, odd, odd, table, lens)
        for d in (12, 264):
            with pytest.raises(RuntimeError):
                paged_attention(torch.zeros(3, 4, d, device=device), *(torch.zeros(5, 2, 4, d, device=device) for _ in range(2)), table, lens)
    ring, rng, done = torch.zeros(5, **i32), torch.zeros(2, dtype=torch.int64, device=device), torch.zeros(3, dtype=torch.bool, device=device)
    ok = dict(page_size=4, max_tokens=3)
    for a, kw, err in [((table.long(), lens, lens, ring, rng), ok, ValueError), ((table, lens[:2], lens, ring, rng), ok, ValueError), ((table, lens, lens.long(), ring, rng), ok, ValueError),
                       ((table, lens, lens, ring[:0], rng), ok, ValueError), ((table, lens, lens, ring, rng.int()), ok, ValueError),
                       ((table, lens, lens, ring, rng), dict(page_size=0, max_tokens=3), ValueError), ((table, lens, lens, ring, rng), dict(page_size=4, max_tokens=-1), ValueError)]:
        with pytest.raises(err):
            append_tokens(*a, **kw)
    with pytest.raises(ValueError):
        release_pages(table, lens, lens, ring, rng, page_size=4)
    release_pages(table, lens, done, ring, rng, page_size=4)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_infinite_values(dtype):
    """an infinite value with a weight above zero is in the output; infinities of both signs are no number; nothing else changes"""
    from returnn_b200.ops.paged import paged_attention

    lens = [1, 40, 2100, 300]
    caches, table, g = _cache(4, 2, 64, 16, lens, dtype, 7)
    kc, vc = caches.cuda().unbind(0)
    q = torch.randn(4, 8, 64, generator=g).to("cuda", dtype)
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    plain = paged_attention(q, kc, vc, table, length)
    assert plain.isfinite().all()
    for places in ([0, 39, 2099, 17], [0, 0, 0, 0], [0, 20, 1024, 299]):
        with_inf = vc.clone()
        for i, t in enumerate(places):
            page, at = table[i, t // 16], t % 16
            with_inf[page, 0, at, 7], with_inf[page, 0, at, 8] = math.inf, -math.inf
            if lens[i] > 1:
                u = (t + 1) % lens[i]
                with_inf[page, 0, at, 9], with_inf[table[i, u // 16], 0, u % 16, 9] = math.inf, -math.inf
        got = paged_attention(q, kc, with_inf, table, length)
        assert (got[:, :4, 7] == math.inf).all() and (got[:, :4, 8] == -math.inf).all() and got[1:, :4, 9].isnan().all()
        same = torch.ones_like(got, dtype=torch.bool)
        same[:, :4, 7:9] = False
        same[1:, :4, 9] = False
        assert torch.equal(got[same], plain[same])


def test_workspace_without_heads():
    """in a process of its own: a division by zero ends it"""
    import os
    import subprocess
    import sys
    from returnn_b200.ops import build

    path = os.path.join(build._BUILD, "librb200.so")
    if not os.path.exists(path):
        pytest.skip("the kernels are not built")
    code = ("import ctypes; f = ctypes.CDLL(%r).rb200_paged_attention_workspace; f.restype = ctypes.c_longlong; "
            "print(f(1, 0, 1, 64, 1), f(0, 8, 2, 64, 1), f(3, 4, 0, 64, 0), f(3, 4, 2, 64, 0) > 0)" % path)
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.split() == ["0", "0", "0", "True"], (res.returncode, res.stdout, res.stderr)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_attention_without_heads_or_requests(device):
    from returnn_b200.ops.paged import paged_attention

    kc = torch.zeros(5, 2, 4, 16, device=device)
    i32 = dict(dtype=torch.int32, device=device)
    for n, heads in ((3, 0), (0, 4), (0, 0)):
        out = paged_attention(torch.zeros(n, heads, 16, device=device), kc, kc, torch.zeros(n, 2, **i32), torch.ones(n, **i32))
        assert out.shape == (n, heads, 16) and out.is_contiguous()


@pytest.mark.parametrize("device,python", [("cpu", False), pytest.param("cuda", False, marks=gpu), pytest.param("cuda", True, marks=gpu)])
def test_tables_written_in_place(monkeypatch, device, python):
    """autograd learns of the writes: a table or a ring that a graph still needs as an index is noticed"""
    from returnn_b200.ops import nodes
    from returnn_b200.ops.paged import append_tokens, release_pages

    if python:
        monkeypatch.setattr(nodes, "active", lambda: None)
    i32 = dict(dtype=torch.int32, device=device)
    table, ring, rng = torch.zeros(2, 3, **i32), torch.arange(6, **i32), torch.tensor([0, 6], device=device)
    x = torch.randn(6, 4, device=device, requires_grad=True)
    by_table, by_ring = x.index_select(0, table.view(-1)).sum(), x.index_select(0, ring).sum()
    r = append_tokens(table, torch.zeros(2, **i32), torch.tensor([5, 4], **i32), ring, rng, page_size=4, max_tokens=9)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        by_table.backward()
    release_pages(table, r.lengths, torch.ones(2, dtype=torch.bool, device=device), ring, r.free_range, page_size=4)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        by_ring.backward()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_slots_beyond_32_bits_are_refused(device):
    from returnn_b200.ops.paged import append_tokens

    i32 = dict(dtype=torch.int32, device=device)
    lens, counts, rng = torch.zeros(1, **i32), torch.ones(1, **i32), torch.tensor([0, 3], device=device)
    with pytest.raises(ValueError):
        append_tokens(torch.full((1, 2), -1, **i32), lens, counts, torch.tensor([2, 1, 0], **i32), rng, page_size=2**30, max_tokens=1)
    r = append_tokens(torch.full((1, 2), -1, **i32), lens, counts, torch.tensor([1, 0], **i32), rng - 1, page_size=2**30, max_tokens=1)
    assert r.slots.tolist() == [0] and r.granted.tolist() == [True]
