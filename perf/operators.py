"""
Operators of language models that are served and scored token by token: the rotation of queries and keys with their norms per head, block
tables of a paged cache, attention of one new token over that cache, log probabilities of given tokens.

Sizes are those of the Transformer configurations of this repository (512 features, 8 heads of 64, 32k and 10k labels, 25k tokens per batch)
and of decoders of 32 query heads over 8 key heads of 128. Requests are ragged, as they are where they come and go. ``run`` computes the plain
form (elementary tensor operations in 32 bits, one rounding at the end) or, with ``own``, calls the framework.
"""

from __future__ import annotations
from typing import Any, Dict, List
import math
import torch

own = False  # True: the framework's operators

DEV = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------- the cases


def listed() -> List[Dict[str, Any]]:
    return [
        # q and k of one decoder layer in a training pass over 25k tokens: slices of a fused projection, every head normed and rotated
        dict(name="rope_train", kind="rope", tokens=25000, heads=8, kv_heads=8, dim=64, rotary=64, interleaved=True, norm=True, dtype="bf16", train=True,
             max_pos=512),
        # grouped heads, a part of each rotated, positions of a long document beyond the trained range, without mixed precision
        dict(name="rope_long_train", kind="rope", tokens=8191, heads=32, kv_heads=8, dim=128, rotary=64, interleaved=False, norm=True, dtype="f32", train=True,
             max_pos=131072),
        # one decoding step: 64 new tokens, keys and values go to their slots in the paged cache
        dict(name="rope_cache_step", kind="rope_cache", tokens=64, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=True, norm=True, dtype="bf16",
             max_pos=4096, page=16, pages=1024),
        # tables and slots of a decoding step: one token for each running request
        dict(name="pages_step", kind="append", requests=64, max_len=4096, new=1, page=16, scarce=False),
        # tables and slots of many prompts at once
        dict(name="pages_prompts", kind="append", requests=256, max_len=0, new=8192, page=16, scarce=False),
        # the pages of finished requests go back
        dict(name="pages_release", kind="release", requests=256, max_len=32768, page=16),
        # one request of this repository's decoder without mixed precision: the smallest attention
        dict(name="attention_one_f32", kind="attention", requests=1, max_len=1000, heads=8, kv_heads=8, dim=64, page=16, dtype="f32", empty=False),
        # an ordinary batch of running requests
        dict(name="attention_batch", kind="attention", requests=64, max_len=4096, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", empty=True),
        # two long documents: few rows, the work is in the length
        dict(name="attention_long", kind="attention", requests=2, max_len=131072, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", empty=False),
        # sequence training: log probability and entropy of every target position of a batch, and the gradient of the logits
        dict(name="score_train", kind="score", rows=6001, vocab=32000, top=0, dtype="bf16", train=True, masked=False),
        # rescoring with alternatives, logits in 32 bits over an odd vocabulary with forbidden labels
        dict(name="score_alternatives", kind="score", rows=1500, vocab=10001, top=8, dtype="f32", train=False, masked=True),
        # the rows of one decoding step
        dict(name="score_step", kind="score", rows=16, vocab=32000, top=5, dtype="bf16", train=False, masked=False),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> Dict[str, Any]:
    kind = rng.choice(["rope", "rope", "rope_cache", "append", "release", "attention", "attention", "attention", "score", "score", "score"])
    if kind in ("rope", "rope_cache"):
        heads, kv_heads, dim = rng.choice([(8, 8, 64), (4, 4, 32), (12, 12, 64), (32, 8, 128), (16, 2, 128), (6, 1, 80), (5, 5, 20), (8, 4, 256)])
        most = min(25000, 80_000_000 // ((heads + 2 * kv_heads) * dim))
        c = dict(kind=kind, tokens=_log_int(rng, 1, most if kind == "rope" else min(most, 4000)), heads=heads, kv_heads=kv_heads, dim=dim,
                 rotary=rng.choice([dim, dim, dim // 2 // 2 * 2]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.7, dtype=rng.choice(["bf16", "bf16", "f32"]),
                 max_pos=_log_int(rng, 10, 131072))
        if kind == "rope":
            c["train"] = rng.random() < 0.7
        else:
            c["page"] = rng.choice([1, 8, 16, 64, 100])
            c["pages"] = c["tokens"] * 2 // c["page"] + rng.randint(1, 40)
        return c
    if kind == "append":
        step = rng.random() < 0.5
        requests = _log_int(rng, 2, 2000 if step else 256)
        return dict(kind=kind, requests=requests, max_len=_log_int(rng, 10, 8192), new=1 if step else _log_int(rng, 2, 8192), page=rng.choice([1, 8, 16, 64, 100]),
                    scarce=rng.random() < 0.3)
    if kind == "release":
        return dict(kind=kind, requests=_log_int(rng, 2, 1000), max_len=_log_int(rng, 10, 8192), page=rng.choice([1, 8, 16, 64, 100]))
    if kind == "attention":
        heads, kv_heads, dim = rng.choice([(8, 8, 64), (4, 4, 32), (12, 12, 64), (32, 8, 128), (16, 2, 128), (6, 1, 80), (20, 1, 128), (40, 8, 96), (8, 4, 256)])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        requests = _log_int(rng, 1, 500)
        most = 230_000_000 // (kv_heads * dim * (2 if dtype == "f32" else 1))  # tokens of all requests, as if each were as long as the longest
        return dict(kind=kind, requests=requests, max_len=_log_int(rng, 1, max(1, min(100_000, most // requests))), heads=heads, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([1, 8, 16, 16, 64, 100]), dtype=dtype, empty=rng.random() < 0.3)
    vocab = rng.choice([80, 1001, 10001, 10025, 32000, 50001, 128000])
    return dict(kind=kind, rows=_log_int(rng, 1, min(6000, 150_000_000 // vocab)), vocab=vocab, top=rng.choice([0, 1, 5, 8, 20, 32]),
                dtype=rng.choice(["bf16", "bf16", "f32"]), train=rng.random() < 0.5, masked=rng.random() < 0.3)


# ---------------------------------------------------------------------------------------------------------------- inputs


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, scale: float = 1.0, dtype=torch.float32) -> torch.Tensor:
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _randint(g, lo: int, hi: int, *shape) -> torch.Tensor:
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)


def _permutation(g, n: int) -> torch.Tensor:
    return torch.argsort(torch.rand(n, generator=g, device=DEV)).to(torch.int32)


def _lengths(g, n: int, most: int, empty: bool) -> torch.Tensor:
    """ragged lengths up to ``most``, one of them that; with ``empty`` a tenth of the requests have none. The seed orders them: their sum is the case's"""
    fixed = _gen(1000 * n + most)
    lens = _randint(fixed, 1, most + 1, n)
    if empty:
        lens = lens * (torch.rand(n, generator=fixed, device=DEV) > 0.1)
    lens[0] = most
    return lens[_permutation(g, n).long()].to(torch.int32)


def _frequencies(rotary: int) -> torch.Tensor:
    return (10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).to(torch.float32).to(DEV)


def _tables(g, have: torch.Tensor, blocks: int, pages: int) -> torch.Tensor:
    """[requests, blocks]: the first ``have`` entries of each row are pages of its own in no order, the others -1"""
    at = torch.arange(blocks, device=DEV)[None, :]
    number = (torch.cumsum(have, 0) - have)[:, None] + at
    perm = _permutation(g, pages)
    return torch.where(at < have[:, None], perm[number.clamp(max=pages - 1).long()], -1).to(torch.int32)


def prepare(case: Dict[str, Any], seed: int) -> Dict[str, Any]:
    g = _gen(seed)
    st: Dict[str, Any] = {"case": case}
    kind = case["kind"]
    dt = _TYPES[case.get("dtype", "bf16")]
    if kind in ("rope", "rope_cache"):
        n, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        qkv = _randn(g, n, (h + 2 * hk) * d, dtype=dt)  # the fused projection; q, k and v are its slices
        if h == hk:  # (q, k, v) of a head side by side, as the attention modules have it
            q, k, v = (x.detach() for x in qkv.view(n, h, 3 * d).split(d, dim=-1))
        else:
            q, k, v = (x.detach() for x in qkv.view(n, h + 2 * hk, d).split([h, hk, hk], dim=1))
        train = bool(case.get("train"))
        if case["norm"]:
            st["q_scale"] = (_randn(g, d, scale=0.2) + 1.0).requires_grad_(train)
            st["k_scale"] = (_randn(g, d, scale=0.2) + 1.0).requires_grad_(train)
        else:
            st["q_scale"] = st["k_scale"] = None
        st.update(q=q.requires_grad_(train), k=k.requires_grad_(train), v=v, frequencies=_frequencies(case["rotary"]),
                  positions=_randint(g, 0, case["max_pos"], n))
        if train:
            st["d_out"] = [_randn(g, n, h, d, dtype=dt), _randn(g, n, hk, d, dtype=dt)]
        if kind == "rope_cache":
            pages, page = case["pages"], case["page"]
            slots = _permutation(g, pages * page)[:n]  # some tokens have no place
            st["slots"] = torch.where(torch.rand(n, generator=g, device=DEV) < 0.05, -1, slots).to(torch.int32)
            st["cache"] = [_randn(g, pages, hk, page, d, dtype=dt) for _ in range(2)]
    elif kind in ("append", "release"):
        r, page = case["requests"], case["page"]
        lens = _lengths(g, r, case["max_len"], True) if case["max_len"] else torch.zeros(r, dtype=torch.int32, device=DEV)
        have = (lens + page - 1) // page
        grow = case.get("new", 0)
        blocks = (case["max_len"] + grow + page - 1) // page
        new = _lengths(g, r, grow, True) if grow else None
        pages = r * blocks + 9
        st.update(lengths=lens, page=page, block_table=_tables(g, have, blocks, pages), free_pages=_permutation(g, pages))
        head = 3 * pages // 4  # the ring's free stretch wraps around its end
        room = pages - int(have.sum())
        if case.get("scarce"):
            room = min(room, int(new.sum()) // page // 2)
        st["free_range"] = torch.tensor([head, head + room], dtype=torch.int64, device=DEV)
        if kind == "append":
            st.update(new=new, tokens=int(new.sum()) + 3)  # the room of a captured step is a little larger
        else:
            st["finished"] = torch.rand(r, generator=g, device=DEV) < 0.5
    elif kind == "attention":
        r, h, hk, d, page = (case[x] for x in ("requests", "heads", "kv_heads", "dim", "page"))
        lens = _lengths(g, r, case["max_len"], case["empty"])
        have = (lens + page - 1) // page
        blocks = (case["max_len"] + page - 1) // page
        pages = int(have.sum()) + 7
        st.update(q=_randn(g, r, h, d, scale=2.0, dtype=dt), lengths=lens, block_table=_tables(g, have, blocks, pages),
                  cache=[torch.empty(pages, hk, page, d, dtype=dt, device=DEV).normal_(generator=g) for _ in range(2)])
    else:
        n, v = case["rows"], case["vocab"]
        logits = torch.empty(n, v, dtype=dt, device=DEV).normal_(generator=g).mul_(2.0)
        if case["masked"]:  # forbidden labels, and rows that allow none
            logits.masked_fill_(torch.rand(v, generator=g, device=DEV) < 0.3, -math.inf)
            logits[:: 50] = -math.inf
        targets = _randint(g, 0, v, n)
        st.update(logits=logits, targets=torch.where(torch.rand(n, generator=g, device=DEV) < 0.05, -1, targets).to(torch.int32))
        if case["train"]:
            logits.requires_grad_(True)
            st["d_out"] = [_randn(g, n), _randn(g, n, scale=0.1)] + ([_randn(g, n, case["top"])] if case["top"] else [])
    return st


# ---------------------------------------------------------------------------------------------------------------- one pass


def _rope_own(st):
    from returnn_b200.ops.norm_rope import norm_rope, norm_rope_to_cache

    c = st["case"]
    opts = dict(q_scale=st["q_scale"], k_scale=st["k_scale"], eps=1e-6, interleaved=c["interleaved"])
    if c["kind"] == "rope_cache":
        q = norm_rope_to_cache(st["q"], st["k"], st["v"], st["positions"], st["frequencies"], st["cache"][0], st["cache"][1], st["slots"], **opts)
        return [q] + st["cache"]
    q, k = norm_rope(st["q"], st["k"], st["positions"], st["frequencies"], **opts)
    if not c["train"]:
        return [q, k]
    leaves = [st["q"], st["k"]] + ([st["q_scale"], st["k_scale"]] if c["norm"] else [])
    return [q.detach(), k.detach()] + list(torch.autograd.grad([q, k], leaves, st["d_out"]))


def _normed(x, scale):
    x = x.float()
    return x if scale is None else x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6) * scale


def _rotated(x, cos, sin, interleaved: bool):
    half = cos.shape[-1]
    rot, rest = x[..., : 2 * half], x[..., 2 * half:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        rot = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([rot, rest], dim=-1)


def _rope_plain(st):
    c = st["case"]
    # the angle of a far position does not fit 24 bits: its product is taken in 64 and only the sine and cosine are rounded
    angle = st["positions"].double()[:, None] * st["frequencies"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotated(_normed(st["q"], st["q_scale"]), cos, sin, c["interleaved"]).to(st["q"].dtype)
    k = _rotated(_normed(st["k"], st["k_scale"]), cos, sin, c["interleaved"]).to(st["k"].dtype)
    if c["kind"] == "rope_cache":
        page = c["page"]
        at = st["slots"].long()
        keep = at >= 0
        at = at[keep]
        for cache, x in zip(st["cache"], (k, st["v"])):
            cache[at // page, :, at % page] = x[keep]
        return [q] + st["cache"]
    if not c["train"]:
        return [q, k]
    leaves = [st["q"], st["k"]] + ([st["q_scale"], st["k_scale"]] if c["norm"] else [])
    return [q.detach(), k.detach()] + list(torch.autograd.grad([q, k], leaves, st["d_out"]))


def _append_own(st):
    from returnn_b200.ops.paged import append_tokens

    r = append_tokens(st["block_table"], st["lengths"], st["new"], st["free_pages"], st["free_range"], page_size=st["page"], max_tokens=st["tokens"])
    return [st["block_table"], r.slots, r.positions, r.requests, r.offsets, r.lengths, r.free_range, r.granted]


def _append_plain(st):
    table, lens, new, ring, page, room = st["block_table"], st["lengths"].long(), st["new"].long(), st["free_pages"], st["page"], st["tokens"]
    head, tail = st["free_range"][0], st["free_range"][1]
    blocks, pages = table.shape[1], ring.shape[0]
    have = (lens + page - 1) // page
    fits = lens + new <= blocks * page
    need = torch.where(fits, (lens + new + page - 1) // page - have, 0)
    granted = fits & ((need == 0) | (torch.cumsum(need, 0) <= tail - head))
    take = torch.where(granted, need, 0)
    first = torch.cumsum(take, 0) - take
    at = torch.arange(blocks, device=DEV)[None, :]
    fresh = ring[((head + first[:, None] + at - have[:, None]) % pages).long()]
    table.copy_(torch.where((at >= have[:, None]) & (at < (have + take)[:, None]), fresh, table))
    offsets = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    token = torch.arange(room, device=DEV)
    request = torch.searchsorted(offsets[1:], token, right=True)
    real = request < lens.shape[0]
    request = request.clamp(max=lens.shape[0] - 1)
    position = lens[request] + token - offsets[request]
    slot = table[request, (position // page).clamp(max=blocks - 1)] * page + position % page
    i32 = torch.int32
    return [table, torch.where(real & granted[request], slot, -1).to(i32), torch.where(real, position, 0).to(i32), torch.where(real, request, -1).to(i32),
            offsets.to(i32), torch.where(granted, lens + new, lens).to(i32), torch.stack([head + take.sum(), tail]), granted]


def _release_own(st):
    from returnn_b200.ops.paged import release_pages

    r = release_pages(st["block_table"], st["lengths"], st["finished"], st["free_pages"], st["free_range"], page_size=st["page"])
    return [st["free_pages"], r.lengths, r.free_range]


def _release_plain(st):
    table, lens, ring, done, page = st["block_table"], st["lengths"].long(), st["free_pages"], st["finished"], st["page"]
    head, tail = st["free_range"][0], st["free_range"][1]
    count = torch.where(done, (lens + page - 1) // page, 0)
    last = torch.cumsum(count, 0)
    number = (torch.arange(ring.shape[0], device=DEV) - tail) % ring.shape[0]  # of the returned page that a place of the ring would get
    request = torch.searchsorted(last, number, right=True).clamp(max=lens.shape[0] - 1)
    block = (number - (last - count)[request]).clamp(min=0, max=table.shape[1] - 1)
    ring.copy_(torch.where(number < last[-1], table[request, block], ring))
    return [ring, torch.where(done, 0, lens).to(torch.int32), torch.stack([head, tail + last[-1]])]


def _attention_own(st):
    from returnn_b200.ops.paged import paged_attention

    return paged_attention(st["q"], st["cache"][0], st["cache"][1], st["block_table"], st["lengths"])


def _attention_plain(st):
    q, lens, table = st["q"], st["lengths"].long(), st["block_table"]
    r, h, d = q.shape
    _, hk, page, _ = st["cache"][0].shape
    t = table.shape[1] * page
    pages = table.clamp(min=0).long()
    k, v = (c[pages].float().permute(0, 2, 1, 3, 4).reshape(r, hk, t, d) for c in st["cache"])
    s = torch.matmul(q.float().view(r, hk, h // hk, d), k.transpose(-1, -2)) * d ** -0.5
    inside = (torch.arange(t, device=DEV)[None, :] < lens[:, None])[:, None, None, :]
    s = torch.where(inside, s, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    e = torch.where(inside, torch.exp(s - top), 0.0)
    total = e.sum(dim=-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, 1.0)  # a request without tokens: zeros
    return o.view(r, h, d).to(q.dtype)


def _score_own(st):
    from returnn_b200.ops.token_log_probs import token_log_probs

    c = st["case"]
    r = token_log_probs(st["logits"], st["targets"], entropy=True, num_top=c["top"])
    outs = [r.log_probs, r.entropy] + ([r.top_log_probs] if c["top"] else [])
    labels = [r.top_labels] if c["top"] else []
    if not c["train"]:
        return outs + labels
    grad = torch.autograd.grad(outs, [st["logits"]], st["d_out"])
    return [x.detach() for x in outs] + labels + list(grad)


def _score_plain(st):
    c = st["case"]
    x, y = st["logits"].detach().float(), st["targets"].long()
    n, v = x.shape
    top = x.amax(dim=-1, keepdim=True)
    z = x - torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(z)
    total = e.sum(dim=-1, keepdim=True)
    some = total > 0  # rows that allow any label
    p = e / torch.where(some, total, 1.0)
    lp = torch.where(z == -math.inf, -math.inf, z - torch.log(torch.where(some, total, 1.0)))
    surprise = torch.where(p > 0, lp, 0.0)
    entropy = -(p * surprise).sum(dim=-1)
    given = (y >= 0) & (y < v)
    label = y.clamp(0, v - 1)[:, None]
    outs = [torch.where(given, lp.gather(-1, label)[:, 0], 0.0), entropy]
    best = []
    if c["top"]:
        best = [torch.sort(x, dim=-1, descending=True, stable=True)[1][:, : c["top"]]]
        outs.append(lp.gather(-1, best[0]))
    labels = [b.to(torch.int32) for b in best]
    if not c["train"]:
        return outs + labels
    # gradients: label minus probability for every log probability, -p (log p + H) for the entropy; none in a row without labels
    g, ge = st["d_out"][0] * given * some[:, 0], st["d_out"][1]
    weight = g[:, None]
    d = torch.zeros_like(x).scatter_add_(-1, label, weight)
    for b, gb in zip(best, st["d_out"][2:]):
        gb = torch.where(some, gb, 0.0)
        d.scatter_add_(-1, b, gb)
        weight = weight + gb.sum(dim=-1, keepdim=True)
    d -= p * (weight + ge[:, None] * (surprise + entropy[:, None]))
    return outs + labels + [d.to(st["logits"].dtype)]


def run(st: Dict[str, Any]):
    kind = st["case"]["kind"].replace("_cache", "")
    return globals()["_%s_%s" % (kind, "own" if own else "plain")](st)


# ---------------------------------------------------------------------------------------------------------------- what a pass cannot do without


def work(case: Dict[str, Any]) -> Dict[str, float]:
    kind = case["kind"]
    size = {"bf16": 2, "f32": 4}[case.get("dtype", "bf16")]
    if kind in ("rope", "rope_cache"):
        qk = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        if kind == "rope_cache":
            return {"bytes": size * (2 * qk + 2 * case["tokens"] * case["kv_heads"] * case["dim"]), "flops": 8.0 * qk}
        times = 2 + (2 + (1 if case["norm"] else 0) if case["train"] else 0)
        return {"bytes": size * times * qk, "flops": (24.0 if case["train"] else 8.0) * qk}
    if kind == "append":
        tokens = 0.45 * case["requests"] * (case["new"] + 1)
        return {"bytes": 12 * tokens + 4 * tokens / case["page"] + 25 * case["requests"] + 32, "flops": 0}
    if kind == "release":
        return {"bytes": 8 * 0.225 * case["requests"] * case["max_len"] / case["page"] + 9 * case["requests"] + 32, "flops": 0}
    if kind == "attention":
        tokens = case["max_len"] + 0.5 * (case["requests"] - 1) * (case["max_len"] + 1) * (0.9 if case["empty"] else 1.0)
        return {"bytes": size * (2.0 * tokens * case["kv_heads"] * case["dim"] + 2 * case["requests"] * case["heads"] * case["dim"]) + 4 * tokens / case["page"],
                "flops": 4.0 * tokens * case["heads"] * case["dim"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": size * n * (2 if case["train"] else 1) + case["rows"] * (12 + 8 * case["top"]), "flops": (14.0 if case["train"] else 6.0) * n}


# ---------------------------------------------------------------------------------------------------------------- the definitions in 64 bits


def exact(case: Dict[str, Any], seed: int):
    st = prepare(case, seed)
    kind = case["kind"]
    f64 = torch.float64
    if kind in ("append", "release"):
        return None  # whole numbers
    if kind in ("rope", "rope_cache"):
        d, rot = case["dim"], case["rotary"]
        # the rotation of every token as a complex number of modulus one
        turn = torch.polar(torch.ones((), dtype=f64, device=DEV), torch.outer(st["positions"].to(f64), st["frequencies"].to(f64)))[:, None, :]
        order = torch.arange(rot, device=DEV).view(-1, 2) if case["interleaved"] else torch.arange(rot, device=DEV).view(2, -1).t()

        def turned(x, by):
            pairs = torch.view_as_complex(x[..., order].contiguous()) * by
            out = x.clone()
            out[..., order] = torch.view_as_real(pairs)
            return out

        outs, grads, scales = [], [], []
        for i, (x, scale) in enumerate(((st["q"], st["q_scale"]), (st["k"], st["k_scale"]))):
            x = x.detach().to(f64)
            inv = 1.0 / torch.sqrt(x.pow(2).sum(dim=-1, keepdim=True) / d + 1e-6) if scale is not None else 1.0
            w = scale.detach().to(f64) if scale is not None else 1.0
            outs.append(turned(x * inv * w, turn))
            if case.get("train"):
                dy = turned(st["d_out"][i].to(f64), turn.conj())
                if scale is not None:
                    unit = x * inv
                    scales.append((dy * unit).flatten(0, 1).sum(dim=0))
                    dy = inv * (dy * w - unit * ((dy * w * unit).sum(dim=-1, keepdim=True) / d))
                grads.append(dy)
        if kind == "rope":
            return outs + grads + scales
        caches = [c.to(f64) for c in st["cache"]]
        for cache, x in zip(caches, (outs[1], st["v"].to(f64))):
            rows = cache.permute(0, 2, 1, 3).reshape(-1, *x.shape[1:])  # by slots
            rows[st["slots"][st["slots"] >= 0].long()] = x[st["slots"] >= 0]
            cache.copy_(rows.view(cache.shape[0], cache.shape[2], *x.shape[1:]).permute(0, 2, 1, 3))
        return [outs[0]] + caches
    if kind == "attention":
        r, h, d = st["q"].shape
        _, hk, page, _ = st["cache"][0].shape
        out = torch.zeros(r, h, d, dtype=f64, device=DEV)
        for i, n in enumerate(st["lengths"].tolist()):
            if n:
                pages = st["block_table"][i, : -(-n // page)].long()
                k, v = (c[pages].transpose(0, 1).reshape(hk, -1, d)[:, :n].to(f64) for c in st["cache"])
                q = st["q"][i].to(f64).view(hk, h // hk, d)
                out[i] = torch.softmax(torch.einsum("hgd,htd->hgt", q, k) / math.sqrt(d), dim=-1).matmul(v).reshape(h, d)
        return out
    n, v = st["logits"].shape
    top = case["top"]
    best = torch.empty(n, top, dtype=f64, device=DEV)
    lp, ent = torch.zeros(n, dtype=f64, device=DEV), torch.zeros(n, dtype=f64, device=DEV)
    grad = torch.zeros(n, v, dtype=f64, device=DEV) if case["train"] else None
    for a in range(0, n, 500):
        x = st["logits"].detach()[a: a + 500].to(f64)
        y = st["targets"][a: a + 500].long()
        rows = torch.arange(x.shape[0], device=DEV)
        empty = torch.isneginf(x).all(dim=-1)
        logp = torch.log_softmax(x, dim=-1)
        logp[empty] = -math.inf
        p = logp.exp()
        plogp = torch.special.entr(p)
        ent[a: a + 500] = plogp.sum(dim=-1)
        asked = (y >= 0) & (y < v)
        lp[a: a + 500][asked] = logp[rows[asked], y[asked]]
        order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top] if top else None
        if top:
            best[a: a + 500] = logp.gather(-1, order)
        if grad is not None:
            gs = [t[a: a + 500].to(f64) * (~empty).view(-1, *[1] * (t.dim() - 1)) for t in st["d_out"]]
            part = plogp * gs[1][:, None] - p * (gs[1] * ent[a: a + 500])[:, None]
            part -= p * (gs[0] * asked)[:, None]
            part[rows[asked], y[asked]] += gs[0][asked]
            if top:
                part -= p * gs[2].sum(dim=-1, keepdim=True)
                part.scatter_add_(-1, order, gs[2])
            grad[a: a + 500] = part
    return [lp, ent] + ([best, None] if top else []) + ([grad] if grad is not None else [])
