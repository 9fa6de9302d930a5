"""
Serving a decoder-only language model (:class:`rf.TransformerDecoder` without an encoder) to requests that come and go: scoring of given texts and greedy
generation over a paged key / value cache.

Keys and values of all running requests lie in pages of ``page_size`` tokens, one pool per layer under one block table; a request takes pages as it grows and gives them back when
it ends (:mod:`returnn_b200.ops.paged`). A step of all running requests is a fixed sequence of kernels on fixed addresses: pages and slots of the new tokens, per layer the
projection, norm and rotation into the cache, attention over the pages, feed-forward; the output layer and its best label with its log probability. On the GPU it is captured
once as a CUDA graph; which rows take part is a tensor, so that requests join and leave between replays. Between two steps the host reads the results of the first.

A serving loop of its own, where :meth:`PagedDecoder.generate` is not what is wanted::

    x = paged.add([row], [prompt])                       # the prompt runs through the layers; paged.logits(x[-1:]) is about its next label
    labels, log_probs, rows, granted = paged.step({row: label, ...})
    paged.end([row])

New requests run through the layers as packed rows, their keys and values going to their pages on the way, with ordinary causal attention inside each prompt.

The reference decodes by the step interface over states that grow by concatenation (returnn/frontend/decoder/transformer.py:216-258); it has no paged form.
"""

from __future__ import annotations
from typing import Dict, List, Mapping, NamedTuple, Optional, Sequence
import torch
import torch.nn.functional as F

from ..ops import attention as _att
from ..ops.norm_rope import norm_rope_to_cache, rope_frequencies
from ..ops.paged import append_tokens, paged_attention, release_pages
from ..ops.status import KernelWaitTimeout, StatusPoller
from ..ops.token_log_probs import token_log_probs
from .decode_graph import _lin, _norm, _apply_norm, _activation

__all__ = ["PagedDecoder", "ScoredText", "GeneratedText"]


class ScoredText(NamedTuple):
    """of one text of :meth:`PagedDecoder.score`"""

    log_probs: torch.Tensor  # [len - 1] fp32: of each label after the first, given those before it
    entropy: torch.Tensor  # [len - 1] fp32
    top_labels: Optional[torch.Tensor]  # [len - 1, num_top] int32
    top_log_probs: Optional[torch.Tensor]


class GeneratedText(NamedTuple):
    """of one prompt of :meth:`PagedDecoder.generate`"""

    labels: List[int]  # without the prompt, with the end label if it was reached
    log_probs: List[float]


class PagedDecoder:
    """see the module docstring"""

    def __init__(self, decoder, *, max_requests: int, max_len: int, page_size: int = 16, num_pages: Optional[int] = None, dtype: Optional[torch.dtype] = None):
        """
        :param decoder: rf TransformerDecoder without cross-attention; self-attention causal, with or without rotary positions
        :param max_requests: rows: requests that run at the same time
        :param max_len: longest request, prompt and new labels
        :param num_pages: of the pool; default: enough for every row to be that long
        """
        from ..frontend.attention import CausalSelfAttention, RotaryPosCausalSelfAttention
        from ..frontend.decoder.transformer import FeedForward, FeedForwardGated

        emb = decoder.input_embedding.weight.raw_tensor
        self.device, self.dtype = emb.device, dtype or emb.dtype
        cast = lambda t: None if t is None else t.detach().to(self.dtype)  # noqa: E731
        if decoder.input_embedding_proj is not None:
            raise TypeError("paged decoder: embed_dim != model_dim is not covered")
        self.emb, self.emb_scale, self.vocab = cast(emb), float(decoder.input_embedding_scale), decoder.vocab_dim.dimension
        self.page_size, self.max_len, self.rows = page_size, max_len, max_requests
        blocks = -(-max_len // page_size)
        self.num_pages = max_requests * blocks if num_pages is None else num_pages
        self.pos_table = None
        if decoder.pos_enc is not None:
            from ..frontend.attention import sinusoidal_positional_encoding
            from ..tensor import Dim

            fn = decoder.pos_enc
            if getattr(fn, "func", fn) is not sinusoidal_positional_encoding:
                raise TypeError("paged decoder: positional encoding %r is not covered" % (fn,))
            steps = Dim(blocks * page_size, name="steps")  # (all positions that have a place)
            self.pos_table = cast(fn(spatial_dim=steps, device=str(self.device)).copy_transpose([steps, decoder.model_dim]).raw_tensor)
        self.layers = []
        for layer in decoder.layers:
            sa = layer.self_att
            if type(sa) not in (CausalSelfAttention, RotaryPosCausalSelfAttention) or layer.cross_att is not None:
                raise TypeError("paged decoder: %r with cross-attention %r is not covered" % (sa, layer.cross_att))
            h, dk, dv = sa.num_heads.dimension, sa.key_dim_per_head.dimension, sa.value_dim_per_head.dimension
            if dk != dv:
                raise TypeError("paged decoder: keys of %i and values of %i features per head are not covered" % (dk, dv))
            rope = dict(frequencies=None)
            if isinstance(sa, RotaryPosCausalSelfAttention):
                given = getattr(sa, "rope", None)
                rope = dict(given) if given is not None else dict(frequencies=rope_frequencies(dk)[0])
                rope["frequencies"] = rope["frequencies"].to(self.device)
                if getattr(sa, "q_norm", None) is not None:
                    rope.update(q_scale=sa.q_norm.scale.raw_tensor.detach(), k_scale=sa.k_norm.scale.raw_tensor.detach(), eps=sa.q_norm.eps)
            ff = layer.ff
            if isinstance(ff, FeedForwardGated):
                acts = (_activation(ff.activation), _activation(ff.gate_activation))
            elif isinstance(ff, FeedForward):
                acts = (_activation(ff.activation), None)
            else:
                raise TypeError("paged decoder: feed-forward %r is not covered" % (ff,))
            pool = torch.zeros(2, self.num_pages, h, page_size, dk, dtype=self.dtype, device=self.device)
            self.layers.append(dict(h=h, d=dk, rope=rope, sa_norm=_norm(layer.self_att_layer_norm), ff_norm=_norm(layer.ff_layer_norm), acts=acts,
                                    qkv=tuple(map(cast, _lin(sa.qkv))), proj=tuple(map(cast, _lin(sa.proj))) if sa.proj else None,
                                    ff1=tuple(map(cast, _lin(ff.linear_ff))), ff2=tuple(map(cast, _lin(ff.linear_out))), k=pool[0], v=pool[1]))
        self.final_norm = _norm(decoder.final_layer_norm)
        self.logits_w, self.logits_b = map(cast, _lin(decoder.logits))
        # what the requests have, on the device
        i32 = dict(dtype=torch.int32, device=self.device)
        self.block_table = torch.full((max_requests, blocks), -1, **i32)
        self.lengths = torch.zeros(max_requests, **i32)
        self.free_pages = torch.arange(self.num_pages, **i32)
        self.free_range = torch.tensor([0, self.num_pages], dtype=torch.int64, device=self.device)
        self._last = torch.zeros(max_requests, dtype=torch.int64, device=self.device)  # label that a row continues with
        self._active = torch.zeros(max_requests, **i32)
        self._ignored = torch.full((max_requests,), -1, **i32)
        self._graph = None
        self._step_out = None
        self._status = StatusPoller(self.device)

    # ---- the layers

    def _embed(self, labels: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        x = self.emb.index_select(0, labels)
        if self.emb_scale != 1.0:
            x = x * self.emb_scale
        if self.pos_table is not None:
            x = x + self.pos_table.index_select(0, positions.long().clamp(max=self.pos_table.shape[0] - 1))
        return x

    def _layer(self, lay, x: torch.Tensor, new, attend) -> torch.Tensor:
        """``x`` [tokens, features]; ``attend(layer, q, k, v)`` -> [tokens, heads * dim], after keys and values went to their slots"""
        w, b = lay["qkv"]
        qkv = F.linear(_apply_norm(x, lay["sa_norm"]), w.t(), b).view(-1, lay["h"], 3 * lay["d"])
        q, k, v = qkv.split(lay["d"], dim=-1)  # (q, k, v) of a head side by side, read in place
        q = norm_rope_to_cache(q, k, v, new.positions, lay["rope"]["frequencies"], lay["k"], lay["v"], new.slots, **{n: o for n, o in lay["rope"].items() if n != "frequencies"})
        att = attend(lay, q, k, v)
        if lay["proj"] is not None:
            w, b = lay["proj"]
            att = F.linear(att, w.t(), b)
        x = x + att
        h = F.linear(_apply_norm(x, lay["ff_norm"]), lay["ff1"][0].t(), lay["ff1"][1])
        act, gate = lay["acts"]
        if gate is None:
            h = act(h)
        else:
            a, g = h.chunk(2, dim=-1)
            h = act(a) * gate(g)
        return x + F.linear(h, lay["ff2"][0].t(), lay["ff2"][1])

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        """output layer for features [tokens, features] that :meth:`add` returned"""
        with torch.autocast(self.device.type, enabled=False):
            return F.linear(_apply_norm(x, self.final_norm), self.logits_w.t(), self.logits_b)

    # ---- requests

    def _check_prompt(self, labels: Sequence[int]):
        if not 0 < len(labels) <= self.max_len:
            raise ValueError("paged decoder: a prompt of %i labels (1 to %i)" % (len(labels), self.max_len))
        self._check_labels(labels)

    def _check_labels(self, labels: Sequence[int]):
        if not (0 <= min(labels) and max(labels) < self.emb.shape[0]):  # (here, not by the lookup on the device)
            raise ValueError("paged decoder: labels %i to %i, the vocabulary has %i" % (min(labels), max(labels), self.emb.shape[0]))

    def _check_rows(self, rows: Sequence[int]):
        if any(not 0 <= r < self.rows for r in rows):
            raise ValueError("paged decoder: rows %s of %i" % (list(rows), self.rows))
        if len(set(rows)) != len(rows):
            raise ValueError("paged decoder: a row twice in %s" % (list(rows),))

    def _empty_rows(self) -> List[int]:
        return [r for r, have in enumerate(self.lengths.tolist()) if have <= 0]

    def _that_fit(self, texts: Sequence[Sequence[int]]) -> int:
        """:return: how many of these, from the first on, have room in the pool together (the host looks at the range of free pages)"""
        head, tail = self.free_range.tolist()
        room = tail - head
        for n, text in enumerate(texts):
            room -= -(-len(text) // self.page_size)
            if room < 0:
                return n
        return len(texts)

    def add(self, rows: Sequence[int], prompts: Sequence[Sequence[int]]) -> torch.Tensor:
        """
        New requests in empty rows (the host looks at the lengths): their prompts take pages and run through the layers.

        :return: [tokens, features] after the last layer, the tokens of the prompts one after another. Rows without room in the pool stay empty (:attr:`lengths`).
        """
        with torch.no_grad(), torch.autocast(self.device.type, enabled=False):
            order = sorted(range(len(rows)), key=lambda i: rows[i])  # (tokens of a call lie in the order of the rows)
            if len(rows) != len(prompts):
                raise ValueError("paged decoder: %i prompts for %i rows" % (len(prompts), len(rows)))
            self._check_rows(rows)
            for prompt in prompts:
                self._check_prompt(prompt)
            if not rows:
                return self.emb.new_zeros(0, self.emb.shape[1])
            held = set(rows) - set(self._empty_rows())
            if held:
                raise ValueError("paged decoder: row %s holds a request" % sorted(held))
            counts = torch.zeros(self.rows, dtype=torch.int32)
            for i in order:
                counts[rows[i]] = len(prompts[i])
            labels = torch.tensor([t for i in order for t in prompts[i]], dtype=torch.int64).to(self.device)
            total = len(labels)
            new = append_tokens(self.block_table, self.lengths, counts.to(self.device), self.free_pages, self.free_range, page_size=self.page_size, max_tokens=total)
            self.lengths.copy_(new.lengths)
            self.free_range.copy_(new.free_range)
            lens = torch.tensor([len(prompts[i]) for i in order], dtype=torch.int32)
            longest, n = int(lens.max()), len(order)
            # where a packed token lies in the padded batch that the attention inside the prompts takes, and back
            place = torch.cat([torch.arange(int(m)) + i * longest for i, m in enumerate(lens)]).to(self.device)
            lens = lens.to(self.device)

            def attend(lay, q, k, v):
                # keys as they are in the cache, normed and rotated
                at = new.slots.long().clamp(min=0)
                k = lay["k"][at // self.page_size, :, at % self.page_size]
                q, k, v = (t.new_zeros(n * longest, lay["h"], lay["d"]).index_copy_(0, place, t).view(n, longest, lay["h"], lay["d"]).transpose(1, 2) for t in (q, k, v))
                out = _att.sdpa(q, k, v, kv_lens=lens[:, None].expand(n, lay["h"]), scale=lay["d"] ** -0.5, causal=True)
                return out.transpose(1, 2).reshape(n * longest, -1).index_select(0, place)

            try:
                x = self._embed(labels, new.positions)
                for lay in self.layers:
                    x = self._layer(lay, x, new, attend)
            except BaseException:
                self.end(rows)
                raise
            return x[self._unsorted(order, [len(p) for p in prompts])] if order != list(range(len(rows))) else x

    def _unsorted(self, order, lens) -> torch.Tensor:
        """of tokens in the given order of prompts: their places in the order of rows"""
        start, at = {}, 0
        for i in order:
            start[i] = at
            at += lens[i]
        return torch.cat([torch.arange(start[i], start[i] + n) for i, n in enumerate(lens)]).to(self.device)

    def _step(self):
        new = append_tokens(self.block_table, self.lengths, self._active, self.free_pages, self.free_range, page_size=self.page_size, max_tokens=self.rows)
        self.lengths.copy_(new.lengths)
        self.free_range.copy_(new.free_range)
        row = new.requests.clamp(min=0).long()  # the rows that take part come first
        table, lengths = self.block_table.index_select(0, row), torch.where(new.requests >= 0, new.lengths.index_select(0, row), 0)
        x = self._embed(self._last.index_select(0, row), new.positions)
        for lay in self.layers:
            x = self._layer(lay, x, new, lambda la, q, k, v: paged_attention(q, la["k"], la["v"], table, lengths).flatten(1))
        best = token_log_probs(self.logits(x), self._ignored, num_top=1)
        return best.top_labels[:, 0], best.top_log_probs[:, 0], new.requests, new.granted

    def step(self, labels: Optional[Mapping[int, int]] = None, *, use_graph: Optional[bool] = None):
        """
        One more token for some rows.

        :param labels: row -> label that it continues with, the last one of its prompt or the one that the step before found; the row may be empty.
            None: the rows and labels of the call before, without those that have ended.
        :return: best label, its log probability and row of each (rows in ascending order, -1 behind the last), and for each row of the decoder whether it was granted its page.
            The next step overwrites them. A row without a page stays as it was, and can take the same label again when another request has ended.
            A kernel of the step that gave up a wait is an error (:class:`returnn_b200.ops.status.KernelWaitTimeout`) in the next call.
        """
        if labels is not None:
            self._check_rows(list(labels))
            if labels:
                self._check_labels(list(labels.values()))
            active, last = torch.zeros(self.rows, dtype=torch.int32), torch.zeros(self.rows, dtype=torch.int64)
            for row, label in labels.items():
                active[row], last[row] = 1, label
            self._active.copy_(active)
            self._last.copy_(last)
        if use_graph is None:
            use_graph = self.device.type == "cuda"
        with torch.no_grad(), torch.autocast(self.device.type, enabled=False):
            if not use_graph:
                out = self._step()
                self._look_at_status()
                return out
            if self._graph is None:
                # lazy initialisation outside the capture, with no row taking part
                active = self._active.clone()
                self._active.zero_()
                side = torch.cuda.Stream(device=self.device)
                side.wait_stream(torch.cuda.current_stream(self.device))
                with torch.cuda.stream(side):
                    self._step()
                torch.cuda.current_stream(self.device).wait_stream(side)
                self._active.copy_(active)
                self._graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(self._graph):
                    self._step_out = self._step()
            self._graph.replay()
            self._look_at_status()
            return self._step_out

    def _look_at_status(self, wait: bool = False):
        """whether a kernel gave up a wait, in what was queued before the last call, or in all so far"""
        try:
            self._status.step(where="paged decoder")
            if wait:
                self._status.flush(where="paged decoder")
        except KernelWaitTimeout:
            self._status = StatusPoller(self.device)  # (copies still under way show the same)
            raise

    def end(self, rows: Sequence[int]):
        """these requests are over: their pages go back to the pool"""
        self._check_rows(rows)
        done = torch.zeros(self.rows, dtype=torch.bool)
        done[list(rows)] = True
        done = done.to(self.device)
        self._active.masked_fill_(done, 0)
        back = release_pages(self.block_table, self.lengths, done, self.free_pages, self.free_range, page_size=self.page_size)
        self.lengths.copy_(back.lengths)
        self.free_range.copy_(back.free_range)

    # ---- what a user calls

    def score(self, texts: Sequence[Sequence[int]], *, num_top: int = 0) -> List[ScoredText]:
        """
        Log probability of every label of each text after its first, the entropy at its position and the best alternatives. The texts run in rows that hold no request.
        """
        res: List[ScoredText] = []
        empty = self._empty_rows()
        if texts and not empty:
            raise RuntimeError("paged decoder: all %i rows hold requests" % self.rows)
        for at in range(0, len(texts), max(len(empty), 1)):
            part = texts[at: at + len(empty)]
            rows = empty[: len(part)]
            if self._that_fit(part) < len(part):
                raise RuntimeError("paged decoder: no room for %i texts in %i pages" % (len(part), self.num_pages))
            x = self.add(rows, part)
            try:
                targets = torch.tensor([y for t in part for y in list(t[1:]) + [-1]], dtype=torch.int32).to(self.device)
                with torch.no_grad():
                    r = token_log_probs(self.logits(x), targets, entropy=True, num_top=num_top)
            finally:
                self.end(rows)
            first = 0
            for t in part:
                cut = slice(first, first + len(t) - 1)
                res.append(ScoredText(r.log_probs[cut], r.entropy[cut], r.top_labels[cut] if num_top else None, r.top_log_probs[cut] if num_top else None))
                first += len(t)
        self._look_at_status(wait=True)
        return res

    def generate(self, prompts: Sequence[Sequence[int]], *, max_new: int, eos: int, use_graph: Optional[bool] = None) -> List[GeneratedText]:
        """
        The best label after each prompt, and so on until ``eos`` or ``max_new`` labels or the longest length. Prompts beyond the number of rows, or without pages at the moment, wait until
        others end. Where none of the running ones can go on for want of a page, the one that began last gives its pages up; it waits, and its prompt and labels so far run through the layers
        again. One that does not fit the pool alone is an error. They run in rows that hold no request.
        """
        for prompt in prompts:
            self._check_prompt(prompt)
            if len(prompt) > self.num_pages * self.page_size:
                raise RuntimeError("paged decoder: a prompt of %i labels does not fit %i pages" % (len(prompt), self.num_pages))
        empty = self._empty_rows()
        if prompts and not empty:
            raise RuntimeError("paged decoder: all %i rows hold requests" % self.rows)
        out = [GeneratedText([], []) for _ in prompts]
        waiting = list(range(len(prompts)))
        running = {}  # row -> prompt, in the order in which they began
        stuck: List[int] = []  # rows that found no page in the last step; others join when there are none
        last: Dict[int, int] = {}  # label that a row continues with

        def take(i: int, label: int, log_prob: float) -> bool:
            """:return: whether the request goes on"""
            out[i].labels.append(label)
            out[i].log_probs.append(log_prob)
            return label != eos and len(out[i].labels) < max_new and len(prompts[i]) + len(out[i].labels) < self.max_len

        held = set()  # rows that may have pages
        try:
            while waiting or running:
                free = [r for r in empty if r not in running]
                batch = waiting[: len(free)] if not stuck else []
                text = {i: list(prompts[i]) + out[i].labels for i in batch}
                batch = batch[: self._that_fit([text[i] for i in batch])] if batch else batch
                if batch:
                    rows = free[: len(batch)]
                    del waiting[: len(batch)]
                    held.update(rows)
                    x = self.add(rows, [text[i] for i in batch])
                    ends = torch.tensor([len(text[i]) for i in batch]).cumsum(0) - 1
                    with torch.no_grad():
                        best = token_log_probs(self.logits(x[ends.to(self.device)]), self._ignored[: len(batch)], num_top=1)
                    over = []
                    for r, i, label, lp in zip(rows, batch, best.top_labels[:, 0].tolist(), best.top_log_probs[:, 0].tolist()):
                        if max_new > 0 and take(i, label, lp):
                            running[r], last[r] = i, label
                        else:
                            over.append(r)
                    if over:
                        self.end(over)
                        held.difference_update(over)
                elif not running:
                    i = waiting[0]
                    raise RuntimeError("paged decoder: a prompt of %i labels and %i more do not fit what is free of %i pages" % (len(prompts[i]), len(out[i].labels), self.num_pages))
                if not running:
                    continue
                labels, log_probs, requests, granted = self.step({r: last[r] for r in running}, use_graph=use_graph)
                over, stuck = [], []
                for r, label, lp, ok in zip(requests.tolist(), labels.tolist(), log_probs.tolist(), granted[requests.clamp(min=0).long()].tolist()):
                    if r < 0:
                        break
                    if not ok:  # no page was left for it in this step; it goes on when another ends
                        stuck.append(r)
                    elif take(running[r], label, lp):
                        last[r] = label
                    else:
                        over.append(r)
                if len(stuck) == len(running):
                    last_row = list(running)[-1]
                    waiting.insert(0, running[last_row])
                    over.append(last_row)
                    stuck.remove(last_row)
                for r in over:
                    del running[r]
                if over:
                    self.end(over)
                    held.difference_update(over)
            self._look_at_status(wait=True)
        finally:
            if held:
                self.end(sorted(held))
        return out
