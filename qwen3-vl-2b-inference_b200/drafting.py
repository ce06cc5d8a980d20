"""Decoding with drafted trees: several tokens of each request per pass.

A draft model (or an n-gram table, or anything else) proposes for every request a
tree of tokens after the one that was chosen last.  One pass over the weights
scores all nodes of all trees, and the path that agrees with the model's own
greedy choices is kept:

    plan_pages -> embedding -> layers x [rms_norm -> q/k/v linear ->
    qknorm_mrope_kv_append -> tree_attention -> o linear + residual ->
    rms_norm -> gate/up linear -> swiglu -> down linear + residual] ->
    rms_norm -> tied LM head -> greedy_decode, token_logprobs -> plan_pages

The linears run as one M = (all nodes) product in the order of the tensor cores
(QVL_SEM_TILED), fewer than 16 rows in the order of a single request's products
(QVL_SEM_LANE8), like TextDecoder with batch_order "auto"; attention sums in fp32 in its
own order, like attn_order "fast".  Requests share one pool of cache pages: a
pass takes pages for its whole draft and hands back what the accepted path does not
need.  No counterpart in the reference, which decodes one token of one request at a
time.
"""
from __future__ import annotations

import dataclasses

import numpy as np
import torch

from . import (AttnDims, PagePlan, Planes, QvlError, SEM_ACCUMULATE, SEM_LANE8, SEM_TILED, Workspace,
               embedding_lookup_i8, greedy_decode, linear_planes_batched, linear_q16, mrope_axes, plan_pages,
               qknorm_mrope_kv_append, quantize_rows_planes, rms_norm_i8_planes, token_logprobs, tree_attention)
from . import swiglu as swiglu_
from .decoder import TextWeights, rope_table

MAX_NODES = 256          # of one request in one pass


class PooledKV:
    """One layer's pages [num_pages, NKV, page_size, D] of a pool that requests share."""

    def __init__(self, k, v, page_table, dims):
        self.k, self.v, self.page_table, self.dims, self.page_size = k, v, page_table, dims, dims.page_size


@dataclasses.dataclass
class Accepted:
    """What a request got from a pass: `tokens`, chosen one after another (the last one is
    its next pass's root), with their log-probabilities and the entropies of the
    distributions they were chosen from; top_ids, top_logprobs [len(tokens), top_k]."""
    tokens: list
    logprobs: np.ndarray
    entropy: np.ndarray
    top_ids: np.ndarray
    top_logprobs: np.ndarray


def check_tree(tokens, parents, vocab: int) -> list:
    """Depths of a tree's nodes: node 0 is its root (parent -1), and every other node's
    parent comes before it."""
    n = len(tokens)
    if not 1 <= n <= MAX_NODES or len(parents) != n:
        raise QvlError(f"a tree has 1 to {MAX_NODES} nodes, each with a parent")
    if parents[0] != -1 or any(not 0 <= p < i for i, p in enumerate(parents) if i):
        raise QvlError("node 0 is the root (parent -1) and a parent comes before its children")
    if any(not 0 <= t < vocab for t in tokens):
        raise QvlError("a drafted token lies outside the vocabulary")
    depth = [0] * n
    for i in range(1, n):
        depth[i] = depth[parents[i]] + 1
    return depth


def accepted_path(tokens, parents, greedy) -> list:
    """Nodes from the root on along which each token is the greedy choice of the one
    before it."""
    path = [0]
    while True:
        step = [i for i in range(path[-1] + 1, len(tokens)) if parents[i] == path[-1] and tokens[i] == greedy[path[-1]]]
        if not step:
            return path
        path.append(step[0])


class TreeDecoder:
    """Requests 0 .. max_requests - 1 over one pool of num_pages cache pages per layer.

    max_tokens: nodes of all requests in one pass.  sections: rotary frequencies per position axis
    (D / 2 in all), None for text positions alone.  A token without positions of its own is at
    its request's largest position so far plus 1, on all axes (a node of a tree at its depth past that),
    which after an image is less than the number of tokens."""

    def __init__(self, weights: TextWeights, max_requests: int, max_ctx: int, num_pages: int, max_tokens: int = 512,
                 page_size: int = 64, sections=None, device="cuda"):
        cfg = self.cfg = weights.cfg
        self.w, self.S, self.max_ctx, self.max_tokens, self.page_size = weights, max_requests, max_ctx, max_tokens, page_size
        dev = self.device = torch.device(device)
        D, H, I, T = cfg.head_dim, cfg.hidden, cfg.intermediate, max_tokens
        maxp = -(-max_ctx // page_size)
        shape = (cfg.layers, num_pages, cfg.kv_heads, page_size, D)
        self.k_all = torch.zeros(shape, dtype=torch.float16, device=dev)
        self.v_all = torch.zeros(shape, dtype=torch.float16, device=dev)
        self.page_table = torch.full((max_requests, maxp), -1, dtype=torch.int32, device=dev)
        dims = AttnDims(cfg.heads, cfg.kv_heads, D, page_size, maxp, max_ctx)
        self.kv = [PooledKV(self.k_all[l], self.v_all[l], self.page_table, dims) for l in range(cfg.layers)]
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=dev)
        self.num_pages, self.lengths = num_pages, [0] * max_requests
        self.next_pos = [0] * max_requests          # each request's largest position so far plus 1
        sections = (D // 2,) if sections is None else sections
        self.axes, self.n_axes = mrope_axes(sections, device=dev), len(sections)
        cos, sin = rope_table(max_ctx, D, cfg.rope_theta)
        self.rope_cos, self.rope_sin = torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev)
        f32, i16 = torch.float32, torch.int16
        self.x = torch.zeros((T, H), dtype=f32, device=dev)
        self.q = torch.zeros((T, cfg.heads * D), dtype=f32, device=dev)
        self.k = torch.zeros((T, cfg.kv_heads * D), dtype=f32, device=dev)
        self.v = torch.zeros((T, cfg.kv_heads * D), dtype=f32, device=dev)
        self.att = torch.zeros((T, cfg.heads * D), dtype=f32, device=dev)
        self.gate = torch.zeros((T, I), dtype=f32, device=dev)
        self.up = torch.zeros((T, I), dtype=f32, device=dev)
        self.q16 = torch.zeros((T, max(H, I, cfg.heads * D)), dtype=i16, device=dev)
        self.qs = torch.zeros((T, 1), dtype=f32, device=dev)
        self.planes = Planes(T, max(H, I, cfg.heads * D), dev)
        self.ws = Workspace(dev)
        self._plans: dict = {}

    def _own_positions(self, s: int, own, n: int) -> np.ndarray:
        """Positions [axes, n] that request s is to have, checked."""
        own = np.asarray(own)
        if own.shape != (self.n_axes, n):
            raise QvlError(f"positions of request {s}: expected [{self.n_axes}, {n}]")
        if own.min() < 0 or own.max() >= self.max_ctx:
            raise QvlError(f"request {s}: a position outside the rotary table's {self.max_ctx} rows")
        return own.astype(np.int32)

    def _check_room(self, after) -> None:
        """The context and the pool have room for requests of these lengths.  (The pool is this decoder's
        alone, so that its free pages follow from the lengths.)"""
        for s, n in enumerate(after):
            if n > self.max_ctx:
                raise QvlError(f"request {s}: {n} tokens pass the context of {self.max_ctx}")
        pages = sum(-(-n // self.page_size) for n in after)
        if pages > self.num_pages:
            raise QvlError(f"the cache pool has {self.num_pages} pages, and the requests would hold {pages}")

    def _plan(self, old, new, free_count, tokens: int, which: str) -> PagePlan:
        """Lengths old -> new; the pass's own plan and the one that gives pages back write
        to buffers of their own, each reading the other's stack size."""
        p = plan_pages(old, new, self.page_table, self.free_pages, free_count, self.page_size, tokens,
                       plan=self._plans.get((which, tokens)))
        if (which, tokens) not in self._plans:
            self._plans = {k: v for k, v in self._plans.items() if k[0] != which}
            self._plans[which, tokens] = p
        return p

    def _product(self, q, qs, names, l, outs, acc=0):
        """Rows quantised last, against matrices of layer l (None: the tied LM head)."""
        t, (M, K) = self.w.t, q.shape
        mats = [(t[n], t[n + "_s"]) if l is None else (t[n][l], t[n + "_s"][l]) for n in names]
        if M >= 16:
            linear_planes_batched(self.planes, qs, mats, outs, M, K, semantics=SEM_TILED | acc)
        else:
            for (w, s), out in zip(mats, outs):
                linear_q16(q, qs, w, s, K, C=out, semantics=SEM_LANE8 | acc)

    def _layers(self, x, T, plan, positions, ctx, parents, max_len, most):
        cfg, t, P, qs = self.cfg, self.w.t, self.planes, self.qs[:T]
        H, I, D, ng, eps = cfg.hidden, cfg.intermediate, cfg.head_dim, cfg.norm_group, cfg.eps
        qh, qi = self.q16.view(-1)[:T * H].view(T, H), self.q16.view(-1)[:T * I].view(T, I)
        qa = self.q16.view(-1)[:T * cfg.heads * D].view(T, cfg.heads * D)
        q, k, v, att = self.q[:T], self.k[:T], self.v[:T], self.att[:T]
        gate, up = self.gate[:T], self.up[:T]
        heads = q.view(T, cfg.heads, D)
        for l in range(cfg.layers):
            rms_norm_i8_planes(x, t["in_norm"][l], t["in_norm_s"][l], ng, eps, qh, qs, P)
            self._product(qh, qs, ("wq", "wk", "wv"), l, [q, k, v])
            qknorm_mrope_kv_append(heads, k.view(T, -1, D), v.view(T, -1, D), self.kv[l], plan.slots, positions, self.axes,
                                   self.rope_cos, self.rope_sin, (t["q_norm"][l], t["q_norm_s"][l], ng),
                                   (t["k_norm"][l], t["k_norm_s"][l], ng), eps, out=heads)
            tree_attention(heads, self.kv[l], ctx, plan.starts, parents, max_len, most, out=att.view(T, cfg.heads, D),
                           workspace=self.ws)
            quantize_rows_planes(att, qa, qs, P)
            self._product(qa, qs, ("wo",), l, [x], SEM_ACCUMULATE)
            rms_norm_i8_planes(x, t["post_norm"][l], t["post_norm_s"][l], ng, eps, qh, qs, P)
            self._product(qh, qs, ("wg", "wu"), l, [gate, up])
            swiglu_(gate, up)
            quantize_rows_planes(gate, qi, qs, P)
            self._product(qi, qs, ("wd",), l, [x], SEM_ACCUMULATE)

    def _pass(self, trees, rows, top_k, positions):
        """All nodes of `trees` {request: (tokens, parents)} through the model; log-probabilities of
        the greedy choices at the nodes `rows` (of all, packed in request order).  Leaves the
        drafts' keys and values in the cache.  (greedy ids, TokenLogprobs, plan, lengths on the
        device and the host, positions by request)"""
        tokens, parents, pos, counts = [], [], {}, [0] * self.S
        for s in sorted(trees):
            if not 0 <= s < self.S:
                raise QvlError(f"no request {s}")
            toks, par = trees[s]
            depth = check_tree(toks, par, self.cfg.vocab)
            tokens += toks
            parents += par
            counts[s] = len(toks)
            own = positions.get(s) if positions else None
            if own is None:
                own = [[self.next_pos[s] + d for d in depth]] * self.n_axes
            pos[s] = self._own_positions(s, own, len(toks))
        T = len(tokens)
        if not 1 <= T <= self.max_tokens:
            raise QvlError(f"a pass takes 1 to {self.max_tokens} tokens, got {T}")
        after = [n + c for n, c in zip(self.lengths, counts)]
        self._check_room(after)
        # one upload: tokens, parents, positions, lengths before and after
        host = np.concatenate([tokens, parents, np.concatenate(list(pos.values()), 1).reshape(-1), self.lengths,
                               after]).astype(np.int32)
        up = torch.from_numpy(host).to(self.device)
        tok, par, dpos, old, new = torch.split(up, [T, T, self.n_axes * T, self.S, self.S])
        plan = self._plan(old, new, self.free_count, T, "grow")
        x = self.x[:T]
        t, cfg = self.w.t, self.cfg
        embedding_lookup_i8(t["embed"], t["embed_s"], tok, x)
        self._layers(x, T, plan, dpos.view(self.n_axes, T), old, par, max(after), max(counts))
        if rows is not None:
            x = x[torch.tensor(rows, device=self.device)]
        R, H = x.shape
        qh, qs = self.q16.view(-1)[:R * H].view(R, H), self.qs[:R]
        rms_norm_i8_planes(x, t["final_norm"], t["final_norm_s"], cfg.norm_group, cfg.eps, qh, qs, self.planes, out=x,
                           inplace_form=True)
        self.logits = torch.empty((R, cfg.vocab), dtype=torch.float32, device=self.device)
        self._product(qh, qs, ("embed",), None, [self.logits])
        greedy = greedy_decode(self.logits)
        scores = token_logprobs(self.logits, greedy, top_k)
        return greedy, scores, plan, new, after, pos

    def _keep(self, plan, new, after, lengths) -> None:
        """The requests' lengths after a pass; pages past them go back to the pool."""
        if lengths != after:
            kept = torch.tensor(lengths, dtype=torch.int32, device=self.device)
            plan = self._plan(new, kept, plan.free_count, 0, "shrink")
        self.free_count = plan.free_count.clone()
        self.lengths = lengths

    def extend(self, prompts: dict, positions: dict | None = None) -> dict:
        """Appends prompts {request: tokens} and returns {request: next greedy token}.  A pass
        takes up to 256 tokens of each request, a chain each; positions: {request: [axes,
        len(prompt)]}.  All of it is checked first: a call that is refused leaves the requests as they were."""
        prompts = {s: list(map(int, p)) for s, p in prompts.items()}
        positions, after = dict(positions or {}), list(self.lengths)
        for s, p in prompts.items():
            if not 0 <= s < self.S:
                raise QvlError(f"no request {s}")
            if not p:
                raise QvlError("an empty prompt")
            if min(p) < 0 or max(p) >= self.cfg.vocab:
                raise QvlError("a token of a prompt lies outside the vocabulary")
            after[s] += len(p)
            text = [range(self.next_pos[s], self.next_pos[s] + len(p))] * self.n_axes
            positions[s] = self._own_positions(s, positions.get(s, text), len(p))
        self._check_room(after)
        at, last = {s: 0 for s in prompts}, {}
        while any(at[s] < len(prompts[s]) for s in at):
            trees, where, ends, room = {}, {}, [], self.max_tokens
            for s in sorted(prompts):
                n = min(len(prompts[s]) - at[s], MAX_NODES, room)
                if n <= 0:
                    continue
                room -= n
                trees[s] = (prompts[s][at[s]:at[s] + n], list(range(-1, n - 1)))
                where[s] = positions[s][:, at[s]:at[s] + n]
                at[s] += n
                ends.append(self.max_tokens - room - 1)
            greedy, _, plan, new, after, pos = self._pass(trees, ends, 0, where)
            self._keep(plan, new, after, after)
            for s, own in pos.items():
                self.next_pos[s] = max(self.next_pos[s], int(own.max()) + 1)
            last.update(zip(sorted(trees), greedy.tolist()))
        return last

    def verify(self, trees: dict, top_k: int = 0, positions: dict | None = None) -> dict:
        """One pass over drafted trees {request: (tokens, parents)}: node 0 is the request's last
        chosen token, not yet in the cache.  Returns {request: Accepted} and keeps
        the accepted nodes' keys and values."""
        greedy, scores, plan, new, after, pos = self._pass(trees, None, top_k, positions)
        ids = greedy.tolist()
        lp, ent = scores.logprobs.cpu().numpy(), scores.entropy.cpu().numpy()
        top_ids, top_lp = scores.top_ids.cpu().numpy(), scores.top_logprobs.cpu().numpy()
        got, lengths, next_pos, moves, first = {}, list(after), list(self.next_pos), [], 0
        for s in sorted(trees):
            tokens, parents = trees[s]
            path = accepted_path(tokens, parents, ids[first:first + len(tokens)])
            rows = [first + p for p in path]
            got[s] = Accepted([ids[r] for r in rows], lp[rows], ent[rows], top_ids[rows], top_lp[rows])
            lengths[s] = self.lengths[s] + len(path)
            next_pos[s] = max(next_pos[s], int(pos[s][:, path].max()) + 1)
            moves += [(r, first + i) for i, r in enumerate(rows) if r != first + i]
            first += len(tokens)
        if moves:
            # the path's keys and values lie side by side from now on
            src, dst = plan.slots[torch.tensor(moves, device=self.device).t()].long()
            P = self.page_size
            for c in (self.k_all, self.v_all):
                c[:, dst // P, :, dst % P] = c[:, src // P, :, src % P]
        self._keep(plan, new, after, lengths)
        self.next_pos = next_pos
        return got

    def release(self, requests) -> None:
        """Ends requests; their pages go back to the pool."""
        lengths = [0 if s in set(requests) else n for s, n in enumerate(self.lengths)]
        old, new = (torch.tensor(v, dtype=torch.int32, device=self.device) for v in (self.lengths, lengths))
        plan = self._plan(old, new, self.free_count, 0, "shrink")
        self.free_count = plan.free_count.clone()
        self.lengths = lengths
        self.next_pos = [p if n else 0 for p, n in zip(self.next_pos, lengths)]
