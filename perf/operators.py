"""Measured cases of the operators that serve drafted (speculative) and multimodal tokens over the paged cache:

=================  =====================================================================================
``pages``          ``plan_pages``: page tables and slot maps from request lengths, on the GPU
``norm_rope``      ``qknorm_mrope_kv_append``: norms of query and key heads, rotary positions with several
                   axes, keys and values written to their cache slots
``tree``           ``tree_attention``: attention of a tree of drafted tokens over the cache
``logprobs``       ``token_logprobs``: log-probabilities of given tokens, entropy and top alternatives
=================  =====================================================================================

``run`` computes a case in its plain form (elementary torch operations, fp32) or, with ``own`` true, with the
package's operators; ``exact`` computes it from the definition in 64 bits.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
_MAX_POS = 40960          # rows of the rotary table
_THETA = 5e6


def _qvl():
    """The package (its folder's name is no identifier), imported as ``qvl_b200``."""
    m = sys.modules.get("qvl_b200")
    if m is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3-vl-2b-inference_b200")
        spec = importlib.util.spec_from_file_location("qvl_b200", os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        m = importlib.util.module_from_spec(spec)
        sys.modules["qvl_b200"] = m
        spec.loader.exec_module(m)
    return m


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one request, one token per step, after an image prompt: nothing but latency
        dict(name="tree_one_token", op="tree", seqs=1, nodes=1, ctx=452, ragged=False, heads=16, kv_heads=8, dim=128,
             page=64, dtype="fp32", cache="fp16"),
        # one interactive request with a drafted tree of an odd size, in the decoder's types
        dict(name="tree_one_request", op="tree", seqs=1, nodes=27, ctx=2011, ragged=False, heads=16, kv_heads=8, dim=128,
             page=64, dtype="fp32", cache="fp16"),
        # a serving batch with small trees, every request at another length, in the decoder's types
        dict(name="tree_batch", op="tree", seqs=32, nodes=16, ctx=4096, ragged=True, heads=16, kv_heads=8, dim=128,
             page=64, dtype="fp32", cache="fp16"),
        # long documents with large trees, half precision
        dict(name="tree_long", op="tree", seqs=16, nodes=64, ctx=32768, ragged=True, heads=16, kv_heads=8, dim=128,
             page=64, dtype="fp16", cache="fp16"),
        # a bf16 cache, small heads, four query heads to a key head, small pages
        dict(name="tree_bf16_d64", op="tree", seqs=12, nodes=33, ctx=6000, ragged=True, heads=32, kv_heads=8, dim=64,
             page=16, dtype="bf16", cache="bf16"),
        # the drafted tokens of one request, on their way into one layer's cache (INT8 norm weights)
        dict(name="norm_rope_draft", op="norm_rope", tokens=27, heads=16, kv_heads=8, dim=128, page=64, dtype="fp32",
             cache="fp16", weights="int8", fused=False),
        # prompts with images, packed, in the decoder's types
        dict(name="norm_rope_prompt", op="norm_rope", tokens=8200, heads=16, kv_heads=8, dim=128, page=64, dtype="fp32",
             cache="fp16", weights="int8", fused=False),
        # the same work in bf16 as rows of one fused projection, float norm weights
        dict(name="norm_rope_fused_bf16", op="norm_rope", tokens=2049, heads=32, kv_heads=8, dim=64, page=16,
             dtype="bf16", cache="bf16", weights="float", fused=True),
        # a decode batch that drafts a tree each: a few pages change hands
        dict(name="pages_draft", op="pages", seqs=64, page=64, max_pages=128, old=4096, new=32, shrink=0.25),
        # a large server's step: prompts arrive, finished requests hand their pages back
        dict(name="pages_prompts", op="pages", seqs=2048, page=16, max_pages=512, old=4096, new=512, shrink=0.2),
        # a small batch of drafted tokens is scored, with the alternatives that a sampler wants
        dict(name="logprobs_draft", op="logprobs", rows=27, vocab=151936, dtype="fp32", top_k=20, masked=False),
        # a prompt is scored token by token
        dict(name="logprobs_prompt", op="logprobs", rows=1024, vocab=151936, dtype="bf16", top_k=5, masked=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "norm_rope", "pages", "logprobs"])
    if op == "tree":
        cache = rng.choice(["fp16", "fp16", "bf16"])
        kv_heads, group = rng.choice([2, 4, 8]), rng.choice([1, 2, 4, 7])
        c = dict(op=op, seqs=_log_int(rng, 1, 48), nodes=_log_int(rng, 1, 128), ctx=_log_int(rng, 1, 32768),
                 ragged=rng.random() < 0.7, heads=kv_heads * group, kv_heads=kv_heads, dim=rng.choice([64, 128]),
                 page=rng.choice([16, 32, 64, 128]), dtype="bf16" if cache == "bf16" else rng.choice(["fp32", "fp16"]),
                 cache=cache)
        most = work(listed()[3])
        while True:       # no more than the largest listed one
            w = work(c)
            if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
                return c
            c["ctx"], c["nodes"] = max(1, c["ctx"] // 2), max(1, (2 * c["nodes"]) // 3)
    if op == "norm_rope":
        dtype = rng.choice(["fp32", "fp16", "bf16"])
        kv_heads, dim = rng.choice([2, 4, 8]), rng.choice([64, 128])
        return dict(op=op, tokens=_log_int(rng, 1, 8192), heads=kv_heads * rng.choice([1, 2, 4]), kv_heads=kv_heads,
                    dim=dim, page=rng.choice([16, 32, 64, 128]), dtype=dtype, cache="bf16" if dtype == "bf16" else "fp16",
                    weights=rng.choice(["int8", "float"]), fused=rng.random() < 0.5)
    if op == "pages":
        return dict(op=op, seqs=_log_int(rng, 1, 2048), page=rng.choice([16, 32, 64, 128]), max_pages=256,
                    old=_log_int(rng, 1, 2048), new=_log_int(rng, 1, 512), shrink=rng.choice([0.0, 0.2, 0.5]))
    rows = _log_int(rng, 1, 1024)
    vocab = _log_int(rng, 1000, 151936)
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    if dtype == "fp32":
        rows = min(rows, 512)
    return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top_k=rng.randint(0, 20), masked=rng.random() < 0.3)


def _spread(n, lo, hi, ragged, turn):
    """n sizes in [lo, hi], all hi unless ragged: they go by the case alone, so that its work does."""
    if not ragged:
        return np.full(n, hi, np.int64)
    f = np.mod((np.arange(n) + 1) * turn, 1.0)
    return (lo + np.floor(f * (hi - lo + 1))).astype(np.int64)


def _tree_sizes(c):
    ctx = _spread(c["seqs"], max(0, c["ctx"] // 8), c["ctx"], c["ragged"], 0.6180339887)
    nodes = _spread(c["seqs"], max(1, c["nodes"] // 2), c["nodes"], c["ragged"], 0.7548776662)
    return ctx, nodes


def work(c):
    """The bytes and operations that a pass cannot do without: each input read once, each output written once."""
    if c["op"] == "tree":
        ctx, nodes = _tree_sizes(c)
        e, ec = _BYTES[c["dtype"]], _BYTES[c["cache"]]
        seen = int((ctx + nodes).sum())
        rows = int(nodes.sum())
        kv = seen * c["kv_heads"] * c["dim"] * 2 * ec
        return {"bytes": kv + 2 * rows * c["heads"] * c["dim"] * e + 4 * int(-(-(ctx + nodes) // c["page"]).sum()),
                "flops": 4 * int((nodes * (ctx + 1)).sum()) * c["heads"] * c["dim"]}
    if c["op"] == "norm_rope":
        e, ec = _BYTES[c["dtype"]], _BYTES[c["cache"]]
        per = (2 * c["heads"] + 2 * c["kv_heads"]) * c["dim"] * e + 2 * c["kv_heads"] * c["dim"] * ec + 16
        return {"bytes": c["tokens"] * per, "flops": c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"] * 7}
    if c["op"] == "pages":
        old, new = _page_sizes(c)
        tokens = int(np.maximum(new - old, 0).sum())
        moved = int(np.abs(-(-new // c["page"]) - -(-old // c["page"])).sum())
        return {"bytes": 12 * tokens + 12 * c["seqs"] + 8 * moved, "flops": 0}
    e = _BYTES[c["dtype"]]
    return {"bytes": c["rows"] * (c["vocab"] * e + 12 + 8 * c["top_k"]), "flops": 5 * c["rows"] * c["vocab"]}


def _page_sizes(c):
    """Lengths before and after a step: most requests grow, some take drafted tokens back, some are done."""
    old = _spread(c["seqs"], 0, c["old"], True, 0.6180339887)
    grow = _spread(c["seqs"], 0, c["new"], True, 0.7548776662)
    f = np.mod((np.arange(c["seqs"]) + 1) * 0.5698402910, 1.0)
    back = f < c["shrink"]
    done = f < c["shrink"] / 4
    new = np.where(done, 0, np.where(back, np.maximum(0, old - grow), old + grow))
    return old, new


# ------------------------------------------------------------------------------------------------ inputs
def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)

    def i32(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()

    def normal(shape, dtype, s=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * s).to(dtype)

    return {"tree": _prepare_tree, "norm_rope": _prepare_norm_rope, "pages": _prepare_pages,
            "logprobs": _prepare_logprobs}[c["op"]](dict(c), g, r, i32, normal)


def _cache(pages, c, g):
    shape = (pages, c["kv_heads"], c["page"], c["dim"])
    return [torch.randn(shape, generator=g, device="cuda", dtype=_DTYPES[c["cache"]]) for _ in range(2)]


def _prepare_tree(c, g, r, i32, normal):
    ctx, nodes = _tree_sizes(c)
    S, P = c["seqs"], c["page"]
    maxp = int(-(-(ctx + nodes).max() // P))
    starts = np.concatenate([[0], np.cumsum(nodes)])
    # parents: a drafter's tree, a node's parent among the few nodes before it
    parents = np.concatenate([np.maximum(-1, np.arange(n) - 1 - r.integers(0, 4, n)) for n in nodes])
    k, v = _cache(S * maxp, c, g)
    T = int(starts[-1])
    dt = _DTYPES[c["dtype"]]
    return dict(c=c, q=normal((T, c["heads"], c["dim"]), dt), k=k, v=v, page_table=i32(r.permutation(S * maxp)).view(S, maxp),
                ctx_lens=i32(ctx), starts=i32(starts), parents=i32(parents), max_ctx=int((ctx + nodes).max()),
                max_nodes=int(nodes.max()), out=torch.empty((T, c["heads"], c["dim"]), dtype=dt, device="cuda"))


def _axes(dim):
    """The position axis (time, height, width) of each frequency: sections of 24, 20, 20 for 64 frequencies, interleaved."""
    sec = (24, 20, 20) if dim == 128 else (12, 10, 10)
    a = np.zeros(dim // 2, np.int32)
    for axis in (1, 2):
        a[axis:3 * sec[axis]:3] = axis
    return a


def _positions(T, r):
    """Three-axis positions of packed prompts: stretches of text, and images as grids of height x width."""
    cols, n, at = [], 0, 0
    while n < T:
        if r.random() < 0.5:
            m = int(r.integers(5, 200))
            cols.append(np.tile(at + np.arange(m), (3, 1)))
            at += m
        else:
            h, w = int(r.integers(2, 20)), int(r.integers(2, 20))
            m = h * w
            y, x = np.divmod(np.arange(m), w)
            cols.append(np.stack([np.full(m, at), at + y, at + x]))
            at += max(h, w)
        n += m
        if at > 16000:
            at = 0
    return np.concatenate(cols, axis=1)[:, :T]


def _prepare_norm_rope(c, g, r, i32, normal):
    T, NH, NKV, D, P = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    dt = _DTYPES[c["dtype"]]
    if c["fused"]:
        qkv = normal((T, (NH + 2 * NKV) * D), dt, 1.5)
        q, k, v = (x.view(T, -1, D) for x in qkv.split([NH * D, NKV * D, NKV * D], dim=1))
    else:
        q, k, v = normal((T, NH, D), dt, 1.5), normal((T, NKV, D), dt, 1.5), normal((T, NKV, D), dt)
    pages = T // P + 2
    perm = r.permutation(pages)
    at = np.arange(T) + int(r.integers(0, P))
    slots = perm[at // P] * P + at % P
    if T > 16:
        slots[T - T // 16:] = -1            # the padding of a captured graph
    kc, vc = _cache(pages, c, g)
    inv = _THETA ** -(np.arange(0, D, 2) / D)
    ang = np.arange(_MAX_POS)[:, None] * inv[None]
    if c["weights"] == "int8":
        norms = [(i32(r.integers(40, 128, D)).to(torch.int8), torch.rand(1, generator=g, device="cuda") * 0.01 + 0.008, D)
                 for _ in range(2)]
    else:
        norms = [(1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt) for _ in range(2)]
    return dict(c=c, q=q, k=k, v=v, k_pages=kc, v_pages=vc, slots=i32(slots), positions=i32(_positions(T, r)),
                axes=i32(_axes(D)), cos=torch.from_numpy(np.cos(ang)).float().cuda(),
                sin=torch.from_numpy(np.sin(ang)).float().cuda(), q_norm=norms[0], k_norm=norms[1], eps=1e-6,
                page_table=torch.arange(pages, dtype=torch.int32, device="cuda").view(1, pages),
                out=torch.empty((T, NH, D), dtype=dt, device="cuda"))


def _prepare_pages(c, g, r, i32, normal):
    old, new = _page_sizes(c)
    # a seed has its own order of requests
    order = r.permutation(c["seqs"])
    old, new = old[order], new[order]
    P, maxp, S = c["page"], c["max_pages"], c["seqs"]
    have, need = -(-old // P), -(-new // P)
    used = int(have.sum())
    total = used + int(np.maximum(need - have, 0).sum()) + 37
    pages = r.permutation(total)
    table = np.full((S, maxp), -1, np.int32)
    at = np.concatenate([[0], np.cumsum(have)])
    for s in range(S):
        table[s, :have[s]] = pages[at[s]:at[s + 1]]
    free = np.zeros(total, np.int32)
    free[:total - used] = pages[used:]
    tokens = -(-int(np.maximum(new - old, 0).sum()) // 64) * 64
    return dict(c=c, old=i32(old), new=i32(new), page_table=i32(table), free=i32(free), free_count=i32([total - used]),
                tokens=max(64, tokens))


def _prepare_logprobs(c, g, r, i32, normal):
    T, V = c["rows"], c["vocab"]
    x = torch.randn((T, V), generator=g, device="cuda") * 2.5
    x += 6.0 * (torch.rand((T, V), generator=g, device="cuda") < 20.0 / V)      # a few likely tokens
    if c["masked"]:
        x.masked_fill_(torch.rand(V, generator=g, device="cuda") < 0.01, -math.inf)
    tokens = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
    tokens = torch.where(torch.rand(T, generator=g, device="cuda") < 0.5, x.argmax(1).to(torch.int32), tokens)
    return dict(c=c, logits=x.to(_DTYPES[c["dtype"]]), tokens=tokens)


# ------------------------------------------------------------------------------------------------ passes
def run(st):
    op = st["c"]["op"]
    if own:
        return {"tree": _own_tree, "norm_rope": _own_norm_rope, "pages": _own_pages, "logprobs": _own_logprobs}[op](st)
    return {"tree": _plain_tree, "norm_rope": _plain_norm_rope, "pages": _plain_pages, "logprobs": _plain_logprobs}[op](st)


def _kv(st, k, v):
    """The program's cache object around its page tensors, made once."""
    kv = st.get("kv")
    if kv is None:
        c, pt = st["c"], st["page_table"]
        kv = st["kv"] = _qvl().PagedKV(pt.shape[0], pt.shape[1] * c["page"], c["heads"], c["kv_heads"], c["dim"], c["page"],
                                       max_pos=_MAX_POS, page_table=pt, k=k, v=v)
    return kv


def _own_tree(st):
    return _qvl().tree_attention(st["q"], _kv(st, st["k"], st["v"]), st["ctx_lens"], st["starts"], st["parents"],
                                 st["max_ctx"], st["max_nodes"], out=st["out"])


def _own_norm_rope(st):
    kv = _kv(st, st["k_pages"], st["v_pages"])
    q = _qvl().qknorm_mrope_kv_append(st["q"], st["k"], st["v"], kv, st["slots"], st["positions"], st["axes"], st["cos"],
                                      st["sin"], st["q_norm"], st["k_norm"], st["eps"], out=st["out"])
    return {"q": q, "k_pages": kv.k, "v_pages": kv.v}


def _own_pages(st):
    p = _qvl().plan_pages(st["old"], st["new"], st["page_table"], st["free"], st["free_count"], st["c"]["page"],
                          st["tokens"], plan=st.get("plan"))
    st["plan"] = p
    return {"table": st["page_table"], "free": st["free"], "free_count": p.free_count, "missing": p.missing,
            "starts": p.starts, "seq_ids": p.seq_ids, "positions": p.positions, "slots": p.slots}


def _own_logprobs(st):
    r = _qvl().token_logprobs(st["logits"], st["tokens"], st["c"]["top_k"], out=st.get("out"))
    st["out"] = r
    return {"logprobs": r.logprobs, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}


def _plain_tree(st):
    c = st["c"]
    S, P, NKV, D = c["seqs"], c["page"], c["kv_heads"], c["dim"]
    G, n = c["heads"] // NKV, st["max_nodes"]
    pt = st["page_table"].long()
    L = pt.shape[1] * P
    K = st["k"][pt].transpose(1, 2).reshape(S, NKV, L, D).float()
    V = st["v"][pt].transpose(1, 2).reshape(S, NKV, L, D).float()
    ctx, starts, parents = st["ctx_lens"].long(), st["starts"].long(), st["parents"].long()
    row = torch.arange(st["q"].shape[0], device="cuda")
    s = torch.searchsorted(starts[1:], row, right=True)
    node = row - starts[s]
    q = torch.zeros((S, n, c["heads"], D), device="cuda")
    q[s, node] = st["q"].float()
    q = q.view(S, n, NKV, G, D).permute(0, 2, 3, 1, 4).reshape(S, NKV, G * n, D)
    # ancestors: the inverse of (1 - parent) is the sum of the parent matrix's powers
    par = torch.zeros((S, n, n + 1), device="cuda")
    par[s, node, torch.where(parents < 0, n, parents)] = 1.0
    eye = torch.eye(n, device="cuda").expand(S, n, n)
    anc = torch.linalg.solve_triangular(eye - par[:, :, :n], eye, upper=False, unitriangular=True) > 0.5
    t = torch.arange(L, device="cuda")
    j = t[None] - ctx[:, None]                                       # the node at cache position t
    tree = torch.gather(anc, 2, j.clamp(0, n - 1)[:, None, :].expand(S, n, L)) & ((j >= 0) & (j < n))[:, None, :]
    seen = ((j < 0)[:, None, :] | tree)[:, None, None]               # [S, 1, 1, n, L]
    sc = torch.matmul(q, K.transpose(2, 3)) * (D ** -0.5)
    del K
    sc = sc.view(S, NKV, G, n, L).masked_fill_(~seen, -math.inf)
    sc -= sc.amax(-1, keepdim=True).clamp_min(-3e38)                 # a padded node sees nothing
    sc.exp_()
    sc /= sc.sum(-1, keepdim=True).clamp_min(1e-37)
    o = torch.matmul(sc.view(S, NKV, G * n, L), V).view(S, NKV, G, n, D).permute(0, 3, 1, 2, 4).reshape(S, n, c["heads"], D)
    return o[s, node].to(st["q"].dtype)


def _plain_norm(x, w, eps):
    x = x.float()
    if isinstance(w, tuple):
        w = w[0].float() * w[1].repeat_interleave(w[2])
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()


def _plain_norm_rope(st):
    c = st["c"]
    P, D = c["page"], c["dim"]
    q, k = _plain_norm(st["q"], st["q_norm"], st["eps"]), _plain_norm(st["k"], st["k_norm"], st["eps"])
    at = st["positions"].long()[st["axes"].long()].t()               # [T, D/2]: each frequency's position
    f = torch.arange(D // 2, device="cuda")[None]
    cos, sin = st["cos"][at, f][:, None], st["sin"][at, f][:, None]

    def rotate(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    slots = st["slots"].long()
    use = torch.where(slots >= 0, torch.arange(len(slots), device="cuda"), 0)      # padding writes token 0's row once more
    to = slots[use]
    st["k_pages"].transpose(1, 2)[to // P, to % P] = rotate(k)[use].to(st["k_pages"].dtype)
    st["v_pages"].transpose(1, 2)[to // P, to % P] = st["v"][use].float().to(st["v_pages"].dtype)
    return {"q": rotate(q).to(st["q"].dtype), "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _plain_pages(st):
    P = st["c"]["page"]
    table, free = st["page_table"], st["free"]
    S, maxp = table.shape
    old, new, fc = st["old"].long(), st["new"].long(), st["free_count"].long()
    have, need = ((old + P - 1) // P).clamp(max=maxp)[:, None], ((new + P - 1) // P).clamp(max=maxp)[:, None]
    col = torch.arange(maxp, device="cuda")[None]
    give, take = ((col >= need) & (col < have)).view(-1), ((col >= have) & (col < need)).view(-1)
    ext = torch.cat([free, torch.zeros(S * maxp + 1, dtype=torch.int32, device="cuda")])
    ext[torch.where(give, fc + give.cumsum(0) - 1, len(ext) - 1)] = table.view(-1)
    R = give.sum()
    at = fc + R - take.cumsum(0)
    table = torch.where(take, torch.where(at >= 0, ext[at.clamp_min(0)], -1), table.view(-1)).view(S, maxp)
    left = (fc + R - take.sum()).clamp_min(0)
    i = torch.arange(len(free), device="cuda")
    free = torch.where((i >= fc) & (i < left), ext[:len(free)], free)
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), (new - old).clamp_min(0).cumsum(0)])
    t = torch.arange(st["tokens"], device="cuda")
    s = torch.searchsorted(starts[1:], t, right=True)
    there = s < S
    s = s.clamp_max(S - 1)
    pos = old[s] + t - starts[s]
    page = table[s, (pos // P).clamp(0, maxp - 1)]
    ok = there & (pos // P < maxp) & (page >= 0)
    out = {"table": table, "free": free, "free_count": left, "missing": (there & ~ok).sum().view(1), "starts": starts,
           "seq_ids": torch.where(there, s, -1), "positions": torch.where(there, pos, -1),
           "slots": torch.where(ok, page * P + pos % P, -1)}
    return {k: x.to(torch.int32) for k, x in out.items()}


def _plain_logprobs(st):
    k = st["c"]["top_k"]
    x = st["logits"].float()
    top = torch.sort(x, dim=1, descending=True, stable=True)
    ids, vals = top.indices[:, :k].to(torch.int32), top.values[:, :k].contiguous()
    m = top.values[:, :1].clone()
    del top
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    ent = lse[:, 0] - torch.where(e > 0, e * x, 0.0).sum(1) / z[:, 0]
    return {"logprobs": x.gather(1, st["tokens"].long()[:, None])[:, 0] - lse[:, 0], "entropy": ent, "top_ids": ids,
            "top_logprobs": vals - lse}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(c, seed):
    st = prepare(c, seed)
    return {"tree": _exact_tree, "norm_rope": _exact_norm_rope, "pages": lambda st: None,
            "logprobs": _exact_logprobs}[c["op"]](st)


def _exact_tree(st):
    """Request by request, key head by key head: a softmax over the positions that each node sees."""
    c = st["c"]
    G, P = c["heads"] // c["kv_heads"], c["page"]
    ctx, starts, parents = (st[n].tolist() for n in ("ctx_lens", "starts", "parents"))
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for s, t0 in enumerate(starts[:-1]):
        n = starts[s + 1] - t0
        hidden = torch.ones((n, ctx[s] + n), dtype=torch.bool)
        hidden[:, :ctx[s]] = False
        for i in range(n):
            j = i
            while j >= 0:
                hidden[i, ctx[s] + j] = False
                j = parents[t0 + j]
        hidden = hidden.cuda()[:, None]
        pages = st["page_table"][s, :-(-(ctx[s] + n) // P)].long()
        for h in range(c["kv_heads"]):
            K = st["k"][pages, h].reshape(-1, c["dim"])[:ctx[s] + n].double()
            V = st["v"][pages, h].reshape(-1, c["dim"])[:ctx[s] + n].double()
            w = torch.einsum("igd,td->igt", st["q"][t0:t0 + n, h * G:(h + 1) * G].double(), K) / math.sqrt(c["dim"])
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            out[t0:t0 + n, h * G:(h + 1) * G] = torch.einsum("igt,td->igd", w, V)
    return out


def _exact_norm_rope(st):
    """Pairs (i, i + D/2) as complex numbers, turned by their axis's angle."""
    c = st["c"]
    P, D = c["page"], c["dim"]
    pos, axes = st["positions"].double(), st["axes"].tolist()
    turn = torch.stack([torch.complex(st["cos"].double()[pos[a].long(), i], st["sin"].double()[pos[a].long(), i])
                        for i, a in enumerate(axes)], -1)[:, None]

    def of(x, w):
        x = x.double()
        w = (w[0].double() * w[1].double()) if isinstance(w, tuple) else w.double()
        x = x * torch.rsqrt(torch.square(x).sum(-1, keepdim=True) / D + st["eps"]) * w
        z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    kc, vc = st["k_pages"].double(), st["v_pages"].double()
    ok = torch.nonzero(st["slots"] >= 0)[:, 0]
    to = st["slots"][ok].long()
    kc[to // P, :, to % P] = of(st["k"], st["k_norm"])[ok]
    vc[to // P, :, to % P] = st["v"][ok].double()
    return {"q": of(st["q"], st["q_norm"]), "k_pages": kc, "v_pages": vc}


def _exact_logprobs(st):
    """Row by row; the order of the alternatives is the logits' own, so only their values are given."""
    k, lp, ent, top = st["c"]["top_k"], [], [], []
    for x, t in zip(st["logits"], st["tokens"].tolist()):
        x = torch.log_softmax(x.double(), 0)
        lp.append(x[t])
        p = x[x > -math.inf]
        ent.append(-(p.exp() * p).sum())
        top.append(torch.topk(x, k).values)
    return {"logprobs": torch.stack(lp), "entropy": torch.stack(ent), "top_ids": None, "top_logprobs": torch.stack(top)}
