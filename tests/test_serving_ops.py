"""The operators that serve drafted and multimodal tokens over the paged cache
(plan_pages, qknorm_mrope_kv_append, tree_attention, token_logprobs) against
plain implementations in 64 bits, and what they refuse.

Tolerances follow from the arithmetic, u = 2^-24 (an fp32 rounding), r the
output type's rounding (0, 2^-11, 2^-8):
  norm + rotation  the sum of squares is at most 21 additions deep, each factor
                   and product is one rounding more: 32 u (|a c| + |b s|) + r |y|
  tree attention   a score is off by at most d = (D + 4) 2u |scale| sum|q k|, a weight by
                   as much relatively, a weighted sum by the depth of its
                   additions: (2 d + (128 + tiles) 2u + r) sum p|v|
  log-probability  Z by its additions' depth (a thread's share, and 20 for the joins)
                   and the exponent's rounding: (n + 60) u, lse by 4 u |lse| more
"""
import ctypes

import numpy as np
import pytest
import torch

from conftest import import_qvl

U = 2.0 ** -24
R = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ plan_pages
def plan_oracle(old, new, table, free, fc, P, max_tokens):
    """Request by request, as the header says it."""
    S, maxp = table.shape
    table, stack = table.copy(), list(free[:fc])
    pages = lambda n: min(-(-max(n, 0) // P), maxp)  # noqa: E731
    for s in range(S):
        stack += [table[s, c] for c in range(pages(new[s]), pages(old[s]))]
    for s in range(S):
        for c in range(pages(old[s]), pages(new[s])):
            table[s, c] = stack.pop() if stack else -1
    out = free.copy()
    out[fc:len(stack)] = stack[fc:]
    starts, rows, missing = [0], [], 0
    for s in range(S):
        o, n = max(old[s], 0), max(new[s], 0)
        for pos in range(o, n):
            page = table[s, pos // P] if pos // P < maxp else -1
            missing += page < 0
            rows.append((s, pos, page * P + pos % P if page >= 0 else -1))
        starts.append(len(rows))
    rows = (rows + [(-1, -1, -1)] * max_tokens)[:max_tokens]
    return table, out, len(stack), missing, starts, np.array(rows).reshape(-1, 3).T


def plan_case(seed, S, P, maxp, old_max, grow, slack, shrink=0.3):
    r = np.random.default_rng(seed)
    old = np.minimum(r.integers(0, old_max + 1, S), maxp * P)
    new = old + r.integers(0, grow + 1, S)
    back = r.random(S) < shrink
    new[back] = old[back] - r.integers(0, old_max + 1, int(back.sum()))
    have = -(-old // P)
    total = int(have.sum()) + max(slack, 0) + 1
    pages = r.permutation(total).astype(np.int32)
    table = np.full((S, maxp), -1, np.int32)
    at = 0
    for s in range(S):
        table[s, :have[s]] = pages[at:at + have[s]]
        at += have[s]
    free = np.zeros(total, np.int32)
    fc = max(0, slack)
    free[:fc] = pages[at:at + fc]
    return old, new, table, free, fc


def check_plan(qvl, old, new, table, free, fc, P, max_tokens):
    dt, df = i32(table), i32(free)
    p = qvl.plan_pages(i32(old), i32(new), dt, df, i32([fc]), P, max_tokens)
    wt, wf, wc, wm, ws, rows = plan_oracle(old, new, table, free, fc, P, max_tokens)
    assert int(p.free_count) == wc and int(p.missing) == wm
    np.testing.assert_array_equal(p.starts.cpu(), ws)
    for got, want in zip((p.seq_ids, p.positions, p.slots), rows):
        np.testing.assert_array_equal(got.cpu(), want)
    np.testing.assert_array_equal(dt.cpu(), wt)
    np.testing.assert_array_equal(df.cpu(), wf)


@pytest.mark.gpu
@pytest.mark.parametrize("S,P,maxp,old_max,grow,slack", [
    (1, 16, 4, 40, 1, 3), (1, 1, 9, 4, 5, 20), (3, 16, 8, 100, 20, 4), (64, 64, 16, 900, 30, 200), (65, 48, 7, 330, 3, 0),
    (257, 16, 40, 500, 120, 900), (1025, 32, 12, 300, 40, 100), (33, 16, 3, 48, 30, 100)])
@pytest.mark.parametrize("seed", [0, 1])
def test_plan_pages(qvl, cuda, S, P, maxp, old_max, grow, slack, seed):
    old, new, table, free, fc = plan_case(seed, S, P, maxp, old_max, grow, slack)
    total = int(np.maximum(np.maximum(new, 0) - old, 0).sum())
    for max_tokens in {total, total + 37, max(0, total - 5)}:
        check_plan(qvl, old, new, table, free, fc, P, max_tokens)


@pytest.mark.gpu
def test_plan_pages_edges(qvl, cuda):
    z = np.zeros(4, np.int64)
    table = np.full((4, 2), -1, np.int32)
    check_plan(qvl, z, z, table, np.arange(5, dtype=np.int32), 5, 16, 8)          # nothing to do
    check_plan(qvl, z, z + 16, table, np.arange(5, dtype=np.int32), 0, 16, 64)    # an empty pool
    check_plan(qvl, z, z + 33, table, np.arange(9, dtype=np.int32), 9, 16, 200)   # wider than the table
    check_plan(qvl, z - 3, z - 1, table, np.arange(9, dtype=np.int32), 9, 16, 8)  # negative lengths count as 0
    old, new, table, free, fc = plan_case(3, 16384, 16, 3, 40, 3, 9000)           # the most requests
    check_plan(qvl, old, new, table, free, fc, 16, 60000)


@pytest.mark.gpu
def test_plan_pages_can_be_dropped(qvl, cuda):
    """A plan that ran out of pages leaves the pool as it was for the caller that keeps the old count."""
    old, new, table, free, fc = plan_case(7, 40, 16, 20, 200, 90, 12)
    dt, df, n = i32(table), i32(free), int(np.maximum(new - old, 0).sum())
    p = qvl.plan_pages(i32(old), i32(new), dt, df, i32([fc]), 16, n)
    assert int(p.missing) > 0
    less = np.where(new > old, old + 1, new)
    q = qvl.plan_pages(i32(old), i32(less), dt, df, i32([fc]), 16, n)
    wt, wf, wc, wm, _, rows = plan_oracle(old, less, table, free, fc, 16, n)
    assert int(q.free_count) == wc and int(q.missing) == wm
    np.testing.assert_array_equal(q.slots.cpu(), rows[2])
    for s in range(40):
        np.testing.assert_array_equal(dt.cpu()[s, :-(-max(less[s], 0) // 16)], wt[s, :-(-max(less[s], 0) // 16)])


# ------------------------------------------------------- qknorm_mrope_kv_append
def norm_rope_oracle(x, w, eps, cos, sin, ok):
    """(y, bound) in 64 bits: norm, then the turn of pairs (i, i + D/2)."""
    x = x.double()
    D = x.shape[-1]
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    a, b = x[..., :D // 2], x[..., D // 2:]
    c, s = cos[:, None].double(), sin[:, None].double()
    y = torch.cat([a * c - b * s, b * c + a * s], -1)
    m = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
    return torch.where(ok[:, None, None], y, 0.0), m


def near(got, want, mag, r, tiny=2.0 ** -24):
    d = (got.double() - want).abs()
    lim = 32 * U * mag + r * want.abs() * (1 + 2.0 ** -8) + (tiny if r else 0.0)
    assert bool((d <= lim).all()), float((d / lim.clamp_min(1e-300)).max())


def mrope_case(qvl, T, NH, NKV, D, dtype, cache, weights, fused, seed, P=16, n_axes=3, group=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    W = (NH + 2 * NKV) * D
    x = (torch.randn((T, W + 16), generator=g, device="cuda") * 3).to(dtype)[:, :W]
    q, k, v = (y.unflatten(1, (-1, D)) for y in x.split([NH * D, NKV * D, NKV * D], 1))
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pages = T // P + 3
    kc = torch.randn((pages, NKV, P, D), generator=g, device="cuda").to(cache)
    vc = torch.randn((pages, NKV, P, D), generator=g, device="cuda").to(cache)
    max_pos = 300
    kv = qvl.PagedKV(1, pages * P, NH, NKV, D, P, max_pos=max_pos, k=kc.clone(), v=vc.clone())
    slots = r.permutation(pages * P)[:T]
    pos = r.integers(0, max_pos, (n_axes, T))
    axes = torch.from_numpy(r.integers(0, n_axes, D // 2).astype(np.int32)).cuda()
    ang = np.arange(max_pos)[:, None] * (1e4 ** -(np.arange(0, D, 2) / D))[None]
    cos, sin = torch.from_numpy(np.cos(ang)).float().cuda(), torch.from_numpy(np.sin(ang)).float().cuda()
    if weights == "int8":
        gr = group or D
        norm = [(i32(r.integers(-127, 128, D)).to(torch.int8),
                 torch.rand(D // gr, generator=g, device="cuda") * 0.02 + 0.001, gr) for _ in range(2)]
        full = [w.double() * s.double().repeat_interleave(gr) for w, s, gr in norm]
    elif weights is None:
        norm, full = [None, None], [None, None]
    else:
        norm = [torch.randn(D, generator=g, device="cuda").to(weights) for _ in range(2)]
        full = norm
    return q, k, v, kv, kc, vc, slots, pos, axes, cos, sin, norm, full


def check_mrope(qvl, case, out=None):
    q, k, v, kv, kc, vc, slots, pos, axes, cos, sin, norm, full = case
    D, P = q.shape[2], kv.page_size
    q0 = q.clone()
    y = qvl.qknorm_mrope_kv_append(q, k, v, kv, i32(slots), i32(pos), axes, cos, sin, norm[0], norm[1], 1e-6, out=out)
    p = i32(pos).long()
    ok = ((p >= 0) & (p < cos.shape[0]))[axes.long()].all(0)
    f = torch.arange(D // 2, device="cuda")[None]
    at = p.clamp(0, cos.shape[0] - 1)[axes.long()].t()
    c, s = cos[at, f], sin[at, f]
    want, m = norm_rope_oracle(q0, full[0], 1e-6, c, s, ok)
    near(y, want, m, R[q.dtype])
    wk, mk = norm_rope_oracle(k, full[1], 1e-6, c, s, ok)
    wkc, wvc, mkc = kc.double(), vc.double(), torch.zeros_like(kc, dtype=torch.float64)
    sl = torch.as_tensor(slots, device="cuda").long()
    use = torch.nonzero(ok & (sl >= 0) & (sl < kc.shape[0] * P))[:, 0]
    to = sl[use]
    wkc[to // P, :, to % P] = wk[use]
    mkc[to // P, :, to % P] = mk[use]
    wvc[to // P, :, to % P] = v[use].to(kc.dtype).double()
    assert torch.equal(kv.v.double(), wvc)                    # a copy, rounded once
    near(kv.k, wkc, mkc, R[kc.dtype])
    untouched = torch.ones(kc.shape[0], P, dtype=torch.bool, device="cuda")
    untouched[to // P, to % P] = False
    assert torch.equal(kv.k.transpose(1, 2)[untouched], kc.transpose(1, 2)[untouched])
    return y


F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 27, 130])
@pytest.mark.parametrize("NH,NKV,D", [(16, 8, 128), (3, 1, 64), (7, 7, 128), (4, 2, 256)])
@pytest.mark.parametrize("dtype,cache,weights,fused", [
    (F32, F16, "int8", False), (F32, F16, None, True), (F16, F16, F16, True), (BF16, BF16, F32, True),
    (BF16, F16, BF16, False), (F32, BF16, F32, False), (F16, BF16, "int8", False)])
def test_mrope_append(qvl, cuda, T, NH, NKV, D, dtype, cache, weights, fused):
    check_mrope(qvl, mrope_case(qvl, T, NH, NKV, D, dtype, cache, weights, fused, seed=T + D))


@pytest.mark.gpu
def test_mrope_append_in_place_axes_groups(qvl, cuda):
    case = mrope_case(qvl, 19, 16, 8, 128, F32, F16, "int8", False, 5, P=48, n_axes=1, group=32)
    y = check_mrope(qvl, case, out=case[0])
    assert y.data_ptr() == case[0].data_ptr()
    check_mrope(qvl, mrope_case(qvl, 5, 2, 2, 64, F16, F16, F32, True, 6, n_axes=4))
    assert qvl.qknorm_mrope_kv_append(case[0][:0], case[1][:0], case[2][:0], case[3], i32([]), i32(np.zeros((1, 0))),
                                      case[8], case[9], case[10]).shape == (0, 16, 128)


@pytest.mark.gpu
def test_mrope_append_padding(qvl, cuda):
    """Slots outside the cache are not written; a position outside the table gives zeros and no write."""
    case = list(mrope_case(qvl, 40, 4, 2, 128, F32, F16, F32, False, 9))
    slots, pos = case[6].copy(), case[7].copy()
    slots[3:9] = [-1, -7, case[3].k.shape[0] * 16, 2 ** 31 - 1, -2 ** 31, -1]
    pos[1, 20], pos[0, 21], pos[2, 22] = -1, 300, 2 ** 31 - 1
    case[6], case[7] = slots, pos
    y = check_mrope(qvl, case)
    assert not y[20:23].any()


@pytest.mark.gpu
def test_mrope_append_is_qknorm_rope_append_on_one_axis(qvl, cuda):
    """Text tokens (all axes alike, slot of the position) get what the text operator gives them."""
    NH, NKV, D, P, n = 16, 8, 128, 64, 33
    r = np.random.default_rng(2)
    q, k, v = (torch.from_numpy(r.standard_normal((n, h, D), dtype=np.float32)).cuda() for h in (NH, NKV, NKV))
    a, b = qvl.PagedKV(1, 128, NH, NKV, D, P), qvl.PagedKV(1, 128, NH, NKV, D, P)
    w = [(i32(r.integers(-127, 128, D)).to(torch.int8), torch.rand(1, device="cuda") * 0.02) for _ in range(2)]
    from qvl_b200.decoder import rope_table
    cos, sin = (torch.from_numpy(x).cuda() for x in rope_table(128))
    pos = torch.arange(70, 70 + n, dtype=torch.int32, device="cuda")
    got = qvl.qknorm_mrope_kv_append(q, k, v, a, pos, pos.repeat(3, 1), qvl.mrope_axes((24, 20, 20)), cos, sin,
                                     (*w[0], 128), (*w[1], 128))
    want = qvl.qknorm_rope_kv_append(q.clone(), k, v, b, torch.zeros_like(pos), pos, cos, sin, *w[0], *w[1], 128, 1e-6)
    assert float((got - want).abs().max() / want.abs().max()) < 64 * U
    assert float((a.k.float() - b.k.float()).abs().max() / b.k.float().abs().max()) < 2.0 ** -10
    assert torch.equal(a.v, b.v)


def test_mrope_axes(qvl):
    a = qvl.mrope_axes((24, 20, 20), device="cpu")
    assert a.tolist() == [0, 1, 2] * 20 + [0] * 4
    assert qvl.mrope_axes((2, 3, 3), False, device="cpu").tolist() == [0, 0, 1, 1, 1, 2, 2, 2]
    with pytest.raises(qvl.QvlError):
        qvl.mrope_axes((1, 5, 2), device="cpu")


# -------------------------------------------------------------- tree_attention
def ancestors(parents, n):
    seen = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while 0 <= j:
            seen[i, j] = True
            p = int(parents[j])
            j = p if p < j else -1
    return seen


def tree_oracle(q, k, v, table, ctx, starts, parents, P, scale, max_nodes, num_pages):
    """(out, sum p|v|, score bound) in 64 bits."""
    T, NH, D = q.shape
    NKV = k.shape[1]
    G = NH // NKV
    out = torch.zeros((T, NH, D), dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    off = torch.zeros((T, NH, 1), dtype=torch.float64, device=q.device)
    cap = table.shape[1] * P
    for s in range(len(ctx)):
        t0, n = starts[s], min(starts[s + 1] - starts[s], max_nodes)
        if n <= 0:
            continue
        seen = torch.from_numpy(ancestors(parents[t0:t0 + n], n)).to(q.device)
        L = min(ctx[s] + n, cap)
        mask = torch.ones((n, L), dtype=torch.bool, device=q.device)
        mask[:, ctx[s]:] = seen[:, :max(0, L - ctx[s])]
        t = torch.arange(L, device=q.device)
        page = torch.as_tensor(np.asarray(table)[s], device=q.device).long()[t // P]
        mask &= ((page >= 0) & (page < num_pages))[None]
        page = page.clamp(0, num_pages - 1)
        for h in range(NH):
            K, V = k[page, h // G, t % P].double(), v[page, h // G, t % P].double()
            qd = q[t0:t0 + n, h].double()
            sc = torch.where(mask, (qd @ torch.nan_to_num(K).t()) * scale + (qd[:, None] * K[None]).sum(-1) * 0, -np.inf)
            p = torch.exp(sc - sc.amax(1, keepdim=True).clamp_min(-1e300))
            z = p.sum(1, keepdim=True)
            p = torch.where(z > 0, p / z, 0.0)
            pv = torch.where(mask[:, :, None], p[:, :, None] * V[None], 0.0)
            out[t0:t0 + n, h] = pv.sum(1)
            mag[t0:t0 + n, h] = pv.abs().sum(1)
            d = (qd.abs()[:, None] * torch.where(mask[:, :, None], K[None].abs(), 0.0)).sum(-1)
            off[t0:t0 + n, h, 0] = (D + 4) * 2 * U * abs(scale) * d.amax(1)
    return out, mag, off


def tree_case(qvl, ctx, nodes, NH, NKV, D, P, dtype, seed, chain=False, pad=0, extra=0, spread=4, q_scale=1.0):
    r = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    ctx, nodes = np.asarray(ctx), np.asarray(nodes)
    S = len(ctx)
    maxp = max(1, int(-(-(ctx + nodes).max() // P)))
    starts = np.concatenate([[0], np.cumsum(nodes)]).tolist()
    T = starts[-1] + pad
    parents = np.concatenate([(np.arange(n) - 1) if chain else np.maximum(-1, np.arange(n) - 1 - r.integers(0, spread, n))
                              for n in nodes] + [np.zeros(pad, np.int64)])
    cache = torch.bfloat16 if dtype == BF16 else torch.float16
    # what no request owns, and what is past a request's last node, holds NaN
    k = torch.full((S * maxp + extra, NKV, P, D), float("nan"), device="cuda", dtype=cache)
    v = k.clone()
    table = r.permutation(S * maxp + extra)[:S * maxp].reshape(S, maxp)
    for s in range(S):
        n = int(ctx[s] + nodes[s])
        t = torch.arange(n, device="cuda")
        pg = torch.as_tensor(table[s], device="cuda")[t // P]
        k[pg, :, t % P] = torch.randn((n, NKV, D), generator=g, device="cuda").to(cache)
        v[pg, :, t % P] = torch.randn((n, NKV, D), generator=g, device="cuda").to(cache)
    q = (torch.randn((T, NH, D), generator=g, device="cuda") * q_scale).to(dtype)
    kv = qvl.PagedKV(S, maxp * P, NH, NKV, D, P, page_table=i32(table), k=k[:S * maxp], v=v[:S * maxp]) if not extra else None
    return dict(q=q, k=k, v=v, kv=kv, table=table, ctx=ctx.tolist(), nodes=nodes.tolist(), starts=starts,
                parents=parents, P=P, D=D)


def run_tree(qvl, c, max_ctx=None, max_nodes=None, scale=None, q=None, **kw):
    return qvl.tree_attention(c["q"] if q is None else q, c["kv"], i32(c["ctx"]), i32(c["starts"]), i32(c["parents"]),
                              max_ctx or max(1, max(a + b for a, b in zip(c["ctx"], c["nodes"]))),
                              max_nodes or max(1, max(c["nodes"])), scale=scale, **kw)


def check_tree(qvl, c, scale=None, max_nodes=None, **kw):
    got = run_tree(qvl, c, scale=scale, max_nodes=max_nodes, **kw)
    sc = c["D"] ** -0.5 if scale is None else scale
    want, mag, off = tree_oracle(c["q"], c["k"], c["v"], c["table"], c["ctx"], c["starts"], c["parents"], c["P"], sc,
                                 max_nodes or 10 ** 9, c["kv"].k.shape[0])
    tiles = max(c["ctx"]) // 64 + 8
    r = R[c["q"].dtype]
    lim = (2 * off + (128 + tiles) * 2 * U) * mag + r * want.abs() * (1 + 2.0 ** -8) + (2.0 ** -24 if r else 1e-30)
    d = (got.double() - want).abs()
    assert bool((d <= lim).all()), float((d / lim).max())
    # the sum of squares: roundings do not all point the same way
    if float(want.norm()):
        assert float((got.double() - want).norm() / want.norm()) <= max(5e-6 * max(1.0, float(off.max()) / 2e-4), r)
    return got


TREES = [([0], [1]), ([1], [1]), ([452], [1]), ([0], [5]), ([63], [2]), ([64], [64]), ([127], [9]), ([128], [33]),
         ([300], [100]), ([0, 5, 700, 0, 129], [3, 0, 17, 1, 40]), ([1000, 20], [1, 128])]


@pytest.mark.gpu
@pytest.mark.parametrize("ctx,nodes", TREES)
@pytest.mark.parametrize("NH,NKV,D,P,dtype", [(16, 8, 128, 64, F32), (4, 4, 64, 16, F16), (14, 2, 128, 48, BF16),
                                              (8, 2, 64, 128, F32), (2, 1, 128, 16, F16), (6, 6, 64, 256, BF16)])
def test_tree_attention(qvl, cuda, ctx, nodes, NH, NKV, D, P, dtype):
    check_tree(qvl, tree_case(qvl, ctx, nodes, NH, NKV, D, P, dtype, seed=len(ctx) + ctx[0] + D))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_tree_attention_long(qvl, cuda, dtype):
    check_tree(qvl, tree_case(qvl, [9000, 1, 4500], [7, 30, 20], 4, 2, 128, 64, dtype, seed=1))
    check_tree(qvl, tree_case(qvl, [5000], [3], 2, 1, 64, 16, dtype, seed=2))


@pytest.mark.gpu
@pytest.mark.parametrize("G", [1, 2, 3, 8, 16])
def test_tree_attention_many_rows(qvl, cuda, G):
    """256 nodes, up to 4096 query rows to a key head; chains as deep as the tree is large."""
    check_tree(qvl, tree_case(qvl, [70, 3], [256, 200], G, 1, 64, 32, F32, seed=G, chain=True))
    check_tree(qvl, tree_case(qvl, [130], [255], 2 * G, 2, 128, 64, F16, seed=G, spread=60))


@pytest.mark.gpu
def test_tree_attention_sharp_and_large_scores(qvl, cuda):
    """Scores up to hundreds: one position takes nearly all of a row; and queries whose size fp16 cannot hold."""
    check_tree(qvl, tree_case(qvl, [700], [20], 4, 2, 128, 64, F32, seed=3, q_scale=30.0))
    check_tree(qvl, tree_case(qvl, [700], [20], 4, 2, 128, 64, F16, seed=4, q_scale=30.0))
    check_tree(qvl, tree_case(qvl, [300], [20], 4, 2, 128, 64, F32, seed=5, q_scale=1e6), scale=1e-6)
    check_tree(qvl, tree_case(qvl, [300], [20], 4, 2, 128, 64, F32, seed=6, q_scale=1e-6), scale=1e5)
    check_tree(qvl, tree_case(qvl, [300], [20], 4, 2, 128, 64, F32, seed=7), scale=-0.1)
    check_tree(qvl, tree_case(qvl, [300], [20], 4, 2, 64, 64, BF16, seed=8), scale=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_tree_attention_masked_values_have_no_influence(qvl, cuda, dtype, bad):
    """Keys and values of nodes that a row does not see, whatever they hold."""
    c = tree_case(qvl, [100, 0], [40, 30], 4, 2, 128, 64, dtype, seed=11, spread=12)
    clean = run_tree(qvl, c).clone()
    hit = [7, 11, 26]
    val = float(torch.finfo(c["k"].dtype).min) if bad == "lowest" else bad
    for s in range(2):
        for j in hit:
            t = c["ctx"][s] + j
            pg = int(c["table"][s][t // 64])
            c["kv"].v[pg, :, t % 64, 5:90] = val
            c["kv"].k[pg, :, t % 64, 3:] = val
    got = run_tree(qvl, c)
    for s in range(2):
        t0, n = c["starts"][s], c["nodes"][s]
        seen = ancestors(c["parents"][t0:t0 + n], n)[:, hit].any(1)
        assert 0 < seen.sum() < n
        assert torch.equal(got[t0:t0 + n][~torch.from_numpy(seen).cuda()], clean[t0:t0 + n][~torch.from_numpy(seen).cuda()])
        if bad != "lowest":
            assert bool(torch.isnan(got[t0:t0 + n][torch.from_numpy(seen).cuda()]).any(-1).all())


@pytest.mark.gpu
def test_tree_attention_visible_infinite_values(qvl, cuda):
    """An infinite value that some rows see is infinite for these alone."""
    c = tree_case(qvl, [80], [24], 2, 1, 64, 16, F32, seed=13, spread=10)
    clean = run_tree(qvl, c).clone()
    t = 80 + 6
    c["kv"].v[int(c["table"][0][t // 16]), 0, t % 16, 9] = float("inf")
    got = run_tree(qvl, c)
    seen = torch.from_numpy(ancestors(c["parents"], 24)[:, 6]).cuda()
    assert bool((got[seen][..., 9] == float("inf")).all())
    clean[seen, :, 9] = float("inf")
    assert torch.equal(got, clean)


@pytest.mark.gpu
def test_tree_attention_rows_without_anything(qvl, cuda):
    """Padding rows, nodes past max_nodes, and requests whose pages do not exist give zeros."""
    c = tree_case(qvl, [50, 10, 200], [6, 9, 0], 4, 2, 128, 16, F32, seed=21, pad=5)
    out = torch.full_like(c["q"], 7.0)
    assert not check_tree(qvl, c, out=out)[15:].any()
    got = check_tree(qvl, c, max_nodes=7, out=out.fill_(7.0))
    assert not got[13:15].any() and got[12].any()
    c["table"] = np.where(np.arange(c["table"].shape[1])[None] % 3 == 1, [[-1], [10 ** 6], [-5]], c["table"])
    c["kv"].page_table = i32(c["table"])
    check_tree(qvl, c)
    c["kv"].page_table = torch.full_like(c["kv"].page_table, -1)
    assert not run_tree(qvl, c).any()
    # more nodes than the page table has room for: those past it do not exist
    c = tree_case(qvl, [30], [10], 4, 2, 128, 16, F32, seed=22)
    c["ctx"] = [45]
    c["kv"].k[:], c["kv"].v[:] = c["kv"].k.nan_to_num(), c["kv"].v.nan_to_num()
    check_tree(qvl, c)
    c["ctx"] = [2000]
    check_tree(qvl, c, max_ctx=48)


@pytest.mark.gpu
def test_tree_attention_parents_strides_streams(qvl, cuda):
    c = tree_case(qvl, [150, 7], [31, 12], 6, 3, 128, 32, F32, seed=31)
    want = check_tree(qvl, c).clone()
    # max_ctx only shapes the launch
    for m in (1, 100, 5000):
        check_tree(qvl, c, max_ctx=m, max_nodes=200)
    # rows of a wider buffer
    wide = torch.randn((43, 6 * 128 + 24), device="cuda")
    view = wide[:, 8:8 + 768].unflatten(1, (6, 128))
    view.copy_(c["q"])
    assert torch.equal(run_tree(qvl, c, q=view), want)
    # a side stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_tree(qvl, c, workspace=qvl.Workspace())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # the same call again: no order of additions is left to chance
    for _ in range(3):
        assert torch.equal(run_tree(qvl, c), want)
    # entries that name no earlier node are roots
    c["parents"] = np.where(np.arange(43) % 5 == 2, -9, c["parents"])
    c["parents"][20], c["parents"][21], c["parents"][3] = 21, 2 ** 31 - 1, 3
    check_tree(qvl, c)


@pytest.mark.gpu
def test_tree_attention_of_a_single_token_is_attention(qvl, cuda):
    """One node per request is a decode step."""
    NH, NKV, D, P = 16, 8, 128, 64
    ctx = [451, 1000, 77]
    c = tree_case(qvl, ctx, [1, 1, 1], NH, NKV, D, P, F32, seed=41)
    for x in (c["kv"].k, c["kv"].v):
        x.nan_to_num_()
    want = qvl.attention(c["q"].clone(), c["kv"], i32([0, 1, 2]), i32(ctx), 1100)
    got = run_tree(qvl, c)
    assert float((got - want).norm() / want.norm()) < 1e-3       # the other one's exponential is a polynomial


# -------------------------------------------------------------- token_logprobs
def logprob_oracle(x, tokens, k):
    x = x.double()
    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - lse[:, None])
    ent = lse - torch.where(p > 0, p * x, 0.0).sum(1)
    empty = (x == -np.inf).all(1)
    ent[empty] = 0.0
    t = tokens.long().clamp(0, x.shape[1] - 1)
    lp = x.gather(1, t[:, None])[:, 0] - lse
    lp[empty] = -np.inf
    lp[(tokens < 0) | (tokens >= x.shape[1])] = 0.0
    top = torch.sort(x, dim=1, descending=True, stable=True)
    v = top.values[:, :k] - lse[:, None]
    v[empty] = -np.inf
    return lp, ent, top.indices[:, :k], v, lse, p, x


def check_logprobs(qvl, x, tokens, k):
    got = qvl.token_logprobs(x, tokens, k)
    lp, ent, ids, v, lse, p, xd = logprob_oracle(x, tokens, k)
    assert torch.equal(got.top_ids.long(), ids)
    depth = -(-x.shape[1] // 256) + 60
    lim = depth * U + 4 * U * lse.abs().nan_to_num(0, 0, 0)

    def close(a, b, lim):
        fin = torch.isfinite(b)
        assert torch.equal(a.double()[~fin], b[~fin])
        d = (a.double() - b).abs()
        assert bool((d <= lim + 2 * U * b.abs())[fin].all()), float(d[fin].max())

    close(got.logprobs, lp, lim)
    close(got.entropy, ent, lim + 2 * depth * U * torch.where(p > 0, p * xd.abs(), 0.0).sum(1).nan_to_num(0))
    close(got.top_logprobs, v, lim[:, None].expand_as(v))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(1, 1), (3, 2), (5, 31), (2, 257), (7, 1000), (4, 4096), (3, 8191), (2, 32003), (33, 5001),
                                 (5, 151936), (1, 151936)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_token_logprobs(qvl, cuda, T, V, dtype):
    g = torch.Generator(device="cuda").manual_seed(T + V)
    x = (torch.randn((T, V), generator=g, device="cuda") * 3).to(dtype)
    tok = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
    for k in {0, 1, min(V, 5), min(V, 20), min(V, 64)}:
        check_logprobs(qvl, x, tok, k)


@pytest.mark.gpu
def test_token_logprobs_ties_and_order(qvl, cuda):
    """Equal logits by the lower index, sorted rows either way, rows with one value."""
    V = 40000
    g = torch.Generator(device="cuda").manual_seed(0)
    rows = [torch.zeros(V, device="cuda"), torch.arange(V, device="cuda") / V, -torch.arange(V, device="cuda") / V,
            torch.randint(0, 3, (V,), generator=g, device="cuda").float(),
            torch.full((V,), -1e30, device="cuda"), torch.randn(V, generator=g, device="cuda").round() * 1e3]
    x = torch.stack(rows)
    tok = i32([0, V - 1, 5, 7, 9, 11])
    for d in (F32, F16, BF16):
        y = x.clamp(-6e4, 6e4).to(d)
        for k in (1, 20, 64):
            check_logprobs(qvl, y, tok, k)
    y = torch.zeros((2, 600), device="cuda")
    y[0, ::2] = -0.0                       # both zeros are one value
    check_logprobs(qvl, y, i32([1, 2]), 8)


@pytest.mark.gpu
def test_token_logprobs_masked_rows(qvl, cuda):
    """-inf logits: a few, all but a few, all; a token that is masked; tokens outside the vocabulary."""
    V = 20011
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((7, V), generator=g, device="cuda")
    x[1, torch.rand(V, generator=g, device="cuda") < 0.5] = -np.inf
    x[2, 3:] = -np.inf
    x[3, :V - 2] = -np.inf
    x[4] = -np.inf
    x[5, :] = -np.inf
    x[5, 12345] = 4.0
    x[6, 0] = -np.inf
    tok = i32([-1, V, 1, 5, 8, 12345, 0])
    for d in (F32, BF16):
        got = check_logprobs(qvl, x.to(d), tok, 20)
        assert float(got.logprobs[0]) == 0.0 and float(got.logprobs[1]) == 0.0
        assert float(got.logprobs[3]) == -np.inf and float(got.logprobs[4]) == -np.inf
        assert float(got.entropy[4]) == 0.0 and float(got.entropy[5]) == 0.0


@pytest.mark.gpu
def test_token_logprobs_not_numbers(qvl, cuda):
    x = torch.randn((4, 3001), device="cuda")
    x[1, 77] = float("nan")
    x[2, 5] = float("inf")
    x[3] = float("nan")
    x[3, 9] = 1.0
    r = qvl.token_logprobs(x, i32([3, 3, 3, 9]), 3)
    assert not bool(torch.isnan(r.logprobs[0])) and bool(torch.isnan(r.logprobs[1:]).all())
    assert bool(torch.isnan(r.entropy[1:]).all())
    assert 77 not in r.top_ids[1].tolist() and r.top_ids[2, 0] == 5
    assert r.top_ids[3].tolist() == [9, -1, -1]


@pytest.mark.gpu
def test_token_logprobs_strides_streams_repeats(qvl, cuda):
    V = 5003
    wide = torch.randn((9, 2 * V + 1), device="cuda")
    for d in (F32, BF16):
        w = wide.to(d)
        x = w[:, 3:3 + V]
        tok = torch.arange(9, dtype=torch.int32, device="cuda")
        a = check_logprobs(qvl, x, tok, 7)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = qvl.token_logprobs(x, tok, 7)
        torch.cuda.current_stream().wait_stream(side)
        c = qvl.token_logprobs(x.contiguous(), tok, 7, out=qvl.TokenLogprobs(9, 7, "cuda"))
        for r in (b, qvl.token_logprobs(x, tok, 7)):
            assert torch.equal(a.logprobs, r.logprobs) and torch.equal(a.entropy, r.entropy)
            assert torch.equal(a.top_ids, r.top_ids) and torch.equal(a.top_logprobs, r.top_logprobs)
        assert torch.equal(a.top_ids, c.top_ids) and float((a.logprobs - c.logprobs).abs().max()) < 1e-5
    assert qvl.token_logprobs(x[:0], tok[:0], 3).logprobs.shape == (0,)


# ------------------------------------------------------------------- refusals
def test_refusals_without_gpu():
    """The C ABI refuses bad arguments before any CUDA call."""
    qvl = import_qvl()
    L = qvl.load_library()
    f = 4096                                     # aligned, never dereferenced
    INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4

    def plan(**o):
        a = dict(old=f, new=f, S=4, table=f, P=16, maxp=4, free=f, fc=f, cap=8, fco=f + 4, missing=f, starts=f, seq=f,
                 pos=f, slots=f, n=10) | o
        return L.qvl_plan_pages(*a.values(), None)

    for o in (dict(old=None), dict(table=None), dict(free=None), dict(missing=None), dict(slots=None), dict(S=0),
              dict(P=0), dict(maxp=0), dict(fco=f), dict(table=f + 2), dict(cap=2 ** 31)):
        assert plan(**o) == INVALID, o
    assert plan(S=16385) == UNSUPPORTED

    d = qvl.AttnDims(16, 8, 128, 64, 4, 256)

    def rope(dims=None, **o):
        dd = dims or d
        a = dict(q=f, k=f, v=f, dt=0, qs=2048, ks=1024, vs=1024, out=f, kp=f, vp=f, kdt=2, pages=8, slots=f, pos=f, ps=5,
                 na=3, axes=f, T=5, cos=f, sin=f, qw=f, qsc=f, kw=f, ksc=f, wd=3, g=128, eps=1e-6) | o
        return L.qvl_qknorm_mrope_kv_append(*a.values(), ctypes.byref(dd), None)

    for o in (dict(q=None), dict(out=None), dict(slots=None), dict(axes=None), dict(qs=2047), dict(qs=2050), dict(q=f + 8),
              dict(kp=f + 8), dict(ps=4), dict(na=0), dict(qw=None), dict(qsc=None), dict(g=0), dict(g=96), dict(eps=-1.0),
              dict(eps=float("nan")), dict(pages=0), dict(dims=qvl.AttnDims(16, 7, 128, 64, 4, 256)),
              dict(dims=qvl.AttnDims(16, 8, 128, 24, 4, 256)), dict(dims=qvl.AttnDims(16, 8, 128, 64, 4, 0))):
        assert rope(**o) == INVALID, o
    for o in (dict(dt=3), dict(dt=1), dict(kdt=0), dict(wd=4), dict(dims=qvl.AttnDims(16, 8, 96, 64, 4, 256))):
        assert rope(**o) == UNSUPPORTED, o
    assert rope(T=0) == 0

    big = L.qvl_tree_attention_workspace_bytes(4, 64, 4096, 16, ctypes.byref(d))

    def tree(dims=None, **o):
        dd = dims or d
        a = dict(q=f, dt=0, qs=2048, kp=f, vp=f, kdt=2, pages=64, table=f, ctx=f, starts=f, par=f, S=4, T=64, mc=4096,
                 mn=16, sc=0.1, out=f) | o
        ws = a.pop("ws", f)
        n = a.pop("n", 1 << 40)
        return L.qvl_tree_attention(*a.values(), ctypes.byref(dd), ws, n, None)

    for o in (dict(q=None), dict(kp=None), dict(table=None), dict(par=None), dict(out=None), dict(qs=100), dict(S=0),
              dict(S=65536), dict(mc=0), dict(mn=0), dict(pages=0), dict(sc=float("nan")), dict(q=f + 4), dict(vp=f + 2),
              dict(dims=qvl.AttnDims(16, 8, 128, 24, 4, 256)), dict(dims=qvl.AttnDims(15, 8, 128, 64, 4, 256))):
        assert tree(**o) == INVALID, o
    for o in (dict(dt=5), dict(kdt=5), dict(dt=0, kdt=0), dict(dt=2, kdt=5), dict(mn=257), dict(pages=2 ** 24),
              dict(dims=qvl.AttnDims(16, 8, 96, 64, 4, 256)), dict(dims=qvl.AttnDims(16, 8, 256, 64, 4, 256))):
        assert tree(**o) == UNSUPPORTED, o
    if big:
        assert tree(ws=None) == WORKSPACE and tree(n=big - 1) == WORKSPACE and tree(ws=f + 16) == WORKSPACE
    assert L.qvl_tree_attention_workspace_bytes(4, 64, 4096, 257, ctypes.byref(d)) == 0

    def lp(**o):
        a = dict(x=f, dt=0, stride=100, tok=f, T=3, V=100, k=5, lp=f, ent=f, ids=f, tl=f) | o
        return L.qvl_token_logprobs(*a.values(), None)

    for o in (dict(x=None), dict(tok=None), dict(lp=None), dict(ids=None), dict(k=-1), dict(V=0), dict(stride=99),
              dict(x=f + 2), dict(V=4, k=5), dict(tok=f + 1)):
        assert lp(**o) == INVALID, o
    for o in (dict(k=65), dict(dt=3), dict(dt=9)):
        assert lp(**o) == UNSUPPORTED, o
    assert lp(T=0, x=None) == 0


@pytest.mark.gpu
def test_python_refusals(qvl, cuda):
    c = tree_case(qvl, [20], [4], 4, 2, 128, 16, F32, seed=1)
    E = qvl.QvlError
    kv, q = c["kv"], c["q"]
    a = (i32([20]), i32([0, 4]), i32([-1, 0, 0, 1]))
    with pytest.raises(E):
        qvl.tree_attention(q[:, :2], kv, *a, 24, 4)
    with pytest.raises(E):
        qvl.tree_attention(q.to(BF16), kv, *a, 24, 4)
    with pytest.raises(E):
        qvl.tree_attention(q, kv, a[0].long(), a[1], a[2], 24, 4)
    with pytest.raises(E):
        qvl.tree_attention(q, kv, a[0], a[1], a[2][:3], 24, 4)
    with pytest.raises(E):
        qvl.tree_attention(q.cpu(), kv, *a, 24, 4)
    with pytest.raises(E):
        qvl.tree_attention(q, kv, *a, 24, 300)
    with pytest.raises(E):
        qvl.tree_attention(q.transpose(0, 1).contiguous().transpose(0, 1), kv, *a, 24, 4)
    with pytest.raises(E):
        qvl.tree_attention(q, kv, *a, 24, 4, out=torch.empty_like(q, dtype=F16))
    with pytest.raises(E):
        qvl.token_logprobs(q[:, 0], i32([0, 1]), 3)
    with pytest.raises(E):
        qvl.token_logprobs(q[:, 0].double(), i32([0, 1, 2, 3]), 3)
    with pytest.raises(E):
        qvl.token_logprobs(q[:, 0], i32([0, 1, 2, 3]), 65)
    with pytest.raises(E):
        qvl.plan_pages(i32([1, 2]), i32([1, 2]), i32([[1]]), i32([1]), i32([1]), 16, 4)
    with pytest.raises(E):
        qvl.plan_pages(i32([1]), i32([1, 2]), i32([[1]]), i32([1]), i32([1]), 16, 4)
    m = mrope_case(qvl, 5, 4, 2, 128, F32, F16, F32, False, 1)
    args = lambda **o: {**dict(q=m[0], k=m[1], v=m[2], kv=m[3], slots=i32(m[6]), positions=i32(m[7]), axes=m[8],  # noqa: E731
                               rope_cos=m[9], rope_sin=m[10], q_norm=m[11][0], k_norm=m[11][1]), **o}
    for o in (dict(k=m[1].half()), dict(slots=i32([1])), dict(positions=i32([1])), dict(axes=m[8][:5]),
              dict(rope_cos=m[9][:3]), dict(q_norm=None), dict(q_norm=m[11][0][:4]), dict(v=m[2][:, :1]),
              dict(out=torch.empty_like(m[0], dtype=F16)), dict(positions=i32(m[7])[:0])):
        with pytest.raises(E):
            qvl.qknorm_mrope_kv_append(**args(**o))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,nodes", [(64, [150, 3]), (128, [70, 129]), (128, [20, 9])])
def test_tree_attention_signs_of_the_scale(qvl, cuda, dtype, D, nodes):
    """A negative scale, and none at all, for tiles of many rows and of few."""
    c = tree_case(qvl, [333, 700], nodes, 4, 2, D, 32, dtype, seed=D + nodes[0])
    for scale in (-0.07, 0.0):
        check_tree(qvl, c, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("T,NH,NKV,D,dtype,cache,weights,fused", [
    (1500, 16, 8, 128, F32, F16, "int8", False), (2100, 5, 1, 64, BF16, BF16, F32, True), (1301, 24, 4, 256, F32, F16, F16, False),
    (700, 64, 8, 128, F16, F16, None, True)])
def test_mrope_append_many_tokens(qvl, cuda, T, NH, NKV, D, dtype, cache, weights, fused):
    """Several tokens to a CTA, among them some without a slot or with a position outside the
    table; heads in several parts."""
    case = list(mrope_case(qvl, T, NH, NKV, D, dtype, cache, weights, fused, seed=T))
    slots, pos = case[6].copy(), case[7].copy()
    r = np.random.default_rng(T)
    slots[r.random(T) < 0.1] = -1
    pos[r.integers(0, 3, 60), r.integers(0, T, 60)] = 300
    pos[0, -1], pos[2, 0] = -1, 10 ** 9
    case[6], case[7] = slots, pos
    check_mrope(qvl, case)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,k", [(300, 3001, 7), (700, 513, 64), (1200, 40, 0), (150, 9000, 3)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_token_logprobs_many_rows(qvl, cuda, T, V, k, dtype):
    """More rows than there are places for CTAs at a time, and the sizes around that."""
    g = torch.Generator(device="cuda").manual_seed(T + V)
    x = (torch.randn((T, V), generator=g, device="cuda") * 4).to(dtype)
    x[torch.rand((T, V), generator=g, device="cuda") < 0.02] = -float("inf")
    x[::17] = 1.5                        # rows of one value: more ties than there is room for candidates
    check_logprobs(qvl, x, torch.arange(T, device="cuda").remainder(V).int(), k)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [2, 9, 700])
def test_token_logprobs_rising_logits(qvl, cuda, V):
    """Every logit far above those before it, up to 40 at a time: the largest's log-probability is nearly 0."""
    steps = torch.linspace(0.5, 40, 300, device="cuda")[:, None] * torch.arange(V, device="cuda").remainder(9)
    for x in (steps, steps.flip(1), steps - 150, steps - steps.amax(1, keepdim=True)):
        check_logprobs(qvl, x.contiguous(), torch.full((300,), V - 1, dtype=torch.int32, device="cuda"), min(V, 12))


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(4, 4001), (2, 151936), (400, 4001)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_token_logprobs_lowest_values(qvl, cuda, T, V, dtype):
    """Logits of the type's lowest value, as masks write them, and others that are as far from the
    row's largest: finite, without weight, and of no influence on the sums."""
    g = torch.Generator(device="cuda").manual_seed(V + T)
    x = (torch.randn((T, V), generator=g, device="cuda") * 3).to(dtype)
    low = torch.finfo(dtype).min
    far = torch.tensor(-1e38 if dtype != F16 else -5e4).to(dtype)
    keep = torch.zeros((6, V), dtype=torch.bool, device="cuda")
    keep[0, V // 3:] = True                         # a masked prefix
    keep[1, ::701] = True                           # all but a few, one at most to a load
    keep[2, :V // 4] = True                         # whole slices and threads of nothing else
    keep[3, V - 1] = True                           # one logit alone
    keep[4] = torch.rand(V, generator=g, device="cuda") < 0.5
    keep[5, :] = True
    keep[5, 0] = False
    tok = torch.arange(T, device="cuda").remainder(V).int()
    for turn in range(0, 6, min(T, 6)):
        m = keep[(torch.arange(T, device="cuda") + turn) % 6]
        for masked in (torch.full_like(x, low), torch.full_like(x, float(far)), torch.where(x > 0, low, far).to(dtype)):
            got = check_logprobs(qvl, torch.where(m, x, masked), tok, 5)
            assert bool(torch.isfinite(got.entropy).all())
        # the largest logit further above than the type holds (its own token: the others' log-probabilities
        # are no fp32 numbers)
        if dtype != F16:
            y = torch.where(m, x, torch.full_like(x, low))
            y[:, V // 2] = 3e38
            assert not bool(check_logprobs(qvl, y, torch.full_like(tok, V // 2), 1).entropy.any())


@pytest.mark.gpu
def test_caches_and_page_tables_of_another_shape_are_refused(qvl, cuda):
    """What the cache's description says has to be what its tensors are: the kernels go by the former."""
    import types
    E = qvl.QvlError
    c = tree_case(qvl, [20], [4], 4, 2, 128, 16, F32, seed=1)
    a = (i32([20]), i32([0, 4]), i32([-1, 0, 0, 1]))
    kv = c["kv"]
    shape = list(kv.k.shape)

    def other(**o):
        return types.SimpleNamespace(**{**dict(k=kv.k, v=kv.v, page_table=kv.page_table, dims=kv.dims,
                                               page_size=kv.page_size), **o})

    pages = [torch.zeros([n + (i == j) * by for j, n in enumerate(shape)], dtype=kv.k.dtype, device="cuda")
             for i, by in ((0, -1), (1, -1), (2, -1), (3, -64))] + [torch.zeros(shape[:3], dtype=kv.k.dtype, device="cuda")]
    m = mrope_case(qvl, 5, 4, 2, 128, F32, F16, F32, False, 1)
    rope = (i32(m[6]), i32(m[7]), m[8], m[9], m[10])
    for i, x in enumerate(pages):
        for o in (dict(v=x), dict(k=x)) + ((dict(k=x, v=x),) if i else ()):      # (fewer pages in both are a cache)
            with pytest.raises(E):
                qvl.tree_attention(c["q"], other(**o), *a, 24, 4)
            with pytest.raises(E):
                qvl.qknorm_mrope_kv_append(m[0], m[1], m[2], other(dims=m[3].dims, **o), *rope, m[11][0], m[11][1])
    t = kv.page_table
    for x in (t[:, :1].contiguous(), torch.cat([t, t], 1), t[0], t[:0]):
        with pytest.raises(E):
            qvl.tree_attention(c["q"], other(page_table=x), *a, 24, 4)
        with pytest.raises(E):
            qvl.tree_attention(c["q"], qvl.PagedKV(1, 2 * 16, 4, 2, 128, 16, k=kv.k, v=kv.v, page_table=x), *a, 24, 4)
    assert bool(torch.isfinite(qvl.tree_attention(c["q"], other(), *a, 24, 4)).all())


def tree_by_definition(c, scale, G):
    """The rows of request 0 and the first key head's G heads in 64 bits, of finite and other values: a
    position whose score is -inf has no weight, every other one a weight above 0, however far its score."""
    ctx, n, kv = c["ctx"][0], c["nodes"][0], c["kv"]
    t = torch.arange(ctx + n, device="cuda")
    page = torch.as_tensor(np.asarray(c["table"])[0], device="cuda")[t // c["P"]]
    K, V = kv.k[page, 0, t % c["P"]].double(), kv.v[page, 0, t % c["P"]].double()
    seen = torch.ones((n, ctx + n), dtype=torch.bool, device="cuda")
    seen[:, ctx:] = torch.from_numpy(ancestors(c["parents"][:n], n)).cuda()
    out = []
    for h in range(G):
        x = (c["q"][:n, h].double()[:, None] * K[None]).sum(-1) * scale
        x = torch.where(seen, x, -np.inf)
        nan = torch.isnan(x).any(1) | (x == np.inf).any(1)
        p = torch.exp(x - x.nan_to_num(0).amax(1, keepdim=True)).clamp_min(1e-300)
        p = torch.where(x > -np.inf, p, 0.0)
        y = torch.where((x > -np.inf)[:, :, None], p[:, :, None] * V[None], 0.0).sum(1) / p.sum(1, keepdim=True).clamp_min(1e-300)
        out.append(torch.where(nan[:, None], np.nan, y))
    return torch.stack(out, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("G,D,nodes", [(2, 128, 1), (2, 64, 12), (4, 128, 16), (2, 128, 50), (4, 64, 40)])
@pytest.mark.parametrize("ctx", [3, 90, 700])
def test_tree_attention_infinities_that_are_seen(qvl, cuda, dtype, G, D, nodes, ctx):
    """Infinite values and keys at cached positions, at drafted nodes and at both, in tiles of few rows and
    of many, whole and in parts: outputs are what the definition says, infinite, NaN or finite."""
    c = tree_case(qvl, [ctx, 5], [nodes, 2], 2 * G, 2, D, 32, dtype, seed=ctx + nodes, spread=6)
    scale = D ** -0.5
    clean = run_tree(qvl, c).clone()
    base_k, base_v = c["kv"].k.clone(), c["kv"].v.clone()

    def put(x, t, h, col, val):
        x[int(c["table"][0][t // 32]), h, t % 32, col] = val

    inf = float("inf")
    last = ctx + nodes - 1
    plants = [[("v", 0, 3, inf)], [("v", ctx - 1, 7, -inf)], [("v", 1, 3, inf), ("v", 2, 3, -inf), ("v", 1, 9, inf)],
              [("v", last, D - 1, -inf), ("v", 2, 0, inf)], [("k", 1, 5, inf)], [("k", ctx - 1, 11, -inf)],
              [("k", last, 2, inf)], [("k", 0, 2, inf), ("v", 0, 6, inf), ("v", ctx - 1, 6, 1.0)],
              [("v", 2, 4, float("nan"))], [("k", 2, 4, float("nan"))]]
    for plant in plants:
        c["kv"].k.copy_(base_k)
        c["kv"].v.copy_(base_v)
        for which, t, col, val in plant:
            put(c["kv"].k if which == "k" else c["kv"].v, t, 0, col, val)
        got = run_tree(qvl, c)
        assert torch.equal(got[:, G:], clean[:, G:])                    # the other key head
        assert torch.equal(got[nodes:], clean[nodes:])                  # the other request
        got, want = got[:nodes, :G], tree_by_definition(c, scale, G)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), plant
        inf_at = torch.isinf(want)
        assert torch.equal(got.double()[inf_at], want[inf_at]), plant
        # what is finite: within the bound of finite inputs, here with |q k| and |v| of the finite ones at
        # most (5.5 sqrt(D))^2 and 5.5
        fin = torch.isfinite(want)
        off = (D + 4) * 2 * U * scale * 30 * D
        lim = (2 * off + 160 * 2 * U) * 5.5 + R[dtype] * want[fin].abs() * (1 + 2.0 ** -8) + 2.0 ** -24
        assert bool(((got.double() - want).abs()[fin] <= lim).all()), plant


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_tree_attention_scores_of_minus_infinity_alone(qvl, cuda, dtype):
    """A row whose every score is -inf has no weights, like one that sees nothing: zeros."""
    c = tree_case(qvl, [4], [3], 2, 1, 64, 16, dtype, seed=3, chain=True)
    c["q"][..., 0] = c["q"][..., 0].abs() + 1
    c["kv"].k[int(c["table"][0][0]), 0, :7, 0] = -float("inf")
    assert not run_tree(qvl, c).any()
    assert not tree_by_definition(c, 0.125, 2).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("D,nodes,ctx", [(128, 1, 40), (64, 20, 300), (128, 60, 300), (128, 5, 3000)])
def test_tree_attention_small_weights_carry_the_output(qvl, cuda, dtype, D, nodes, ctx):
    """One position that takes nearly all of every row's weight and whose value is 0, as an attention sink's
    is: the output is made of weights 2^-17 to 2^-29 of that one, and as exact as any."""
    for below in (12.0, 14.0, 17.0, 20.0):
        c = tree_case(qvl, [ctx], [nodes], 4, 2, D, 32, dtype, seed=int(below), chain=True)
        # scores of the sink: `below` + the others', which are random with a deviation of 1/4
        c["q"].mul_(0.25)
        c["q"][..., 0] = 4.0
        page = int(c["table"][0][0])
        t = torch.arange(ctx + nodes, device="cuda")
        pg = torch.as_tensor(c["table"][0], device="cuda")[t // 32]
        c["kv"].k[pg, :, t % 32, 0] = 0.0
        c["kv"].k[page, :, 0, :] = 0.0
        c["kv"].k[page, :, 0, 0] = below * D ** 0.5 / 4.0
        # (values of a size at which fp16 outputs are normal numbers)
        c["kv"].v[pg, :, t % 32, :] *= 8192.0
        c["kv"].v[page, :, 0, :] = 0.0
        check_tree(qvl, c)


@pytest.mark.gpu
def test_default_scratch_of_streams_and_threads(qvl, cuda):
    """Calls without a workspace on two streams at a time, and from two threads on one stream: each has
    its own parts."""
    import threading
    cases = [tree_case(qvl, [ctx], [n], 8, 4, 128, 64, F32, seed=n) for ctx, n in ((9000, 40), (7000, 9))]
    args = [(c["q"], c["kv"], i32(c["ctx"]), i32(c["starts"]), i32(c["parents"]), c["ctx"][0] + c["nodes"][0], c["nodes"][0])
            for c in cases]
    want = [qvl.tree_attention(*a, workspace=qvl.Workspace()) for a in args]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(40):
        for i in range(2):
            got[i].append(qvl.tree_attention(*args[i], stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])

    def work(i):
        got[i] = [qvl.tree_attention(*args[i]) for _ in range(40)]

    got = [[], []]
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 40 and all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.gpu
def test_captured_call_keeps_its_scratch(qvl, cuda):
    """A graph that was captured without a workspace, replayed after other calls have asked for more
    scratch and other tensors have taken what was given back."""
    c = tree_case(qvl, [5000, 300], [20, 3], 8, 4, 128, 64, F32, seed=5)
    a = (c["q"], c["kv"], i32(c["ctx"]), i32(c["starts"]), i32(c["parents"]), 5020, 20)
    want = qvl.tree_attention(*a).clone()
    out = torch.empty_like(want)
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        qvl.tree_attention(*a, out=out)
    x, w = torch.randn((3000, 8192), device="cuda"), torch.ones((32, 8192), dtype=torch.int8, device="cuda")
    for st in (None, side):
        qvl.linear(x, w, torch.ones((32, 1), device="cuda"), group_quantized=False, stream=st)
    torch.cuda.synchronize()
    hold = [torch.full((1 << 18,), 7.0, device="cuda") for _ in range(200)]
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert all(bool((h == 7.0).all()) for h in hold)


@pytest.mark.gpu
def test_memory_comes_from_the_stream_of_the_call(qvl, cuda, monkeypatch):
    """Outputs and scratch that a call on another stream allocates are that stream's: what is free on the
    current one may still be in use there."""
    side, made, real = torch.cuda.Stream(), [], torch.empty
    c = tree_case(qvl, [20], [4], 4, 2, 128, 16, F32, seed=1)
    a = (i32(c["ctx"]), i32(c["starts"]), i32(c["parents"]))
    m = mrope_case(qvl, 30, 4, 2, 128, F32, F16, None, False, 1)
    x, w, s = torch.randn((64, 256), device="cuda"), torch.ones((32, 256), dtype=torch.int8, device="cuda"), torch.ones((32, 1), device="cuda")
    slots, pos, tok = i32(m[6]), i32(m[7]), torch.zeros(64, dtype=torch.int32, device="cuda")
    plan = (i32([0]), i32([9]), i32([[-1]]), i32([0]), i32([1]))
    side.wait_stream(torch.cuda.current_stream())

    def recorded(*args, **kw):
        made.append(torch.cuda.current_stream().cuda_stream)
        return real(*args, **kw)

    monkeypatch.setattr(torch, "empty", recorded)
    for call in (lambda: qvl.tree_attention(c["q"], c["kv"], *a, 24, 4, stream=side),
                 lambda: qvl.qknorm_mrope_kv_append(m[0], m[1], m[2], m[3], slots, pos, m[8], m[9], m[10], stream=side),
                 lambda: qvl.token_logprobs(x, tok, 5, stream=side), lambda: qvl.plan_pages(*plan, 16, 40, stream=side),
                 lambda: qvl.greedy_decode(x, stream=side), lambda: qvl.quantize_rows(x, 256, stream=side),
                 lambda: qvl.linear(x, w, s, group_quantized=False, stream=side),
                 lambda: qvl.attention(c["q"], c["kv"], tok[:4], tok[:4], 24, stream=side)):
        made.clear()
        call()
        assert made and set(made) <= {side.cuda_stream}
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("D,P,NH", [(128, 8, 4), (64, 24, 4), (128, 16, 3)])
def test_tree_attention_after_a_refused_call(qvl, cuda, monkeypatch, D, P, NH):
    """What the library refuses says nothing about the scratch of later calls."""
    import qvl_b200
    monkeypatch.setattr(qvl_b200, "_tree_bytes", {})
    c = tree_case(qvl, [20], [4], 4, 2, D, 16, F32, seed=1)
    a = (i32(c["ctx"]), i32(c["starts"]), i32(c["parents"]), 24, 4)
    with pytest.raises(qvl.QvlError):
        qvl.tree_attention(torch.zeros((4, NH, D), device="cuda"), qvl.PagedKV(1, 48, NH, 2, D, P), *a,
                           workspace=qvl.Workspace())
    check_tree(qvl, c, workspace=qvl.Workspace())


@pytest.mark.gpu
def test_plan_pages_of_different_sizes_from_two_threads(qvl, cuda):
    """Plans of many and of fewer requests at once: what one launch needs of shared memory does not
    take away the other's."""
    import threading
    args, errors = [], []
    for S in (16384, 3600):
        z = torch.zeros(S, dtype=torch.int32, device="cuda")
        args.append((z, z, torch.full((S, 1), -1, dtype=torch.int32, device="cuda"), i32([0]), i32([0]), 16, 0, qvl.PagePlan(S, 0, "cuda")))

    def work(a):
        stream = torch.cuda.Stream()
        try:
            for _ in range(20000):
                qvl.plan_pages(*a, stream=stream)
        except qvl.QvlError as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(a,)) for a in args]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors


def test_plan_pages_refuses_more_tokens_than_its_indexes_hold():
    """A warp's stretch of tokens ends up to 150,000 past the last one, in 32 bits."""
    L = import_qvl().load_library()
    f = 4096                                     # aligned, never dereferenced
    for n in (2 ** 31 - 1 - 4096, 2 ** 31 - 150_000, 2 ** 31 - 2 ** 18, 2 ** 31, 2 ** 40):
        assert L.qvl_plan_pages(f, f, 4, f, 16, 4, f, f, 8, f + 4, f, f, f, f, f, n, None) == 1, n


def test_no_read_only_loads_beside_the_launch_that_writes():
    """The operators' launches begin before those ahead of them have ended (pdl_wait), so that what they
    read is written in their lifetime: nothing for the read-only path."""
    import os
    import re
    from conftest import PKG_DIR
    for f in ("page_plan", "mrope_append", "tree_attention", "token_logprobs"):
        with open(os.path.join(PKG_DIR, "csrc", f + ".cu")) as h:
            src = h.read()
        assert "pdl_wait();" in src
        assert not re.search(r"__ldg|ld\.global\.nc|__restrict__|ld_stream", src), f
