"""Decoding with drafted trees (TreeDecoder: plan_pages, qknorm_mrope_kv_append,
tree_attention and token_logprobs in one path) against the decoder that takes one
token of a request at a time.

Tokens are those of the other decoder, exactly.  Logits are no continuous function of
what the operators compute: with random weights one activation that is quantised to
the next step moves them by 3e-3 of the largest, and noise of 1e-6 on the attention
is enough for that.  So each call of an operator within the path is held
against 64-bit code on the same inputs instead.  Its bars: norms and rotations are a
sum of 128 squares and a few roundings, 128 2^-24 = 2^-17 of the largest at most;
attention has queries and probabilities of 22 bits and fp32 sums of 128 products, so that a
score is off by 2^-17 of |q| |k| scale at most and an output by that and 2^-17 of the
largest value.  One layer, for the reason that the decoder's own tests give.  The cache is
compared with the other decoder's, whose products have another order.  2048 additions
of a random walk, each rounded to 2^-25 of a partial sum (root mean square), are
sqrt(2048) 2^-25 = 2^-19.5 of the heads' root mean square apart; 8 times that for the
furthest of some 10^5 values is 2^-16.5, and no head's largest value is below its root
mean square: 2^-16 of the largest.  Beside it an fp16 value may differ by its last
bit, 2^-10 of the value."""
import numpy as np
import pytest
import torch


def _setup(qvl, cuda, seed, max_ctx=320):
    import qvl_b200.decoder as D
    import qvl_b200.drafting as F
    cfg = D.TextConfig(layers=1, vocab=4096)
    w = D.TextWeights.random(cfg, seed=seed, device=cuda)
    one = D.TextDecoder(w, max_batch=1, max_ctx=max_ctx, device=cuda, batch_order="lane8", attn_order="fast")
    return D, F, cfg, w, one


def _checked(F, monkeypatch):
    """Has every call of the path's rotation and attention compared with 64-bit torch code."""
    own_rope, own_tree, calls = F.qknorm_mrope_kv_append, F.tree_attention, [0]

    def rope(q, k, v, kv, slots, positions, axes, cos, sin, q_norm, k_norm, eps, out):
        half = q.shape[2] // 2
        at = positions.long()[axes.long(), :].t()                       # [T, D / 2]
        c, s = (t.double().gather(0, at)[:, None] for t in (cos, sin))

        def turn(x, norm):
            w = norm[0].double() * norm[1].double().repeat_interleave(norm[2])
            x = x.double()
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
            a, b = x[..., :half], x[..., half:]
            return torch.cat([a * c - b * s, b * c + a * s], -1)

        q_ref, k_ref = turn(q, q_norm), turn(k, k_norm)
        own_rope(q, k, v, kv, slots, positions, axes, cos, sin, q_norm, k_norm, eps, out=out)
        assert (out - q_ref).abs().max() <= 2.0 ** -17 * q_ref.abs().max()
        P, to = kv.page_size, slots.long()
        got = kv.k[to // P, :, to % P]
        assert ((got - k_ref).abs() <= 2.0 ** -11 * k_ref.abs() + 2.0 ** -17 * k_ref.abs().max()).all()
        assert torch.equal(kv.v[to // P, :, to % P], v.to(kv.v.dtype))
        calls[0] += 1
        return out

    def attend(q, kv, ctx, starts, parents, max_ctx, max_nodes, out, workspace):
        own_tree(q, kv, ctx, starts, parents, max_ctx, max_nodes, out=out, workspace=workspace)
        G = q.shape[1] // kv.dims.num_kv_heads
        scale = q.shape[2] ** -0.5
        for s in range(ctx.numel()):
            a, n, c = int(starts[s]), int(starts[s + 1] - starts[s]), int(ctx[s])
            if n == 0:
                continue
            pages = kv.page_table[s, :-(-(c + n) // kv.page_size)].long()
            K, V = (x[pages].double().transpose(0, 1).flatten(1, 2)[:, :c + n].repeat_interleave(G, 0) for x in (kv.k, kv.v))
            sees = torch.zeros((n, c + n), dtype=torch.bool)
            sees[:, :c] = True
            for i in range(n):
                if int(parents[a + i]) >= 0:
                    sees[i] = sees[int(parents[a + i])]
                sees[i, c + i] = True
            Q = q[a:a + n].double()
            x = torch.einsum("nhd,htd->nht", Q, K) * scale
            x = x.masked_fill(~sees[:, None].to(x.device), float("-inf"))
            ref = torch.einsum("nht,htd->nhd", torch.softmax(x, -1), V)
            size = scale * float(Q.norm(dim=-1).max() * K.norm(dim=-1).max())
            assert (out[a:a + n] - ref).abs().max() <= 2.0 ** -17 * (1 + 2 * size) * V.abs().max()
        calls[0] += 1
        return out

    monkeypatch.setattr(F, "qknorm_mrope_kv_append", rope)
    monkeypatch.setattr(F, "tree_attention", attend)
    return calls


def _greedy(one, prompt, steps, cuda):
    """The other decoder's tokens after a prompt."""
    one.prefill(torch.tensor(prompt, dtype=torch.int32, device=cuda), order="tiled" if len(prompt) >= 16 else "lane8")
    toks = [int(one.tokens[0])]
    for _ in range(steps):
        one.step()
        toks.append(int(one.tokens[0]))
    return toks


def test_tree_checks():
    from conftest import import_qvl
    qvl = import_qvl()
    import qvl_b200.drafting as F
    assert F.check_tree([5, 6, 7, 8], [-1, 0, 0, 2], 10) == [0, 1, 1, 2]
    for tokens, parents in (([], []), ([1], [0]), ([1, 2], [-1, -1]), ([1, 2], [-1, 1]), ([1, 10], [-1, 0]), ([1, 2], [-1]),
                            ([-1], [-1]), ([1] * 257, list(range(-1, 256)))):
        with pytest.raises(qvl.QvlError):
            F.check_tree(tokens, parents, 10)


def test_accepted_path():
    from conftest import import_qvl
    import_qvl()
    import qvl_b200.drafting as F
    # two children with the greedy token: the first; a match below a rejected node does not count
    assert F.accepted_path([1, 2, 3, 4, 4, 9], [-1, 0, 0, 1, 2, 4], [3, 7, 4, 0, 9, 5]) == [0, 2, 4, 5]
    assert F.accepted_path([1, 2, 3], [-1, 0, 1], [9, 3, 1]) == [0]
    assert F.accepted_path([1], [-1], [1]) == [0]


@pytest.mark.gpu
def test_tree_decoding_equals_token_by_token(qvl, cuda, monkeypatch):
    """Three requests, prompts of 70, 1 and 300 tokens (two chunks), trees with the true
    continuation hidden among wrong branches, and drafts that go wrong."""
    D, F, cfg, w, one = _setup(qvl, cuda, seed=33)
    prompts = {0: [(7 * i + 3) % cfg.vocab for i in range(70)], 1: [17], 3: [(11 * i + 5) % cfg.vocab for i in range(300)]}
    tree = F.TreeDecoder(w, max_requests=4, max_ctx=320, num_pages=12, max_tokens=400, device=cuda)
    calls = _checked(F, monkeypatch)
    first = tree.extend(prompts)
    assert tree.lengths == [70, 1, 0, 300]
    want, cache = {}, {}
    for s in prompts:
        want[s] = _greedy(one, prompts[s], 9, cuda)
        pt = one.kv[0].page_table[0].long()
        cache[s] = [c[pt].float().transpose(0, 1).reshape(cfg.kv_heads, -1, cfg.head_dim).cpu().numpy()
                    for c in (one.kv[0].k, one.kv[0].v)]
        assert first[s] == want[s][0]
    done = {s: 1 for s in prompts}          # tokens chosen so far
    last = {s: want[s][0] for s in prompts}
    for good in (3, 0, 2):                  # how much of the draft is right
        trees, roots, base = {}, [], 0
        for s in sorted(prompts):
            n = done[s]
            true = want[s][n:n + good]
            # wrong siblings first, so that the accepted nodes do not lie side by side
            toks, par, at = [last[s]], [-1], 0
            for t in true:
                toks += [(t + 1) % cfg.vocab, t]
                par += [at, at]
                at = len(toks) - 1
            toks += [(want[s][n + good] + 2) % cfg.vocab] * 2
            par += [at, len(toks) - 2]
            trees[s] = (toks, par)
            roots.append(base)
            base += len(toks)
        got = tree.verify(trees, top_k=3)
        for b, s in zip(roots, sorted(prompts)):
            n, a = done[s], got[s]
            assert a.tokens == want[s][n:n + good + 1], (s, good)
            x = tree.logits[b].double().cpu()
            lse = torch.logsumexp(x, 0)
            assert abs(a.logprobs[0] - float(x.max() - lse)) < 1e-5 * max(1.0, float(x.abs().max()))
            assert a.top_ids[0, 0] == a.tokens[0] and a.top_logprobs[0, 0] == a.logprobs[0]
            done[s] += good + 1
            last[s] = a.tokens[-1]
    assert calls[0] == 2 * (2 + 3)
    assert tree.lengths == [70 + 8, 1 + 8, 0, 300 + 8]
    # the pool: each request's pages, the rest free, no page twice
    held = [-(-n // 64) for n in tree.lengths]
    table, free = tree.page_table.cpu().numpy(), tree.free_pages[:int(tree.free_count)].tolist()
    used = [int(p) for s in range(4) for p in table[s, :held[s]]]
    assert sorted(used + free) == list(range(12))
    for s in prompts:
        L = tree.lengths[s]
        pt = torch.from_numpy(table[s, :held[s]]).long().to(cuda)
        for c, ref in zip((tree.k_all[0], tree.v_all[0]), cache[s]):
            x = c[pt].float().transpose(0, 1).reshape(cfg.kv_heads, -1, cfg.head_dim)[:, :L].cpu().numpy()
            r = ref[:, :L]
            assert (np.abs(x - r) <= 2.0 ** -10 * np.abs(r) + 2.0 ** -16 * np.abs(r).max()).all(), s
    tree.release([0, 3])
    assert int(tree.free_count) == 11 and tree.lengths == [0, 9, 0, 0]


@pytest.mark.gpu
def test_pool_out_of_pages_keeps_the_state(qvl, cuda):
    D, F, cfg, w, one = _setup(qvl, cuda, seed=5)
    tree = F.TreeDecoder(w, max_requests=2, max_ctx=320, num_pages=2, max_tokens=300, device=cuda)
    first = tree.extend({0: list(range(60))})
    chain = ([first[0]] + [1] * 79, list(range(-1, 79)))
    with pytest.raises(qvl.QvlError):
        tree.verify({0: chain, 1: ([3], [-1])})
    assert tree.lengths == [60, 0] and int(tree.free_count) == 1
    want = _greedy(one, list(range(60)), 1, cuda)
    got = tree.verify({0: ([first[0]], [-1])})
    assert first[0] == want[0] and got[0].tokens == [want[1]]
    assert tree.lengths == [61, 0] and int(tree.free_count) == 1


@pytest.mark.gpu
def test_positions_with_three_axes(qvl, cuda):
    """Equal positions on all axes are text positions: the same tokens as with one axis."""
    D, F, cfg, w, one = _setup(qvl, cuda, seed=8)
    prompt = [(3 * i + 1) % cfg.vocab for i in range(20)]
    a = F.TreeDecoder(w, 1, 64, 2, max_tokens=64, device=cuda)
    b = F.TreeDecoder(w, 1, 64, 2, max_tokens=64, sections=(24, 20, 20), device=cuda)
    fa, fb = a.extend({0: prompt}), b.extend({0: prompt}, positions={0: np.tile(np.arange(20), (3, 1))})
    assert fa == fb and torch.equal(a.logits, b.logits)
    assert torch.equal(a.k_all, b.k_all)
    # an image's rows and columns differ from the text's positions
    grid = np.stack([np.zeros(20), np.arange(20) // 5, np.arange(20) % 5]).astype(np.int32)
    c = F.TreeDecoder(w, 1, 64, 2, max_tokens=64, sections=(24, 20, 20), device=cuda)
    c.extend({0: prompt}, positions={0: grid})
    assert not torch.equal(a.k_all, c.k_all) and torch.equal(a.v_all, c.v_all)


@pytest.mark.gpu
def test_tree_decoder_refusals(qvl, cuda):
    D, F, cfg, w, one = _setup(qvl, cuda, seed=8)
    t = F.TreeDecoder(w, 2, 64, 2, max_tokens=40, device=cuda)
    for call in (lambda: t.extend({0: []}), lambda: t.extend({2: [1]}), lambda: t.extend({0: [cfg.vocab]}),
                 lambda: t.extend({0: [1] * 65}), lambda: t.verify({}),
                 lambda: t.verify({0: ([1] * 41, list(range(-1, 40)))}),
                 lambda: t.verify({0: ([1, 2], [-1, 0])}, positions={0: [[0]]})):
        with pytest.raises(qvl.QvlError):
            call()
        t.release([0, 1])
    assert t.lengths == [0, 0] and int(t.free_count) == 2


@pytest.mark.gpu
def test_tokens_after_a_prompt_with_its_own_positions(qvl, cuda):
    """After an image prompt the next position is the largest one so far plus 1, for a drafted tree as for
    more of the prompt; the accepted path's depth counts, not the number of its nodes."""
    D, F, cfg, w, one = _setup(qvl, cuda, seed=8)
    prompt = [(3 * i + 1) % cfg.vocab for i in range(20)]
    grid = np.stack([np.zeros(20), np.arange(20) // 5, np.arange(20) % 5]).astype(np.int32)      # largest: 4
    a, b = (F.TreeDecoder(w, 2, 64, 4, max_tokens=64, sections=(24, 20, 20), device=cuda) for _ in range(2))
    roots = [d.extend({1: prompt}, positions={1: grid})[1] for d in (a, b)]
    assert roots[0] == roots[1]

    def same(x, y):
        assert x[1].tokens == y[1].tokens and torch.equal(a.logits, b.logits)
        assert torch.equal(a.k_all, b.k_all) and torch.equal(a.v_all, b.v_all)

    # a tree: root and two children side by side, a grandchild of the second
    tree = ([roots[0], 5, 6, 7], [-1, 0, 0, 2])
    same(a.verify({1: tree}), b.verify({1: tree}, positions={1: [[5, 6, 6, 7]] * 3}))
    kept = a.lengths[1] - 20
    # a chain whose first child is the model's own choice: two nodes at least are kept
    root = a.verify({1: ([9], [-1])})[1].tokens
    assert b.verify({1: ([9], [-1])}, positions={1: [[5 + kept]] * 3})[1].tokens == root
    chain = ([root[0], 1], [-1, 0])
    nxt = 5 + kept + 1
    same(a.verify({1: chain}), b.verify({1: chain}, positions={1: [[nxt, nxt + 1]] * 3}))
    nxt += a.lengths[1] - 20 - kept - 1
    # more text after it, in an extend()
    assert a.extend({1: [4, 5, 6]}) == b.extend({1: [4, 5, 6]}, positions={1: [list(range(nxt, nxt + 3))] * 3})
    assert torch.equal(a.logits, b.logits) and torch.equal(a.k_all, b.k_all)
    # a request that ended and another one in its place begin at 0
    a.release([1])
    c = F.TreeDecoder(w, 2, 64, 4, max_tokens=64, sections=(24, 20, 20), device=cuda)
    assert a.extend({1: prompt[:7]}) == c.extend({1: prompt[:7]}, positions={1: np.tile(np.arange(7), (3, 1))})
    assert torch.equal(a.logits, c.logits)


@pytest.mark.gpu
def test_positions_outside_the_rotary_table_are_refused(qvl, cuda):
    """The table has max_ctx rows; a token outside it would get no query and no place in the cache."""
    D, F, cfg, w, one = _setup(qvl, cuda, seed=8)
    t = F.TreeDecoder(w, 1, 64, 2, max_tokens=64, sections=(24, 20, 20), device=cuda)
    good = np.tile(np.arange(5), (3, 1))
    for axis, at, value in ((0, 4, 64), (2, 0, -1), (1, 2, 2 ** 31 - 1)):
        bad = good.copy()
        bad[axis, at] = value
        with pytest.raises(qvl.QvlError):
            t.extend({0: [1, 2, 3, 4, 5]}, positions={0: bad})
        with pytest.raises(qvl.QvlError):
            t.verify({0: ([1, 2, 3, 4, 5], [-1, 0, 1, 2, 3])}, positions={0: bad})
    assert t.lengths == [0] and int(t.free_count) == 2
    t.extend({0: [1, 2, 3, 4, 5]}, positions={0: good + 59})       # up to the table's last row
    with pytest.raises(qvl.QvlError):
        t.verify({0: ([1], [-1])})
    assert t.lengths == [5]


@pytest.mark.gpu
def test_a_refused_prompt_leaves_nothing_behind(qvl, cuda):
    """What is wrong with a prompt, or with one of several, in a chunk after the first as well: lengths and
    pool are as they were, and the requests go on as if nothing had been asked."""
    D, F, cfg, w, one = _setup(qvl, cuda, seed=8)
    a, b = (F.TreeDecoder(w, 3, 256, 4, max_tokens=40, device=cuda) for _ in range(2))
    assert a.extend({1: [5, 6, 7]}) == b.extend({1: [5, 6, 7]})
    v = cfg.vocab
    long = [1] * 50
    for call in (lambda: a.extend({0: [1] * 257}), lambda: a.extend({1: [1] * 254}), lambda: a.extend({0: long + [v]}),
                 lambda: a.extend({0: [1] * 45, 2: [1] * 30 + [-1]}), lambda: a.extend({0: long, 3: [1]}),
                 lambda: a.extend({0: [1] * 60, 2: []}), lambda: a.extend({-1: [1], 0: [1]}),
                 lambda: a.extend({0: long}, positions={0: [list(range(49))]}),
                 lambda: a.extend({0: long}, positions={0: [list(range(50))] * 2}),
                 lambda: a.extend({0: long}, positions={0: [list(range(49)) + [256]]}),
                 # pages: the second chunk of one, and the second of two, find none
                 lambda: a.extend({0: [1] * 193}), lambda: a.extend({0: [1] * 129, 2: [1] * 30}),
                 lambda: a.verify({0: ([1] * 40, list(range(-1, 39))), 3: ([1], [-1])})):
        with pytest.raises(qvl.QvlError):
            call()
        assert a.lengths == [0, 3, 0] and int(a.free_count) == 3
    prompt = [(5 * i + 2) % v for i in range(70)]
    assert a.extend({0: prompt, 1: [9]}) == b.extend({0: prompt, 1: [9]})
    assert a.lengths == b.lengths == [70, 4, 0] and torch.equal(a.logits, b.logits)
    tree = {0: ([3, 4], [-1, 0]), 1: ([8], [-1])}
    x, y = a.verify(tree), b.verify(tree)
    assert [x[s].tokens for s in x] == [y[s].tokens for s in y] and torch.equal(a.logits, b.logits)
