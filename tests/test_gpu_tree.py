"""Verify steps over trees of drafted tokens: the conv and the gated delta rule of every
node, and the accepted paths' way into the pools, against 64-bit forms that keep a state
per node; chains against the token-by-token calls; steps in a row, in a captured graph
and through the mixer."""
import pytest
import torch

import tree_ref as ref
from helpers import BF16

pytestmark = pytest.mark.gpu


def _inputs(gen, B, T, Hk, Hv, D, slow=False):
    C = 2 * Hk * D + Hv * D
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16)  # noqa: E731
    g = -torch.nn.functional.softplus(torch.randn(B, T, Hv, generator=gen)) * (0.02 if slow else 2.0)
    return dict(y=n(B, T, C), x=n(B, T, C), g=g, beta=torch.sigmoid(torch.randn(B, T, Hv, generator=gen)).to(BF16),
                u=torch.randn(B, T, Hv, D, generator=gen) * 0.5)


def _qkv(y, Hk, Hv, D):
    kd = Hk * D
    return (y[..., :kd].unflatten(-1, (Hk, D)), y[..., kd:2 * kd].unflatten(-1, (Hk, D)),
            y[..., 2 * kd:].unflatten(-1, (Hv, D)))


def _close(got, want, bound, tag):
    d = (got.detach().cpu().double() - want).abs()
    worst = float((d / bound.clamp(min=1e-300)).max()) if d.numel() else 0.0
    assert bool((d <= bound).all()), f"{tag}: max |diff| / bound {worst:.2f}"


# one node, chains, bushy trees, the most nodes; one and several value heads per key head; both head dims
RULE = [(1, 1, 1, 1, 128, 1), (2, 2, 2, 4, 128, 1), (3, 8, 2, 2, 128, 3), (2, 16, 1, 4, 128, 4), (3, 17, 2, 2, 64, 2),
        (1, 33, 1, 2, 128, 1), (2, 48, 2, 2, 128, 8), (1, 64, 1, 1, 128, 1), (2, 64, 2, 2, 64, 5), (5, 7, 1, 3, 64, 2)]


@pytest.mark.parametrize("B,T,Hk,Hv,D,back", RULE)
@pytest.mark.parametrize("pending", [False, True])
@pytest.mark.parametrize("slow", [False, True])
def test_rule_against_a_state_per_node(pkg, dev, B, T, Hk, Hv, D, back, pending, slow):
    gen = torch.Generator().manual_seed(1000 * B + T + Hv + 7 * pending)
    i, last = _inputs(gen, B, T, Hk, Hv, D, slow), _inputs(gen, B, T + 3 if T + 3 <= 64 else T, Hk, Hv, D, slow)
    parents, _ = ref.tree(gen, B, T, back, ragged=B > 1)
    last_parents, accepted = ref.tree(gen, B, last["y"].shape[1], back, ragged=True)
    slots = B + 2
    pool = torch.randn(slots, 2, Hv, D, D, generator=gen) * 0.3          # two layers: strided slots
    ids = torch.randperm(slots, generator=gen)[:B]
    pool_d = pool.to(dev)
    q, k, v = _qkv(i["y"].to(dev), Hk, Hv, D)
    last_k = _qkv(last["y"], Hk, Hv, D)[1]
    pend = tuple(t.to(dev) for t in (last_k, last["g"], last["u"], last_parents, accepted)) if pending else None
    o, u = pkg.recurrent_gdn_tree(q, k, v, i["g"].to(dev), i["beta"].to(dev), pool_d[:, 1], ids.to(dev),
                                  parents.to(dev), pending=pend)
    torch.cuda.synchronize()
    after = pool_d.cpu()
    q, k, v = _qkv(i["y"], Hk, Hv, D)
    for b in range(B):
        S, extra = pool[ids[b], 1].double(), torch.zeros(Hv, D, D, dtype=torch.float64)
        if pending and accepted[b] >= 0:
            S, extra = ref.advanced(S, last_k[b], last["g"][b], last["u"][b], last_parents[b], int(accepted[b]))
            _close(after[ids[b], 1], S, extra, f"row {b}: state")
            S = after[ids[b], 1].double()      # the tree starts from the state as it was stored
        else:
            assert torch.equal(after[ids[b], 1], pool[ids[b], 1])
        ro, ru, _, eo, eu = ref.rule(q[b], k[b], v[b], i["g"][b], i["beta"][b], S, parents[b])
        _close(u[b], ru, eu, f"row {b}: u")
        _close(o[b], ro, eo + ref.HALF_BF16 * (ro.abs() + eo) + 1e-30, f"row {b}: o")
    others = [s for s in range(slots) if s not in ids.tolist()]
    assert torch.equal(after[others], pool[others]) and torch.equal(after[:, 0], pool[:, 0])


def test_rule_states_follow_from_u(pkg, dev):
    """commit_tree's state after any node is the 64-bit state of that node."""
    gen = torch.Generator().manual_seed(5)
    B, T, Hk, Hv, D = 4, 13, 2, 4, 128
    i = _inputs(gen, B, T, Hk, Hv, D)
    parents, _ = ref.tree(gen, 1, T, 3)
    parents = parents.expand(B, T).contiguous()
    pool = torch.randn(B, Hv, D, D, generator=gen) * 0.3
    ids = torch.arange(B)
    q, k, v = _qkv(i["y"].to(dev), Hk, Hv, D)
    gd = i["g"].to(dev)
    o, u = pkg.recurrent_gdn_tree(q, k, v, gd, i["beta"].to(dev), pool.to(dev), ids.to(dev), parents[0].to(dev))
    conv_pool = torch.zeros(B, i["x"].shape[2], 3, dtype=BF16, device=dev)
    nodes = torch.tensor([0, 5, T - 1, 7])
    got = pool.to(dev)
    pkg.commit_tree(got, conv_pool, ids.to(dev), parents.to(dev), nodes.to(dev), i["x"].to(dev), k, gd, u)
    torch.cuda.synchronize()
    qc, kc, vc = _qkv(i["y"], Hk, Hv, D)
    for b in range(B):
        _, ru, states, _, eu = ref.rule(qc[b], kc[b], vc[b], i["g"][b], i["beta"][b], pool[b], parents[b])
        P, A, depth = states[int(nodes[b])]
        bound = (2 * D + 3 * T + 64) * (depth + 2) * ref.U32 * A
        _close(got[b], P, bound, f"row {b}")


@pytest.mark.parametrize("B,T,C,back", [(1, 1, 64, 1), (3, 5, 384, 2), (2, 16, 1032, 4), (1, 64, 8192, 1), (7, 33, 200, 6),
                                        (25, 18, 8192, 3), (40, 64, 6152, 30), (1600, 4, 96, 2), (1600, 11, 96, 4)])
@pytest.mark.parametrize("pending", [False, True])
def test_conv_against_64_bits(pkg, dev, B, T, C, back, pending):
    gen = torch.Generator().manual_seed(B + T + C)
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16)  # noqa: E731
    slots = B + 3
    x, last_x, pool, w = n(B, T, C), n(B, min(64, T + 2), C), n(slots, 2, C, 3), n(C, 4)
    parents, _ = ref.tree(gen, B, T, back, ragged=B > 1)
    last_parents, accepted = ref.tree(gen, B, last_x.shape[1], back, ragged=True)
    ids = torch.randperm(slots, generator=gen)[:B]
    pool_d = pool.to(dev)
    pend = tuple(t.to(dev) for t in (last_x, last_parents, accepted)) if pending else None
    y = pkg.conv_tree_step(x.to(dev), pool_d[:, 1], ids.to(dev), w.to(dev), parents.to(dev), pending=pend)
    torch.cuda.synchronize()
    after = pool_d.cpu()
    want_pool = pool.clone()
    for b in range(B):
        if pending and accepted[b] >= 0:
            want_pool[ids[b], 1] = ref.taps_after(pool[ids[b], 1], last_x[b], last_parents[b], int(accepted[b]))
        ry, e = ref.conv(x[b], want_pool[ids[b], 1], w, parents[b])
        _close(y[b], ry, e, f"row {b}")
    assert torch.equal(after.view(torch.int16), want_pool.view(torch.int16))


@pytest.mark.parametrize("T,Hk,Hv,D", [(6, 2, 4, 128), (9, 2, 2, 64)])
def test_a_chain_is_the_decode_steps(pkg, dev, T, Hk, Hv, D):
    """A chain's conv rows are conv_decode_step's one after the other, bit for bit, and its
    outputs and final state those of recurrent_gdn_multitoken up to fp32's rounding."""
    gen = torch.Generator().manual_seed(T)
    B = 3
    C = 2 * Hk * D + Hv * D
    i = _inputs(gen, B, T, Hk, Hv, D)
    w = torch.randn(C, 4, generator=gen).to(BF16).to(dev)
    conv_pool = torch.randn(B, C, 3, generator=gen).to(BF16).to(dev)
    pool = (torch.randn(B, Hv, D, D, generator=gen) * 0.3).to(dev)
    pool_before = pool.clone()
    ids = torch.tensor([2, 0, 1], device=dev)
    chain = torch.arange(-1, T - 1, device=dev)
    x, g, beta = i["x"].to(dev), i["g"].to(dev), i["beta"].to(dev)
    y = pkg.conv_tree_step(x, conv_pool, ids, w, chain)
    step_pool = conv_pool.clone()
    steps = torch.stack([pkg.conv_decode_step(x[:, t].contiguous(), step_pool, ids, w) for t in range(T)], 1)
    q, k, v = _qkv(y, Hk, Hv, D)
    o, u = pkg.recurrent_gdn_tree(q, k, v, g, beta, pool, ids, chain)
    chain_pool = pool.clone()
    want = pkg.recurrent_gdn_multitoken(q, k, v, g, beta, chain_pool, ids)
    all_of_it = torch.full((B,), T - 1, device=dev)
    pkg.commit_tree(pool, conv_pool, ids, chain, all_of_it, x, k, g, u)
    torch.cuda.synchronize()
    assert torch.equal(y.view(torch.int16), steps.view(torch.int16))
    assert torch.equal(conv_pool.float(), step_pool.float())
    # two fp32 evaluations, each within the 64-bit form's bounds
    before = pool_before.cpu()
    for n in range(B):
        ro, _, states, eo, _ = ref.rule(*(t[n].cpu() for t in (q, k, v, g, beta)), before[ids[n]], chain.cpu())
        bound = eo + ref.HALF_BF16 * (ro.abs() + eo)
        _close(o[n], ro, bound, "tree o")
        _close(want[n], ro, bound, "multitoken o")
        P, A, depth = states[T - 1]
        bound = (2 * D + 3 * T + 64) * (depth + 2) * ref.U32 * A
        _close(pool[ids[n]], P, bound, "tree state")
        _close(chain_pool[ids[n]], P, bound, "multitoken state")


def test_unused_nodes_ids_out_of_range_and_nothing_accepted(pkg, dev):
    """Links that lead nowhere, slots that are none and accepted nodes that are none: zeros
    out, pools as they were, the other rows as without them."""
    gen = torch.Generator().manual_seed(11)
    B, T, Hk, Hv, D, slots = 6, 9, 1, 2, 128, 7
    C = 2 * Hk * D + Hv * D
    i, last = _inputs(gen, B, T, Hk, Hv, D), _inputs(gen, B, T, Hk, Hv, D)
    parents, _ = ref.tree(gen, B, T, 3)
    parents[1] = torch.tensor([-1, 0, 7, 2, -2, 4, 1, -5, 200])     # 2 waits on 7, 3 on 2; 4 unused, 5 on 4; -5, 200
    parents[2] = -2                                                # no node at all
    parents[3, 0] = 0                                              # its own parent: the whole tree hangs on it
    ids = torch.tensor([3, 5, 0, 1, -1, slots])
    accepted = torch.tensor([-1, 3, 4, T, 2, 2])                   # 3 of row 1 is unused; row 2's tree below is whole
    last_parents = parents.clone()
    last_parents[2] = torch.arange(-1, T - 1)
    pool = torch.randn(slots, Hv, D, D, generator=gen)
    conv_pool = torch.randn(slots, C, 3, generator=gen).to(BF16)
    w = torch.randn(C, 4, generator=gen).to(BF16)
    pd, cd = pool.to(dev), conv_pool.to(dev)
    dv = lambda *ts: tuple(t.to(dev) for t in ts)  # noqa: E731
    last_k = _qkv(last["y"], Hk, Hv, D)[1]
    y = pkg.conv_tree_step(*dv(i["x"]), cd, *dv(ids, w, parents), pending=dv(last["x"], last_parents, accepted))
    o, u = pkg.recurrent_gdn_tree(*_qkv(*dv(i["y"]), Hk, Hv, D), *dv(i["g"], i["beta"]), pd, *dv(ids, parents),
                                  pending=dv(last_k, last["g"], last["u"], last_parents, accepted))
    torch.cuda.synchronize()
    y, o, u, pc, cc = y.cpu(), o.cpu(), u.cpu(), pd.cpu(), cd.cpu()
    assert ref.used(parents[1].tolist()) == [True, True, False, False, False, False, True, False, False]
    for b in range(B):
        ok = torch.tensor(ref.used(parents[b].tolist())) & (0 <= int(ids[b]) < slots)
        for t in (y[b], o[b], u[b]):
            assert bool((t[~ok] == 0).all()) and (not ok.any() or bool((t[ok] != 0).any()))
    keep = [s for s in range(slots) if s != 0]                     # row 2 alone committed (slot 0)
    assert torch.equal(pc[keep], pool[keep]) and torch.equal(cc[keep], conv_pool[keep])
    S, e = ref.advanced(pool[0], last_k[2], last["g"][2], last["u"][2], last_parents[2], 4)
    _close(pc[0], S, e, "row 2")
    assert torch.equal(cc[0], ref.taps_after(conv_pool[0], last["x"][2], last_parents[2], 4))
    # the same through commit_tree
    p2, c2 = pool.to(dev), conv_pool.to(dev)
    pkg.commit_tree(p2, c2, *dv(ids, last_parents, accepted, last["x"], last_k, last["g"], last["u"]))
    torch.cuda.synchronize()
    assert torch.equal(c2.cpu(), cc) and torch.equal(p2.cpu()[keep], pool[keep])
    _close(p2.cpu()[0], S, e, "row 2 by commit_tree")


def test_extreme_decays(pkg, dev):
    """g of -inf (all forgotten), of -1e4 and of 0: no NaN, the 64-bit values."""
    gen = torch.Generator().manual_seed(13)
    B, T, Hk, Hv, D = 2, 12, 1, 2, 128
    i = _inputs(gen, B, T, Hk, Hv, D)
    g = i["g"]
    g[0, 3], g[0, 7], g[1, 5], g[1, 1] = float("-inf"), -1e4, 0.0, -200.0
    parents = torch.arange(-1, T - 1, dtype=torch.int32)
    pool = torch.randn(B, Hv, D, D, generator=gen)
    q, k, v = _qkv(i["y"], Hk, Hv, D)
    o, u = pkg.recurrent_gdn_tree(*_qkv(i["y"].to(dev), Hk, Hv, D), g.to(dev), i["beta"].to(dev), pool.to(dev),
                                  torch.arange(B, device=dev), parents.to(dev))
    torch.cuda.synchronize()
    for b in range(B):
        ro, ru, _, eo, eu = ref.rule(q[b], k[b], v[b], g[b], i["beta"][b], pool[b], parents)
        _close(u[b], ru, eu, "u")
        _close(o[b], ro, eo + ref.HALF_BF16 * (ro.abs() + eo), "o")


def _mixer(pkg, gen, dev, weights, Hk, Hv, D, hidden):
    C, V = 2 * Hk * D + Hv * D, Hv * D
    n = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).to(BF16).to(dev)  # noqa: E731
    ws = [n(r, hidden, std=hidden ** -0.5) for r in (C, V, Hv, Hv)] + [n(hidden, V, std=V ** -0.5)]
    return pkg.GatedDeltaNetLayer(*ws, Hk, Hv, D, n(C, 4, std=0.5), n(Hv), n(Hv), n(D, std=0.1) + 1, weights=weights)


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
@pytest.mark.parametrize("Hk,Hv,D,hidden", [(2, 16, 128, 256), (8, 16, 64, 256)])  # (bf16 rows of 16-byte pieces)
def test_mixer_steps_in_a_row(pkg, dev, weights, Hk, Hv, D, hidden):
    """Three verify steps through the mixer, each committing the one before, then a commit
    and a plain decode step: every node's output, the pools and the decode row are those of
    a second layer's plain decode steps along each path (bf16 rounding of two ways)."""
    gen = torch.Generator().manual_seed(17)
    layer = _mixer(pkg, gen, dev, weights, Hk, Hv, D, hidden)
    B, T, slots = 3, 6, 5
    C = layer.core.conv_dim
    pool = (torch.randn(slots, Hv, D, D, generator=gen) * 0.1).to(dev)
    cpool = torch.randn(slots, C, 3, generator=gen).to(BF16).to(dev)
    plain_pool, plain_cpool = pool.clone(), cpool.clone()
    ids = torch.tensor([4, 1, 2], device=dev)

    def decode(row, b, s, c):
        """One token of sequence b on scratch pools."""
        return layer.forward(row[None], torch.tensor([0, 1], dtype=torch.int32, device=dev), 1, ids[b:b + 1], c, s)[0]

    step, worst = None, 0.0
    for _ in range(3):
        hidden_rows = torch.randn(B, T, hidden, generator=gen).to(BF16).to(dev)
        parents, accepted = ref.tree(gen, B, T, 2)
        y, step = layer.verify_tree(hidden_rows, ids, cpool, pool, parents.to(dev), pending=step)
        step.accept(accepted.to(dev))
        for b in range(B):
            for t in range(T):
                s, c = plain_pool.clone(), plain_cpool.clone()
                for n in ref.path(parents[b].tolist(), t):
                    out = decode(hidden_rows[b, n], b, s, c)
                worst = max(worst, float((y[b, t].float() - out.float()).norm() / out.float().norm()))
        for b in range(B):
            for n in ref.path(parents[b].tolist(), int(accepted[b])):
                decode(hidden_rows[b, n], b, plain_pool, plain_cpool)
    layer.commit_tree(step, ids, cpool, pool)
    torch.cuda.synchronize()
    # Two evaluations in bf16 (or e4m3) of the same numbers: the projections of a row differ
    # by a rounding now and then, each of relative 2^-8 (2^-4) on some of the values; the mixer's
    # output is a sum over hundreds of them.
    assert worst < (2e-2 if weights == "bf16" else 6e-2), worst
    rel = float((pool - plain_pool).norm() / plain_pool.norm())
    assert rel < (1e-2 if weights == "bf16" else 3e-2), rel
    assert float((cpool.float() - plain_cpool.float()).norm() / plain_cpool.float().norm()) < 1e-2
    untouched = [0, 3]
    assert torch.equal(pool[untouched], plain_pool[untouched]) and torch.equal(cpool[untouched], plain_cpool[untouched])


def test_pending_is_commit_then_verify(pkg, dev):
    """A verify with the last step pending is commit_tree followed by one without."""
    gen = torch.Generator().manual_seed(19)
    B, T, Hk, Hv, D = 5, 16, 2, 4, 128
    C = 2 * Hk * D + Hv * D
    core = pkg.GatedDeltaNetCore(Hk, Hv, D, torch.randn(C, 4, generator=gen).to(BF16).to(dev),
                                 *(torch.randn(Hv, generator=gen).to(BF16).to(dev) for _ in range(2)),
                                 torch.ones(D, dtype=BF16, device=dev))
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16).to(dev)  # noqa: E731
    s1 = (torch.randn(B + 1, Hv, D, D, generator=gen) * 0.1).to(dev)
    c1 = n(B + 1, C, 3)
    s2, c2 = s1.clone(), c1.clone()
    ids = torch.randperm(B + 1, generator=gen)[:B].to(dev)
    rows = [(n(B, T, C), n(B, T, Hv * D), n(B, T, Hv), n(B, T, Hv)) for _ in range(2)]
    trees = [ref.tree(gen, B, T, 3, ragged=True) for _ in range(2)]
    _, step = core.verify_tree(*rows[0], ids, c1, s1, trees[0][0].to(dev))
    step.accept(trees[0][1].to(dev))
    got, after = core.verify_tree(*rows[1], ids, c1, s1, trees[1][0].to(dev), pending=step)
    core.commit_tree(step, ids, c2, s2)
    want, other = core.verify_tree(*rows[1], ids, c2, s2, trees[1][0].to(dev))
    torch.cuda.synchronize()
    assert torch.equal(s1, s2) and torch.equal(c1, c2)
    assert torch.equal(got, want) and torch.equal(after.u, other.u) and torch.equal(after.k, other.k)


def test_graph_replays_equal_eager_steps(pkg, dev):
    """Two alternating verify steps captured in one graph, each committing the other's accepted
    paths, replayed with new rows, trees and accepted nodes; other work between the replays."""
    gen = torch.Generator().manual_seed(23)
    B, T, Hk, Hv, D, hidden = 4, 8, 2, 4, 128, 256
    layer = _mixer(pkg, gen, dev, "fp8", Hk, Hv, D, hidden)
    C = layer.core.conv_dim
    pool = (torch.randn(B + 1, Hv, D, D, generator=gen) * 0.1).to(dev)
    cpool = torch.randn(B + 1, C, 3, generator=gen).to(BF16).to(dev)
    ids = torch.tensor([2, 0, 4, 1], device=dev)
    hid = [torch.zeros(B, T, hidden, dtype=BF16, device=dev) for _ in range(2)]
    par = [torch.zeros(B, T, dtype=torch.int32, device=dev) for _ in range(2)]
    acc = [torch.full((B,), -1, device=dev) for _ in range(2)]

    def both(step):
        outs = []
        for n in range(2):
            y, step = layer.verify_tree(hid[n], ids, cpool, pool, par[n], pending=step)
            step.accept(acc[n])
            outs.append(y)
        return outs, step

    def load():
        for n in range(2):
            p, a = ref.tree(gen, B, T, 3, ragged=True)
            hid[n].copy_(torch.randn(B, T, hidden, generator=gen).to(BF16))
            par[n].copy_(p)
            acc[n].copy_(a)

    load()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(None)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs, step = both(None)
        layer.commit_tree(step, ids, cpool, pool)
    for _ in range(3):
        load()
        start = pool.clone(), cpool.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (*outs, pool, cpool)]
        pool.copy_(start[0])
        cpool.copy_(start[1])
        eager, step = both(None)
        layer.commit_tree(step, ids, cpool, pool)
        torch.cuda.synchronize()
        for r, e in zip(replayed, (*eager, pool, cpool)):
            assert torch.equal(r, e)


def test_other_stream(pkg, dev):
    gen = torch.Generator().manual_seed(29)
    B, T, Hk, Hv, D = 3, 10, 1, 2, 128
    i = _inputs(gen, B, T, Hk, Hv, D)
    parents, _ = ref.tree(gen, B, T, 3)
    pool = torch.randn(B, Hv, D, D, generator=gen).to(dev)
    args = (*_qkv(i["y"].to(dev), Hk, Hv, D), i["g"].to(dev), i["beta"].to(dev), pool, torch.arange(B, device=dev),
            parents.to(dev))
    want = pkg.recurrent_gdn_tree(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = pkg.recurrent_gdn_tree(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_not_finite_stays_on_its_branch(pkg, dev):
    """Infinities and NaN in the rows of some nodes, of unused ones among them: every value
    that the 64-bit form has finite is within its bound, the others are not finite."""
    gen = torch.Generator().manual_seed(31)
    B, T, Hk, Hv, D = 4, 40, 1, 2, 128
    i = _inputs(gen, B, T, Hk, Hv, D, slow=True)
    parents, _ = ref.tree(gen, B, T, 6)
    parents[:, 1::9] = 0                                 # branches from the root's child on
    parents[:, 20] = -2                                  # unused, and what follows it
    q, k, v = _qkv(i["y"], Hk, Hv, D)
    nan, inf = float("nan"), float("inf")
    k[0, 3, 0, 5], v[0, 20], k[0, 20], q[0, 9, 0, 1] = nan, nan, inf, nan
    v[1, 2, 1, 77], v[1, 18, 0, 3] = inf, nan
    i["g"][2, 7], i["beta"][2, 30, 1] = nan, nan
    k[3, 20], q[3, 20], v[3, 20], i["g"][3, 20], i["beta"][3, 20] = nan, nan, nan, nan, nan
    pool = torch.randn(B, Hv, D, D, generator=gen) * 0.3
    o, u = pkg.recurrent_gdn_tree(*_qkv(i["y"].to(dev), Hk, Hv, D), i["g"].to(dev), i["beta"].to(dev), pool.to(dev),
                                  torch.arange(B, device=dev), parents.to(dev))
    torch.cuda.synchronize()
    o, u = o.cpu().double(), u.cpu().double()
    for b in range(B):
        ro, ru, _, eo, eu = ref.rule(q[b], k[b], v[b], i["g"][b], i["beta"][b], pool[b], parents[b])
        for got, want, bound in ((u[b], ru, eu), (o[b], ro, eo + ref.HALF_BF16 * (ro.abs() + eo))):
            ok = want.isfinite()
            assert 0 < int(ok.sum()) and (b == 3) == bool(ok.all())
            assert torch.equal(got.isfinite(), ok)
            _close(got[ok], want[ok], bound[ok] + 1e-30, f"row {b}")


def test_a_decay_of_zero_forgets_what_is_not_finite(pkg, dev):
    """A state and corrections that are not finite, behind a decay of 0: outputs and committed
    states are those of the 64-bit form on a state of zeros."""
    gen = torch.Generator().manual_seed(37)
    B, T, Hk, Hv, D = 2, 19, 1, 2, 128
    i = _inputs(gen, B, T, Hk, Hv, D, slow=True)
    parents = torch.arange(-1, T - 1, dtype=torch.int32)
    parents[9] = -1                                      # a second root: 9, and the chain behind it
    q, k, v = _qkv(i["y"], Hk, Hv, D)
    i["g"][:, 9], i["g"][:, 4] = float("-inf"), float("-inf")
    v[0, 2] = float("nan")                               # a correction that node 4 forgets
    pool = torch.full((B, Hv, D, D), float("nan"))
    ids, node = torch.arange(B), torch.tensor([T - 1, 6])
    dv = lambda *ts: tuple(t.to(dev) for t in ts)  # noqa: E731
    kd = _qkv(i["y"].to(dev), Hk, Hv, D)
    pd, cd = pool.to(dev), torch.zeros(B, i["x"].shape[2], 3, dtype=BF16, device=dev)
    o, u = pkg.recurrent_gdn_tree(*kd, *dv(i["g"], i["beta"]), pd, *dv(ids, parents))
    pkg.commit_tree(pd, cd, *dv(ids, parents, node, i["x"]), kd[1], i["g"].to(dev), u)
    torch.cuda.synchronize()
    o, u, pd = o.cpu().double(), u.cpu().double(), pd.cpu()
    v = v.clone()
    v[0, 2] = 0
    for b in range(B):
        ro, ru, states, eo, eu = ref.rule(q[b], k[b], v[b], i["g"][b], i["beta"][b], torch.zeros(Hv, D, D), parents)
        seen = torch.arange(T) >= 4
        _close(u[b][seen], ru[seen], eu[seen], f"row {b}: u")
        _close(o[b][seen], ro[seen], (eo + ref.HALF_BF16 * (ro.abs() + eo))[seen], f"row {b}: o")
        assert not u[b][~seen].isfinite().any() and not o[b][~seen].isfinite().any()
        P, A, depth = states[int(node[b])]
        _close(pd[b], P, (2 * D + 3 * T + 64) * (depth + 2) * ref.U32 * A + 1e-30, f"row {b}: state")


@pytest.mark.parametrize("taps,lead", [(4, 0), (3, 2), (8, 6), (3, 1)])
def test_conv_pools_of_other_layouts(pkg, dev, taps, lead):
    """Taps that lie apart, and pools that begin in the middle of a 16- or 4-byte piece."""
    gen = torch.Generator().manual_seed(41)
    B, T, C, slots = 3, 9, 264, 4
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16)  # noqa: E731
    x, last_x, w = n(B, T, C), n(B, T, C), n(C, 4)
    parents, _ = ref.tree(gen, B, T, 3)
    accepted = torch.tensor([4, 8, 0])
    flat = n(slots * C * taps + lead)
    view = lambda t: t[lead:].view(slots, C, taps)[..., :3]  # noqa: E731
    ids = torch.tensor([2, 0, 3])
    flat_d, flat_2 = flat.to(dev), flat.to(dev)
    dv = lambda *ts: tuple(t.to(dev) for t in ts)  # noqa: E731
    y = pkg.conv_tree_step(*dv(x), view(flat_d), *dv(ids, w, parents), pending=dv(last_x, parents, accepted))
    Hv, D = 1, 64                                        # commit_tree beside a small state
    k, g, u = n(B, T, 1, D), torch.zeros(B, T, Hv), torch.zeros(B, T, Hv, D)
    pkg.commit_tree(torch.zeros(slots, Hv, D, D, device=dev), view(flat_2),
                    *dv(ids, parents, accepted, last_x, k, g, u))
    torch.cuda.synchronize()
    want = flat.clone()
    for b in range(B):
        view(want)[ids[b]] = ref.taps_after(view(want)[ids[b]], last_x[b], parents[b], int(accepted[b]))
        ry, e = ref.conv(x[b], view(want)[ids[b]], w, parents[b])
        _close(y[b], ry, e, f"row {b}")
    assert torch.equal(flat_d.cpu(), want) and torch.equal(flat_2.cpu(), want)


def test_no_sequences(pkg, dev):
    gen = torch.Generator().manual_seed(43)
    for weights in ("bf16", "fp8"):
        layer = _mixer(pkg, gen, dev, weights, 2, 16, 64, 256)
        pool, cpool = torch.ones(2, 16, 64, 64, device=dev), torch.ones(2, layer.core.conv_dim, 3, dtype=BF16, device=dev)
        none = torch.empty(0, dtype=torch.int64, device=dev)
        parents = torch.empty(0, 5, dtype=torch.int32, device=dev)
        y, step = layer.verify_tree(torch.empty(0, 5, 256, dtype=BF16, device=dev), none, cpool, pool, parents)
        y, step = layer.verify_tree(torch.empty(0, 5, 256, dtype=BF16, device=dev), none, cpool, pool, parents,
                                    pending=step.accept(none))
        layer.commit_tree(step.accept(none), none, cpool, pool)
        torch.cuda.synchronize()
        assert y.shape == (0, 5, 256) and bool((pool == 1).all()) and bool((cpool == 1).all())


def test_rows_of_a_slot_that_is_read_only_twice(pkg, dev):
    """The same slot in several rows, with nothing accepted in all but one of them."""
    gen = torch.Generator().manual_seed(47)
    B, T, Hk, Hv, D = 4, 6, 1, 2, 128
    i, last = _inputs(gen, B, T, Hk, Hv, D), _inputs(gen, B, T, Hk, Hv, D)
    parents, _ = ref.tree(gen, B, T, 2)
    pool = torch.randn(2, Hv, D, D, generator=gen) * 0.3
    ids, accepted = torch.tensor([1, 0, 0, 0]), torch.tensor([3, -1, -1, -1])
    dv = lambda *ts: tuple(t.to(dev) for t in ts)  # noqa: E731
    pd = pool.to(dev)
    kk = _qkv(last["y"], Hk, Hv, D)[1]
    o, _ = pkg.recurrent_gdn_tree(*_qkv(i["y"].to(dev), Hk, Hv, D), *dv(i["g"], i["beta"]), pd, *dv(ids, parents),
                                  pending=dv(kk, last["g"], last["u"], parents, accepted))
    torch.cuda.synchronize()
    assert torch.equal(pd[0].cpu(), pool[0])
    q, k, v = _qkv(i["y"], Hk, Hv, D)
    for b in range(B):
        ro, _, _, eo, _ = ref.rule(q[b], k[b], v[b], i["g"][b], i["beta"][b], pd[ids[b]].cpu(), parents[b])
        _close(o[b], ro, eo + ref.HALF_BF16 * (ro.abs() + eo), f"row {b}")


def _layer_inputs(gen, B, T, Hk, Hv, D, f32=False):
    """What stands around the rule in the layer: b, a, A_log, dt_bias, z's rows among 16 others, w."""
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16)  # noqa: E731
    params = [torch.randn(Hv, generator=gen) for _ in range(2)]
    return (n(B, T, Hv), n(B, T, Hv), *(p if f32 else p.to(BF16) for p in params), n(B, T, Hv * D + 16),
            (1 + 0.1 * torch.randn(D, generator=gen)).to(BF16))


@pytest.mark.parametrize("B,T,Hk,Hv,D,back", RULE)
@pytest.mark.parametrize("pending", [False, True])
def test_rule_with_gates_and_norm_is_the_three_calls(pkg, dev, B, T, Hk, Hv, D, back, pending):
    """Bit for bit on used nodes, zeros on the others and on rows of a slot that is none."""
    gen = torch.Generator().manual_seed(7 * B + T + Hv + pending)
    i, last = _inputs(gen, B, T, Hk, Hv, D), _inputs(gen, B, T, Hk, Hv, D)
    b, a, A_log, dt, z, w = (t.to(dev) for t in _layer_inputs(gen, B, T, Hk, Hv, D, f32=T % 2 == 0))
    z = z[..., 8:-8]
    parents, _ = ref.tree(gen, B, T, back, ragged=B > 1)
    last_parents, accepted = ref.tree(gen, B, T, back, ragged=True)
    pools = [(torch.randn(B + 1, Hv, D, D, generator=torch.Generator().manual_seed(3)) * 0.3).to(dev) for _ in range(3)]
    ids = torch.randperm(B + 1, generator=gen)[:B]
    if B > 2:
        ids[1] = -1
    q, k, v = _qkv(i["y"].to(dev), Hk, Hv, D)
    pend = (tuple(t.to(dev) for t in (_qkv(last["y"], Hk, Hv, D)[1], last["g"], last["u"], last_parents, accepted))
            if pending else None)
    ids, par = ids.to(dev), parents.to(dev)
    g, beta = pkg.fused_g_beta(b, a, A_log, dt, None)
    o, u = pkg.recurrent_gdn_tree(q, k, v, g, beta, pools[0], ids, par, pending=pend)
    want = pkg.rms_norm_gated(o, z.reshape(B, T, Hv, D), w, 1e-6)
    on = torch.tensor([ref.used(p.tolist()) for p in parents], device=dev) & (ids >= 0)[:, None]

    def same(got, ref_, tag):
        assert torch.equal(got[on].contiguous().view(torch.uint8), ref_[on].contiguous().view(torch.uint8)), tag
        assert bool((got[~on].float() == 0).all()), tag

    y, u1, g1 = pkg.recurrent_tree_fused(q, k, v, b, a, A_log, dt, z, w, pools[1], ids, par, pending=pend)
    same(y, want, "y")
    same(u1, u, "u")
    assert torch.equal(g1[ids >= 0], g[ids >= 0]) and bool((g1[ids < 0] == 0).all())
    assert torch.equal(pools[0], pools[1])
    if D == 128:
        want, ws = pkg.rms_norm_gated_fp8(o, z.reshape(B, T, Hv, D), w, 1e-6)
        (y, ys), u2, g2 = pkg.recurrent_tree_fused(q, k, v, b, a, A_log, dt, z, w, pools[2], ids, par, pending=pend,
                                                   fp8=True)
        same(y, want, "y8")
        assert torch.equal(ys.view(B, T, Hv)[on], ws.view(B, T, Hv)[on]) and ys.shape == ws.shape
        assert torch.equal(u1, u2) and torch.equal(g1, g2) and torch.equal(pools[0], pools[2])
    torch.cuda.synchronize()


def test_rule_with_gates_and_norm_where_not_finite(pkg, dev):
    """A NaN in one head of one sequence: its rows are not finite in the norm, the other rows
    are those of the separate calls, bit for bit elsewhere and within rounding in that head
    (the rule takes another order of sums there)."""
    gen = torch.Generator().manual_seed(59)
    B, T, Hk, Hv, D = 2, 37, 1, 2, 128
    i = _inputs(gen, B, T, Hk, Hv, D)
    b, a, A_log, dt, z, w = _layer_inputs(gen, B, T, Hk, Hv, D)
    z = z[..., 8:-8]
    parents, _ = ref.tree(gen, B, T, 5)
    parents[:, 5::7] = 0
    q, k, v = _qkv(i["y"], Hk, Hv, D)
    v[0, 3, 1, 70] = float("nan")
    pool = torch.randn(B, Hv, D, D, generator=gen) * 0.3
    dv = lambda *ts: tuple(t.to(dev) for t in ts)  # noqa: E731
    ids = torch.arange(B)
    y, u, g = pkg.recurrent_tree_fused(*_qkv(i["y"].to(dev), Hk, Hv, D), *dv(b, a, A_log, dt, z, w, pool, ids, parents))
    g0, beta = pkg.fused_g_beta(*dv(b, a, A_log, dt), None)
    o, u0 = pkg.recurrent_gdn_tree(*_qkv(i["y"].to(dev), Hk, Hv, D), g0, beta, *dv(pool, ids, parents))
    want = pkg.rms_norm_gated(o, z.to(dev).reshape(B, T, Hv, D), w.to(dev), 1e-6)
    torch.cuda.synchronize()
    y, want, o, beta, g = (t.cpu() for t in (y, want, o, beta, g))
    assert torch.equal(y[1], want[1]) and torch.equal(y[0, :, 0], want[0, :, 0])
    hit = ~o[0, :, 1].float().isfinite().all(-1)
    assert 1 < int(hit.sum()) < T - 5
    assert torch.equal(y[0, :, 1].isnan().all(-1), hit) and torch.equal(y[0, :, 1].isfinite().all(-1), ~hit)
    # both o are within eo and half a step of the 64-bit one, so 2 (eo + 2^-8 |o|) of each other; that
    # through x r w silu(z), r from the row, and three roundings of the norm on either side
    ro, _, _, eo, _ = ref.rule(q[0], k[0], v[0], g[0], beta[0], pool[0], parents[0])
    ro, eo = ro[~hit, 1], eo[~hit, 1]
    d = 2 * (eo + ref.HALF_BF16 * (ro.abs() + eo))
    r = (ro.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    zz = z.double().view(B, T, Hv, D)[0, ~hit, 1]
    gain = (w.double() * zz * torch.sigmoid(zz)).abs()
    rel = d.norm(dim=-1, keepdim=True) / ro.norm(dim=-1, keepdim=True)
    bound = r * gain * (d + ro.abs() * rel) * 1.1 + 6 * ref.HALF_BF16 * (want[0, ~hit, 1].double().abs() + r * gain * d)
    _close(y[0, ~hit, 1], want[0, ~hit, 1].double(), bound + 1e-30, "head 1")


class _NoQuick:
    def __getattr__(self, name):
        return lambda *a: None


def test_quick_and_checked_calls_agree(pkg, dev, monkeypatch):
    """The calls by way of C++ and those by way of the Python wrappers: the same bits, errors of the
    same type; memory that comes back; what the kernel does not take as it is goes the other way."""
    gen = torch.Generator().manual_seed(61)
    B, T, Hk, Hv, D, slots = 3, 9, 1, 2, 128, 5
    C = 2 * Hk * D + Hv * D
    i, last = _inputs(gen, B, T, Hk, Hv, D), _inputs(gen, B, T, Hk, Hv, D)
    parents, accepted = (t.to(dev) for t in ref.tree(gen, B, T, 3))
    ids = torch.tensor([4, 0, 2], device=dev)
    x, y, g, beta = (i[n].to(dev) for n in ("x", "y", "g", "beta"))
    q, k, v = _qkv(y, Hk, Hv, D)
    lk, lg, lu, lx = _qkv(last["y"].to(dev), Hk, Hv, D)[1], last["g"].to(dev), last["u"].to(dev), last["x"].to(dev)
    b, a, A_log, dt, z, w = (t.to(dev) for t in _layer_inputs(gen, B, T, Hk, Hv, D))
    z, cw = z[..., 8:-8], torch.randn(C, 4, generator=gen).to(BF16).to(dev)
    pend = (lk, lg, lu, parents, accepted)
    pools = (torch.randn(slots, 2, Hv, D, D, generator=gen) * 0.3, torch.randn(slots, 2, C, 3, generator=gen).to(BF16))
    x8, xs = pkg.quantize_fp8(torch.randn(40, 256, generator=gen).to(BF16).to(dev))
    w8, ws = pkg.quantize_weight_fp8(torch.randn(300, 256, generator=gen).to(BF16).to(dev))
    rows = torch.randn(5, 8, 256, generator=gen).to(BF16).to(dev)

    def run():
        s, c = (p.to(dev)[:, 1] for p in pools)
        out = [pkg.conv_tree_step(x, c, ids, cw, parents, pending=(lx, parents, accepted)),
               pkg.conv_tree_step(x, c, ids, cw, parents[0]),
               *pkg.recurrent_gdn_tree(q, k, v, g, beta, s, ids, parents, pending=pend),
               *pkg.recurrent_gdn_tree(q, k, v, g, beta, s, ids, parents)]
        y8, *rest = pkg.recurrent_tree_fused(q, k, v, b, a, A_log, dt, z, w, s, ids, parents, 1e-6, pending=pend, fp8=True)
        out += [*y8, *rest, *pkg.recurrent_tree_fused(q, k, v, b, a, A_log, dt, z, w, s, ids, parents)]
        pkg.commit_tree(s, c, ids, parents, accepted, lx, lk, lg, lu)
        out += [s, c, pkg.linear_fp8(x8, w8, ws, x_scale=xs), pkg.linear_fp8(rows, w8, ws), pkg.linear_fp8(rows[:1], w8, ws),
                *pkg.rms_norm_gated_fp8(v, v, w, 1e-6)]
        return [t.contiguous().view(torch.uint8).cpu() for t in out], [t.shape for t in out], [t.stride() for t in out]

    quick = pkg._lib.quick()
    assert quick.conv_tree(x, pools[1].to(dev)[:, 1], ids, cw, parents, None) is not None
    assert quick.linear_fp8(rows, w8, ws, None) is not None and quick.norm_fp8(v.contiguous(), v.contiguous(), w, 1e-6)
    got = run()
    before = torch.cuda.memory_allocated()
    for _ in range(50):
        pkg.recurrent_tree_fused(q, k, v, b, a, A_log, dt, z, w, pools[0].to(dev)[:, 1], ids, parents, pending=pend)
        pkg.linear_fp8(rows, w8, ws)
    assert torch.cuda.memory_allocated() == before
    # int32 ids, int64 parents, strided gates: the wrappers copy
    for bad in (quick.conv_tree(x, pools[1].to(dev)[:, 1], ids.int(), cw, parents, None),
                quick.conv_tree(x, pools[1].to(dev)[:, 1], ids, cw, parents.long(), None),
                quick.rule_tree(q, k, v, torch.cat([g, g], 2)[..., :Hv], beta, pools[0].to(dev)[:, 1], ids, parents, None),
                quick.rule_tree(q, k, v, g, beta, pools[0].to(dev)[:, 1], ids.cpu(), parents, None),
                quick.linear_fp8(rows[..., :128], w8, ws, None), quick.linear_fp8(x8, w8, ws, None)):
        assert bad is None
    with pytest.raises(pkg._lib.GDNKernelError):         # head dim 32
        pkg.recurrent_gdn_tree(q[..., :32].contiguous(), k[..., :32].contiguous(), v[..., :32].contiguous(), g, beta,
                               torch.zeros(slots, Hv, 32, 32, device=dev), ids, parents)
    monkeypatch.setattr(pkg._lib, "quick", lambda: _NoQuick())
    want = run()
    torch.cuda.synchronize()
    assert got[1] == want[1] and got[2] == want[2]
    assert all(torch.equal(p, r) for p, r in zip(got[0], want[0]))


def test_slots_past_four_gigabytes(pkg, dev):
    """Slots whose bytes begin past 2^32 (and past 2^31 values): the results of the same slots in
    small pools."""
    gen = torch.Generator().manual_seed(67)
    B, T, Hk, Hv, D = 2, 5, 16, 32, 128
    C = 2 * Hk * D + Hv * D
    slots = [2 ** 32 // (4 * Hv * D * D) + 3, 2 ** 32 // (2 * 3 * C) + 3]
    i, last = _inputs(gen, B, T, Hk, Hv, D), _inputs(gen, B, T, Hk, Hv, D)
    parents, accepted = ref.tree(gen, B, T, 2)
    accepted[:] = torch.tensor([3, 2])
    dv = lambda *ts: tuple(t.to(dev) for t in ts)  # noqa: E731
    parents, accepted = dv(parents, accepted)
    S = torch.randn(B, Hv, D, D, generator=gen) * 0.3
    taps = torch.randn(B, C, 3, generator=gen).to(BF16)
    w = torch.randn(C, 4, generator=gen).to(BF16).to(dev)
    lk = _qkv(last["y"].to(dev), Hk, Hv, D)[1]
    kk = _qkv(i["y"].to(dev), Hk, Hv, D)
    lx, lg, lu, x, g, beta = dv(last["x"], last["g"], last["u"], i["x"], i["g"], i["beta"])
    results = []
    for far in (False, True):
        n = slots if far else [B, B]
        s_pool = torch.zeros(n[0], Hv, D, D, device=dev)
        c_pool = torch.zeros(n[1], C, 3, dtype=BF16, device=dev)
        s_ids, c_ids = (torch.arange(m - B, m, device=dev) for m in n)
        s_pool[s_ids], c_pool[c_ids] = dv(S, taps)
        y = pkg.conv_tree_step(x, c_pool, c_ids, w, parents, pending=(lx, parents, accepted))
        o, u = pkg.recurrent_gdn_tree(*kk, g, beta, s_pool, s_ids, parents, pending=(lk, lg, lu, parents, accepted))
        pkg.commit_tree(s_pool, c_pool[:n[0]], s_ids, parents, accepted, x, kk[1], g, u)
        results.append([t.cpu() for t in (y, o, u, s_pool[s_ids], c_pool[c_ids], c_pool[s_ids])])
        if far:
            assert not s_pool[:8].any() and not c_pool[:8].any()
        del s_pool, c_pool
    near, far = results
    assert all(torch.equal(a, b) for a, b in zip(near[:4], far[:4]))


@pytest.mark.parametrize("C,T,accepted", [(192, 64, 63), (200, 40, 35), (8, 34, 33), (264, 64, 50)])
@pytest.mark.parametrize("taps", [3, 4])                      # (channels' taps side by side, and apart)
def test_commit_of_few_channels_and_far_nodes(pkg, dev, C, T, accepted, taps):
    """The accepted node and its path lie past the lanes that have channels: the taps bit for bit."""
    gen = torch.Generator().manual_seed(C + T)
    B, Hk, Hv, D = 3, 1, 1, 64
    n = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, cpool = n(B, T, C).to(BF16), n(B, C, taps).to(BF16)
    k, g, u = n(B, T, Hk, D).to(BF16), -n(B, T, Hv).abs(), n(B, T, Hv, D)
    pool = n(B, Hv, D, D)
    parents = torch.arange(-1, T - 1, dtype=torch.int32).expand(B, T).clone()
    parents[1, accepted] = accepted - 3
    parents[2, accepted] = -1                                 # (a root: two of the old taps stay)
    nodes = torch.full((B,), accepted)
    cd = cpool.to(dev)
    pkg.commit_tree(pool.to(dev), cd[..., :3], torch.arange(B, device=dev), parents.to(dev), nodes.to(dev), x.to(dev),
                    k.to(dev), g.to(dev), u.to(dev))
    torch.cuda.synchronize()
    want = cpool.clone()
    for b in range(B):
        want[b, :, :3] = ref.taps_after(cpool[b, :, :3], x[b], parents[b], accepted)
    assert torch.equal(cd.cpu().view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("Hk,Hv,D,fp8,timed", [(2, 4, 128, False, False), (2, 4, 128, True, False), (2, 4, 64, True, False),
                                               (2, 4, 128, True, True), (1, 1, 64, False, True)])
def test_a_refused_verify_leaves_the_pools(pkg, dev, monkeypatch, Hk, Hv, D, fp8, timed):
    """A verify whose rule is refused leaves the taps too, so that the call repeated with what was
    wrong mended is commit_tree followed by a verify (which goes through the Python wrappers)."""
    gen = torch.Generator().manual_seed(71 + D)
    B, T = 3, 7
    C = (2 * Hk + Hv) * D
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16).to(dev)  # noqa: E731
    core = pkg.GatedDeltaNetCore(Hk, Hv, D, n(C, 4), n(Hv), n(Hv), torch.ones(D, dtype=BF16, device=dev))
    if timed:
        class Timer:
            names = []
            start = lambda self, name: self.names.append(name)  # noqa: E731
            stop = lambda self, *a: None  # noqa: E731
        core.timer = Timer()
    s1, c1 = (torch.randn(B + 1, Hv, D, D, generator=gen) * 0.1).to(dev), n(B + 1, C, 3)
    ids = torch.tensor([3, 0, 2], device=dev)
    rows = [(n(B, T, C), n(B, T, Hv * D), n(B, T, Hv), n(B, T, Hv)) for _ in range(2)]
    trees = [ref.tree(gen, B, T, 3) for _ in range(2)]
    _, step = core.verify_tree(*rows[0], ids, c1, s1, trees[0][0].to(dev), fp8=fp8)
    step.accept(torch.tensor([2, -1, T - 1], device=dev))
    before = s1.clone(), c1.clone()
    x, z, b, a = rows[1]
    par = trees[1][0].to(dev)
    whole = torch.zeros(s1.numel() + 1, device=dev)[1:].view(s1.shape)      # not 16-byte aligned: the entry point's refusal
    wrong = pkg.TreeStep(step.x, step.k, step.g, step.u[..., :D // 2], step.parents, step.accepted)
    for args, pending in (((x, z[..., 8:], b, a, ids, c1, s1), step), ((x, z, b.float(), a, ids, c1, s1), step),
                          ((x, z, b, a, ids, c1, whole), step), ((x, z, b, a, ids, c1, s1[:B]), step),
                          ((x, z, b, a, ids, c1, s1), wrong)):
        with pytest.raises((ValueError, TypeError, RuntimeError, AssertionError)):
            core.verify_tree(*args, par, pending=pending, fp8=fp8)
        torch.cuda.synchronize()
        assert torch.equal(s1, before[0]) and torch.equal(c1, before[1])
    got, after = core.verify_tree(x, z, b, a, ids, c1, s1, par, pending=step, fp8=fp8)
    monkeypatch.setattr(pkg._lib, "quick", lambda: _NoQuick())
    core.commit_tree(step, ids, before[1], before[0])
    want, other = core.verify_tree(x, z, b, a, ids, before[1], before[0], par, fp8=fp8)
    torch.cuda.synchronize()
    pairs = [(s1, before[0]), (c1, before[1]), (after.u, other.u), (after.k, other.k), (after.g, other.g)]
    pairs += [(got[0].float(), want[0].float()), (got[1], want[1])] if fp8 else [(got, want)]
    assert all(torch.equal(p, r) for p, r in pairs)
    assert not timed or {"conv_tree", "recurrent_tree"} <= set(core.timer.names)


@pytest.mark.parametrize("fp8", [False, True])
def test_padded_rows_share_a_slot_of_which_nothing_is_accepted(pkg, dev, fp8):
    """The rows of a padded batch on the dummy slot, between rows that commit their last step: the
    slot stays, and every row's outputs are those that it has alone."""
    gen = torch.Generator().manual_seed(73)
    B, T, Hk, Hv, D, slots = 6, 9, 2, 4, 128, 5
    C = (2 * Hk + Hv) * D
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16).to(dev)  # noqa: E731
    core = pkg.GatedDeltaNetCore(Hk, Hv, D, n(C, 4), n(Hv), n(Hv), n(D))
    pools = (torch.randn(slots, Hv, D, D, generator=gen) * 0.1).to(dev), n(slots, C, 3)
    ids, accepted = torch.tensor([4, 1, 4, 0, 4, 4], device=dev), torch.tensor([-1, 5, -1, 2, -1, T], device=dev)
    rows = [(n(B, T, C), n(B, T, Hv * D), n(B, T, Hv), n(B, T, Hv)) for _ in range(2)]
    par = [ref.tree(gen, B, T, 3)[0].to(dev) for _ in range(2)]

    def steps(at):
        s, c = (p.clone() for p in pools)
        pick = lambda r: [t[at] for t in r]  # noqa: E731
        _, step = core.verify_tree(*pick(rows[0]), ids[at], c, s, par[0][at], fp8=fp8)
        out, after = core.verify_tree(*pick(rows[1]), ids[at], c, s, par[1][at], pending=step.accept(accepted[at]), fp8=fp8)
        return [t.float() for t in ((out[0], out[1].unflatten(0, (-1, T))) if fp8 else (out,))] + [after.u, after.k], s, c

    got, s, c = steps(slice(0, B))
    for b in range(B):
        want, s1, c1 = steps(slice(b, b + 1))
        assert all(torch.equal(g[b:b + 1], w) for g, w in zip(got, want)), b
        assert torch.equal(s[ids[b]], s1[ids[b]]) and torch.equal(c[ids[b]], c1[ids[b]])
    assert all(torch.equal(a[[2, 3, 4]], p[[2, 3, 4]]) for a, p in zip((s, c), pools))


@pytest.mark.parametrize("lead", [1, 4])
def test_conv_weight_that_begins_anywhere(pkg, dev, lead):
    """A contiguous weight that is not 16-byte aligned (a view into a flat buffer) is copied."""
    gen = torch.Generator().manual_seed(79)
    B, T, C = 2, 5, 264
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16).to(dev)  # noqa: E731
    x, pool, w = n(B, T, C), n(B, C, 3), n(C, 4)
    flat = torch.cat([n(lead), w.flatten()])[lead:].view(C, 4)
    assert flat.is_contiguous() and flat.data_ptr() % 16
    args = torch.arange(B, device=dev), torch.arange(-1, T - 1, dtype=torch.int32, device=dev)
    got, want = pkg.conv_tree_step(x, pool, args[0], flat, args[1]), pkg.conv_tree_step(x, pool, args[0], w, args[1])
    torch.cuda.synchronize()
    assert torch.equal(got, want)
