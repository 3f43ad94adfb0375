"""The mixer between its norms (GatedDeltaNetBlock) and with low-rank adapters beside its
projections (GatedDeltaNetLayer.add_adapters), as a server runs them: prompts, decode steps, verify
steps, replayed graphs.  The projections are held to 64 bits with every sequence's adapter merged into
the weights, and the whole to its parts, bit for bit."""
import pytest
import torch

from helpers import BF16, assert_state
from test_gpu_layer_proj import _weights

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _layer(pkg, dev, gen, hidden, Hk, Hv, D, weights="bf16", **kw):
    ws = _weights(gen, hidden, Hk, Hv, D)
    return pkg.GatedDeltaNetLayer(*(t.to(dev) for t in ws[1:6]), Hk, Hv, D, *(t.to(dev) for t in ws[6:]), weights=weights,
                                  **kw), ws


def _adapter(gen, layer, r):
    """(A, B) for every projection, by name; A and B so that the adapter is about as large as the projection."""
    c = layer.core
    pair = lambda rows, cols: ((torch.randn(r, cols, generator=gen) * cols ** -0.5).to(BF16),  # noqa: E731
                               (torch.randn(rows, r, generator=gen) * r ** -0.5).to(BF16))
    return dict(qkv=pair(c.conv_dim, layer.hidden), z=pair(c.value_dim, layer.hidden), b=pair(c.Hv, layer.hidden),
                a=pair(c.Hv, layer.hidden), out=pair(layer.hidden, c.value_dim))


def _state(pkg, dev, gen, layer, slots):
    c = layer.core
    return (torch.randn(slots, c.conv_dim, 3, generator=gen).to(BF16).to(dev),
            (torch.randn(slots, c.Hv, c.D, c.D, generator=gen) * 0.1).to(dev))


def _cu(lens, dev):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=I32, device=dev)


def test_layer_with_adapters_against_merged_weights(pkg, dev):
    """A decode prefix and prompts, each with an adapter, without one, or with one that has no part for
    some projections: the projections of merged weights, in 64 bits."""
    gen = torch.Generator().manual_seed(91)
    Hk = Hv = 16
    D, hidden = 128, 1024
    layer, (_, w_qkv, w_z, w_b, w_a, w_out, *_) = _layer(pkg, dev, gen, hidden, Hk, Hv, D)
    layer.add_adapters(4, 12)
    full = [_adapter(gen, layer, r) for r in (12, 5, 8)]
    part = dict(full[2], qkv=None, a=None)
    adapters = [(full[0], 0.5), (full[1], 2.0), (part, 1.0)]
    for slot, (ad, scale) in zip((0, 1, 3), adapters):
        layer.load_adapter(slot, scale, **{k: None if p is None else tuple(t.to(dev) for t in p) for k, p in ad.items()})
    of = {0: adapters[0], 1: adapters[1], 3: adapters[2]}
    lens, seq = [1, 1, 1, 130, 64, 200, 9], [1, -1, 3, 0, 7, 3, 1]        # (7: no slot; slot 2 stays empty)
    N = sum(lens)
    ids = torch.tensor([7, 2, 0, 5, 8, 3, 6])
    conv0, s0 = (t.cpu() for t in _state(pkg, dev, gen, layer, 9))
    x = torch.randn(N, hidden, generator=gen).to(BF16)
    cu = _cu(lens, dev)
    rows = pkg.adapter_rows(torch.tensor(seq, device=dev), cu, N)
    cp, sp = conv0.to(dev), s0.to(dev)
    out = layer.forward(x.to(dev), cu, max(lens), ids.to(dev), cp, sp, lens_q=lens, adapters=rows)

    def product(x, w, name, size=False):
        """x W^T with each row's adapter merged, float64; size: of the magnitudes."""
        f = (lambda t: t.double().abs()) if size else (lambda t: t.double())
        x = f(x)
        y = x @ f(w).t()
        at = 0
        for n, s in zip(lens, seq):
            if s in of and of[s][0][name] is not None:
                A, B = of[s][0][name]
                y[at:at + n] += of[s][1] * (x[at:at + n] @ f(A).t()) @ f(B).t()
            at += n
        return y

    def held(y, x, w, name):
        """Half a bf16 step, and of the magnitudes: K + R roundings of a sum (2^-24 each, doubled: under
        2^-12) and 2^-16 of the shrunk values."""
        want, size = product(x, w, name), product(x, w, name, True)
        assert bool(((y.cpu().double() - want).abs() <= 2.0 ** -8 * (want.abs() + size * 2.0 ** -12) + size * 2.0 ** -12).all()), name

    # (1) in_proj
    got = layer.project_in(x.to(dev), adapters=rows)[:4]
    for y, w, name in zip(got, (w_qkv, w_z, w_b, w_a), ("qkv", "z", "b", "a")):
        held(y, x, w, name)
    # (2) the core on these, whose rows and pools are what they are without adapters, and out_proj on its rows
    pools = conv0.to(dev), s0.to(dev)
    own = layer.core.forward(*got, cu, max(lens), ids.to(dev), *pools, lens_q=lens)
    assert torch.equal(pools[0], cp) and torch.equal(pools[1], sp)
    held(out, own.cpu(), w_out, "out")
    # rows without an adapter: those of the layer without any, up to the products' own sizes
    layer.clear_adapter(1)
    again = layer.project_in(x.to(dev), adapters=rows)[:4]
    plain = layer.project_in(x.to(dev), adapters=torch.full_like(rows, -1))[:4]
    bare = (rows != 0) & (rows != 3)
    assert all(torch.equal(p[bare], q[bare]) for p, q in zip(again, plain))


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
@pytest.mark.parametrize("sw", [{}, {"fused_prefill": False, "fused_decode": False}], ids=["fused", "unfused"])
def test_layer_with_adapters_is_its_parts(pkg, dev, weights, sw):
    """forward and verify_tree with adapters: the products with adapters around the core, bit for bit,
    the gates that the product yields among them."""
    gen = torch.Generator().manual_seed(92)
    Hk, Hv, D, hidden, S = 8, 16, 128, 512, 5
    layer, _ = _layer(pkg, dev, gen, hidden, Hk, Hv, D, weights, switches=pkg.Switches(**sw))
    layer.add_adapters(S, 16)
    for s in range(S):
        layer.load_adapter(s, 0.7, **{k: tuple(t.to(dev) for t in p) for k, p in _adapter(gen, layer, 16).items()})
    lens = [1, 1, 90, 3, 130]
    N, c = sum(lens), layer.core
    cu, ids = _cu(lens, dev), torch.tensor([4, 1, 6, 0, 3], device=dev)
    x = torch.randn(N, hidden, generator=gen).to(BF16).to(dev)
    rows = pkg.adapter_rows(torch.tensor([2, -1, 0, 4, 2], device=dev), cu, N)
    conv0, s0 = _state(pkg, dev, gen, layer, 8)
    pools = [conv0.clone(), s0.clone()], [conv0.clone(), s0.clone()]
    got = layer.forward(x, cu, max(lens), ids, *pools[0], lens_q=lens, adapters=rows)
    pin, pout = layer.lora_in, layer.lora_out
    lora, widths = (pin.a, pin.b, pin.scale, rows), [c.conv_dim, c.value_dim, Hv, Hv]
    if weights == "fp8":
        y = pkg.linear_fp8_lora(x, layer.w_in, layer.w_in_scale, *lora, widths=widths, wide=layer.w_ba)
    else:
        y = pkg.linear_lora(x, layer.w_in, *lora, widths=widths)
    core = c.forward(*y, cu, max(lens), ids, *pools[1], lens_q=lens, fp8=weights == "fp8")
    lora = pout.a, pout.b, pout.scale, rows
    if weights == "fp8":
        core, scale = core if isinstance(core, tuple) else (core, None)
        want = pkg.linear_fp8_lora(core.reshape(N, -1), layer.w_out, layer.w_out_scale, *lora, x_scale=scale)
    else:
        want = pkg.linear_lora(core, layer.w_out, *lora)
    assert torch.equal(got, want) and all(torch.equal(p, q) for p, q in zip(*pools))
    if sw:
        return
    B, T = 3, 6
    x = torch.randn(B, T, hidden, generator=gen).to(BF16).to(dev)
    rows = torch.tensor([1, -1, 3], dtype=I32, device=dev).repeat_interleave(T)
    parents = torch.arange(-1, T - 1, dtype=I32, device=dev)
    got, step = layer.verify_tree(x, ids[:B], *pools[0], parents, adapters=rows)
    y = layer.project_in(x.view(B * T, hidden), adapters=rows)[:4]
    core, other = c.verify_tree(*(t.view(B, T, -1) for t in y), ids[:B], *pools[1], parents, fp8=weights == "fp8")
    lora = pout.a, pout.b, pout.scale, rows
    if weights == "fp8":
        want = pkg.linear_fp8_lora(core[0].reshape(B, T, -1), layer.w_out, layer.w_out_scale, *lora, x_scale=core[1])
    else:
        want = pkg.linear_lora(core.reshape(B, T, -1), layer.w_out, *lora)
    assert torch.equal(got, want) and torch.equal(step.u, other.u)


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
@pytest.mark.parametrize("wide", [False, True], ids=["bf16 stream", "fp32 stream"])
@pytest.mark.parametrize("lens", [[1, 1, 1], [1, 1, 40, 300], [700, 600, 50]], ids=["decode", "mixed", "prompts"])
def test_block_is_its_parts(pkg, dev, weights, wide, lens):
    """The block: norm, mixer, norm, bit for bit, with the stream in either type; past 1024 rows of
    8-bit weights the first norm's e4m3 rows go into in_proj."""
    gen = torch.Generator().manual_seed(93)
    Hk, Hv, D, hidden = 8, 16, 128, 512
    layer, _ = _layer(pkg, dev, gen, hidden, Hk, Hv, D, weights)
    n1, n2 = ((torch.randn(hidden, generator=gen) * 0.1).to(BF16).to(dev) for _ in range(2))
    block = pkg.GatedDeltaNetBlock(layer, n1, n2, eps=1e-5)
    N, cu = sum(lens), _cu(lens, dev)
    ids = torch.tensor([4, 1, 6, 0][:len(lens)], device=dev)
    x = torch.randn(N, hidden, generator=gen).to(BF16).to(dev)
    res = torch.randn(N, hidden, generator=gen).to(torch.float32 if wide else BF16).to(dev)
    conv0, s0 = _state(pkg, dev, gen, layer, 8)
    for residual in (res, None):
        pools = [conv0.clone(), s0.clone()], [conv0.clone(), s0.clone()]
        keep = None if residual is None else residual.clone()
        got = block.forward(x, residual, cu, max(lens), ids, *pools[0], lens_q=lens)
        if weights == "fp8" and N > 1024:
            y8, scale, stream, y = pkg.add_rms_norm_fp8(x, residual, n1, 1e-5, keep=True)
            mixed, z = pkg.ops.linear_fp8_cols(y8, layer.w_in, layer.w_in_scale, [layer.core.conv_dim, layer.core.value_dim],
                                               x_scale=scale)
            b, a = pkg.linear(y, layer.w_ba).split(Hv, -1)
            core = layer.core.forward(mixed, z, b.contiguous(), a.contiguous(), cu, max(lens), ids, *pools[1], lens_q=lens, fp8=True)
            out = layer._project_out(core, x.shape)
        else:
            y, stream = pkg.add_rms_norm(x, residual, n1, 1e-5)
            out = layer.forward(y, cu, max(lens), ids, *pools[1], lens_q=lens)
        want = pkg.add_rms_norm(out, stream, n2, 1e-5)
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and all(torch.equal(p, q) for p, q in zip(*pools))
        assert got[1].dtype == (BF16 if residual is None else residual.dtype)
        assert residual is None or torch.equal(residual, keep)


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
def test_blocks_served(pkg, dev, weights):
    """Two blocks behind each other, as a server runs them: prompts with adapters, then decode steps as a
    replayed graph whose rows, adapters and slots change between the replays, an adapter loaded and
    one cleared between them, then a verify step and its commit; every step against the eager one."""
    gen = torch.Generator().manual_seed(94)
    Hk, Hv, D, hidden, S, slots = 8, 16, 128, 512, 4, 10
    blocks = []
    for _ in range(2):
        layer, _ = _layer(pkg, dev, gen, hidden, Hk, Hv, D, weights)
        layer.add_adapters(S, 16)
        norms = ((torch.randn(hidden, generator=gen) * 0.1).to(BF16).to(dev) for _ in range(2))
        blocks.append(pkg.GatedDeltaNetBlock(layer, *norms))
    loads = [[{k: tuple(t.to(dev) for t in p) for k, p in _adapter(gen, b.layer, 16).items()} for b in blocks] for _ in range(3)]

    def load(slot, which, scale):
        for block, ad in zip(blocks, loads[which]):
            block.layer.load_adapter(slot, scale, **ad)

    def run(x, cu, T, ids, pools, lens, rows):
        residual = None
        for block, (conv, s) in zip(blocks, pools):
            x, residual = block.forward(x, residual, cu, T, ids, conv, s, lens_q=lens, adapters=rows)
        return x, residual

    load(0, 0, 1.0)
    load(2, 1, 0.5)
    lens = [70, 5, 129, 64]
    N, n, cu = sum(lens), len(lens), _cu(lens, dev)
    ids = torch.tensor([7, 2, 5, 9], device=dev)
    pools = [_state(pkg, dev, gen, b.layer, slots) for b in blocks]
    copies = [tuple(t.clone() for t in p) for p in pools]
    x = torch.randn(N, hidden, generator=gen).to(BF16).to(dev)
    rows = pkg.adapter_rows(torch.tensor([0, 2, -1, 0], device=dev), cu, N)
    one, two = run(x, cu, max(lens), ids, pools, lens, rows), run(x, cu, max(lens), ids, copies, lens, rows)
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    # the decode step as a graph
    xs, at, who = torch.zeros(n, hidden, dtype=BF16, device=dev), ids.clone(), torch.full((n,), -1, dtype=I32, device=dev)
    cu1 = torch.arange(n + 1, dtype=I32, device=dev)
    side = torch.cuda.Stream(dev)
    warm = [tuple(t.clone() for t in p) for p in pools]
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        run(xs, cu1, 1, at, warm, None, who)
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, stream = run(xs, cu1, 1, at, pools, None, who)
    for step in range(4):
        if step == 2:
            load(1, 2, 2.0)
            for block in blocks:
                block.layer.clear_adapter(2)
        now = torch.randn(n, hidden, generator=gen).to(BF16).to(dev)
        seq = torch.randperm(slots, generator=gen)[:n].to(dev)
        lora = torch.tensor([[0, 2, -1, 0], [2, 2, 2, 2], [1, 2, 0, 9], [-1, -1, -1, -1]][step], dtype=I32, device=dev)
        xs.copy_(now)
        at.copy_(seq)
        who.copy_(lora)
        graph.replay()
        want = run(now, cu1, 1, seq, copies, None, lora)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(stream, want[1]), step
        assert all(torch.equal(p, q) for a, b in zip(pools, copies) for p, q in zip(a, b)), step
    # a verify step over chains, its accepted nodes committed: the decode steps of the same tokens
    B, T = 2, 4
    x = torch.randn(B, T, hidden, generator=gen).to(BF16).to(dev)
    who = torch.tensor([1, 0], dtype=I32, device=dev)
    parents = torch.arange(-1, T - 1, dtype=I32, device=dev)
    acc = torch.tensor([T - 1, -1], device=dev)
    y, residual, steps = x, None, []
    for block, pool in zip(blocks, pools):
        y, residual, step = block.verify_tree(y, residual, ids[:B], *pool, parents, adapters=who.repeat_interleave(T))
        steps.append(step.accept(acc))
    for block, pool, step in zip(blocks, pools, steps):
        block.commit_tree(step, ids[:B], *pool)
    cu1 = torch.arange(2, dtype=I32, device=dev)
    for t in range(T):
        run(x[0, t:t + 1], cu1, 1, ids[:1], copies, None, who[:1])
    torch.cuda.synchronize()
    for a, b in zip(pools, copies):
        assert torch.equal(a[1][ids[1]], b[1][ids[1]])                    # (nothing accepted: as it was)
        assert_state(a[1][ids[0]], b[1][ids[0]], "committed state")


def test_adapters_refused(pkg, dev):
    gen = torch.Generator().manual_seed(95)
    layer, _ = _layer(pkg, dev, gen, 128, 1, 1, 64)
    with pytest.raises(ValueError, match="16"):
        layer.add_adapters(2, 8)
    layer, _ = _layer(pkg, dev, gen, 128, 8, 16, 64)
    x, cu = torch.zeros(2, 128, dtype=BF16, device=dev), torch.arange(3, dtype=I32, device=dev)
    pools, ids = _state(pkg, dev, gen, layer, 4), torch.arange(2, device=dev)
    rows = torch.zeros(2, dtype=I32, device=dev)
    before = [t.clone() for t in pools]
    for call in (lambda: layer.load_adapter(0, 1.0), lambda: layer.clear_adapter(0),
                 lambda: layer.forward(x, cu, 1, ids, *pools, adapters=rows)):
        with pytest.raises(ValueError, match="add_adapters"):
            call()
    layer.add_adapters(2, 8)
    ad = {k: tuple(t.to(dev) for t in p) for k, p in _adapter(gen, layer, 8).items()}
    layer.load_adapter(1, 1.0, **ad)
    keep = [t.clone() for pool in (layer.lora_in, layer.lora_out) for t in (pool.a, pool.b, pool.scale)]
    wide = (torch.zeros(9, 1024, device=dev), torch.zeros(128, 9, device=dev))
    for bad in (dict(slot=2), dict(slot=-1), dict(slot=1, qkv=ad["z"]), dict(slot=1, **{**ad, "out": wide})):
        with pytest.raises(ValueError):
            layer.load_adapter(bad.pop("slot"), 1.0, **bad)
    now = [t for pool in (layer.lora_in, layer.lora_out) for t in (pool.a, pool.b, pool.scale)]
    assert all(torch.equal(p, q) for p, q in zip(keep, now))
    for bad in (rows.long(), rows[:1], rows.float()):
        with pytest.raises(ValueError):
            layer.forward(x, cu, 1, ids, *pools, adapters=bad)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(before, pools))
    for norms in ((torch.zeros(64), torch.zeros(128)), (torch.zeros(128), torch.zeros(1, 128))):
        with pytest.raises(ValueError):
            pkg.GatedDeltaNetBlock(layer, *norms)


@pytest.mark.parametrize("lens", [[1, 1, 40, 300], [700, 600, 50]], ids=["mixed", "prompts"])
def test_block_with_gates_from_the_product(pkg, dev, lens):
    """8-bit weights and a path that takes its gates from in_proj: the e4m3 rows of the first norm give
    the same gates as its bf16 rows."""
    gen = torch.Generator().manual_seed(96)
    Hk, Hv, D, hidden = 8, 16, 128, 512
    layer, _ = _layer(pkg, dev, gen, hidden, Hk, Hv, D, "fp8", switches=pkg.Switches(fused_prefill=False, fused_decode=False))
    assert layer.gates_in_gemm()
    n1, n2 = ((torch.randn(hidden, generator=gen) * 0.1).to(BF16).to(dev) for _ in range(2))
    block = pkg.GatedDeltaNetBlock(layer, n1, n2)
    N, cu, ids = sum(lens), _cu(lens, dev), torch.tensor([4, 1, 6, 0][:len(lens)], device=dev)
    x, res = (torch.randn(N, hidden, generator=gen).to(BF16).to(dev) for _ in range(2))
    conv0, s0 = _state(pkg, dev, gen, layer, 8)
    pools = [conv0.clone(), s0.clone()], [conv0.clone(), s0.clone()]
    y, stream = block.forward(x, res, cu, max(lens), ids, *pools[0], lens_q=lens)
    y8, scale, r, h = pkg.add_rms_norm_fp8(x, res, n1, 1e-6, keep=True)
    rows = layer.project_in(h, gates=True, fp8=(y8, scale) if N > 1024 else None)
    g, beta = pkg.fused_g_beta(rows[2].contiguous(), rows[3].contiguous(), layer.core.A_log, layer.core.dt_bias, None)
    assert torch.equal(rows[4][0], g) and torch.equal(rows[4][1], beta)
    core = layer.core.forward(*(t.contiguous() for t in rows[:4]), cu, max(lens), ids, *pools[1], lens_q=lens, gb=rows[4],
                              fp8=True)
    want = pkg.add_rms_norm(layer._project_out(core, x.shape), r, n2, 1e-6)
    assert torch.equal(y, want[0]) and torch.equal(stream, want[1]) and all(torch.equal(p, q) for p, q in zip(*pools))
