"""Projections with low-rank adapters (linear_lora, linear_fp8_lora) against 64 bits.

Tolerances.  u = 2^-24; the matrix cores add with an error of at most a rounding per product, the
partial sums with one each.  With X = |x| |A_s|^T, S = |scale|:
  v       off by 2 K u S X, and held to 2^-16 of itself (a bf16 value and the bf16 value of its rest)
  y       off by 2 (K + 2 R) u (|x| |W|^T + S X |B_s|^T) and by (2^-16 + 2 K u) S X |B_s|^T, then bf16's half step, 2^-8
8-bit products: what tree_ref.linear says of them in the first term's place."""
import pytest
import torch

import tree_ref as ref
from helpers import BF16

pytestmark = pytest.mark.gpu
F32, FP8 = torch.float32, torch.float8_e4m3fn
U, HALF = 2.0 ** -24, 2.0 ** -8


def _ids(gen, M, S, how):
    if how == "none":
        return torch.full((M,), -1, dtype=torch.int32)
    if how == "one":
        return torch.full((M,), S - 1, dtype=torch.int32)
    if how == "each":
        return (torch.arange(M) * 7 % S).to(torch.int32)
    if how == "mixed":                                       # with rows without one, by ids on both sides of the slots
        ids = torch.randint(-1, S + 1, (M,), generator=gen)
        return torch.where(torch.rand(M, generator=gen) < 0.1, torch.tensor(-(1 << 31)), ids).to(torch.int32)
    cuts = torch.randint(0, M, (max(1, M // 90),), generator=gen)    # sequences
    seq = torch.zeros(M, dtype=torch.int64).index_fill_(0, cuts, 1).cumsum(0)
    return torch.randint(-1, S, (int(seq.max()) + 1,), generator=gen)[seq].to(torch.int32)


def _adapters(gen, S, widths, K, R):
    P, N = len(widths), sum(widths)
    a = (torch.randn(S, P * R, K, generator=gen) * K ** -0.5).to(BF16)
    b = (torch.randn(S, N, R, generator=gen) * R ** -0.5).to(BF16)
    return a, b, torch.rand(S, generator=gen) * 2 + 0.25


def _delta(x, a, b, scale, ids, widths, K):
    """What the adapters add, and how far it may be off, in 64 bits on x's device; x as they read it."""
    x = x.double()
    R = b.shape[2]
    out = torch.zeros(x.shape[0], sum(widths), dtype=torch.float64, device=x.device)
    size = out.clone()
    for s in ids.unique().tolist():
        if 0 <= s < len(a):
            rows = (ids == s).nonzero()[:, 0]
            A, B = a[s].double(), b[s].double().split(widths)
            v, X = float(scale[s]) * (x[rows] @ A.t()), abs(float(scale[s])) * (x[rows].abs() @ A.abs().t())
            out[rows] = torch.cat([v[:, p * R:p * R + R] @ t.t() for p, t in enumerate(B)], 1)
            size[rows] = torch.cat([X[:, p * R:p * R + R] @ t.abs().t() for p, t in enumerate(B)], 1)
    return out, size * (2.0 ** -16 + 2 * (2 * K + 2 * R) * U)


def _check(y, want, slack, tag=""):
    d = (y.double() - want).abs()
    bound = HALF * (want.abs() + slack) + slack
    worst = float((d / bound.clamp(min=1e-300)).max()) if d.numel() else 0.0
    assert bool((d <= bound).all()), f"{tag}: max |diff| / bound {worst:.3f}"


# M, N or widths, K, R, S, ids: each kernel of the product (16, 32 and 64 rows x 32 columns, 64-row tiles, 128 x 128
# blocks, 256 x 256 tiles with and without a rest), each of the shrink, ranks below, at and past a product's depth
SHAPES = [
    (1, [2048], 2048, 16, 4, "one"), (1, [8192, 4096, 32, 32], 2048, 16, 8, "one"), (1, [16], 64, 8, 1, "one"),
    (3, [48, 16], 128, 24, 5, "each"), (5, [33], 192, 256, 3, "mixed"), (16, [2048], 4096, 8, 16, "each"),
    (17, [1000], 1152, 16, 40, "each"), (33, [2048], 2048, 32, 9, "mixed"), (37, [6144, 2048, 16, 16], 2048, 16, 37, "each"),
    (64, [8192, 4096, 32, 32], 2048, 16, 64, "each"), (64, [2048], 2048, 64, 3, "none"), (65, [512], 512, 16, 70, "each"),
    (100, [96, 32, 48, 80], 320, 40, 6, "mixed"), (129, [4096], 2048, 128, 5, "mixed"), (200, [8192, 2048], 2048, 32, 32, "mixed"),
    (256, [2048], 2048, 16, 256, "each"), (300, [8224], 2048, 8, 7, "sequences"), (511, [513], 896, 16, 9, "mixed"),
    (900, [4096], 2048, 16, 4, "sequences"), (1949, [6144, 2048, 32, 32], 2048, 16, 5, "sequences"),
    (2049, [256], 1024, 48, 6, "sequences"), (2500, [8192, 4096, 32, 32], 2048, 64, 12, "mixed"),
    (4100, [2048], 2048, 16, 3, "sequences"), (5000, [2064], 576, 72, 8, "sequences"), (6000, [64], 2048, 16, 9, "mixed"),
]


def _case(M, widths, K, R, S, how):
    gen = torch.Generator().manual_seed(M * 13 + sum(widths) + K + R)
    return gen, _ids(gen, M, S, how), _adapters(gen, S, widths, K, R)


@pytest.mark.parametrize("M,widths,K,R,S,how", SHAPES)
def test_linear_lora(pkg, dev, M, widths, K, R, S, how):
    gen, ids, lora = _case(M, widths, K, R, S, how)
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = (torch.randn(sum(widths), K, generator=gen) * K ** -0.5).to(BF16).to(dev)
    ids, lora = ids.to(dev), [t.to(dev) for t in lora]
    y = pkg.linear_lora(x, w, *lora, ids, widths=widths)
    torch.cuda.synchronize()
    assert [tuple(t.shape) for t in y] == [(M, n) for n in widths] and all(t.is_contiguous() for t in y)
    delta, loose = _delta(x, *lora, ids, widths, K)
    base, size = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    _check(torch.cat(y, 1), base + delta, 2 * (K + 2 * R) * U * size + loose)
    if len(widths) == 1:
        assert torch.equal(pkg.linear_lora(x, w, *lora, ids), y[0])


@pytest.mark.parametrize("M,widths,K,R,S,how", [
    (1, [2048], 2048, 16, 4, "one"), (1, [8192, 4096], 2048, 16, 8, "one"), (3, [200], 128, 24, 5, "each"),
    (16, [256, 256], 384, 8, 16, "each"), (17, [2048], 4096, 16, 16, "each"), (37, [2048], 4096, 16, 16, "mixed"),
    (64, [1008], 1152, 64, 64, "each"), (65, [130], 2048, 16, 9, "mixed"), (128, [2048], 2048, 32, 50, "each"),
    (200, [8192, 4096], 2048, 32, 32, "mixed"), (257, [384], 256, 128, 4, "sequences"), (400, [2048], 2176, 16, 7, "mixed"),
    (700, [8192], 2048, 16, 5, "sequences"), (1025, [2048], 1920, 16, 6, "mixed"), (2049, [4096, 2048], 2048, 32, 8, "sequences"),
    (4100, [320, 13], 640, 16, 6, "sequences"), (5000, [8192], 1024, 64, 9, "none")])
@pytest.mark.parametrize("ready", [False, True])
def test_linear_fp8_lora(pkg, dev, M, widths, K, R, S, how, ready):
    gen, ids, lora = _case(M, widths, K, R, S, how)
    x = (torch.randn(M, K, generator=gen) * torch.exp(2 * torch.rand(M, 1, generator=gen) - 1)).to(BF16)
    x8, xs = ref.to_e4m3(x.float(), 1)
    w8, ws = ref.to_e4m3(torch.randn(sum(widths), K, generator=gen) * K ** -0.5, 128)
    x, x8, xs, w8, ws, ids = (t.to(dev) for t in (x, x8, xs, w8, ws, ids))
    lora = [t.to(dev) for t in lora]
    if ready:
        y = pkg.linear_fp8_lora(x8, w8, ws, *lora, ids, x_scale=xs, widths=widths)
        seen = (x8.double().unflatten(-1, (-1, 128)) * xs.double()[..., None]).flatten(-2)
        other = pkg.linear_fp8_lora(x8, w8, ws, *lora, ids, x_scale=xs.t().contiguous().t(), widths=widths)
        assert all(torch.equal(p, q) for p, q in zip(y, other))
    else:
        y, seen = pkg.linear_fp8_lora(x, w8, ws, *lora, ids, widths=widths), x
    torch.cuda.synchronize()
    delta, loose = _delta(seen, *lora, ids, widths, K)
    want, slack = ref.linear(x8, xs, w8, ws)
    _check(torch.cat(y, 1), want + delta, slack + loose + 4 * R * U * (want.abs() + delta.abs()))


@pytest.mark.parametrize("M", [5, 300, 1500])
def test_wide_columns_and_gates(pkg, dev, M):
    """The 8-bit product's bf16 columns and their gates; the bf16 product's gates: those of the gate
    kernel on the adapted columns, bit for bit."""
    widths, K, R, S = [512, 256, 32, 32], 512, 16, 6
    gen, ids, lora = _case(M, widths, K, R, S, "mixed")
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = (torch.randn(832, K, generator=gen) * K ** -0.5).to(BF16).to(dev)
    ids, lora = ids.to(dev), [t.to(dev) for t in lora]
    A_log, dt = torch.randn(32, generator=gen).to(dev), torch.randn(32, generator=gen).to(dev)
    delta, loose = _delta(x, *lora, ids, widths, K)
    base, size = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    y, g, beta = pkg.linear_lora(x, w, *lora, ids, widths=widths, gates=dict(gate_col=768, A_log=A_log, dt_bias=dt))
    _check(torch.cat(y, 1), base + delta, 2 * (K + 2 * R) * U * size + loose)
    eg, eb = pkg.fused_g_beta(y[2], y[3], A_log, dt, None)
    assert torch.equal(g, eg) and torch.equal(beta, eb)
    w8, ws = pkg.quantize_weight_fp8(w[:768])
    y8, g, beta = pkg.linear_fp8_lora(x, w8, ws, *lora, ids, widths=widths, wide=w[768:],
                                      gates=dict(gate_col=0, A_log=A_log, dt_bias=dt))
    _check(torch.cat(y8[2:], 1), (base + delta)[:, 768:], (2 * (K + 2 * R) * U * size + loose)[:, 768:])
    eg, eb = pkg.fused_g_beta(y8[2], y8[3], A_log, dt, None)
    assert torch.equal(g, eg) and torch.equal(beta, eb)
    narrow = pkg.linear_fp8_lora(x, w8, ws, lora[0][:, :2 * R].contiguous(), lora[1][:, :768].contiguous(), lora[2], ids,
                                 widths=widths[:2])
    assert all(torch.equal(p, q) for p, q in zip(narrow, y8))


@pytest.mark.parametrize("M,N,K", [(20, 256, 512), (64, 12352, 2048), (300, 8224, 2048), (3000, 4096, 2048)])
def test_rows_stand_alone(pkg, dev, M, N, K):
    """A row's bits do not depend on the others' adapters: not on which they are, nor on infinities and NaN in them;
    and rows without an adapter are never touched by one."""
    gen = torch.Generator().manual_seed(M)
    R, S = 16, 6
    a, b, scale = (t.to(dev) for t in _adapters(gen, S, [N], K, R))
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = (torch.randn(N, K, generator=gen) * K ** -0.5).to(BF16).to(dev)
    w8, ws = pkg.quantize_weight_fp8(w)
    ids = torch.randint(-1, 4, (M,), generator=gen).to(torch.int32).to(dev)
    keep = torch.rand(M, generator=gen).to(dev) < 0.5
    other = torch.where(keep, ids, 4 + (torch.arange(M, device=dev) % 2).int())
    clean = pkg.linear_lora(x, w, a, b, scale, ids), pkg.linear_fp8_lora(x, w8, ws, a, b, scale, ids)
    a[4, 3], b[4, ::5], b[5], scale[5] = float("inf"), float("nan"), float("inf"), float("nan")
    dirty = pkg.linear_lora(x, w, a, b, scale, other), pkg.linear_fp8_lora(x, w8, ws, a, b, scale, other)
    torch.cuda.synchronize()
    for p, q in zip(clean, dirty):
        assert torch.equal(p[keep], q[keep]) and bool(torch.isfinite(p).all())
        assert bool(torch.isnan(q[other == 5]).all())


def test_values_past_bf16(pkg, dev):
    """Shrunk values that bf16 does not hold are infinite, not NaN: their high part is, and has no low one."""
    K = 64
    x = torch.full((2, K), 1e19, dtype=BF16, device=dev)
    w = torch.zeros(32, K, dtype=BF16, device=dev)
    a = torch.full((1, 8, K), 1e19, dtype=BF16, device=dev)
    b = torch.zeros(1, 32, 8, dtype=BF16, device=dev)
    b[:, :, 0] = 1.0
    scale = torch.ones(1, device=dev)
    y = pkg.linear_lora(x, w, a, b, scale, torch.tensor([0, -1], dtype=torch.int32, device=dev))
    # (a sum of 64 * 1e38; the other row has no adapter.  An infinity times B's zeros is NaN, as in the formula)
    assert not bool(torch.isfinite(y[0]).any()) and not bool(y[1].any())
    b = b[:, :, :].clone().fill_(1.0)
    top = torch.zeros(1, 8, K, dtype=BF16, device=dev)
    top[0, 0, 0] = 1.0
    x = torch.zeros(1, K, dtype=BF16, device=dev)
    x[0, 0] = torch.finfo(BF16).max
    y = pkg.linear_lora(x, w, top, b, torch.full((1,), 1.003, device=dev), torch.zeros(1, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    assert bool(torch.isinf(y).all())


def test_views_batches_and_nothing(pkg, dev):
    """Rows of a wider buffer and leading dims; adapters as views of a pool for several layers; no rows,
    no slots; weights that are not laid out as the kernel reads them."""
    M, widths, K, R, S = 42, [64, 32], 256, 16, 5
    gen, ids, lora = _case(M, widths, K, R, S, "mixed")
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = (torch.randn(96, K, generator=gen) * K ** -0.5).to(BF16).to(dev)
    ids, (a, b, scale) = ids.to(dev), (t.to(dev) for t in lora)
    want = pkg.linear_lora(x, w, a, b, scale, ids, widths=widths)
    pool_a, pool_b = (torch.zeros(S, 3, *t.shape[1:], dtype=BF16, device=dev) for t in (a, b))
    pool_a[:, 1], pool_b[:, 1] = a, b
    buf = torch.zeros(M, 2 * K, dtype=BF16, device=dev)
    buf[:, K:] = x
    odd = torch.empty(M * K + 1, dtype=BF16, device=dev)[1:].view(M, K).copy_(x)
    for xv in (buf[:, K:], odd, x.view(6, 7, K), x.t().contiguous().t()):
        for wv in (w, w.t().contiguous().t()):
            i = ids.view(xv.shape[:-1]) if xv.dim() == 3 else ids.repeat_interleave(2)[::2]
            y = pkg.linear_lora(xv, wv, pool_a[:, 1], pool_b[:, 1], scale, i, widths=widths)
            assert all(torch.equal(p.reshape(M, -1), q) and p.shape[:-1] == xv.shape[:-1] for p, q in zip(y, want))
    y = pkg.linear_lora(x[:0], w, a, b, scale, ids[:0], widths=widths)
    assert [tuple(t.shape) for t in y] == [(0, 64), (0, 32)]
    y = torch.cat(pkg.linear_lora(x, w, a[:0], b[:0], scale[:0], ids, widths=widths), 1)
    base = x.double() @ w.double().t()
    _check(y, base, 2 * K * U * (x.double().abs() @ w.double().abs().t()))


def test_pool(pkg, dev):
    """LoraPool: smaller ranks, projections that an adapter leaves out, slots that are loaded again and cleared."""
    gen = torch.Generator().manual_seed(5)
    K, widths = 128, [64, 48]
    pool = pkg.LoraPool(3, 12, K, widths, device=dev)
    assert pool.rank == 16 and pool.a.shape == (3, 32, K) and pool.b.shape == (3, 112, 16)
    r = lambda *s: torch.randn(*s, generator=gen).to(BF16)  # noqa: E731
    x, w = r(6, K).to(dev), r(112, K).to(dev)
    ids = torch.tensor([0, 1, 2, 0, 1, -1], dtype=torch.int32, device=dev)
    parts = {0: ([(r(12, K), r(64, 12)), (r(5, K), r(48, 5))], 0.5), 1: ([None, (r(16, K), r(48, 16))], 2.0)}
    pool.load(0, [(r(16, K), r(64, 16)), (r(16, K), r(48, 16))], 3.0)
    for s, (p, scale) in parts.items():
        pool.load(s, p, scale)

    def check():
        want = x.double() @ w.double().t()
        size = x.double().abs() @ w.double().abs().t()
        for m, s in enumerate(ids.tolist()):
            col = 0
            for i, part in enumerate(parts[s][0] if s in parts else []):
                if part is not None:
                    A, B = (t.double().to(dev) for t in part)
                    want[m, col:col + widths[i]] += parts[s][1] * (x[m].double() @ A.t() @ B.t())
                    size[m, col:col + widths[i]] += parts[s][1] * (x[m].double().abs() @ A.t().abs() @ B.t().abs())
                col += widths[i]
        y = pkg.linear_lora(x, w, pool.a, pool.b, pool.scale, ids, widths=widths)
        torch.cuda.synchronize()
        _check(torch.cat(y, 1), want, (2 * (K + 32) * U + 2.0 ** -16 + 4 * K * U) * size)

    check()
    pool.clear(0)
    parts.pop(0)
    check()


def test_graph_streams_and_reloading(pkg, dev):
    """A captured step replayed on new rows, ids and adapters; two graphs; another stream; each equal to the eager call."""
    widths, K, R, S, M = [2048, 512], 1024, 16, 8, 48
    gen, ids, lora = _case(M, widths, K, R, S, "mixed")
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = (torch.randn(2560, K, generator=gen) * K ** -0.5).to(BF16).to(dev)
    w8, ws = pkg.quantize_weight_fp8(w)
    ids, (a, b, scale) = ids.to(dev), [t.to(dev) for t in lora]
    both = lambda: (*pkg.linear_lora(x, w, a, b, scale, ids, widths=widths),  # noqa: E731
                    *pkg.linear_fp8_lora(x, w8, ws, a, b, scale, ids, widths=widths))
    eager = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(eager, other))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both())
        graphs.append(g)
    for i in range(4):
        x.copy_(torch.randn(M, K, generator=gen))
        ids.copy_(_ids(gen, M, S, "mixed"))
        b[i].normal_()
        for g in graphs:
            g.replay()
        eager = both()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(p, q) for p, q in zip(eager, o)), i


def test_adapter_rows(pkg, dev):
    cu = torch.tensor([0, 3, 3, 7, 8], device=dev)
    rows = pkg.adapter_rows(torch.tensor([2, 5, -1, 0], device=dev), cu, 8)
    assert rows.dtype == torch.int32 and rows.tolist() == [2, 2, 2, -1, -1, -1, -1, 0]


class _NoQuick:
    def __getattr__(self, name):
        return lambda *a: None


def _bits(out):
    return [t.view(torch.uint8) if t.dtype == FP8 else t for t in (out if isinstance(out, (list, tuple)) else [out])]


def test_quick_and_checked_calls_agree(pkg, dev, monkeypatch):
    """The calls by way of C++ and those by way of the Python wrappers: the same bits, shapes and
    strides; memory that comes back; what the kernels do not take as it is goes the other way."""
    gen = torch.Generator().manual_seed(47)
    M, N, K, R, S = 37, 96, 256, 16, 3
    x, w = torch.randn(M, K, generator=gen).to(BF16).to(dev), (torch.randn(N, K, generator=gen) * 0.1).to(BF16).to(dev)
    w8, ws = pkg.quantize_weight_fp8(w)
    x8, xs = pkg.quantize_fp8(x)
    ids = _ids(gen, M, S, "mixed").to(dev)
    one = [t.to(dev) for t in _adapters(gen, S, [N], K, R)]
    two = [t.to(dev) for t in _adapters(gen, S, [64, 32], K, R)]
    res, nw = torch.randn(M, K, generator=gen).to(dev), torch.randn(K, generator=gen).to(BF16).to(dev)
    gates = torch.randn(M, 1, generator=gen).to(dev), torch.randn(K, generator=gen).to(BF16).to(dev), x.clone()
    calls = [lambda: pkg.linear_lora(x, w, *one, ids), lambda: pkg.linear_lora(x, w, *two, ids, widths=[64, 32]),
             lambda: pkg.linear_lora(x.view(1, M, K), w, *two, ids.view(1, M), widths=[64, 32]),
             lambda: pkg.linear_fp8_lora(x, w8, ws, *one, ids), lambda: pkg.linear_fp8_lora(x, w8, ws, *two, ids, widths=[64, 32]),
             lambda: pkg.linear_fp8_lora(x8, w8, ws, *two, ids, x_scale=xs, widths=[64, 32]),
             lambda: pkg.linear_fp8_lora(x8, w8, ws, *one, ids, x_scale=xs.contiguous()),
             lambda: pkg.add_rms_norm(x, None, nw, 1e-6), lambda: pkg.add_rms_norm(x, res, nw.float(), 1e-6),
             lambda: pkg.add_rms_norm(x, x, nw, 1e-6, post_weight=nw, gate=gates[0], gate_sigmoid=True, scale=0.5, offset=0.0),
             *(lambda g=g: pkg.add_rms_norm(x, res, nw, 1e-6, gate=g) for g in gates),
             lambda: pkg.add_rms_norm(x[0], x[1], nw, 1e-6),
             *(lambda k=k: pkg.add_rms_norm_fp8(x, res, nw, 1e-6, post_weight=nw, keep=k) for k in (False, True))]
    got = [call() for call in calls]
    quick = pkg._lib.quick()
    q = lambda t: t[:, :128]  # noqa: E731
    taken = [quick.linear_lora(x, w, *one, ids, None), quick.linear_fp8_lora(x8, w8, ws, *one, ids, xs, None),
             quick.add_norm(x, res, nw, 1e-6, nw, None, False, 1.0, 1.0, True, True)]
    assert all(t is not None for t in taken)
    left = [quick.linear_lora(q(x), q(w), *one, ids, None), quick.linear_lora(x, w, *one, ids.long(), None),
            quick.linear_lora(x, w, *one, ids[1:], None), quick.linear_lora(x, w, *two, ids, None),
            quick.linear_lora(x, w, *two, ids, [64, 31]), quick.linear_lora(x, w, *two, ids, [60, 36]),
            quick.linear_lora(x, w, one[0], one[1], one[2].cpu(), ids, None), quick.linear_lora(x[:0], w, *one, ids[:0], None),
            quick.linear_fp8_lora(x, w8, ws[:, :1], *one, ids, None, None), quick.linear_fp8_lora(x8, w8, ws, *one, ids, None, None),
            quick.linear_fp8_lora(x8, w8, ws, *one, ids, xs[1:], None),
            quick.add_norm(q(x), None, nw[:128], 1e-6, None, None, False, 1.0, 1.0, True, False),
            quick.add_norm(x, res[1:], nw, 1e-6, None, None, False, 1.0, 1.0, True, False),
            quick.add_norm(x, res, nw, 1e-6, nw.float(), None, False, 1.0, 1.0, True, False),
            quick.add_norm(x, res, nw, 1e-6, None, ids.view(M, 1), False, 1.0, 1.0, True, False)]
    assert all(t is None for t in left), [t is None for t in left]
    before = torch.cuda.memory_allocated(dev)
    for _ in range(3):
        for call in calls:
            call()
    assert torch.cuda.memory_allocated(dev) == before
    monkeypatch.setattr(pkg._lib, "quick", lambda: _NoQuick())
    for i, (call, g) in enumerate(zip(calls, got)):
        for a, b in zip(_bits(g), _bits(call()), strict=True):
            assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b), i
    assert calls[7]()[1] is x and got[7][1] is x


def test_out_of_memory_is_torchs_error(pkg, dev):
    """Outputs that do not fit raise torch's own error, and the next call is right."""
    from test_gpu_no_memory import _memory_left
    S, R, K = 1, 8, 128
    x, w = torch.ones(16384, K, dtype=BF16, device=dev), torch.ones(8192, K, dtype=BF16, device=dev)
    w8, ws = torch.ones(8192, K, device=dev).to(FP8), torch.ones(64, 1, device=dev)
    a, b = torch.ones(S, R, K, dtype=BF16, device=dev), torch.ones(S, 8192, R, dtype=BF16, device=dev)
    scale, ids = torch.ones(S, device=dev), torch.zeros(16384, dtype=torch.int32, device=dev)
    rows = torch.zeros(8192, 8192, dtype=BF16, device=dev)
    norm_w = torch.ones(8192, dtype=BF16, device=dev)
    calls = (lambda: pkg.linear_lora(x, w, a, b, scale, ids),                     # 256 MiB
             lambda: pkg.linear_fp8_lora(x, w8, ws, a, b, scale, ids),
             lambda: pkg.add_rms_norm(rows, rows, norm_w, 1e-6),                  # twice 128 MiB
             lambda: pkg.add_rms_norm_fp8(rows, rows, norm_w, 1e-6))
    with _memory_left(dev, 32):
        for call in calls:
            with pytest.raises(torch.OutOfMemoryError):
                call()
    assert bool((calls[0]() == K + K * R).all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("M", [2, 15, 16, 17, 63, 64, 65, 127, 129, 200, 255, 256, 257, 300])
@pytest.mark.parametrize("N,S,how", [(96, 3, "mixed"), (96, 300, "mixed"), (12352, 8, "mixed"), (96, 5, "one"), (160, 1, "mixed"), (2048, 30, "mixed")])
def test_rows_in_the_order_of_their_adapters(pkg, dev, M, N, S, how, fp8):
    """Few rows are taken in their adapters' order: at the sizes where that begins, ends and changes, with more
    adapters than rows and with one, each row stays its own, and the gates with it."""
    gen = torch.Generator().manual_seed(M + N + S)
    K, R = 256, 8
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = (torch.randn(N, K, generator=gen) * K ** -0.5).to(BF16).to(dev)
    a, b, scale = (t.to(dev) for t in _adapters(gen, S, [N], K, R))
    ids = _ids(gen, M, S, how).to(dev)
    delta, slack = _delta(x, a, b, scale, ids, [N], K)
    if fp8:
        w8, ws = pkg.quantize_weight_fp8(w)
        x8, xs = pkg.quantize_fp8(x)
        y = pkg.linear_fp8_lora(x, w8, ws, a, b, scale, ids)
        want, base = ref.linear(x8, xs, w8, ws)
        base = base + 4 * R * U * (want.abs() + delta.abs())
    else:
        y = pkg.linear_lora(x, w, a, b, scale, ids)
        want, base = x.double() @ w.double().t(), 2 * (K + 2 * R) * U * (x.double().abs() @ w.double().abs().t())
    _check(y, want + delta, slack + base)
    # an adapter's rows alone, at the same size: the same bits
    for s in ids[[0, M // 2, M - 1]].tolist():
        rows = ids == s
        only = torch.where(rows, ids, -1)
        again = pkg.linear_fp8_lora(x, w8, ws, a, b, scale, only) if fp8 else pkg.linear_lora(x, w, a, b, scale, only)
        assert torch.equal(again[rows], y[rows])
    if not fp8 and N == 96:
        gates = dict(A_log=torch.randn(16, generator=gen).to(dev), dt_bias=torch.randn(16, generator=gen).to(dev), gate_col=64)
        y2, g, beta = pkg.linear_lora(x, w, a, b, scale, ids, gates=gates)
        assert torch.equal(y2, y)
        eg, eb = pkg.fused_g_beta(y[:, 64:80].contiguous(), y[:, 80:].contiguous(), gates["A_log"], gates["dt_bias"], None)
        assert torch.equal(g, eg) and torch.equal(beta, eb)


@pytest.mark.parametrize("M", [1, 40, 300, 2000, 2500])
def test_no_slots_and_the_rows_quantized_on_the_way(pkg, dev, M):
    """A pool without slots: the products alone, bit for bit, bf16 rows for 8-bit weights quantized all the same;
    and the e4m3 rows that come out of the adapters' launch are quantize_fp8's."""
    gen = torch.Generator().manual_seed(M)
    N, K, R = 96, 384, 16
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = (torch.randn(N, K, generator=gen) * K ** -0.5).to(BF16).to(dev)
    w8, ws = pkg.quantize_weight_fp8(w)
    empty = pkg.LoraPool(0, R, K, [N], dev)
    ids = torch.zeros(M, dtype=torch.int32, device=dev)
    assert torch.equal(pkg.linear_lora(x, w, empty.a, empty.b, empty.scale, ids), pkg.linear(x, w))
    assert torch.equal(pkg.linear_fp8_lora(x, w8, ws, empty.a, empty.b, empty.scale, ids), pkg.linear_fp8(x, w8, ws))
    a, b, scale = (t.to(dev) for t in _adapters(gen, 2, [N], K, R))
    x8, xs = pkg.quantize_fp8(x)
    to, to_s = torch.zeros_like(x8), torch.zeros_like(xs)
    v, _ = pkg.ops._lora_shrink(dev.index or 0, x, K, None, a, scale, ids, M, K, 1, R, to, to_s)
    alone, _ = pkg.ops._lora_shrink(dev.index or 0, x, K, None, a, scale, ids, M, K, 1, R)
    assert torch.equal(to.view(torch.uint8), x8.view(torch.uint8)) and torch.equal(to_s, xs) and torch.equal(v, alone)


def test_slots_past_32_bits(pkg, dev):
    """Slots whose offsets pass 2^32 bytes, of A and of B: the same bits as from a pool of two.  (Which wave adds
    an adapter goes by its slot's number modulo 8 at most: 8 for 0 and 33 for 1.)"""
    gen = torch.Generator().manual_seed(53)
    N, K, R, S = 384, 128, 16, 34
    two = _adapters(gen, 2, [N], K, R)
    far = [torch.empty(S, 1 << 26, dtype=BF16, device=dev) for _ in range(2)]
    views = [t.as_strided((S, *s.shape[1:]), (1 << 26, s.shape[2], 1)) for t, s in zip(far, two)]
    for t, s in zip(views, two):
        t[8].copy_(s[0])
        t[33].copy_(s[1])
    scale = torch.zeros(S, device=dev)
    scale[8], scale[33] = two[2][0], two[2][1]
    near = [t.to(dev) for t in two]
    assert 33 * (2 << 26) > 1 << 32
    for M in (1, 20, 300, 2500, 5000):
        x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
        w = torch.randn(N, K, generator=gen).to(BF16).to(dev)
        ids = torch.randint(0, 2, (M,), generator=gen).sort().values.to(torch.int32).to(dev)
        moved = torch.where(ids == 0, 8, 33).to(torch.int32)
        assert torch.equal(pkg.linear_lora(x, w, *views, scale, moved), pkg.linear_lora(x, w, *near, ids)), M
        w8, ws = pkg.quantize_weight_fp8(w)
        assert torch.equal(pkg.linear_fp8_lora(x, w8, ws, *views, scale, moved), pkg.linear_fp8_lora(x, w8, ws, *near, ids)), M


@pytest.mark.parametrize("S", [15, 16, 34])
def test_large_tiles_of_far_slots(pkg, dev, S):
    """Tiles of several adapters whose slots in B lie up to, at and past 2^31 bytes: the same bits as from a pool side by side."""
    gen = torch.Generator().manual_seed(S)
    M, N, K, R = 2000, 12352, 1024, 16
    a, b, scale = (t.to(dev) for t in _adapters(gen, S, [N], K, R))
    far = torch.empty(S, 1 << 26, dtype=BF16, device=dev).as_strided(b.shape, (1 << 26, R, 1))
    for s in range(S):
        far[s].copy_(b[s])
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = torch.randn(N, K, generator=gen).to(BF16).to(dev)
    ids = torch.randint(-1, S, (40,), generator=gen).repeat_interleave(50).to(torch.int32).to(dev)
    assert torch.equal(pkg.linear_lora(x, w, a, far, scale, ids), pkg.linear_lora(x, w, a, b, scale, ids))
    w8, ws = pkg.quantize_weight_fp8(w)
    assert torch.equal(pkg.linear_fp8_lora(x, w8, ws, a, far, scale, ids), pkg.linear_fp8_lora(x, w8, ws, a, b, scale, ids))


def test_two_streams_at_once(pkg, dev):
    """Calls that overlap on two streams, and two graphs replayed in turn and at once: each has rows of its own."""
    gen = torch.Generator().manual_seed(59)
    N, K, R, S = 2048, 1024, 16, 8
    w = torch.randn(N, K, generator=gen).to(BF16).to(dev)
    lora = [t.to(dev) for t in _adapters(gen, S, [N], K, R)]
    sides = [torch.cuda.Stream(dev) for _ in range(2)]
    for M in (37, 3000):
        xs = [torch.randn(M, K, generator=gen).to(BF16).to(dev) for _ in range(2)]
        ids = [_ids(gen, M, S, how).to(dev) for how in ("mixed", "sequences")]
        want = [pkg.linear_lora(x, w, *lora, i) for x, i in zip(xs, ids)]
        torch.cuda.synchronize()
        for _ in range(5):
            got = []
            for side, x, i in zip(sides, xs, ids):
                with torch.cuda.stream(side):
                    got.append(pkg.linear_lora(x, w, *lora, i))
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        graphs, out = [], []
        for x, i in zip(xs, ids):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                out.append(pkg.linear_lora(x, w, *lora, i))
        for _ in range(3):
            for side, g, y in zip(sides, graphs, out):
                with torch.cuda.stream(side):
                    y.zero_()
                    g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("R", [8, 16, 40, 72])
@pytest.mark.parametrize("n", [2, 3, 6, 7, 12, 13, 20, 21, 40])
def test_large_tiles_of_several_adapters(pkg, dev, n, R, fp8):
    """256 rows with n adapters each, in runs and row by row: up to, at and past what a tile takes as more steps, in whole tiles
    and in a last one of two slices; a row's bits are those that it has when the others have no adapter, whatever theirs hold."""
    gen = torch.Generator().manual_seed(n + R)
    M, K, S, widths = 1300, 256, 48, [8192, 4096, 32, 32]
    N = sum(widths)
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = (torch.randn(N, K, generator=gen) * K ** -0.5).to(BF16).to(dev)
    a, b, scale = (t.to(dev) for t in _adapters(gen, S, widths, K, R))
    row = torch.arange(M)
    ids = torch.where(row < 768, row // 256 * n + row % 256 * n // 256, row * 7 % n) % (S - 1)
    ids = torch.where(row % 50 == 9, torch.tensor(-1), ids).to(torch.int32).to(dev)
    delta, slack = _delta(x, a, b, scale, ids, widths, K)
    if fp8:
        w8, ws = pkg.quantize_weight_fp8(w)
        x8, xs = pkg.quantize_fp8(x)
        call = lambda i: torch.cat(pkg.linear_fp8_lora(x, w8, ws, a, b, scale, i, widths=widths), 1)  # noqa: E731
        want, base = ref.linear(x8, xs, w8, ws)
        base = base + 4 * R * U * (want.abs() + delta.abs())
    else:
        call = lambda i: torch.cat(pkg.linear_lora(x, w, a, b, scale, i, widths=widths), 1)  # noqa: E731
        want, base = x.double() @ w.double().t(), 2 * (K + 2 * R) * U * (x.double().abs() @ w.double().abs().t())
    y = call(ids)
    _check(y, want + delta, slack + base)
    for s in ids[[0, 300, 1299]].tolist():
        rows = ids == s
        assert torch.equal(call(torch.where(rows, ids, -1))[rows], y[rows])
    b[S - 1, ::3] = float("inf")
    last = torch.where(ids == int(ids[100]), S - 1, ids).int()
    rows = last != S - 1
    assert torch.equal(call(last)[rows], y[rows])
