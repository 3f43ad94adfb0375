"""The norms around a block (add_rms_norm, add_rms_norm_fp8) against the formula in 64 bits.

Tolerances.  u = 2^-24.  A sum of H squares and the steps around it (each a rounding, rsqrt and
the exponential a few) are off by at most c u with c = H / 64 + 64: a thread adds at most H / 64
of them one after the other (the narrowest launch), the rest in a tree.  The stream r = residual +
scale h is off by c u (|scale h| + |residual|) in all, and rounded once to its type; y by what r
is off times |rstd (offset + w)|, by c u of itself, and by bf16's half step, 2^-8."""
import pytest
import torch

from helpers import BF16

pytestmark = pytest.mark.gpu
F32, F64, FP8 = torch.float32, torch.float64, torch.float8_e4m3fn
U = 2.0 ** -24
HALF = {BF16: 2.0 ** -8, F32: U}
EPS = 1e-6


def _inputs(M, H, form, wide, dev, seed=0, w_dtype=BF16):
    gen = torch.Generator().manual_seed(1000 * M + H + seed)
    r = lambda *s, std=1.0: torch.randn(*s, generator=gen) * std  # noqa: E731
    x = (r(M, H) * torch.exp(2 * torch.rand(M, 1, generator=gen) - 1)).to(BF16)
    kw = {}
    res = None
    if "first" not in form:
        res = (r(M, H) * torch.where(torch.rand(H, generator=gen) < 0.02, 20.0, 1.0)).to(F32 if wide else BF16)
    if "post" in form:
        kw["post_weight"] = r(H, std=0.2).to(w_dtype)
    if "row" in form:
        kw["gate"] = r(M, 1).to(BF16)
    if "column" in form:
        kw["gate"] = r(H).to(F32)
    if "value" in form:
        kw["gate"] = r(M, H).to(BF16)
    if "sigmoid" in form:
        kw["gate_sigmoid"] = True
        kw["gate"] = kw["gate"] * 4
    if "scale" in form:
        kw["scale"] = 0.22
    if "bare" in form:
        kw["offset"] = 0.0
    w = r(H, std=0.2).to(w_dtype)
    put = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    return put(x), put(res), put(w), {k: put(v) for k, v in kw.items()}


def _oracle(x, res, w, post_weight=None, gate=None, gate_sigmoid=False, scale=1.0, offset=1.0):
    """(r, y, |scale h| + |residual|, rstd |offset + w|) in 64 bits."""
    def rstd(t):
        return (t.square().mean(-1, keepdim=True) + EPS) ** -0.5

    h = x.double()
    if post_weight is not None:
        h = h * rstd(h) * (offset + post_weight.double())
    if gate is not None:
        h = h * (torch.sigmoid(gate.double()) if gate_sigmoid else gate.double())
    h = h * scale
    r = h if res is None else res.double() + h
    size = h.abs() + (0 if res is None else res.double().abs())
    gain = rstd(r) * (offset + w.double()).abs()
    return r, r * rstd(r) * (offset + w.double()), size, gain


def _within(got, want, bound, tag):
    d = (got.double() - want).abs()
    worst = float((d / bound.clamp(min=1e-300)).max()) if d.numel() else 0.0
    assert bool((d <= bound).all()), f"{tag}: max |diff| / bound {worst:.3f}"


def _check(y, r, x, res, w, kw, tag=""):
    want_r, want_y, size, gain = _oracle(x, res, w, **kw)
    c = (x.shape[-1] / 64 + 64) * U
    if r is not None:
        # (a residual of -scale h leaves what the fp32 sum is off by)
        _within(r, want_r, (1 + HALF[r.dtype]) * c * size + HALF[r.dtype] * want_r.abs(), tag + " r")
    if y is not None:
        # (r off by c u size moves the mean of its squares by at most twice that of itself, and so y)
        loose = c * size * gain + (c + 2 * c * size.amax(-1, keepdim=True) * gain.amax(-1, keepdim=True)) * want_y.abs()
        _within(y, want_y, (1 + HALF[BF16]) * loose + HALF[BF16] * want_y.abs(), tag + " y")
    return want_y


# every launch: one to many rows, one column to the most, whole 16-byte pieces and not
SIZES = [(1, 2048), (1, 16384), (3, 8), (7, 64), (5, 1), (4, 127), (201, 2048), (33, 1000), (2, 1025), (9, 4099), (2, 16383),
         (300, 4096), (17, 8192), (2048, 512), (2500, 520), (2100, 2048), (2050, 4096), (2049, 1024), (2049, 130), (70000, 64)]


@pytest.mark.parametrize("M,H", SIZES)
def test_sizes(pkg, dev, M, H):
    for wide in (False, True):
        x, res, w, kw = _inputs(M, H, "plain", wide, dev)
        y, r = pkg.add_rms_norm(x, res, w, EPS)
        torch.cuda.synchronize()
        assert y.dtype == BF16 and r.dtype == res.dtype and y.shape == r.shape == x.shape
        _check(y, r, x, res, w, kw, f"wide {wide}")


FORMS = ["first", "first scale", "post", "post scale bare", "row", "row sigmoid scale", "column", "column sigmoid", "value",
         "value sigmoid post", "first post value scale"]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("M,H", [(3, 2048), (2051, 1024), (5, 333)])
def test_forms(pkg, dev, M, H, form):
    for wide, w_dtype in ((False, BF16), (True, F32)):
        x, res, w, kw = _inputs(M, H, form, wide, dev, w_dtype=w_dtype)
        y, r = pkg.add_rms_norm(x, res, w, EPS, **kw)
        torch.cuda.synchronize()
        _check(y, r, x, res, w, kw, f"wide {wide}")
        if form == "first":
            assert r.data_ptr() == x.data_ptr()


@pytest.mark.parametrize("M,H", [(1, 128), (1, 2048), (37, 640), (2100, 2048), (2049, 256), (5, 16384), (300, 4096)])
@pytest.mark.parametrize("form", ["plain", "post row sigmoid scale", "first", "value"])
def test_e4m3(pkg, dev, M, H, form):
    """The scales within fp32's error of amax / 448; the values within e4m3's half step (2^-4, or half of its
    smallest step, 2^-10, times the scale) of y; the bf16 rows and the stream are add_rms_norm's, bit for bit."""
    x, res, w, kw = _inputs(M, H, form, "row" in form, dev)
    y8, ys, r, y = pkg.add_rms_norm_fp8(x, res, w, EPS, keep=True, **kw)
    b8, bs, br = pkg.add_rms_norm_fp8(x, res, w, EPS, **kw)
    y16, r16 = pkg.add_rms_norm(x, res, w, EPS, **kw)
    torch.cuda.synchronize()
    assert y8.dtype == FP8 and ys.shape == (M, H // 128) and ys.dtype == F32
    assert torch.equal(y, y16) and torch.equal(r, r16) and torch.equal(br, r16) and torch.equal(bs, ys)
    assert torch.equal(b8.view(torch.uint8), y8.view(torch.uint8))
    want = _check(y, r, x, res, w, kw)
    _, _, size, gain = _oracle(x, res, w, **kw)
    c = (H / 64 + 66) * U
    loose = c * size * gain + (c + 2 * c * size.amax(-1, keepdim=True) * gain.amax(-1, keepdim=True)) * want.abs()
    groups = lambda t: t.unflatten(-1, (-1, 128))  # noqa: E731
    top = groups(want).abs().amax(-1)
    _within(ys, top / 448, groups(loose).amax(-1) / 448 + 3 * U * top / 448, "scales")
    s = ys.double()[..., None]
    _within(groups(y8.double()) * s, groups(want),
            groups(loose) * (1 + 2.0 ** -4) + (2.0 ** -4 + 4 * U) * groups(want).abs() + 2.0 ** -10 * s, "values")


def test_views_and_batches(pkg, dev):
    """Rows of a wider buffer, leading dims, unaligned rows, expanded weights and gates."""
    M, H = 24, 512
    x, res, w, kw = _inputs(M, H, "value post", False, dev)
    want_y, want_r = pkg.add_rms_norm(x, res, w, EPS, **kw)

    def wider(t, at):
        b = torch.zeros(M, H + 24, dtype=t.dtype, device=dev)
        b[:, at:at + H] = t
        return b[:, at:at + H]

    for at in (8, 3):
        y, r = pkg.add_rms_norm(wider(x, at), wider(res, at), w, EPS, gate=wider(kw["gate"], at),
                                post_weight=wider(kw["post_weight"].expand(M, H), at)[0])
        torch.cuda.synchronize()
        _check(y, r, x, res, w, kw, f"at {at}")
        if at == 8:
            assert torch.equal(y, want_y) and torch.equal(r, want_r)
        y8, ys, r = pkg.add_rms_norm_fp8(wider(x, at), wider(res, at), w, EPS, gate=wider(kw["gate"], at),
                                         post_weight=kw["post_weight"])
        e8, es, er = pkg.add_rms_norm_fp8(x, res, w, EPS, **kw)
        assert torch.equal(ys, es) and torch.equal(r, er) and torch.equal(y8.view(torch.uint8), e8.view(torch.uint8))
    y, r = pkg.add_rms_norm(x.view(4, 6, H), res.view(4, 6, H), w, EPS, gate=kw["gate"].view(4, 6, H),
                            post_weight=kw["post_weight"])
    assert y.shape == (4, 6, H) and torch.equal(y.view(M, H), want_y) and torch.equal(r.view(M, H), want_r)
    y, r = pkg.add_rms_norm(x.t().contiguous().t(), res.t().contiguous().t(), w, EPS, **kw)
    assert torch.equal(y, want_y) and torch.equal(r, want_r)
    g = torch.randn(4, 6, 1, device=dev)
    y, r = pkg.add_rms_norm(x.view(4, 6, H), res.view(4, 6, H), w.expand(2, H)[1], EPS, gate=g)
    _check(y.view(M, H), r.view(M, H), x, res, w, dict(gate=g.view(M, 1)))
    y, r = pkg.add_rms_norm(x[0], res[0], w, EPS)
    assert y.shape == (H,)
    _check(y[None], r[None], x[:1], res[:1], w, {})


def test_residual_out(pkg, dev):
    """The stream in place, and into another tensor; the bits of the call that allocates it."""
    for M, H, wide in ((5, 2048, False), (2100, 1024, True), (3, 333, False)):
        x, res, w, kw = _inputs(M, H, "row sigmoid", wide, dev)
        want_y, want_r = pkg.add_rms_norm(x, res, w, EPS, **kw)
        other, mine = torch.empty_like(res), res.clone()
        y, r = pkg.add_rms_norm(x, res, w, EPS, residual_out=other, **kw)
        assert r is other and torch.equal(other, want_r) and torch.equal(y, want_y)
        y, r = pkg.add_rms_norm(x, mine, w, EPS, residual_out=mine, **kw)
        assert r is mine and torch.equal(mine, want_r) and torch.equal(y, want_y)
        out = torch.empty_like(x)
        y, r = pkg.add_rms_norm(x, None, w, EPS, residual_out=out)
        assert r is out and torch.equal(out, x)


def test_nothing_and_non_finite(pkg, dev):
    x, res, w, kw = _inputs(4, 1024, "row", False, dev)
    y, r = pkg.add_rms_norm(x[:0], res[:0], w, EPS, gate=kw["gate"][:0])
    assert y.shape == r.shape == (0, 1024)
    y8, ys, r = pkg.add_rms_norm_fp8(x[:0], res[:0], w, EPS)
    assert y8.shape == (0, 1024) and ys.shape == (0, 8)
    clean, _ = pkg.add_rms_norm(x, res, w, EPS, **kw)
    x[1, 7], x[2, 9] = float("nan"), float("inf")
    y, r = pkg.add_rms_norm(x, res, w, EPS, **kw)
    torch.cuda.synchronize()
    assert torch.equal(y[[0, 3]], clean[[0, 3]])                    # the other rows
    assert bool(torch.isnan(y[1]).all()) and torch.isnan(y[2, 9]).item() and torch.isinf(r[2, 9]).item()
    # rows of zeros, and a gate that closes a row: y is 0 where the stream is
    z = torch.zeros(3, 1024, dtype=BF16, device=dev)
    y, r = pkg.add_rms_norm(z, z, w, EPS, post_weight=w, gate=torch.full((3, 1), -200.0, device=dev), gate_sigmoid=True)
    assert not y.any() and not r.any()
    big = torch.full((2, 1024), 3e4, dtype=BF16, device=dev)
    y, r = pkg.add_rms_norm(big, z[:2], w, EPS, gate=torch.tensor([[-200.0], [200.0]], device=dev), gate_sigmoid=True)
    assert not r[0].any() and torch.equal(r[1], big[1])


def test_graph_and_stream(pkg, dev):
    """Replays on new data beside eager work; a stream that is not the tensors' own."""
    x, res, w, kw = _inputs(64, 2048, "value sigmoid", True, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, r = pkg.add_rms_norm(x, res, w, EPS, **kw)
    torch.cuda.current_stream().wait_stream(side)
    _check(y, r, x, res, w, kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gr = pkg.add_rms_norm(x, res, w, EPS, residual_out=res, **kw)
        g8, gs, _ = pkg.add_rms_norm_fp8(x, gr, w, EPS)
    stream = res.clone()
    for i in range(4):
        x.copy_(torch.randn(64, 2048, device=dev))
        graph.replay()
        ey, stream = pkg.add_rms_norm(x, stream, w, EPS, **kw)
        e8, es, _ = pkg.add_rms_norm_fp8(x, stream, w, EPS)
        torch.cuda.synchronize()
        assert torch.equal(gy, ey) and torch.equal(gr, stream)
        assert torch.equal(gs, es) and torch.equal(g8.view(torch.uint8), e8.view(torch.uint8))
