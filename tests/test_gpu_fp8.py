"""The 8-bit projections: quantize_fp8 and quantize_weight_fp8 bit for bit against the
same fp32 steps in torch on the CPU; linear_fp8 against a 64-bit product of the values
that its operands stand for; the gated norm in e4m3 against 64 bits; the mixer with
8-bit weights against its own parts."""
import pytest
import torch

import tree_ref as ref
from helpers import BF16

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def _rows(gen, M, K):
    """Rows of very different sizes with a few loud columns."""
    x = torch.randn(M, K, generator=gen) * torch.exp(4 * torch.rand(M, 1, generator=gen) - 2)
    x[:, torch.rand(K, generator=gen) < 0.02] *= 30
    return x


def _bits(t):
    return t.cpu().contiguous().view(torch.uint8)


@pytest.mark.parametrize("M,K", [(1, 128), (1, 2048), (37, 4096), (257, 640), (1000, 1152)])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_quantize_rows(pkg, dev, M, K, dtype):
    x = _rows(torch.Generator().manual_seed(M + K), M, K).to(dtype)
    x[0, :128] = 0                      # a group of zeros
    if M > 3:
        x[1, 0:128] = 1e-38             # below the smallest scale's range
        x[2, 128 % K] = 3e38 if dtype == torch.float32 else 3.3e38
    q, s = pkg.quantize_fp8(x.to(dev))
    torch.cuda.synchronize()
    rq, rs = ref.to_e4m3(x.float(), 1)
    assert q.dtype == FP8 and q.shape == x.shape and tuple(s.shape) == (M, K // 128)
    assert torch.equal(s.cpu(), rs)
    assert torch.equal(_bits(q), _bits(rq))


def test_quantize_rows_views_and_batches(pkg, dev):
    gen = torch.Generator().manual_seed(3)
    x = _rows(gen, 60, 1024).to(BF16)
    rq, rs = ref.to_e4m3(x[:, 128:640].float(), 1)
    xd = x.to(dev)
    for view in (xd[:, 128:640], xd.view(5, 12, 1024)[..., 128:640], xd.t().contiguous().t()[:, 128:640]):
        q, s = pkg.quantize_fp8(view)
        torch.cuda.synchronize()
        assert q.shape == view.shape
        assert torch.equal(s.cpu(), rs) and torch.equal(_bits(q.view(60, 512)), _bits(rq))
    odd = torch.empty(60 * 512 + 1, dtype=BF16, device=dev)[1:].view(60, 512)   # not 16-byte aligned
    odd.copy_(xd[:, 128:640])
    q, s = pkg.quantize_fp8(odd)
    assert torch.equal(s.cpu(), rs) and torch.equal(_bits(q), _bits(rq))
    q, s = pkg.quantize_fp8(xd[:0])
    assert q.shape == (0, 1024) and tuple(s.shape) == (0, 8)


def test_quantize_non_finite(pkg, dev):
    """NaN stays NaN and does not count; an infinity makes the scale infinite, itself NaN, the rest 0."""
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(4)).to(BF16)
    clean_q, clean_s = pkg.quantize_fp8(x.to(dev))
    x[1, 5], x[2, 200] = float("nan"), float("-inf")
    q, s = pkg.quantize_fp8(x.to(dev))
    qf = q.float().cpu()
    keep = torch.ones(4, 256, dtype=torch.bool)
    keep[1, 5] = False
    keep[2, 128:] = False
    assert torch.equal(_bits(q)[keep], _bits(clean_q)[keep])
    assert torch.isnan(qf[1, 5]) and torch.isnan(qf[2, 200])
    rest = torch.cat([qf[2, 128:200], qf[2, 201:]])
    assert bool((rest == 0).all()) and torch.isinf(s[2, 1]).item() and torch.equal(s[1].cpu(), clean_s[1].cpu())


@pytest.mark.parametrize("N,K", [(1, 128), (128, 256), (200, 1152), (2048, 2048)])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_quantize_weight_blocks(pkg, dev, N, K, dtype):
    w = _rows(torch.Generator().manual_seed(N + K), N, K).to(dtype)
    q, s = pkg.quantize_weight_fp8(w.to(dev))
    torch.cuda.synchronize()
    rq, rs = ref.to_e4m3(w.float(), 128)
    assert torch.equal(s.cpu(), rs) and torch.equal(_bits(q), _bits(rq))


def _check(y, want, slack, tag):
    d = (y.to(want.device).double() - want).abs()
    bound = ref.HALF_BF16 * (want.abs() + slack) + slack
    worst = float((d / bound.clamp(min=1e-300)).max()) if d.numel() else 0.0
    assert bool((d <= bound).all()), f"{tag}: max |diff| / bound {worst:.2f}"


# one row to thousands, K of one block, odd counts of blocks and many, N below, at and past the blocks' edges
SHAPES = [(1, 1, 128), (1, 2048, 2048), (1, 12288, 2048), (3, 200, 128), (16, 256, 384), (17, 2048, 4096),
          (33, 72, 640), (37, 8192, 2048), (64, 1000, 1152), (65, 130, 2048), (100, 520, 4992), (129, 2048, 2048),
          (200, 12288, 2048), (256, 2048, 4096), (257, 384, 256), (300, 8192, 2048), (511, 513, 896),
          (400, 2048, 4096), (129, 3000, 2176), (500, 2000, 2304), (65, 8192, 2048), (700, 4096, 2048), (1024, 12288, 2048), (1025, 2048, 1920), (2049, 2048, 2048), (4100, 333, 640)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_fp8(pkg, dev, M, N, K):
    gen = torch.Generator().manual_seed(M * 7 + N + K)
    x = _rows(gen, M, K).to(BF16)
    w8, ws = ref.to_e4m3(_rows(gen, N, K) * K ** -0.5, 128)
    x8, xs = ref.to_e4m3(x.float(), 1)
    w8d, wsd = w8.to(dev), ws.to(dev)
    y = pkg.linear_fp8(x.to(dev), w8d, wsd)
    ready = pkg.linear_fp8(x8.to(dev), w8d, wsd, x_scale=xs.to(dev))
    out = torch.full((M, N + 9), 7.0, dtype=BF16, device=dev)
    pkg.linear_fp8(x8.to(dev), w8d, wsd, x_scale=xs.t().contiguous().t().to(dev), out=out[:, :N])
    torch.cuda.synchronize()
    assert y.shape == (M, N) and y.dtype == BF16
    _check(y, *ref.linear(*(t.to(dev) for t in (x8, xs, w8, ws))), "from bf16")
    assert torch.equal(ready, y)
    # some rows and columns, the last ones among them, by the tight bound
    rows = torch.cat([torch.randint(0, M, (8,), generator=gen), torch.arange(max(0, M - 8), M)])
    cols = torch.cat([torch.randint(0, N, (100,), generator=gen), torch.arange(max(0, N - 40), N)])
    _check(y[rows][:, cols], *ref.linear_tight(x8, xs, w8, ws, rows, cols), "tight")
    assert torch.equal(out[:, :N], ready) and bool((out[:, N:] == 7).all())


@pytest.mark.parametrize("M", [5, 300, 2000])
def test_linear_fp8_cols(pkg, dev, M):
    gen = torch.Generator().manual_seed(M)
    K, widths = 512, [256, 144, 48, 100]
    N = sum(widths)
    x = _rows(gen, M, K).to(BF16).to(dev)
    w8, ws = (t.to(dev) for t in ref.to_e4m3(_rows(gen, N, K), 128))
    y = pkg.linear_fp8(x, w8, ws)
    parts = pkg.ops.linear_fp8_cols(x.view(M, 1, K), w8, ws, widths)
    torch.cuda.synchronize()
    assert [tuple(p.shape) for p in parts] == [(M, 1, w) for w in widths]
    assert torch.equal(torch.cat(parts, -1).view(M, N), y)


@pytest.mark.parametrize("M,N,K,N2", [(1, 12288, 2048, 64), (1, 2048, 128, 16), (5, 256, 384, 32), (37, 12288, 2048, 64),
                                      (37, 2048, 4096, 48), (200, 8192, 2048, 32), (1000, 512, 640, 64),
                                      (1025, 1024, 512, 64), (3000, 2048, 2048, 64), (3, 80, 256, 32), (16, 48, 384, 16),
                                      (40, 144, 512, 16), (70, 8208, 256, 32), (1100, 2064, 640, 48)])
def test_linear_fp8_with_bf16_columns(pkg, dev, M, N, K, N2):
    """The 8-bit columns are linear_fp8's; the bf16 ones within bf16's half step and fp32's
    error (K products and K / 128 partial sums, each a rounding) of the 64-bit product."""
    gen = torch.Generator().manual_seed(M + N2)
    x = _rows(gen, M, K).to(BF16).to(dev)
    w8, ws = (t.to(dev) for t in ref.to_e4m3(_rows(gen, N, K) * K ** -0.5, 128))
    wide = (torch.randn(N2, 2 * K, generator=gen) * K ** -0.5).to(BF16).to(dev)[:, K:]
    widths = [N - 16, 16, N2] if N2 < 32 else [N, N2 - 16, 16]
    parts = pkg.ops.linear_fp8_cols(x, w8, ws, widths, wide=wide)
    torch.cuda.synchronize()
    y = torch.cat(parts, 1)
    assert torch.equal(y[:, :N], pkg.linear_fp8(x, w8, ws))
    a, b = x.double(), wide.double()
    want, slack = a @ b.t(), (a.abs() @ b.abs().t()) * (K + K // 128) * ref.U32
    _check(y[:, N:], want, slack, "bf16 columns")


def test_linear_fp8_views_empty_and_non_finite(pkg, dev):
    gen = torch.Generator().manual_seed(8)
    M, N, K = 70, 300, 512
    big = _rows(gen, M, 2 * K).to(BF16).to(dev)
    w8, ws = ref.to_e4m3(_rows(gen, N, 2 * K), 128)
    w8, ws = w8.to(dev), ws.to(dev)
    x, w, s = big[:, K:], w8[:, K:], ws[:, K // 128:]                    # strided operands and scales
    y = pkg.linear_fp8(x, w, s)
    assert torch.equal(y, pkg.linear_fp8(x.contiguous(), w.contiguous(), s.contiguous()))
    x8, xs = pkg.quantize_fp8(big)
    assert torch.equal(y, pkg.linear_fp8(x8[:, K:], w, s, x_scale=xs[:, K // 128:]))
    assert pkg.linear_fp8(x[:0], w, s).shape == (0, N)
    assert pkg.linear_fp8(x, w[:0], s[:0]).shape == (M, 0)
    # a row with a NaN or an infinity is NaN, the others are what they were
    bad = big.clone()
    bad[3, K + 7], bad[9, K + 300] = float("nan"), float("inf")
    z = pkg.linear_fp8(bad[:, K:], w, s)
    rows = [r for r in range(M) if r not in (3, 9)]
    assert torch.isnan(z[[3, 9]]).all().item() and torch.equal(z[rows], y[rows])


def test_linear_fp8_same_bits_again(pkg, dev):
    gen = torch.Generator().manual_seed(9)
    w8, ws = (t.to(dev) for t in ref.to_e4m3(_rows(gen, 2048, 4096), 128))
    for M in (1, 37, 600):
        x = _rows(gen, M, 4096).to(BF16).to(dev)
        y = pkg.linear_fp8(x, w8, ws)
        for _ in range(3):
            assert torch.equal(pkg.linear_fp8(x, w8, ws), y)


@pytest.mark.parametrize("M,H,D", [(1, 1, 128), (1, 32, 128), (5, 2, 64), (33, 6, 64), (201, 32, 128), (1000, 16, 128)])
def test_norm_fp8(pkg, dev, M, H, D):
    """Scales within 64 half steps of fp32 of the 64-bit ones (the mean square over D
    values, its root, exp and four products: under 48), values within half an e4m3 step (2^-4 of the value, 2^-10 of the
    scale where steps are smallest) and the scaled value's own fp32 error."""
    gen = torch.Generator().manual_seed(M + H)
    x = (torch.randn(M, H, D, generator=gen) * torch.exp(-4 * torch.rand(M, H, 1, generator=gen))).to(BF16)
    z = torch.randn(M, H, D, generator=gen).to(BF16) * 3
    w = (1 + 0.1 * torch.randn(D, generator=gen)).to(BF16)
    x[0] = 0                                                   # rows of zeros: smallest scale, zero values
    y8, s = pkg.rms_norm_gated_fp8(x.to(dev), z.to(dev), w.to(dev), 1e-6)
    strided = pkg.rms_norm_gated_fp8(torch.cat([x, x], 1).to(dev)[:, H:], torch.cat([z, z], 1).to(dev)[:, :H],
                                     w.to(dev), 1e-6)
    torch.cuda.synchronize()
    xd, zd = x.double(), z.double()
    want = xd / (xd.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double() * zd * torch.sigmoid(zd)
    flat = want.view(M, -1, 128)
    scale = (flat.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
    assert y8.dtype == FP8 and y8.shape == x.shape and s.shape == scale.shape
    assert bool(((s.cpu().double() - scale).abs() <= 64 * ref.U32 * scale).all())
    got = y8.float().cpu().double().view(M, -1, 128) * s.cpu().double()[..., None]
    bound = (2.0 ** -4 + 1e-5) * flat.abs() + (2.0 ** -10 + 1e-5) * scale[..., None]
    assert bool(((got - flat).abs() <= bound).all())
    assert torch.equal(_bits(strided[0]), _bits(y8)) and torch.equal(strided[1], s)


def _layer(pkg, gen, dev, Hk, Hv, D, hidden, **kw):
    C, V = 2 * Hk * D + Hv * D, Hv * D
    n = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).to(BF16).to(dev)  # noqa: E731
    ws = [n(r, hidden, std=hidden ** -0.5) for r in (C, V, Hv, Hv)] + [n(hidden, V, std=V ** -0.5)]
    rest = (Hk, Hv, D, n(C, 4, std=0.5), n(Hv), n(Hv), n(D, std=0.1) + 1)
    return pkg.GatedDeltaNetLayer(*ws, *rest, weights="fp8", **kw), ws, rest


@pytest.mark.parametrize("Hk,Hv,D,hidden", [(2, 4, 128, 256), (16, 16, 128, 2048), (2, 2, 64, 384)])
def test_mixer_with_8_bit_weights(pkg, dev, Hk, Hv, D, hidden):
    """The mixer's steps (prompts, one-token rows, both at once) are its parts called one by
    one: linear_fp8 on the quantized weights, the core, linear_fp8 on the core's output."""
    gen = torch.Generator().manual_seed(Hv + D)
    layer, (w_qkv, w_z, w_b, w_a, w_out), rest = _layer(pkg, gen, dev, Hk, Hv, D, hidden)
    C, V = layer.core.conv_dim, Hv * D
    w_in8, w_in_s = pkg.quantize_weight_fp8(torch.cat([w_qkv, w_z]))
    w_out8, w_out_s = pkg.quantize_weight_fp8(w_out)
    if C % 128 == 0:      # a checkpoint's pairs give the same layer
        pairs = [(w_in8[:C], w_in_s[:C // 128]), (w_in8[C:], w_in_s[C // 128:]), w_b, w_a, (w_out8, w_out_s)]
        again = pkg.GatedDeltaNetLayer(*pairs, *rest, weights="fp8")
        assert torch.equal(_bits(again.w_in), _bits(layer.w_in)) and torch.equal(again.w_in_scale, layer.w_in_scale)
    core = pkg.GatedDeltaNetCore(*rest)
    slots = 12
    pools = [(torch.randn(slots, Hv, D, D, generator=gen) * 0.1).to(dev),
             torch.randn(slots, C, 3, generator=gen).to(BF16).to(dev)]
    for lens in ([1] * 5, [70, 3, 130], [1, 1, 1, 90, 20]):
        N = sum(lens)
        hidden_rows = torch.randn(N, hidden, generator=gen).to(BF16).to(dev)
        ids = torch.randperm(slots, generator=gen)[:len(lens)].to(dev)
        cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
        mine, theirs = [t.clone() for t in pools], [t.clone() for t in pools]
        y = layer.forward(hidden_rows, cu, max(lens), ids, mine[1], mine[0], lens_q=lens)
        if Hv % 16 == 0:
            mixed, z, b, a = pkg.ops.linear_fp8_cols(hidden_rows, w_in8, w_in_s, [C, V, Hv, Hv],
                                                     wide=torch.cat([w_b, w_a]))
        else:
            mixed, z = pkg.ops.linear_fp8_cols(hidden_rows, w_in8, w_in_s, [C, V])
            ba = pkg.linear(hidden_rows, torch.cat([w_b, w_a]))
            b, a = ba[:, :Hv].contiguous(), ba[:, Hv:].contiguous()
        o = core.forward(mixed, z, b, a, cu, max(lens), ids, theirs[1], theirs[0], lens_q=lens, fp8=True)
        o, s = o if isinstance(o, tuple) else (o, None)
        want = pkg.linear_fp8(o.reshape(N, V), w_out8, w_out_s, x_scale=s)
        torch.cuda.synchronize()
        assert (s is not None) == (1 not in lens or (D == 128 and max(lens) == 1))
        assert torch.equal(y, want) and torch.equal(mine[0], theirs[0]) and torch.equal(mine[1], theirs[1])


def test_other_stream_and_one_scale_for_all(pkg, dev):
    """On a second stream the same bits; a broadcast scale is its copies."""
    gen = torch.Generator().manual_seed(53)
    x, w = _rows(gen, 40, 384).to(BF16).to(dev), (torch.randn(300, 384, generator=gen) * 0.05).to(BF16).to(dev)
    o, z = (torch.randn(33, 4, 128, generator=gen).to(BF16).to(dev) for _ in range(2))
    weight = torch.rand(128, generator=gen).to(BF16).to(dev)

    def run():
        x8, xs = pkg.quantize_fp8(x)
        w8, ws = pkg.quantize_weight_fp8(w)
        one = torch.full((1, 1), 0.25, device=dev)
        return (x8.view(torch.uint8), xs, pkg.linear_fp8(x, w8, ws), pkg.linear_fp8(x8, w8, ws, x_scale=xs),
                pkg.linear_fp8(x8, w8, one.expand(3, 3), x_scale=one.expand(40, 3)),
                pkg.linear_fp8(x8, w8, torch.full((3, 3), 0.25, device=dev),
                               x_scale=torch.full((40, 3), 0.25, device=dev)),
                pkg.rms_norm_gated_fp8(o, z, weight, 1e-6)[0].view(torch.uint8))

    want = run()
    torch.cuda.synchronize()
    assert torch.equal(want[4], want[5])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("M", [1, 2, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("N,K", [(40, 128), (256, 896), (2048, 2048), (512, 2176), (1024, 4096), (64, 4224), (12288, 2048),
                                 (8200, 640), (8320, 4096), (8320, 2304)])
def test_linear_fp8_few_rows(pkg, dev, M, N, K):
    """Few bf16 rows, also strided, with a NaN, an infinity and a row of zeros among them: the
    bits of quantize_fp8 and a call with its result; rows past M are not there; bf16 columns."""
    gen = torch.Generator().manual_seed(M + N + K)
    big = _rows(gen, M + 1, K + 8).to(BF16)
    w8, ws = (t.to(dev) for t in ref.to_e4m3(_rows(gen, N, K) * K ** -0.5, 128))
    for bad in (False, True):
        if bad:
            big[0, 8 + K - 3] = float("nan")
            big[M // 2, 9] = float("-inf")
            big[M - 1] = 0
        x = big.to(dev)[:M, 8:]
        x8, xs = pkg.quantize_fp8(x)
        want = pkg.linear_fp8(x8, w8, ws, x_scale=xs)
        out = torch.full((M + 1, N + 3), 7.0, dtype=BF16, device=dev)
        pkg.linear_fp8(x, w8, ws, out=out[:M, :N])
        wide = torch.randn(32, K, generator=gen).to(BF16).to(dev)
        parts = pkg.ops.linear_fp8_cols(x, w8, ws, [N, 16, 16], wide=wide) if N % 16 == 0 else None
        torch.cuda.synchronize()
        rows = [r for r in range(M) if not bad or r not in (0, M // 2)] + ([M - 1] if bad else [])
        assert torch.equal(out[rows, :N], want[rows]) and bool(want[rows].isfinite().all())
        if bad and M > 2:
            assert bool(out[[0, M // 2], :N].isnan().all())
        assert bool((out[M:] == 7).all()) and bool((out[:, N:] == 7).all())
        if parts is not None:
            assert torch.equal(parts[0][rows], want[rows])
            a, b = x[rows].double(), wide.double()
            slack = (a.abs() @ b.abs().t()) * (K + K // 64) * ref.U32
            _check(torch.cat(parts[1:], 1)[rows], a @ b.t(), slack, "bf16 columns")


@pytest.mark.parametrize("B,Hk,Hv", [(1, 16, 32), (5, 2, 2), (33, 4, 8), (7, 2, 8), (130, 16, 16), (170, 16, 32)])
@pytest.mark.parametrize("params", [BF16, torch.float32])
def test_decode_step_to_e4m3(pkg, dev, B, Hk, Hv, params):
    """The decode step's norm in e4m3, in each of its forms (whole step in one launch with one or
    two value heads per key head, at small and at large batches; behind the q/k conv): the bits
    of rms_norm_gated_fp8 on the core output, the pools those of the bf16 step."""
    gen = torch.Generator().manual_seed(B + Hv)
    D = 128
    C, kd = 2 * Hk * D + Hv * D, Hk * D
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16).to(dev)  # noqa: E731
    mixed, z, b, a, conv_w = n(B, C), n(B, Hv * D + 8)[:, :Hv * D], n(B, Hv), n(B, Hv), n(C, 4)
    a_log, dt = (torch.randn(Hv, generator=gen).to(params).to(dev) for _ in range(2))
    w = (1 + 0.1 * torch.randn(D, generator=gen)).to(BF16).to(dev)
    pools = [((torch.randn(B + 2, Hv, D, D, generator=torch.Generator().manual_seed(1)) * 0.2).to(dev),
              torch.randn(B + 2, C, 3, generator=torch.Generator().manual_seed(2)).to(BF16).to(dev)) for _ in range(2)]
    ids = torch.randperm(B + 2, generator=gen)[:B].to(dev)
    z[0] = 0                                             # a row of zeros: the smallest scale

    def step(s_pool, c_pool, whole, **kw):
        qk = None if whole else pkg.conv_decode_step(mixed[:, :2 * kd], c_pool[:, :2 * kd], ids, conv_w[:2 * kd])
        return pkg.ops.recurrent_decode_fused(qk, mixed, c_pool, conv_w, b, a, a_log, dt, s_pool, ids, Hk, Hv, D,
                                              grouped=whole, **kw)

    core = step(*pools[0], False)
    want, ws = pkg.rms_norm_gated_fp8(core, z.reshape(B, 1, Hv, D), w, 1e-6)
    for whole in ([True, False] if Hv <= 2 * Hk else [False]):
        s_pool, c_pool = (t.clone() for t in pools[1])
        y, scale = step(s_pool, c_pool, whole, z=z, norm_weight=w, fp8=True)
        torch.cuda.synchronize()
        assert y.shape == (B, 1, Hv, D) and torch.equal(y.view(torch.uint8), want.view(torch.uint8))
        assert torch.equal(scale, ws) and scale.shape == (B, Hv)
        assert torch.equal(s_pool, pools[0][0]) and torch.equal(c_pool.view(torch.int16), pools[0][1].view(torch.int16))


@pytest.mark.parametrize("M,N,K", [(1, 2048, 256), (3, 72, 128), (16, 520, 384), (37, 2048, 4096), (300, 512, 2048),
                                   (600, 2048, 256), (1500, 2048, 384), (4100, 2056, 128)])
@pytest.mark.parametrize("lead", [1, 2, 4, 8])
def test_linear_fp8_into_columns_that_begin_anywhere(pkg, dev, M, N, K, lead):
    """out: columns of a wider buffer, its rows of 16-byte pieces, that begin between them."""
    gen = torch.Generator().manual_seed(M + N + lead)
    x = _rows(gen, M, K).to(BF16).to(dev)
    w8, ws = (t.to(dev) for t in ref.to_e4m3(_rows(gen, N, K) * K ** -0.5, 128))
    buf = torch.full((M, N + 16), 7.0, dtype=BF16, device=dev)
    pkg.linear_fp8(x, w8, ws, out=buf[:, lead:lead + N])
    torch.cuda.synchronize()
    assert torch.equal(buf[:, lead:lead + N], pkg.linear_fp8(x, w8, ws))
    assert bool((buf[:, :lead] == 7).all()) and bool((buf[:, lead + N:] == 7).all())


@pytest.mark.parametrize("lead", [1, 4])
def test_norm_weight_that_begins_anywhere(pkg, dev, lead):
    gen = torch.Generator().manual_seed(83)
    x, z, w = (torch.randn(*s, generator=gen).to(BF16).to(dev) for s in ((5, 2, 128), (5, 2, 128), (128,)))
    flat = torch.cat([w[:lead], w])[lead:]
    assert flat.is_contiguous() and flat.data_ptr() % 16
    got, want = pkg.rms_norm_gated_fp8(x, z, flat, 1e-6), pkg.rms_norm_gated_fp8(x, z, w, 1e-6)
    torch.cuda.synchronize()
    assert torch.equal(_bits(got[0]), _bits(want[0])) and torch.equal(got[1], want[1])


# odd numbers of 128-column blocks: a ring, tiles in two halves of K, 256-row tiles with whole ones and quarters alone
@pytest.mark.parametrize("M,N,K", [(3, 512, 384), (500, 2000, 2176), (4100, 2056, 640), (8492, 2304, 384), (200, 8192, 640),
                                   (1500, 2048, 640)])
def test_linear_fp8_infinite_row_scales(pkg, dev, M, N, K):
    """A caller's infinite scale of a row's last block, whose values are positive as the weight's are,
    makes the row infinite, not NaN; the other rows are what they were."""
    gen = torch.Generator().manual_seed(M + K)
    x8, xs = (t.to(dev) for t in ref.to_e4m3(_rows(gen, M, K), 1))
    w8, ws = (t.to(dev) for t in ref.to_e4m3(_rows(gen, N, K).abs() + 0.1, 128))
    x8.view(torch.uint8)[:, -128:] = 0x38                      # 1.0
    y = pkg.linear_fp8(x8, w8, ws, x_scale=xs)
    rows = torch.randperm(M, generator=gen)[:max(1, M // 7)].to(dev)
    xs[rows, -1] = float("inf")
    z = pkg.linear_fp8(x8, w8, ws, x_scale=xs)
    torch.cuda.synchronize()
    assert bool((z[rows] == float("inf")).all())
    others = torch.ones(M, dtype=torch.bool, device=dev)
    others[rows] = False
    assert torch.equal(z[others], y[others]) and bool(y.isfinite().all())


@pytest.mark.parametrize("lens", [[1] * 4, [1, 1, 30, 70]])
def test_steps_that_write_bf16_take_any_heads(pkg, dev, lens):
    """Three value heads of 64 (no whole groups of 128): decode rows, and decode rows ahead of prompts,
    give bf16 with fp8 too, and the same."""
    gen = torch.Generator().manual_seed(97)
    Hk, Hv, D, N = 1, 3, 64, sum(lens)
    C = (2 * Hk + Hv) * D
    n = lambda *s: torch.randn(*s, generator=gen).to(BF16).to(dev)  # noqa: E731
    core = pkg.GatedDeltaNetCore(Hk, Hv, D, n(C, 4), n(Hv), n(Hv), n(D))
    rows = n(N, C), n(N, Hv * D), n(N, Hv), n(N, Hv)
    pools = torch.randn(4, Hv, D, D, generator=gen).to(dev) * 0.1, n(4, C, 3)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(dev)
    got = []
    for fp8 in (False, True):
        s, c = (p.clone() for p in pools)
        got.append((core.forward(*rows, cu, max(lens), torch.arange(4, device=dev), c, s, lens_q=lens, fp8=fp8), s, c))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*got)) and got[0][0].dtype == BF16
