"""The norms around a block where their arguments end: gates past what an exponential holds, rows past one launch."""
import pytest
import torch

from helpers import BF16
from test_gpu_block_norm import EPS, F32, _check, _inputs

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
GATES = [INF, -INF, 3e38, -3e38, 2.4e38, 500.0, 89.0, 88.0, -88.0, -500.0, 0.0, NAN]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", ["row", "column", "value"])
def test_gates_of_any_size(pkg, dev, form, dtype):
    """sigmoid is 1 far above 0, up to an infinity, and 0 far below; a NaN is one where it gates and, as a part of the
    mean, in its row's y."""
    M, H = len(GATES), 640
    x, res, w, _ = _inputs(M, H, "plain", True, dev)
    g = torch.tensor(GATES, device=dev).to(dtype)
    if form == "row":
        gate, spread = g[:, None], g[:, None].expand(M, H)
    elif form == "column":
        gate = torch.zeros(H, dtype=dtype, device=dev)
        gate[5:5 + M - 1] = g[:-1]          # (no NaN, which would be in every row)
        spread = gate.expand(M, H)
    else:
        gate = torch.zeros(M, H, dtype=dtype, device=dev)
        gate[torch.arange(M), torch.arange(M) * 50] = g
        spread = gate
    kw = dict(gate=gate, gate_sigmoid=True, scale=0.5)
    y, r = pkg.add_rms_norm(x, res, w, EPS, **kw)
    y8, ys, r8, keep = pkg.add_rms_norm_fp8(x, res, w, EPS, keep=True, **kw)
    torch.cuda.synchronize()
    same = lambda a, b: torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))  # noqa: E731
    assert same(y, keep) and same(r, r8)
    nan = spread.isnan()
    assert torch.equal(r.isnan(), nan) and torch.equal(y.isnan(), nan.any(1, keepdim=True).expand(M, H))
    rows = ~nan.any(1)
    _check(y[rows], r[rows], x[rows], res[rows], w, dict(kw, gate=spread[rows]), form)
    shut = spread <= -500
    assert torch.equal(r[shut], res[shut])
    open_ = spread >= 500
    assert torch.equal(r[open_], torch.add(res, x.float(), alpha=0.5)[open_])
    # the same by rows that are not whole pieces
    odd = 333
    part = gate if form == "row" else gate[..., :odd].contiguous()
    y, r = pkg.add_rms_norm(x[:, :odd].contiguous(), res[:, :odd].contiguous(), w[:odd], EPS, gate=part, gate_sigmoid=True,
                            scale=0.5)
    torch.cuda.synchronize()
    assert torch.equal(r.isnan(), nan[:, :odd])


def test_more_rows_than_a_launch_has(pkg, dev):
    """Narrow rows past what one launch's threads number: the bits of the calls with a part of the rows."""
    M, H, part = (1 << 26) + 5, 8, 1 << 22
    gen = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(M, H, generator=gen, device=dev, dtype=BF16)
    res = torch.randn(M, H, generator=gen, device=dev)
    gate = torch.randn(M, 1, generator=gen, device=dev, dtype=BF16)
    w = torch.randn(H, generator=gen, device=dev, dtype=BF16)
    y, r = pkg.add_rms_norm(x, res, w, EPS, gate=gate, gate_sigmoid=True)
    torch.cuda.synchronize()
    for at in range(0, M, part):
        to = min(M, at + part)
        if to - at < 2048:
            at = to - 2048
        ey, er = pkg.add_rms_norm(x[at:to], res[at:to], w, EPS, gate=gate[at:to], gate_sigmoid=True)
        assert torch.equal(y[at:to], ey) and torch.equal(r[at:to], er), at
    last = slice(M - 2048, M)
    _check(y[last], r[last], x[last], res[last], w, dict(gate=gate[last], gate_sigmoid=True))
