"""Adapters of large ranks and several parts against 64 bits, the tolerances those of test_gpu_lora."""
import pytest
import torch

import tree_ref as ref
from helpers import BF16
from test_gpu_block import _layer
from test_gpu_lora import U, _adapters, _check, _delta, _ids

pytestmark = pytest.mark.gpu


def _products(pkg, dev, M, widths, K, R, S, how, forms):
    """The calls named by forms, each checked."""
    gen = torch.Generator().manual_seed(M * 7 + R + sum(widths))
    ids, lora = _ids(gen, M, S, how).to(dev), [t.to(dev) for t in _adapters(gen, S, widths, K, R)]
    x = torch.randn(M, K, generator=gen).to(BF16).to(dev)
    w = (torch.randn(sum(widths), K, generator=gen) * K ** -0.5).to(BF16).to(dev)
    w8, ws = pkg.quantize_weight_fp8(w)
    x8, xs = pkg.quantize_fp8(x)
    for form in forms:
        if form == "bf16":
            y = pkg.linear_lora(x, w, *lora, ids, widths=widths)
            want, slack = x.double() @ w.double().t(), 2 * (K + 2 * R) * U * (x.double().abs() @ w.double().abs().t())
            delta, loose = _delta(x, *lora, ids, widths, K)
        else:
            ready = form == "e4m3"
            y = pkg.linear_fp8_lora(x8 if ready else x, w8, ws, *lora, ids, x_scale=xs if ready else None, widths=widths)
            seen = (x8.double().unflatten(-1, (-1, 128)) * xs.double()[..., None]).flatten(-2) if ready else x
            want, slack = ref.linear(x8, xs, w8, ws)
            delta, loose = _delta(seen, *lora, ids, widths, K)
            slack = slack + 4 * R * U * (want.abs() + delta.abs())
        torch.cuda.synchronize()
        _check(torch.cat(y, 1), want + delta, slack + loose, f"{form} M {M} R {R}")


@pytest.mark.parametrize("R", [224, 232, 240, 256])
@pytest.mark.parametrize("M", [224, 225, 240, 241, 256])
def test_decode_batches_of_four_parts(pkg, dev, M, R):
    """The rows that are taken in their adapters' order, at the widths where the shrink's tiles are many."""
    _products(pkg, dev, M, [96, 32, 48, 80], 256, R, 9, "mixed", ("bf16", "quantized", "e4m3"))


@pytest.mark.parametrize("weights", ["bf16", "fp8"])
def test_layer_with_the_largest_adapters(pkg, dev, weights):
    """A decode batch of 256 rows through a layer whose adapters have rank 256."""
    gen = torch.Generator().manual_seed(256)
    Hk, Hv, D, hidden, S, M = 8, 16, 128, 512, 7, 256
    layer, (C, w_qkv, w_z, w_b, w_a, *_) = _layer(pkg, dev, gen, hidden, Hk, Hv, D, weights)
    layer.add_adapters(S, 256)
    pool = layer.lora_in
    a, b, scale = _adapters(gen, S, pool.widths, hidden, 256)
    pool.a.copy_(a)
    pool.b.copy_(b)
    pool.scale.copy_(scale)
    ids = _ids(gen, M, S, "mixed").to(dev)
    x = torch.randn(M, hidden, generator=gen).to(BF16).to(dev)
    y = torch.cat(layer.project_in(x, adapters=ids)[:4], 1)
    w = torch.cat([t.to(dev) for t in (w_qkv, w_z, w_b, w_a)]).double()
    want, slack = x.double() @ w.t(), 2 * (hidden + 512) * U * (x.double().abs() @ w.abs().t())
    delta, loose = _delta(x, pool.a, pool.b, pool.scale, ids, pool.widths, hidden)
    if weights == "fp8":
        x8, xs = pkg.quantize_fp8(x)
        n = layer.w_in.shape[0]
        want[:, :n], slack[:, :n] = ref.linear(x8, xs, layer.w_in, layer.w_in_scale)
        slack = slack + 4 * 256 * U * (want.abs() + delta.abs())
    torch.cuda.synchronize()
    _check(y, want + delta, slack + loose)


@pytest.mark.parametrize("M,widths,R", [
    # the last shapes of the few rows' shrink (tiles of 16 x 16 up to 896) and the first ones past them
    (257, [96, 32, 48, 80], 208), (257, [96, 32, 48, 80], 216), (1024, [96, 32, 48, 80], 56), (1024, [64, 48, 16], 80),
    (1025, [96, 32, 48, 80], 56), (2048, [80, 16], 56), (2048, [80, 16], 64), (2049, [80, 16], 56),
    # ranks past 128: small products, 256 x 256 tiles with a rest, a last tile of two slices
    (257, [512], 256), (300, [8192, 4096, 32, 32], 136), (900, [4096, 4096], 200), (1300, [8192, 4096, 32, 32], 256),
    (2500, [2048, 4096, 16, 32], 248), (4100, [2064], 192)])
@pytest.mark.parametrize("how", ["mixed", "sequences"])
def test_more_rows_and_large_ranks(pkg, dev, M, widths, R, how):
    _products(pkg, dev, M, widths, 256, R, 6, how, ("bf16", "quantized", "e4m3"))
