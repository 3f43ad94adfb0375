"""Calls whose outputs do not fit: torch's own error, and nothing moved on."""
import contextlib

import pytest
import torch

from helpers import BF16

pytestmark = pytest.mark.gpu
MIB = 1 << 20


@contextlib.contextmanager
def _memory_left(dev, mib):
    """This process has mib MiB left, by the allocator's own limit: no new segments, and what is free
    inside of those that are there (pieces below 16 MiB apart) is held meanwhile."""
    torch.cuda.synchronize()
    take = lambda size: torch.empty(size, dtype=torch.uint8, device=dev)  # noqa: E731
    left, held, size = take(mib * MIB), [], 4096 * MIB
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(dev).total_memory
    torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved(dev) / total, dev)
    try:
        while size >= 16 * MIB:
            try:
                held.append(take(size))
            except torch.OutOfMemoryError:
                size //= 2
        del left
        yield
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0, dev)
        held.clear()


def test_out_of_memory_is_torchs_error(pkg, dev):
    x8 = torch.zeros(8192, 128, dtype=torch.float8_e4m3fn, device=dev)
    w8 = torch.zeros(16384, 128, dtype=torch.float8_e4m3fn, device=dev)
    xs, ws = torch.ones(8192, 1, device=dev), torch.ones(128, 1, device=dev)
    rows = torch.zeros(16, 8192, 8, 128, dtype=BF16, device=dev)
    weight = torch.ones(128, dtype=BF16, device=dev)
    with _memory_left(dev, 32):
        for call in (lambda: pkg.linear_fp8(x8, w8, ws, x_scale=xs),                       # 256 MiB
                     lambda: pkg.rms_norm_gated_fp8(rows, rows, weight, 1e-6)):             # 128 MiB and scales
            with pytest.raises(torch.OutOfMemoryError):
                call()
    assert pkg.linear_fp8(x8, w8, ws, x_scale=xs).shape == (8192, 16384)


def test_a_verify_without_memory_leaves_the_pools(pkg, dev):
    """Room for the conv's rows (512 MiB) but not for the rule's outputs (768 MiB) behind them: neither
    pool has moved on."""
    gen = torch.Generator(device=dev).manual_seed(89)
    B, T, Hk, Hv, D = 512, 64, 16, 32, 128
    C = (2 * Hk + Hv) * D
    n = lambda *s: torch.randn(*s, generator=gen, device=dev, dtype=BF16)  # noqa: E731
    core = pkg.GatedDeltaNetCore(Hk, Hv, D, n(C, 4), n(Hv), n(Hv), n(D))
    s, c = torch.randn(B, Hv, D, D, generator=gen, device=dev) * 0.1, n(B, C, 3)
    ids, par = torch.arange(B, device=dev), torch.arange(-1, T - 1, dtype=torch.int32, device=dev)
    rows = n(B, T, C), n(B, T, Hv * D), n(B, T, Hv), n(B, T, Hv)
    _, step = core.verify_tree(*rows, ids, c, s, par)
    step.accept(torch.full((B,), 2, device=dev))
    before = s.clone(), c.clone()
    with _memory_left(dev, 640):
        with pytest.raises(torch.OutOfMemoryError):
            core.verify_tree(*rows, ids, c, s, par, pending=step)
    torch.cuda.synchronize()
    assert torch.equal(s, before[0]) and torch.equal(c, before[1])
    got, _ = core.verify_tree(*rows, ids, c, s, par, pending=step)
    core.commit_tree(step, ids, before[1], before[0])
    want, _ = core.verify_tree(*rows, ids, before[1], before[0], par)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(s, before[0]) and torch.equal(c, before[1])
