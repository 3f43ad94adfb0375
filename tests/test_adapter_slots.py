"""Slots of adapters and the block's norms: what is refused before anything changes (CPU tensors)."""
from types import SimpleNamespace

import pytest
import torch


def test_clear_refuses_slots_that_are_not_there(pkg):
    """-1 is the slot of rows without an adapter: clearing it leaves the last one as it was."""
    pool = pkg.LoraPool(3, 8, 64, [32, 16], device="cpu")
    for slot in range(3):
        pool.load(slot, [(torch.ones(8, 64), torch.ones(32, 8)), (torch.ones(8, 64), torch.ones(16, 8))], 1.0 + slot)
    before = [t.clone() for t in (pool.a, pool.b, pool.scale)]
    for slot in (-1, -3, 3, 100):
        with pytest.raises(ValueError, match="slot"):
            pool.clear(slot)
        assert all(torch.equal(p, q) for p, q in zip(before, (pool.a, pool.b, pool.scale))), slot
    pool.clear(1)
    assert not pool.a[1].any() and not pool.b[1].any() and pool.scale.tolist() == [1.0, 0.0, 3.0]
    assert torch.equal(pool.a[2], before[0][2]) and torch.equal(pool.b[0], before[1][0])


def test_block_refuses_norms_before_a_step(pkg):
    """What the second norm's call would refuse only after the mixer has moved its pools on."""
    layer = SimpleNamespace(hidden=64, w_in=torch.zeros(8, 64))
    good = torch.zeros(64, dtype=torch.bfloat16)
    for norm in (good, good.float()):
        block = pkg.GatedDeltaNetBlock(layer, good, norm)
        assert block.post_norm is norm
    for bad, error in ((good.half(), TypeError), (good.double(), TypeError), (good.to(torch.int16), TypeError),
                       (good.to("meta"), ValueError), (good[:32], ValueError), (good[None], ValueError)):
        for norms in ((good, bad), (bad, good)):
            with pytest.raises(error):
                pkg.GatedDeltaNetBlock(layer, *norms)


def test_room_for_adapters_stays(pkg):
    """Captured graphs read the pools: a second add_adapters empties them in place or is refused."""
    hidden, Hk, Hv, D = 64, 8, 16, 64
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    C = (2 * Hk + Hv) * D
    layer = pkg.GatedDeltaNetLayer(z(C, hidden), z(Hv * D, hidden), z(Hv, hidden), z(Hv, hidden), z(hidden, Hv * D), Hk, Hv, D,
                                   z(C, 4), z(Hv), z(Hv), z(D))
    layer.add_adapters(3, 12)
    held = [t for pool in (layer.lora_in, layer.lora_out) for t in (pool.a, pool.b, pool.scale)]
    layer.load_adapter(2, 0.5, z=(torch.ones(12, hidden), torch.ones(Hv * D, 12)), out=(torch.ones(8, Hv * D), torch.ones(hidden, 8)))
    assert all(bool(t[2].any()) for t in held)
    kept = [t.clone() for t in held]
    for slots, rank in ((4, 12), (2, 12), (3, 8), (3, 17), (0, 12), (3, 0)):
        with pytest.raises(ValueError, match="room for 3 adapters of rank 16"):
            layer.add_adapters(slots, rank)
    now = lambda: [t for pool in (layer.lora_in, layer.lora_out) for t in (pool.a, pool.b, pool.scale)]  # noqa: E731
    assert all(p is q and torch.equal(p, k) for p, q, k in zip(held, now(), kept))
    layer.add_adapters(3, 16)
    assert all(p is q and not p.any() for p, q in zip(held, now()))
    layer.lora_in = layer.lora_out = None
    layer.add_adapters(4, 40)
    assert layer.lora_in.a.shape == (4, 160, hidden) and layer.lora_out.b.shape == (4, hidden, 40)
    layer.load_adapter(3, 1.0)


def test_adapter_rows_of_64_bits(pkg):
    """Numbers that 32 bits do not hold name no slot, whatever their low bits are."""
    far = torch.tensor([3, (1 << 32) + 3, -(1 << 32), 1 << 40, (1 << 31) - 1, -1, -(1 << 63), 0])
    rows = pkg.adapter_rows(far, torch.arange(9), 8)
    assert rows.dtype == torch.int32
    for slots in (4, 1 << 20):
        named = [int(r) if 0 <= r < slots else None for r in rows]
        assert named == [3, None, None, None, None, None, None, 0]
    assert pkg.adapter_rows(far[5:6], torch.arange(2), 1).tolist() == [-1]
