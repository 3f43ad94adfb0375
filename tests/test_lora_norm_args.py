"""What the calls around the projections refuse before any launch: the wrappers with the device
check and the launch stubbed (CPU tensors), the C entry points with NULL or, where no GPU is
visible, dummy aligned addresses."""
import ctypes

import pytest
import torch

BF16, FP8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


class Launched(Exception):
    pass


@pytest.fixture
def ops(pkg, monkeypatch):
    def fake_call(*a, **k):
        raise Launched()

    monkeypatch.setattr(pkg.ops, "_device_of", lambda *ts: 0)
    monkeypatch.setattr(pkg.ops, "_call_on", fake_call)
    monkeypatch.setattr(pkg._lib, "call", fake_call)
    monkeypatch.setattr(pkg._lib, "stream_of", lambda index: 0)

    class Quick:
        def __getattr__(self, name):
            return lambda *a: None

    monkeypatch.setattr(pkg._lib, "quick", lambda: Quick())
    return pkg.ops


def _refused(fn, good, **bad):
    """fn with good arguments reaches the launch; with each bad one it does not."""
    with pytest.raises(Launched):
        fn(**good)
    for name, values in bad.items():
        for value in values:
            with pytest.raises((ValueError, TypeError)):
                fn(**{**good, name: value})


@pytest.mark.parametrize("fp8", [False, True])
def test_add_rms_norm_refuses(ops, fp8):
    M, H = 4, 256
    x, w = torch.zeros(M, H, dtype=BF16), torch.zeros(H, dtype=BF16)
    fn = ops.add_rms_norm_fp8 if fp8 else ops.add_rms_norm
    _refused(fn, dict(x=x, residual=x, weight=w, eps=1e-6, post_weight=w, gate=torch.zeros(M, 1)),
             x=[x.float(), x[:, :128], torch.zeros((), dtype=BF16)], residual=[x[:2], x.half(), x[:, :1]],
             weight=[w[:128], w.half(), w[None]], post_weight=[w[:1], w.double(), w[None]],
             gate=[torch.zeros(M), torch.zeros(1, H), torch.zeros(M, 2), torch.zeros(M, 1, dtype=torch.half),
                   torch.zeros(M, H, 1)],
             residual_out=[x.float(), x[:2], torch.zeros(H, M, dtype=BF16).t(), torch.zeros(M, 2 * H, dtype=BF16)[:, ::2]])
    for wide in (0, 16385 if not fp8 else 16384 + 128):
        with pytest.raises(ValueError):
            fn(torch.zeros(1, wide, dtype=BF16), None, torch.zeros(wide, dtype=BF16), 1e-6)
    if fp8:
        with pytest.raises(ValueError, match="128"):
            fn(x[:, :200], None, w[:200], 1e-6)


def _lora(S=3, P=2, R=16, K=128, N=96):
    return dict(lora_a=torch.zeros(S, P * R, K, dtype=BF16), lora_b=torch.zeros(S, N, R, dtype=BF16),
                lora_scale=torch.zeros(S))


def _bad_lora(S=3, P=2, R=16, K=128, N=96):
    z = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    return dict(
        lora_a=[z(S, R, K), z(S, P * R, K - 64), z(S + 1, P * R, K), z(P * R, K), z(S, P * R, K).float(),
                z(S, K, P * R).transpose(1, 2), z(S, P * R, 2 * K)[..., :K]],
        lora_b=[z(S, N - 16, R), z(S, N, 12), z(S, N, 8), z(S, N, 264), z(N, R), z(S, N, R).float(), z(S, R, N).transpose(1, 2),
                z(S * N * R + 1)[1:].view(S, N, R)],
        lora_scale=[torch.zeros(S, dtype=BF16), torch.zeros(S + 1), torch.zeros(S, 1), torch.zeros(2 * S)[::2]])


def test_linear_lora_refuses(ops):
    M, N, K = 5, 96, 128
    x, w, ids = torch.zeros(M, K, dtype=BF16), torch.zeros(N, K, dtype=BF16), torch.zeros(M, dtype=I32)
    _refused(ops.linear_lora, dict(x=x, weight=w, ids=ids, widths=[64, 32], **_lora()),
             x=[x.float(), x[:, :64], x[:4]], weight=[w.float(), w[:80], w[:, :64], w[0]],
             ids=[ids.long(), ids[:4], ids[None], ids.float()],
             widths=[[64, 16], [60, 36], [96, 0], [32, 16, 16, 16, 16], [], None, [128, -32]], **_bad_lora())
    with pytest.raises(ValueError, match="64"):
        ops.linear_lora(x[:, :96], w[:, :96], ids=ids, **_lora(P=1, K=96))


def test_linear_fp8_lora_refuses(ops):
    M, N, K = 5, 96, 128
    x, ids = torch.zeros(M, K, dtype=BF16), torch.zeros(M, dtype=I32)
    w, ws = torch.zeros(N, K, dtype=torch.uint8).view(FP8), torch.zeros(1, 1)
    good = dict(x=x, weight=w, weight_scale=ws, ids=ids, widths=[64, 32], **_lora())
    _refused(ops.linear_fp8_lora, good, x=[x.float(), x[:, :64], x.to(FP8)], weight=[w.view(torch.uint8), w[:80]],
             weight_scale=[ws.double(), torch.zeros(2, 1)], x_scale=[torch.zeros(M, 1)],
             ids=[ids.long(), ids[:4]], widths=[[64, 16], [60, 36], []], gates=[dict(gate_col=0)], **_bad_lora())
    wide = torch.zeros(32, K, dtype=BF16)
    more = dict(good, wide=wide, widths=[96, 32], **_lora(N=128))
    _refused(ops.linear_fp8_lora, more, wide=[wide.float(), wide[:20], wide[:0], wide[:, :64]],
             widths=[[64, 64], [128], [96, 16, 20]])
    with pytest.raises(TypeError):   # (the wide columns read bf16 rows)
        ops.linear_fp8_lora(**{**more, "x": x.to(FP8), "x_scale": torch.zeros(M, 1)})


def _bad_gates(N, Hv=8):
    z = torch.zeros
    good = dict(A_log=z(Hv), dt_bias=z(Hv), gate_col=N - 2 * Hv)
    return good, [dict(good, **bad) for bad in (
        dict(dt_bias=z(Hv - 1)), dict(dt_bias=z(Hv + 1)), dict(A_log=z(Hv - 1)), dict(A_log=z(0), dt_bias=z(0)), dict(gate_col=-1),
        dict(gate_col=N - 2 * Hv + 1), dict(A_log=z(Hv, dtype=I32)), dict(dt_bias=z(Hv, dtype=torch.int64)))]


def test_gates_refuse(ops, monkeypatch):
    """Gates' parameters of another length, or whose columns are not the product's; all of them
    go through the device check."""
    M, N, K = 5, 96, 128
    x, w, ids = torch.zeros(M, K, dtype=BF16), torch.zeros(N, K, dtype=BF16), torch.zeros(M, dtype=I32)
    gates, bad = _bad_gates(N)
    _refused(ops.linear_lora, dict(x=x, weight=w, ids=ids, widths=[64, 32], gates=gates, **_lora()), gates=bad)
    wide = dict(x=x, weight=torch.zeros(N, K, dtype=torch.uint8).view(FP8), weight_scale=torch.zeros(1, 1), ids=ids, widths=[96, 32],
                wide=torch.zeros(32, K, dtype=BF16), **_lora(N=128))
    gates, bad = _bad_gates(32)
    _refused(ops.linear_fp8_lora, dict(wide, gates=gates), gates=bad)
    seen = []
    monkeypatch.setattr(ops, "_device_of", lambda *ts: seen.extend(map(id, ts)) or 0)
    for call in (lambda: ops.linear_fp8_lora(gates=gates, **wide),
                 lambda: ops.linear_lora(x, w, ids=ids, widths=[64, 32], gates=gates, **_lora())):
        seen.clear()
        with pytest.raises(Launched):
            call()
        assert {id(gates["A_log"]), id(gates["dt_bias"])} <= set(seen)


def test_pool_refuses(pkg):
    with pytest.raises(ValueError):
        pkg.LoraPool(2, 0, 64, [32], device="cpu")
    with pytest.raises(ValueError):
        pkg.LoraPool(2, 257, 64, [32], device="cpu")
    for widths in ([], [24, 8], [16, 0], [16] * 5):
        with pytest.raises(ValueError):
            pkg.LoraPool(2, 8, 64, widths, device="cpu")
    pool = pkg.LoraPool(2, 5, 64, [32, 16], device="cpu")
    assert pool.rank == 8
    z = lambda *s: torch.ones(*s)  # noqa: E731
    pool.load(0, [(z(8, 64), z(32, 8)), None], 1.0)
    before = pool.a.clone(), pool.b.clone()
    for slot, parts in ((2, [None, None]), (-1, [None, None]), (0, [None]), (0, [(z(9, 64), z(32, 9)), None]),
                        (0, [(z(4, 32), z(32, 4)), None]), (0, [(z(4, 64), z(16, 4)), None]), (0, [None, (z(4, 64), z(16, 3))])):
        with pytest.raises(ValueError):
            pool.load(slot, parts, 1.0)
    assert torch.equal(pool.a, before[0]) and torch.equal(pool.b, before[1])   # (a refused load changes nothing)


def test_c_entries_refuse(pkg):
    lib, bad = pkg._lib.load(), pkg._lib.GDN_ERR_INVALID_ARG
    norm = lambda M=4, H=256, g_col=0, y=None, y8=None: lib.gdn_add_rms_norm(  # noqa: E731
        None, H, None, 0, 0, None, None, 0, 1.0, None, 0, 0, g_col, 0, 1.0, 1e-6, None, y, y8, None, 1, M, M, H, None)
    assert norm() == bad and norm(M=-1) == bad and norm(H=0) == bad and norm(g_col=2) == bad
    assert norm(H=16385) == pkg._lib.GDN_ERR_UNSUPPORTED and norm(M=0) == 0
    shrink = lambda slots=2, slices=1, rank=16, M=4, K=128: lib.gdn_lora_shrink(  # noqa: E731
        None, 1, K, None, 0, 0, None, 0, None, None, slots, slices, rank, M, K, None, 32, None, None, 0, None, 0, 0, None)
    for kw in (dict(), dict(slots=-1), dict(slices=0), dict(slices=5), dict(rank=12), dict(rank=264), dict(rank=0), dict(K=96),
               dict(M=-1), dict(K=0)):
        assert shrink(**kw) == bad, kw
    assert shrink(M=0) == 0 and shrink(slots=0) == 0
    n = ctypes.c_int * 4
    parts = (ctypes.c_void_p * 4)(*[1 << 20] * 4), (ctypes.c_int64 * 4)(*[128] * 4)
    if torch.cuda.device_count() > 0:
        pytest.skip("dummy device addresses are passed only where no GPU is visible")
    P = ctypes.c_void_p(1 << 20)

    def bf16(M=4, N=96, K=64, ends=(96,), slice_ends=(96,), v=P, ldv=32, groups=P, lb=P, lb_slot=96 * 16, ids=P, slots=2, rank=16):
        return lib.gdn_gemm_bf16_lora(P, K, P, K, M, N, K, len(ends), *parts, n(*ends), None, None, None, None, 0, 0, 0, v, ldv,
                                      groups, lb, lb_slot, ids, slots, rank, len(slice_ends), n(*slice_ends), None)

    def fp8(M=4, N=96, K=128, ends=(96,), slice_ends=(96,), v=P, ldv=32, groups=P, lb=P, lb_slot=96 * 16, ids=P, slots=2, rank=16):
        return lib.gdn_gemm_fp8_lora(P, K, P, 1, M, P, K, P, 1, M, N, K, len(ends), *parts, n(*ends), v, ldv, groups, lb, lb_slot, ids,
                                     slots, rank, len(slice_ends), n(*slice_ends), None)

    def shrink(x_is_bf16=1, M=4, K=128, x8=P, sx8=128, s8=P, ids=P):
        return lib.gdn_lora_shrink(P, x_is_bf16, K, P, 1, M, P, 16 * K, P, ids, 2, 1, 16, M, K, P, 32, P, x8, sx8, s8, 1, M, None)

    for kw in (dict(x_is_bf16=0), dict(K=64), dict(x8=ctypes.c_void_p((1 << 20) + 4)), dict(sx8=120), dict(sx8=132), dict(s8=None),
               dict(s8=ctypes.c_void_p((1 << 20) + 2)), dict(ids=None)):
        assert shrink(**kw) == bad, kw
    odd, byte = ctypes.c_void_p((1 << 20) + 2), ctypes.c_void_p((1 << 20) + 1)
    for call in (bf16, fp8):
        for kw in (dict(v=None), dict(v=odd), dict(groups=None), dict(groups=byte), dict(lb=None), dict(lb=odd), dict(ids=None), dict(ids=odd), dict(slots=-1),
                   dict(rank=12), dict(rank=264), dict(ldv=24), dict(ldv=36), dict(lb_slot=95 * 16), dict(lb_slot=96 * 16 + 4),
                   dict(slice_ends=(90,)), dict(slice_ends=(24, 96)), dict(slice_ends=(96, 96), ldv=64), dict(slice_ends=()),
                   dict(slice_ends=(48, 96)), dict(M=1 << 30), dict(K=100), dict(ends=(90,))):
            assert call(**kw) == bad, (call.__name__, kw)
    assert bf16(M=0) == 0 and fp8(N=0) == 0
    good = dict(x=P, sx=256, res=P, sr=256, w=P, post=None, gate=None, g_row=0, g_col=0, out=P, y=P, y8=None, ys=None, H=256)

    def norm(**kw):
        a = {**good, **kw}
        return lib.gdn_add_rms_norm(a["x"], a["sx"], a["res"], a["sr"], 0, a["w"], a["post"], 0, 1.0, a["gate"], 0, a["g_row"],
                                    a["g_col"], 0, 1.0, 1e-6, a["out"], a["y"], a["y8"], a["ys"], 1, 4, 4, a["H"],
                                    ctypes.c_void_p(-1))
    assert norm() == 0 and norm(y8=P, ys=P) == 0 and norm(y=None, y8=P, ys=P) == 0     # (checked only: nothing is launched)
    for kw in (dict(x=None), dict(w=None), dict(y=None), dict(y8=P), dict(sx=255), dict(sr=255), dict(x=byte), dict(res=byte),
               dict(gate=P, g_col=1, g_row=255), dict(gate=byte), dict(y8=P, ys=P, H=200), dict(y8=P, ys=P, x=odd),
               dict(y8=P, ys=P, sx=260), dict(y8=odd, ys=P), dict(y8=P, ys=P, gate=odd, g_col=1)):
        assert norm(**kw) == bad, kw


def test_quick_calls_leave_the_rest_to_the_wrappers(pkg):
    """What is not a tensor on the device as the kernel takes it is not taken, and said to be None."""
    quick = pkg._lib.quick()
    t, f = torch.zeros(2, 128, dtype=BF16), torch.zeros(128)
    for name, n in (("add_norm", 11), ("linear_lora", 7), ("linear_fp8_lora", 9)):
        call = getattr(quick, name)
        for arg in (t, f, None, 3, "x", (), torch.nn.Parameter(f), [t], [1 << 70], 1.5, True):
            assert call(*[arg] * n) is None, (name, arg)
        for wrong in (0, n - 1, n + 1):
            with pytest.raises(TypeError):
                call(*[t] * wrong)
    assert quick.add_norm(t, t, f, 1e-6, None, None, False, 1.0, 1.0, True, False) is None   # (not on the device)


def test_adapter_rows(pkg):
    """Each row its sequence's adapter, empty sequences none of them; rows behind the last one none."""
    cu = torch.tensor([0, 3, 3, 4, 9], dtype=I32)
    got = pkg.adapter_rows(torch.tensor([5, 7, -1, 2]), cu, 11)
    assert got.dtype == I32 and got.tolist() == [5, 5, 5, -1, 2, 2, 2, 2, 2, -1, -1]
    assert pkg.adapter_rows(torch.zeros(0, dtype=I32), cu[:1], 2).tolist() == [-1, -1]
    for bad in ((torch.zeros(3), cu), (torch.zeros(4, 1), cu), (torch.zeros(4), cu[None])):
        with pytest.raises(ValueError):
            pkg.adapter_rows(*bad, 9)
