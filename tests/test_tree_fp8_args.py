"""What the tree verify's and the 8-bit projections' entry points refuse, before any
launch: the wrappers with the device check and the launch stubbed (CPU tensors), the C
entry points with NULL or, where no GPU is visible, dummy aligned addresses."""
import ctypes

import pytest
import torch

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


class Launched(Exception):
    pass


@pytest.fixture
def ops(pkg, monkeypatch):
    def fake_call(*a, **k):
        raise Launched()

    monkeypatch.setattr(pkg.ops, "_device_of", lambda *ts: 0)
    monkeypatch.setattr(pkg.ops, "_call_on", fake_call)
    monkeypatch.setattr(pkg.ops, "_launch_on", fake_call)
    monkeypatch.setattr(pkg._lib, "stream_of", lambda index: 0)
    return pkg.ops


def _refused(fn, good, **bad):
    """fn with good arguments reaches the launch; with each bad one it does not."""
    with pytest.raises(Launched):
        fn(**good)
    for name, values in bad.items():
        for value in values:
            with pytest.raises((ValueError, TypeError)):
                fn(**{**good, name: value})


def test_conv_tree_step_refuses(ops):
    B, T, C = 3, 5, 64
    x, pool, w = torch.zeros(B, T, C, dtype=BF16), torch.zeros(6, C, 3, dtype=BF16), torch.zeros(C, 1, 4, dtype=BF16)
    ids, par = torch.arange(B), torch.zeros(B, T, dtype=torch.int32)
    acc = torch.zeros(B, dtype=torch.int64)
    _refused(ops.conv_tree_step, dict(x=x, conv_pool=pool, ids=ids, weight=w, parents=par, pending=(x, par, acc)),
             x=[x.float(), x[0], torch.zeros(B, 65, C, dtype=BF16), x[..., :60]],
             conv_pool=[pool.float(), pool[:, :60], pool[..., :2], pool.permute(0, 2, 1)],
             ids=[ids[:2], ids.float(), ids[None]], weight=[w.float(), w[:60], torch.zeros(C, 3, dtype=BF16)],
             parents=[par.float(), par[:2], par[:, :4], torch.zeros(T + 1, dtype=torch.int32)],
             pending=[(x[:2], par, acc), (x, par[:, :4], acc), (x, par, acc[:2]), (x.float(), par, acc),
                      (x, par, acc.float())])
    for good in (torch.zeros(T, dtype=torch.int64), par.long(), par.expand(B, T)):
        with pytest.raises(Launched):
            ops.conv_tree_step(x, pool, ids, w, good)


def test_recurrent_gdn_tree_refuses(ops):
    B, T, Hk, Hv, D = 2, 4, 2, 4, 64
    q, v = torch.zeros(B, T, Hk, D, dtype=BF16), torch.zeros(B, T, Hv, D, dtype=BF16)
    g, beta, pool = torch.zeros(B, T, Hv), torch.zeros(B, T, Hv, dtype=BF16), torch.zeros(5, Hv, D, D)
    ids, par, u = torch.arange(B), torch.zeros(B, T, dtype=torch.int32), torch.zeros(B, T, Hv, D)
    _refused(ops.recurrent_gdn_tree, dict(q=q, k=q, v=v, g=g, beta=beta, s_pool=pool, ids=ids, parents=par,
                                          pending=(q, g, u, par, ids)),
             q=[q.float(), q[:, :3], q[..., :32]], k=[q[:1], q[:, :, :1], q[0]],
             v=[v.float(), v[:, :, :3], v[..., :32]], g=[g.double(), g[..., :2], g[:1]],
             beta=[beta.float(), beta[..., :2]], s_pool=[pool.double(), pool[:, :2], pool.transpose(2, 3)],
             ids=[ids[:1], ids.float()], parents=[par[:1], par.bool()],
             pending=[(q[:, :, :1], g, u, par, ids), (q, g[:, :3], u, par, ids), (q, g, u.double(), par, ids),
                      (q, g, u, par[:, :2], ids), (q, g, u, par, ids[:1])])


def test_recurrent_tree_fused_refuses(ops):
    B, T, Hk, Hv, D = 2, 4, 1, 2, 128
    q, v = torch.zeros(B, T, Hk, D, dtype=BF16), torch.zeros(B, T, Hv, D, dtype=BF16)
    b, z, w = torch.zeros(B, T, Hv, dtype=BF16), torch.zeros(B, T, Hv * D, dtype=BF16), torch.ones(D)
    p, pool, ids = torch.zeros(Hv), torch.zeros(5, Hv, D, D), torch.arange(B)
    par, g, u = torch.zeros(B, T, dtype=torch.int32), torch.zeros(B, T, Hv), torch.zeros(B, T, Hv, D)
    good = dict(q=q, k=q, v=v, b=b, a=b, a_log=p, dt_bias=p.to(BF16), z=z, norm_weight=w, s_pool=pool, ids=ids,
                parents=par, pending=(q, g, u, par, ids), fp8=True)
    _refused(ops.recurrent_tree_fused, good,
             q=[q.float()], v=[v[:, :3]], b=[b.float(), b[:1]], a=[b.float(), b[..., :1]], a_log=[p[:1]],
             dt_bias=[p[:1]], z=[z.float(), z[..., :128], v], norm_weight=[w[:64]], s_pool=[pool.double()],
             ids=[ids.float()], parents=[par[:1]], pending=[(q, g, u, par, ids[:1])])
    half = dict(good, q=q[..., :64], k=q[..., :64], v=v[..., :64], z=z[..., :128], norm_weight=w[:64],
                s_pool=torch.zeros(5, Hv, 64, 64), pending=None)
    with pytest.raises(ValueError):      # heads of 64 share a scale
        ops.recurrent_tree_fused(**half)
    with pytest.raises(Launched):
        ops.recurrent_tree_fused(**dict(half, fp8=False))


def test_commit_tree_refuses(ops):
    B, T, Hk, Hv, D, C = 2, 4, 2, 4, 64, 512
    k, u = torch.zeros(B, T, Hk, D, dtype=BF16), torch.zeros(B, T, Hv, D)
    x, g, pool = torch.zeros(B, T, C, dtype=BF16), torch.zeros(B, T, Hv), torch.zeros(5, Hv, D, D)
    cpool, ids, par = torch.zeros(5, C, 3, dtype=BF16), torch.arange(B), torch.zeros(B, T, dtype=torch.int32)
    _refused(ops.commit_tree, dict(s_pool=pool, conv_pool=cpool, ids=ids, parents=par, accepted=ids, x=x, k=k, g=g,
                                   u=u),
             s_pool=[pool[:4], pool[:, :2]], conv_pool=[cpool[:, :8], cpool.float()], ids=[ids[:1]],
             parents=[par[:, :2]], accepted=[ids[:1], ids.float()], x=[x[:, :3], x[0]], k=[k[:1], k.float()],
             g=[g[:1]], u=[u[..., :32], u[0]])


def test_8_bit_calls_refuse(ops):
    M, N, K = 5, 200, 256
    x, w8, ws = torch.zeros(M, K, dtype=BF16), torch.zeros(N, K, dtype=FP8), torch.ones(2, 2)
    x8, xs = torch.zeros(M, K, dtype=FP8), torch.ones(M, 2)
    out = torch.zeros(M, N, dtype=BF16)
    _refused(ops.quantize_fp8, dict(x=x), x=[x.half(), x[:, :100], x[:, :0], x8])
    _refused(ops.quantize_weight_fp8, dict(weight=out.new_zeros(N, K)),
             weight=[x[0], x.half(), x[:, :130], w8])
    _refused(ops.linear_fp8, dict(x=x8, weight=w8, weight_scale=ws, x_scale=xs, out=out),
             x=[x, x8[:, :128], x.float()], weight=[w8.float(), w8[:, :128], w8[0]],
             weight_scale=[ws[:1], ws[:, :1], ws.to(BF16)], x_scale=[None, xs[:4], xs[:, :1], xs.double()],
             out=[out.float(), out[:4], out.t(), out.expand(M, N)[:, :100], out[:1].expand(M, N)])
    _refused(ops.linear_fp8_cols, dict(x=x, weight=w8, weight_scale=ws, widths=[96, 104]),
             widths=[[100, 100], [], [96, 96], [16] * 5 + [120], [-16, 216]])
    w9, wide = torch.zeros(192, K, dtype=FP8), torch.zeros(32, K, dtype=BF16)
    _refused(ops.linear_fp8_cols, dict(x=x, weight=w9, weight_scale=ws, widths=[192, 16, 16], wide=wide),
             x=[x8], weight=[w8], widths=[[192], [176, 48], [192, 24, 8], [192, 48]],
             wide=[wide.float(), wide[:24], wide[:, :128], wide[:0], wide[0]])
    n = torch.zeros(M, 4, 64, dtype=BF16)
    _refused(ops.rms_norm_gated_fp8, dict(hidden_states=n, gate=n, weight=torch.ones(64), eps=1e-6),
             hidden_states=[n.float(), n[:, :3], n[0, 0]], gate=[n.float(), n[:, :2]], weight=[torch.ones(32)])
    odd = n[:, :3]
    with pytest.raises(ValueError):      # 192 columns: no whole groups
        ops.rms_norm_gated_fp8(odd, odd, torch.ones(64), 1e-6)


def test_no_cpu_path(pkg):
    with pytest.raises(ValueError):
        pkg.quantize_fp8(torch.zeros(1, 128, dtype=BF16))
    with pytest.raises(ValueError):
        pkg.linear_fp8(torch.zeros(1, 128, dtype=BF16), torch.zeros(1, 128, dtype=FP8), torch.ones(1, 1))


def test_steps_without_accepted_nodes_are_refused(pkg):
    Hk = Hv = 2
    D, C = 64, 384
    core = pkg.GatedDeltaNetCore(Hk, Hv, D, torch.zeros(C, 4, dtype=BF16), torch.zeros(Hv), torch.zeros(Hv),
                                 torch.ones(D), switches=pkg.Switches())
    z = torch.zeros(1, 3, C, dtype=BF16)
    step = pkg.TreeStep(z, z, z, z, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        core.commit_tree(step, None, None, None)
    with pytest.raises(ValueError):
        core.verify_tree(z, z, z, z, None, None, None, None, pending=step)
    with pytest.raises(ValueError):
        step.accept(torch.zeros(2, dtype=torch.int64))
    off = pkg.GatedDeltaNetCore(Hk, Hv, D, torch.zeros(C, 4, dtype=BF16), torch.zeros(Hv), torch.zeros(Hv),
                                torch.ones(D), switches=pkg.Switches(conv_kernel=False))
    with pytest.raises(NotImplementedError):
        off.verify_tree(z, z, z, z, None, None, None, None)
    with pytest.raises(ValueError):
        pkg.GatedDeltaNetLayer(*[torch.zeros(1, 1)] * 5, Hk, Hv, D, torch.zeros(C, 4), torch.zeros(Hv),
                               torch.zeros(Hv), torch.ones(D), weights="int8")


def test_c_entry_points_reject_before_launch(pkg):
    lib, _lib = pkg._lib.load(), pkg._lib
    inv, uns, ok = _lib.GDN_ERR_INVALID_ARG, _lib.GDN_ERR_UNSUPPORTED, _lib.GDN_OK
    if torch.cuda.device_count() > 0:
        pytest.skip("dummy device addresses are passed only where no GPU is visible")
    P, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
    # quantizer
    q = lambda x=P, sx=256, y=P, sy=256, s=P, M=4, K=256, rows=1: lib.gdn_quantize_fp8(  # noqa: E731
        x, 0, sx, y, sy, s, 2, 1, M, K, rows, None)
    assert q(M=0) == ok and q(K=0) == ok
    for bad in (dict(x=None), dict(x=odd), dict(sx=252), dict(sx=128), dict(y=None), dict(sy=250), dict(s=None),
                dict(K=200), dict(rows=64), dict(M=-1)):
        assert q(**bad) == inv, bad
    # product
    C1, ld1, end1 = (ctypes.c_void_p * 1)(1 << 20), (ctypes.c_int64 * 1)(96), (ctypes.c_int * 1)(96)
    f = lambda A=P, lda=256, sa=P, ar=1, B=P, ldb=256, sb=P, br=2, M=4, N=96, K=256, n=1, C=C1, ld=ld1, e=end1, q=0, ws=None, wb=0, b2=None, l2=256, n2=0: (  # noqa: E731,E501
        lib.gdn_gemm_fp8(A, q, lda, sa, ar, 4, B, ldb, sb, br, b2, l2, n2, M, N, K, n, C, ld, e, ws, wb, None))
    assert f(M=0) == ok and f(N=0) == ok
    for bad in (dict(A=None), dict(A=odd), dict(lda=248), dict(lda=128), dict(sa=None), dict(B=None), dict(B=odd),
                dict(ldb=250), dict(sb=None), dict(br=1), dict(K=0), dict(K=192), dict(n=0), dict(n=5), dict(C=None),
                dict(ld=(ctypes.c_int64 * 1)(90)), dict(e=(ctypes.c_int * 1)(90)), dict(M=1 << 24), dict(ar=-1),
                dict(ar=1 << 28)):
        assert f(**bad) == inv, bad
    # from bf16 rows: the workspace that the size says, of rows that no kernel quantizes itself
    size = lib.gdn_gemm_fp8_workspace_size
    assert size(5000, 96, 256, 0) == 0 and size(0, 96, 256, 1) == 0 and size(-1, 96, 256, 1) == -1
    assert size(4, 96, 200, 1) == -1
    need = size(5000, 96, 256, 1)
    assert need == 5000 * (256 + 8)
    for bad in (dict(ws=None, wb=need), dict(ws=odd, wb=need), dict(ws=P, wb=need - 1), dict(lda=252)):
        assert f(**{**dict(q=1, M=5000, ws=P, wb=need), **bad}) == inv, bad
    # bf16 columns behind them: on bf16 rows, in 16s, with a part that ends at N
    C2, ld2 = (ctypes.c_void_p * 2)(1 << 20, 1 << 20), (ctypes.c_int64 * 2)(96, 96)
    wide = dict(q=1, b2=P, n2=32, n=2, C=C2, ld=ld2, e=(ctypes.c_int * 2)(96, 128), ws=P, wb=4 * 264)
    for bad in (dict(q=0), dict(b2=None), dict(b2=odd), dict(n2=24), dict(l2=252), dict(l2=128), dict(n2=-16),
                dict(e=(ctypes.c_int * 2)(80, 128)), dict(e=(ctypes.c_int * 2)(96, 112)), dict(n=1, e=end1)):
        assert f(**{**wide, **bad}) == inv, bad
    # norm
    n = lambda x=P, sx=256, w=P, y=P, s=P, N=4, H=2, D=128: lib.gdn_rmsnorm_gated_fp8(  # noqa: E731
        x, sx, P, 256, w, y, s, 1, 4, N, H, D, 1e-6, None)
    assert n(N=0) == ok and n(D=96) == uns
    for bad in (dict(x=None), dict(sx=252), dict(w=odd), dict(y=None), dict(s=None), dict(H=0), dict(H=3, D=64),
                dict(N=-1)):
        assert n(**bad) == inv, bad
    # trees
    C = 512
    cv = lambda x=P, xb=8 * C, xt=C, pool=P, slot=3 * C, ch=3, y=P, B=2, T=8, Cc=C, lx=P, lt=C, acc=P, lT=8: (  # noqa: E731,E501
        lib.gdn_conv_tree(x, xb, xt, pool, slot, ch, 4, P, P, P, 8, lx, 8 * C, lt, P, 8, acc, lT, y, B, T, Cc, None))
    assert cv(B=0) == ok and cv(T=0) == ok and cv(T=65) == uns and cv(lT=65) == uns and cv(Cc=516) == uns
    for bad in (dict(x=None), dict(x=odd), dict(xt=C - 8), dict(xb=4), dict(pool=None), dict(slot=3 * C - 3),
                dict(ch=2), dict(y=None), dict(lx=None), dict(lt=C - 8), dict(lT=0), dict(B=-1)):
        assert cv(**bad) == inv, bad
    slot = 4 * 64 * 64
    r = lambda q=P, qt=128, vt=256, g=P, s=P, st=slot, o=P, u=P, B=2, T=8, Hk=2, Hv=4, D=64, lu=P, lT=8: (  # noqa: E731,E501
        lib.gdn_rule_tree(q, 8 * 128, qt, P, 8 * 128, 128, P, 8 * 256, vt, g, P, s, st, 4, P, P, 8, P, 8 * 128, 128,
                          P, lu, P, 8, P, lT, o, u, B, T, Hk, Hv, D, 1.0, None))
    assert r(B=0) == ok and r(T=65) == uns and r(D=96) == uns and r(lT=65) == uns
    for bad in (dict(q=None), dict(qt=120), dict(qt=1 << 24), dict(vt=248), dict(g=None), dict(s=odd), dict(st=slot - 4), dict(o=None),
                dict(u=odd), dict(Hk=3), dict(Hk=0), dict(lu=None), dict(lT=0), dict(T=-1)):
        assert r(**bad) == inv, bad
    f = lambda q=P, b=P, a=P, al=P, z=P, zt=256, w=P, y=P, y8=None, ys=None, u=P, g=P, B=2, T=8, D=64: (  # noqa: E731
        lib.gdn_rule_tree_layer(q, 8 * 128, 128, P, 8 * 128, 128, P, 8 * 256, 256, b, a, al, P, 0, P, slot, 4, P, P, 8,
                                None, 0, 0, None, None, None, 0, None, 0, z, 8 * 256, zt, w, 1e-6, y, y8, ys, u, g, B,
                                T, 2, 4, D, 1.0, None))
    assert f(B=0) == ok and f(T=65) == uns and f(y=None, y8=P, ys=P) == uns
    for bad in (dict(q=None), dict(b=None), dict(a=None), dict(al=None), dict(z=None), dict(z=odd), dict(zt=248),
                dict(w=odd), dict(y=None), dict(y8=P, ys=P), dict(y=None, y8=P), dict(y=odd), dict(u=odd),
                dict(g=None)):
        assert f(**bad) == inv, bad
    c = lambda s=P, st=slot, cp=P, cs=3 * C, x=P, k=P, u=P, acc=P, B=2, T=8, Hk=2, Hv=4, D=64, Cc=C: (  # noqa: E731
        lib.gdn_commit_tree(s, st, cp, cs, 3, 4, P, P, 8, acc, x, 8 * C, C, k, 8 * 128, 128, P, u, B, T, Hk, Hv, D,
                            Cc, None))
    assert c(B=0) == ok and c(T=65) == uns and c(D=32) == uns and c(Cc=500) == uns
    for bad in (dict(s=None), dict(st=slot - 4), dict(cp=None), dict(cs=3 * C - 3), dict(x=None), dict(k=odd),
                dict(u=None), dict(acc=None), dict(Hk=3)):
        assert c(**bad) == inv, bad


def test_calls_by_words(pkg):
    """An entry point's arguments as words: the same answers as the call itself; wrong heads,
    counts and integers that do not fit are refused."""
    lib, _lib = pkg._lib.load(), pkg._lib
    inv, uns, ok = _lib.GDN_ERR_INVALID_ARG, _lib.GDN_ERR_UNSUPPORTED, _lib.GDN_OK
    assert lib.gdn_call_words(None) == inv
    for name, (pack, head) in _lib.WORDS.items():
        n = head >> 32
        types = _lib.SIGNATURES[name]
        assert n == len(types)
        zeros = [0.0 if t is ctypes.c_float else 0 for t in types]
        assert lib.gdn_call_words(pack(head, *zeros)) == getattr(lib, name)(
            *(None if t is ctypes.c_void_p else z for t, z in zip(types, zeros))), name
        for wrong in (head + (1 << 32), head - (1 << 32), head & 0xffffffff, head + 64, n << 32):
            assert lib.gdn_call_words(pack(wrong, *zeros)) == inv
    pack, head = _lib.WORDS["gdn_conv_tree"]
    conv = lambda B=0, T=8, C=64: lib.gdn_call_words(pack(head, *[0] * 19, B, T, C, 0))  # noqa: E731
    assert conv() == ok and conv(T=65) == uns and conv(C=1 << 23) == uns and conv(C=0) == inv and conv(B=1) == inv
    assert conv(B=1 << 32) == inv and conv(T=(1 << 32) + 8) == inv       # 0 and 8 if they were cut
    for n in range(1, 5):
        pack, head = _lib.GEMM_FP8_WORDS[n]
        args = lambda M, N, parts: [0] * 13 + [M, N, 128, parts, 0, 0, 0] + [0, 64, 64] * n  # noqa: E731
        assert lib.gdn_call_words(pack(head, *args(0, 64, n))) == ok
        assert lib.gdn_call_words(pack(head, *args(1 << 32, 64, n))) == inv
        assert lib.gdn_call_words(pack(head, *args(0, 64, n % 4 + 1))) == inv
        assert lib.gdn_call_words(pack(head, *args(0, 64, 0))) == inv
        assert lib.gdn_call_words(pack(head, *args(2, 64, n))) == inv     # no operands


def test_decode_step_to_e4m3_refuses(pkg, monkeypatch):
    monkeypatch.setattr(pkg.ops, "_check_cuda", lambda *ts: torch.device("cpu"))
    monkeypatch.setattr(pkg._lib, "call", lambda *a: (_ for _ in ()).throw(Launched()))
    monkeypatch.setattr(pkg.ops, "_stream", lambda dev: 0)
    B, Hk, Hv, D = 2, 1, 2, 128
    C = 2 * Hk * D + Hv * D
    n = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    good = dict(qk=None, mixed=n(B, C), conv_pool=n(4, C, 3), conv_weight=n(C, 4), b=n(B, Hv), a=n(B, Hv), a_log=n(Hv),
                dt_bias=n(Hv), s_pool=torch.zeros(4, Hv, D, D), ids=torch.arange(B), Hk=Hk, Hv=Hv, D=D, z=n(B, Hv * D),
                norm_weight=n(D), grouped=True, fp8=True)
    _refused(pkg.ops.recurrent_decode_fused, good, z=[None], out=[n(B, Hv * D)])
    with pytest.raises(ValueError):
        pkg.ops.recurrent_decode_fused(**dict(good, qk=n(B, 2 * Hk * D), fuse_norm=False))
    lib, _lib = pkg._lib.load(), pkg._lib
    P, odd = 1 << 20, (1 << 20) + 2
    f = lambda q=None, k=None, x=P, y=P, s=P, ss=8, B=4, Hk=2, Hv=4, D=128, z=P, w=P, sx=1024: (  # noqa: E731
        lib.gdn_decode_fp8(q, 1024, k, 1024, x, sx, P, 3 * 1024, 3, P, P, P, P, P, 0, P, Hv * D * D, P, y, s, ss, B, Hk,
                           Hv, D, 1.0, 1, z, 512, w, 1e-6, None))
    assert f(B=0) == _lib.GDN_OK and f(D=64) == _lib.GDN_ERR_UNSUPPORTED
    for bad in (dict(q=P), dict(k=P), dict(Hk=1), dict(Hv=5), dict(x=None), dict(x=odd), dict(y=None), dict(y=odd),
                dict(s=None), dict(ss=3), dict(z=None), dict(z=odd), dict(w=None), dict(sx=1020), dict(B=-1)):
        assert f(**bad) == _lib.GDN_ERR_INVALID_ARG, bad


def test_quick_calls_leave_the_rest_to_the_wrappers(pkg):
    """What is not a tensor on the device as the kernel takes it is not taken, and said to be None."""
    quick = pkg._lib.quick()
    t, f = torch.zeros(1, 2, 8, dtype=BF16), torch.zeros(1, 2, 2, 64)
    for name, n in (("conv_tree", 6), ("rule_tree", 9), ("rule_tree_layer", 15), ("commit_tree", 9), ("linear_fp8", 4),
                    ("norm_fp8", 4)):
        call = getattr(quick, name)
        for arg in (t, f, None, 3, "x", (), torch.nn.Parameter(f), [t]):
            assert call(*[arg] * n) is None, (name, arg)
        for wrong in (0, n - 1, n + 1):
            with pytest.raises(TypeError):
                call(*[t] * wrong)


@pytest.mark.parametrize("D,fp8", [(128, False), (128, True), (64, False), (64, True)])
def test_a_refused_verify_launches_nothing(pkg, monkeypatch, D, fp8):
    """The conv of a verify step moves the conv pool on: it is not launched where a later call of the
    same step is refused, by its wrapper or by its entry point."""
    launched = []
    monkeypatch.setattr(pkg.ops, "_device_of", lambda *ts: 0)
    monkeypatch.setattr(pkg.ops, "_call_on", lambda idx, name, *a: launched.append(name))
    none = type("Nothing", (), {"__getattr__": lambda self, name: lambda *a: None})()
    monkeypatch.setattr(pkg._lib, "quick", lambda: none)
    B, T, Hk, Hv, slots = 2, 5, 1, 2, 6
    C = (2 * Hk + Hv) * D
    n = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    f = lambda *s: torch.zeros(*s)  # noqa: E731
    core = pkg.GatedDeltaNetCore(Hk, Hv, D, n(C, 4), f(Hv), f(Hv), n(D))
    core._g_beta = lambda b, a, mask: (f(*b.shape), b)
    step = lambda **kw: pkg.TreeStep(**{**dict(x=n(B, T, C), k=n(B, T, Hk, D), g=f(B, T, Hv), u=f(B, T, Hv, D),  # noqa: E731
                                               parents=torch.zeros(T, dtype=torch.int32)), **kw})
    acc = torch.zeros(B, dtype=torch.int64)
    good = dict(mixed=n(B, T, C), z=n(B, T, Hv * D), b=n(B, T, Hv), a=n(B, T, Hv), ids=torch.arange(B),
                conv_cache=n(slots, C, 3), s_cache=f(slots, Hv, D, D), parents=torch.zeros(B, T, dtype=torch.int32),
                pending=step().accept(acc), fp8=fp8)
    fused = not fp8 or D == 128
    core.verify_tree(**good)
    assert launched == ["gdn_conv_tree", "gdn_rule_tree_layer"] if fused else \
        launched == ["gdn_conv_tree", "gdn_rule_tree", "gdn_rmsnorm_gated_fp8"]
    bad = dict(z=[n(B, T, Hv * D + 8), n(B, T + 1, Hv * D)], b=[n(B, T, Hv + 1)[..., 1:].float()],
               s_cache=[f(slots, Hv, D, D).double(), f(slots, Hv + 1, D, D), f(slots, Hv, D, D).transpose(2, 3),
                        f(slots * Hv * D * D + 1)[1:].view(slots, Hv, D, D),                # not 16-byte aligned
                        f(slots, Hv * D * D + 2)[:, :-2].unflatten(1, (Hv, D, D)),          # slots neither
                        f(0, Hv, D, D)],
               pending=[step(k=n(B, T, Hk + 1, D)).accept(acc), step(u=f(B, T, Hv, D).double()).accept(acc),
                        step(g=f(B, T + 1, Hv)).accept(acc)],
               mixed=[n(B, T, C + 64), n(B, T, C).float()], parents=[torch.zeros(B, T + 1, dtype=torch.int32)],
               conv_cache=[n(slots + 1, C, 3)])
    for name, values in bad.items():
        for value in values:
            launched.clear()
            with pytest.raises((ValueError, TypeError, RuntimeError)):
                core.verify_tree(**{**good, name: value})
            assert launched == [], name
    small = pkg.GatedDeltaNetCore(Hk, Hv, 32, n(4 * 32, 4), f(Hv), f(Hv), n(32))     # no such head dim
    launched.clear()
    with pytest.raises(pkg._lib.GDNKernelError):
        small.verify_tree(n(B, T, 4 * 32), n(B, T, Hv * 32), n(B, T, Hv), n(B, T, Hv), torch.arange(B),
                          n(slots, 4 * 32, 3), f(slots, Hv, 32, 32), good["parents"])
    assert launched == []


def test_checks_without_a_launch(pkg):
    """CHECK_ONLY in the stream's place: the entry point's own answers, for arguments that it takes as
    well (dummy addresses: nothing is launched)."""
    lib, _lib = pkg._lib.load(), pkg._lib
    inv, uns, ok, only = _lib.GDN_ERR_INVALID_ARG, _lib.GDN_ERR_UNSUPPORTED, _lib.GDN_OK, ctypes.c_void_p(-1)
    P, odd, C, slot = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8), 512, 4 * 64 * 64
    cv = lambda x=P, B=2, T=8, Cc=C: lib.gdn_conv_tree(  # noqa: E731
        x, 8 * C, C, P, 3 * C, 3, 4, P, P, P, 8, P, 8 * C, C, P, 8, P, 8, P, B, T, Cc, only)
    assert cv() == ok and cv(B=0) == ok and cv(x=odd) == inv and cv(T=65) == uns and cv(B=65536) == uns
    r = lambda q=P, s=P, st=slot, T=8, Hv=4: lib.gdn_rule_tree(  # noqa: E731
        q, 8 * 128, 128, P, 8 * 128, 128, P, 8 * 256, 256, P, P, s, st, 4, P, P, 8, P, 8 * 128, 128, P, P, P, 8, P, 8, P, P,
        2, T, 2, Hv, 64, 1.0, only)
    assert r() == ok and r(q=None) == inv and r(s=odd) == inv and r(st=slot + 2) == inv and r(T=65) == uns
    f = lambda z=P, w=P, D=64: lib.gdn_rule_tree_layer(  # noqa: E731
        P, 8 * 128, 128, P, 8 * 128, 128, P, 8 * 256, 256, P, P, P, P, 0, P, slot, 4, P, P, 8, None, 0, 0, None, None, None,
        0, None, 0, z, 8 * 256, 256, w, 1e-6, P, None, None, P, P, 2, 8, 2, 4, D, 1.0, only)
    assert f() == ok and f(z=None) == inv and f(w=odd) == inv and f(D=32) == uns
    c = lambda s=P, T=8: lib.gdn_commit_tree(s, slot, P, 3 * C, 3, 4, P, P, 8, P, P, 8 * C, C, P, 8 * 128, 128, P, P, 2, T,  # noqa: E731
                                             2, 4, 64, C, only)
    assert c() == ok and c(s=None) == inv and c(T=65) == uns
    n = lambda w=P, H=2: lib.gdn_rmsnorm_gated_fp8(P, 256, P, 256, w, P, P, 1, 4, 4, H, 128, 1e-6, only)  # noqa: E731
    assert n() == ok and n(w=odd) == inv and n(H=0) == inv
    quick, t = pkg._lib.quick(), torch.zeros(1, 2, 8, dtype=BF16)
    for arg in (t, None, 3, (), [t]):
        assert quick.verify_tree(*[arg] * 20) is None and quick.verify_tree_norm(*[arg] * 17) is None
    for call, n in ((quick.verify_tree, 20), (quick.verify_tree_norm, 17)):
        for wrong in (0, n - 1, n + 1):
            with pytest.raises(TypeError):
                call(*[t] * wrong)


def _between(t):
    """The same values at an address that is no multiple of 16."""
    flat = torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)
    assert flat.is_contiguous() and flat.data_ptr() % 16
    return flat


def test_conv_weight_reaches_the_kernel_aligned(pkg, monkeypatch):
    monkeypatch.setattr(pkg.ops, "_device_of", lambda *ts: 0)
    B, T, C = 2, 3, 64
    z = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    pkg.ops._conv_tree_ready(z(B, T, C), z(4, C, 3), torch.arange(B), _between(z(C, 1, 4)),
                             torch.zeros(T, dtype=torch.int32), None).check()


def test_norm_weight_reaches_the_kernel_aligned(pkg, monkeypatch):
    monkeypatch.setattr(pkg.ops, "_device_of", lambda *ts: 0)
    n = torch.zeros(5, 2, 128, dtype=BF16)
    pkg.ops._norm_fp8_ready(n, n, _between(torch.ones(128, dtype=BF16)), 1e-6).check()


def test_quick_calls_of_another_version_or_place_are_refused(pkg, tmp_path):
    """The module is the one beside the library that is loaded, and of the bindings' version: its calls
    are compiled against a header's argument lists."""
    import shutil
    import subprocess
    import sys
    import sysconfig
    from pathlib import Path

    lib = pkg._lib.LIB_PATH
    shutil.copy(lib, tmp_path / lib.name)
    code = ("import os, sys; sys.path.insert(0, %r); os.environ['GDN_MI355X_LIB'] = %r\n"
            "import __graft_entry__ as ge\npkg = ge.load_package()\n"
            "try:\n    print('TAKEN', pkg._lib.quick().__file__)\nexcept pkg._lib.GDNLibraryError as e:\n    print('LOUD', e)\n"
            % (str(Path(__file__).resolve().parents[1]), str(tmp_path / lib.name)))
    run = lambda: subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120).stdout  # noqa: E731
    assert "LOUD" in run()                                           # none beside it
    module = tmp_path / pkg._lib.QUICK_NAME
    for constant in ("", f'if (m) PyModule_AddIntConstant(m, "ABI_VERSION", {pkg._lib.ABI_VERSION - 1});'):
        src = tmp_path / "old.c"
        src.write_text('#include <Python.h>\nstatic struct PyModuleDef d = {PyModuleDef_HEAD_INIT, "gdn_quick_calls", 0, -1};\n'
                       "PyMODINIT_FUNC PyInit_gdn_quick_calls(void) {\n  PyObject* m = PyModule_Create(&d);\n"
                       f"  {constant}\n  return m;\n}}\n")
        subprocess.run(["gcc", "-shared", "-fPIC", f"-I{sysconfig.get_paths()['include']}", str(src), "-o", str(module)],
                       check=True)
        out = run()
        assert "LOUD ABI mismatch" in out, out
    shutil.copy(lib.parent / module.name, module)
    out = run()
    assert f"TAKEN {module}" in out, out


def test_e4m3_rows_without_whole_groups_launch_nothing(pkg, monkeypatch):
    """Three value heads of 64: 192 columns.  The core refuses them before its conv and rule have moved
    the pools on, not in the norm behind them."""
    launched = []
    for where, name in ((pkg._lib, "call"), (pkg.ops, "_call_on"), (pkg.ops, "_launch_on")):
        monkeypatch.setattr(where, name, lambda *a: launched.append(a))
    monkeypatch.setattr(pkg.ops, "_device_of", lambda *ts: 0)
    monkeypatch.setattr(pkg.ops, "_check_cuda", lambda *ts: torch.device("cpu"))
    Hk, Hv, D, N = 1, 3, 64, 6
    C, V = (2 * Hk + Hv) * D, Hv * D
    n = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    core = pkg.GatedDeltaNetCore(Hk, Hv, D, n(C, 4), n(Hv), n(Hv), n(D))
    pools, cu = (n(2, C, 3), torch.zeros(2, Hv, D, D)), torch.tensor([0, 4, 6], dtype=torch.int32)
    rows, ids = (n(N, C), n(N, V), n(N, Hv), n(N, Hv)), torch.arange(2)
    for call in (lambda: core.forward(*rows, cu, 4, ids, *pools, lens_q=[4, 2], fp8=True),
                 lambda: core.prefill_varlen(*rows, [4, 2], ids, *pools, fp8=True),
                 lambda: core.verify_tree(*(t.view(2, 3, -1) for t in rows), ids, *pools, torch.zeros(3, dtype=torch.int32),
                                          fp8=True)):
        with pytest.raises(ValueError, match="192 columns"):
            call()
    with pytest.raises(ValueError, match="head dim of 128"):       # (two launches: the conv's is the first)
        core.decode(*rows, torch.arange(6), *pools, fp8=True)
    assert launched == []
    monkeypatch.setattr(pkg.ops, "_stream", lambda dev: 0)
    # decode rows are bf16 with heads of 64: nothing to refuse
    out = core.forward(*rows, torch.arange(7), 1, torch.arange(6) % 2, *pools, lens_q=[1] * 6, fp8=True)
    assert out.dtype == BF16 and out.shape == (N, V) and launched


def test_a_checkpoints_out_projection_is_laid_out_once(pkg):
    """An e4m3 w_out that comes as a view (columns of a wider tensor, a transposed one) is contiguous in the
    layer, which would copy it in every call else."""
    Hk = Hv = 1
    D, hidden, C = 128, 256, 384
    z = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    e = lambda *s: z(*s).to(FP8)  # noqa: E731
    rest = (z(Hv, hidden), z(Hv, hidden))
    for w8, scale in ((e(hidden, 136)[:, :D], torch.ones(2, 1)), (e(D, hidden).t(), torch.ones(1, 2).t())):
        layer = pkg.GatedDeltaNetLayer((e(C, hidden), torch.ones(3, 2)), (e(D, hidden), torch.ones(1, 2)), *rest, (w8, scale),
                                       Hk, Hv, D, z(C, 4), z(Hv), z(Hv), z(D), weights="fp8")
        assert layer.w_out.is_contiguous() and layer.w_out_scale.is_contiguous() and layer.w_in.is_contiguous()
