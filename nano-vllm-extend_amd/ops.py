"""GDN operators with the reference's Python signatures, backed by the gfx950
HIP kernels of libgdn_mi355x.so.

Each function mirrors a module-level function of
nanovllm/models/qwen3_5.py (cited per function): same argument meaning,
same output allocation (torch.empty on the input's device), same in-place
mutation of the state pools, and the reference's shape asserts.  There is no
CPU or eager fallback: a CPU tensor or a missing library raises.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import os

import torch

from . import _lib


def _check_cuda(*ts: torch.Tensor | None) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("GDN ops run on the GPU only (got a CPU tensor; there is no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    return dev


def _bf16(t: torch.Tensor, name: str) -> None:
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")


def _out(t: torch.Tensor, numel: int, dev: torch.device) -> torch.Tensor:
    """A caller's output tensor, checked."""
    _bf16(t, "out")
    if t.device != dev or t.numel() != numel or not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError("out must be a contiguous, 16-byte aligned tensor of the result's size on its device")
    return t


def _stream(dev: torch.device) -> int:
    return _lib.stream_handle(dev)


def _device_of(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """The index of the device that all of them are on (as _check_cuda; a few lookups
    cheaper)."""
    idx = first.get_device()
    for t in others:
        if t is not None and t.get_device() != idx:
            _check_cuda(first, *others)
    if idx < 0 or not first.is_cuda:
        _check_cuda(first, *others)
    return idx


def _call_on(idx: int, name: str, *args) -> None:
    """An entry point of _lib.WORDS on device idx's current stream, which is appended to
    args (NULL is 0): a launch goes to its stream's device, so that one is made current
    where it is not."""
    pack, head = _lib.WORDS[name]
    _launch_on(idx, name, pack(head, *args, _lib.stream_of(idx)))


def _launch_on(idx: int, name: str, words: bytes) -> None:
    if idx == _current_device():
        _lib.call_words(name, words)
    else:
        with torch.cuda.device(idx):
            _lib.call_words(name, words)


class _Ready:
    """A call whose arguments are checked and whose outputs are there: launch() makes it.  keep: the
    tensors that the arguments point into."""
    __slots__ = ("idx", "name", "args", "out", "keep")

    def __init__(self, idx, name, args, out, keep):
        self.idx, self.name, self.args, self.out, self.keep = idx, name, args, out, keep

    def check(self):
        """What the entry point itself would refuse, without a launch."""
        pack, head = _lib.WORDS[self.name]
        _lib.call_words(self.name, pack(head, *self.args, _lib.CHECK_ONLY))

    def launch(self):
        _call_on(self.idx, self.name, *self.args)
        return self.out


# (0.2 us cheaper than the public call, which checks that CUDA is initialised: a tensor on
# the device says so)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


# ------------------------------------------------------- fp16 operand range --
# The chunk kernels run their state-path products on fp16 matrix cores: the
# raw k and v rows (after the conv), Q', the block inverses, A, the state S
# and Vn = U - W S become fp16 operands, so each must stay below the fp16
# maximum.  Q' and A are bounded by the L2 norm (|Q'| <= scale, |A| <= scale);
# the inputs a caller controls are checked here on request.
FP16_MAX = 65504.0


def range_check_enabled() -> bool:
    """NANOVLLM_GDN_CHECK_RANGE=1 turns on the input range check of the
    prefill wrappers (a device reduction and a host sync per call)."""
    return os.environ.get("NANOVLLM_GDN_CHECK_RANGE", "0") == "1"


def fp16_range_violation(rows: torch.Tensor | None = None, conv_weight: torch.Tensor | None = None,
                         states: torch.Tensor | None = None) -> str | None:
    """Why a prefill call's inputs could leave the fp16 operand range, or None.

    rows: the rows that feed the kernels -- raw q|k|v rows when conv_weight
    [C, 4] is given (the conv output of channel c is at most
    sum_i |w[c, i]| * max |x| in magnitude, SiLU not increasing it), else the
    q, k, v rows themselves; states: the initial states that will be read.
    Non-finite values count as violations.  Works on any device."""
    if rows is not None and rows.numel():
        m = rows.detach().float().abs().amax()
        if not torch.isfinite(m):
            return "non-finite input rows"
        bound = float(m)
        if conv_weight is not None:
            gain = float(conv_weight.detach().float().reshape(conv_weight.shape[0], -1).abs().sum(1).amax())
            bound *= gain
        if bound >= FP16_MAX:
            return (f"input rows reach {bound:.4g} after the conv" if conv_weight is not None
                    else f"input rows reach {bound:.4g}") + f" (fp16 operands must stay below {FP16_MAX:g})"
    if states is not None and states.numel():
        m = float(states.detach().abs().amax())
        if not m < FP16_MAX:  # also catches NaN / inf
            return f"initial states reach {m:.4g} (fp16 operands must stay below {FP16_MAX:g})"
    return None


def _check_range(**kw) -> None:
    why = fp16_range_violation(**kw)
    if why is not None:
        raise ValueError(f"GDN chunk prefill: {why}")


# ----------------------------------------------------------------- g / beta --
def fused_g_beta(b: torch.Tensor, a: torch.Tensor, a_log: torch.Tensor, dt_bias: torch.Tensor,
                 mask: torch.Tensor | None):
    """g = -exp(A_log) * softplus(a + dt_bias) (fp32, 0 on padding rows),
    beta = sigmoid(b) (bf16).  b/a [.., Vh] bf16 contiguous; a_log/dt_bias
    [Vh] (bf16 or fp32); mask [n, T] bool or None.
    Reference: fused_g_beta, nanovllm/models/qwen3_5.py:345-360."""
    dev = _check_cuda(b, a, a_log, dt_bias, mask)
    _bf16(a, "a")
    _bf16(b, "b")
    assert a.is_contiguous() and b.is_contiguous() and a.shape == b.shape
    vh = a.shape[-1]
    if a_log.dtype != dt_bias.dtype or a_log.dtype not in (torch.bfloat16, torch.float32):
        a_log = a_log.float()
        dt_bias = dt_bias.float()
    a_log = a_log.contiguous()
    dt_bias = dt_bias.contiguous()
    assert a_log.numel() == vh and dt_bias.numel() == vh
    g = torch.empty_like(a, dtype=torch.float32)
    beta = torch.empty_like(a)
    flat_mask = None
    if mask is not None:
        flat_mask = mask.reshape(-1).contiguous()
        if flat_mask.dtype != torch.bool:
            flat_mask = flat_mask.to(torch.bool)
        assert flat_mask.numel() * vh == a.numel()
    _lib.call("gdn_g_beta", _lib.ptr(b), _lib.ptr(a), _lib.ptr(a_log), _lib.ptr(dt_bias),
              int(a_log.dtype == torch.float32), _lib.ptr(flat_mask), _lib.ptr(g), _lib.ptr(beta),
              a.numel(), vh, _stream(dev))
    return g, beta


# --------------------------------------------------------------------- conv --
def _conv_varlen(x, state, weight, lens, cuseq, key_dim, state_ids):
    dev = _check_cuda(x, state, weight, lens, cuseq, state_ids)
    _bf16(x, "x")
    _bf16(state, "state")
    N, C = x.shape
    K = weight.shape[-1]
    w = weight.reshape(C, K)
    _bf16(w, "weight")
    w = w.contiguous()
    assert x.stride(1) == 1 and state.stride(2) == 1 and tuple(state.shape[1:]) == (C, K - 1)
    n = lens.shape[0]
    lens32 = lens.to(torch.int32).contiguous()
    cu32 = cuseq.to(torch.int32).contiguous()
    assert cu32.shape[0] >= n
    ids = None
    if state_ids is not None:
        ids = state_ids.to(torch.int64).contiguous()
        assert ids.shape[0] == n
    y = torch.empty(N * C, dtype=x.dtype, device=x.device)
    _lib.call("gdn_conv_varlen", _lib.ptr(x), x.stride(0), _lib.ptr(state), state.stride(0),
              state.stride(1), _lib.ptr(ids), _lib.ptr(w), _lib.ptr(y), key_dim, _lib.ptr(lens32),
              _lib.ptr(cu32), n, N, C, K, _stream(dev))
    return y


def causal_conv_silu_varlen_parts(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor,
                                  lens: torch.Tensor, cuseq: torch.Tensor, key_dim: int,
                                  state_ids: torch.Tensor | None = None):
    """Varlen conv + SiLU returning the (q, k, v) parts [N, key_dim],
    [N, key_dim], [N, C - 2*key_dim], each contiguous (one allocation), so
    grouped-value layouts (C != 3*key_dim) are covered.  state: conv states
    [n, C, K-1], or with state_ids the slot pool [slots, C, K-1] updated in
    place at those rows."""
    N, C = x.shape
    y = _conv_varlen(x, state, weight, lens, cuseq, key_dim, state_ids)
    q = y[: N * key_dim].view(N, key_dim)
    k = y[N * key_dim: 2 * N * key_dim].view(N, key_dim)
    v = y[2 * N * key_dim:].view(N, C - 2 * key_dim)
    return q, k, v


def causal_conv_silu_varlen(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor,
                            lens: torch.Tensor, cuseq: torch.Tensor) -> torch.Tensor:
    """x [N, C] bf16 contiguous varlen; state [n, C, K-1] (updated in place);
    lens int32 [n]; cuseq int32 [n] (per-row starts).  Returns [3, N, C//3]:
    the q/k/v thirds, each contiguous.
    Reference: causal_conv_silu_varlen, nanovllm/models/qwen3_5.py:459-473."""
    N, C = x.shape
    d3 = C // 3
    assert d3 * 3 == C and d3 % 64 == 0
    return _conv_varlen(x, state, weight, lens, cuseq, d3, None).view(3, N, d3)


def conv_decode_step(x: torch.Tensor, state_pool: torch.Tensor, ids: torch.Tensor,
                     weight: torch.Tensor) -> torch.Tensor:
    """x [n, C] (decode rows); state_pool [slots, C, K-1] rolled in place at
    rows `ids`; weight [C, K] (or [C, 1, K]).  Returns y [n, C].
    Reference: conv_decode_step, nanovllm/models/qwen3_5.py:546-558."""
    dev = _check_cuda(x, state_pool, ids, weight)
    _bf16(x, "x")
    _bf16(state_pool, "state_pool")
    n, C = x.shape
    K = weight.shape[-1]
    w = weight.reshape(C, K).contiguous()
    assert x.stride(1) == 1 and state_pool.stride(2) == 1
    ids64 = ids.to(torch.int64).contiguous()
    assert ids64.shape == (n,), "one slot id per row"
    y = torch.empty(n, C, dtype=x.dtype, device=x.device)
    _lib.call("gdn_conv_decode", _lib.ptr(x), x.stride(0), _lib.ptr(state_pool), state_pool.stride(0),
              state_pool.stride(1), _lib.ptr(ids64), _lib.ptr(w), _lib.ptr(y), y.stride(0), n, C, K,
              _stream(dev))
    return y


def causal_conv_silu(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor,
                     endp: torch.Tensor) -> torch.Tensor:
    """x [n, C, T] (arbitrary strides), state [n, C, K-1] (updated in place
    at each row's endp), weight [C, K].  Returns y [n, C, T] contiguous;
    endp int32 [n] (-1 = skip writeback).
    Reference: causal_conv_silu, nanovllm/models/qwen3_5.py:300-317."""
    dev = _check_cuda(x, state, weight, endp)
    _bf16(x, "x")
    _bf16(state, "state")
    n, C, T = x.shape
    K = weight.shape[-1]
    w = weight.reshape(C, K).contiguous()
    assert state.stride(2) == 1
    e32 = endp.to(torch.int32).contiguous()
    y = torch.empty(n, C, T, dtype=x.dtype, device=x.device)
    _lib.call("gdn_conv_padded", _lib.ptr(x), x.stride(0), x.stride(1), x.stride(2), _lib.ptr(state),
              state.stride(0), state.stride(1), _lib.ptr(w), _lib.ptr(y), _lib.ptr(e32), n, C, T, K,
              _stream(dev))
    return y


# -------------------------------------------------------------- chunk rule --
def _host_offsets(cu_cpu, n: int):
    """int64 host copy of the sequence offsets [n + 1], or None."""
    if cu_cpu is None:
        return None
    if (isinstance(cu_cpu, torch.Tensor) and cu_cpu.dtype == torch.int64
            and cu_cpu.device.type == "cpu" and cu_cpu.is_contiguous()):
        assert cu_cpu.shape == (n + 1,)
        return cu_cpu
    t = torch.as_tensor(cu_cpu)
    if t.device.type != "cpu":
        raise ValueError("cu_seqlens_cpu must be in host memory")
    t = t.to(torch.int64).contiguous()
    assert t.shape == (n + 1,)
    return t


def _host_ptr(t):
    """Host pointer of a CPU tensor (the caller keeps the tensor alive)."""
    return None if t is None else t.data_ptr()


def _state_view_ok(s: torch.Tensor, H: int, D: int) -> bool:
    return (s.dtype == torch.float32 and s.dim() == 4 and tuple(s.shape[1:]) == (H, D, D)
            and s.stride(1) == D * D and s.stride(2) == D and s.stride(3) == 1)


def _rows16(t: torch.Tensor, D: int) -> torch.Tensor:
    if t.stride(2) != 1 or t.stride(1) != D or t.stride(0) % 8 or t.data_ptr() % 16:
        return t.contiguous() if not t.is_contiguous() else t.clone()
    return t


def chunk_gated_delta_rule_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                                  beta: torch.Tensor, cu_seqlens: torch.Tensor,
                                  initial_state: torch.Tensor | None = None, *,
                                  output_final_state: bool = True,
                                  use_qk_l2norm_in_kernel: bool = True, scale: float | None = None,
                                  state_ids: torch.Tensor | None = None,
                                  final_state: torch.Tensor | None = None,
                                  cu_seqlens_cpu: torch.Tensor | None = None, max_segments: int = 0):
    """Varlen chunked gated delta rule (chunk 64) on packed rows.

    q, k [N, Hk, D]; v [N, Hv, D] (bf16, head dim contiguous, any token
    stride); g [N, Hv] fp32; beta [N, Hv] bf16; cu_seqlens [n+1] (device).
    Value head h uses key head h // (Hv // Hk).
    initial_state: [n, Hv, D, D] fp32, or with state_ids a slot pool
    [slots, Hv, D, D] (any slot stride) read at rows state_ids.
    Final states go to `final_state` (same indexing; may be the pool itself
    for an in-place update) or to a new [n, Hv, D, D] tensor.
    cu_seqlens_cpu: the offsets on the host (as the fla call passes them);
    with them a call of few long sequences is cut into segments that run in
    parallel (max_segments: 0 automatic, 1 never, k up to k per sequence).
    Returns (o [N, Hv, D] bf16, final or None)."""
    dev = _check_cuda(q, k, v, g, beta, cu_seqlens, initial_state, state_ids, final_state)
    for t, nm in ((q, "q"), (k, "k"), (v, "v"), (beta, "beta")):
        _bf16(t, nm)
    N, Hk, D = k.shape
    Hv = v.shape[1]
    assert q.shape == k.shape and v.shape[0] == N and v.shape[2] == D and Hv % Hk == 0
    # the kernels read 16-byte row pieces: head-contiguous rows, 16-byte
    # aligned, token stride a multiple of 8 elements (else copy once)
    q, k, v = (_rows16(t, D) for t in (q, k, v))
    g = g.float().contiguous() if g.dtype != torch.float32 else g.contiguous()
    beta = beta.contiguous()
    assert g.shape == (N, Hv) and beta.shape == (N, Hv)
    cu = cu_seqlens.to(torch.int64).contiguous()
    n = cu.shape[0] - 1
    ids = None
    if state_ids is not None:
        ids = state_ids.to(torch.int64).contiguous()
        assert ids.shape[0] == n
    h0 = initial_state
    if h0 is not None and not _state_view_ok(h0, Hv, D):
        assert state_ids is None, "pool-indexed initial state must be an fp32 [slots, H, D, D] view"
        h0 = h0.float().contiguous()
    hT = None
    if output_final_state:
        if final_state is not None:
            assert _state_view_ok(final_state, Hv, D)
            hT = final_state
        else:
            assert state_ids is None or h0 is not None
            hT = torch.empty(n, Hv, D, D, dtype=torch.float32, device=q.device)
    if ids is not None and hT is not None and final_state is None:
        raise ValueError("state_ids requires final_state (the pool) for the output state")
    sstride = 0
    for st in (h0, hT):
        if st is not None:
            sstride = st.stride(0)
    if h0 is not None and hT is not None:
        assert h0.stride(0) == hT.stride(0), "initial and final state must share the slot stride"
    if range_check_enabled():
        read = None
        if h0 is not None:
            read = h0.index_select(0, ids) if ids is not None else h0
        _check_range(rows=torch.cat([q.reshape(N, -1), k.reshape(N, -1), v.reshape(N, -1)], 1), states=read)
    if scale is None:
        scale = D ** -0.5
    o = torch.empty(N, Hv, D, dtype=v.dtype, device=v.device)
    # per-(chunk, head) records of the chunk-local phase; the caching
    # allocator's blocks are 512-byte aligned, the kernels need 256
    ws_bytes = _lib.load().gdn_chunk_prefill_workspace_size(N, n, Hv, D)
    if ws_bytes < 0:
        raise ValueError(f"unsupported chunk shape N={N} n_seqs={n} Hv={Hv} D={D}")
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=q.device)
    cu_host = _host_offsets(cu_seqlens_cpu, n)
    _lib.call("gdn_chunk_prefill", _lib.ptr(q), q.stride(0), _lib.ptr(k), k.stride(0), _lib.ptr(v),
              v.stride(0), _lib.ptr(g), _lib.ptr(beta), _lib.ptr(h0), _lib.ptr(hT), _lib.ptr(ids),
              sstride, _lib.ptr(cu), _host_ptr(cu_host), int(max_segments), n, N, Hk, Hv, D, float(scale),
              int(bool(use_qk_l2norm_in_kernel)), _lib.ptr(o), _lib.ptr(ws), ws_bytes, _stream(dev))
    return o, hT


def conv_chunk_prefill_varlen(mixed: torch.Tensor, conv_state: torch.Tensor, conv_weight: torch.Tensor,
                              b: torch.Tensor, a: torch.Tensor, a_log: torch.Tensor, dt_bias: torch.Tensor,
                              cu_seqlens: torch.Tensor, state: torch.Tensor, state_ids: torch.Tensor | None,
                              num_k_heads: int, num_v_heads: int, head_dim: int,
                              scale: float | None = None, fresh: torch.Tensor | None = None,
                              cu_seqlens_cpu: torch.Tensor | None = None, max_segments: int = 0,
                              late: list[bool] | None = None, side_stream=None, keep: list | None = None):
    """Gates, varlen causal conv1d + SiLU and the chunked gated delta rule in
    one call (two kernels), the prefill sequence of _gdn_prefill_varlen
    (nanovllm/models/qwen3_5.py:934-961): the same results as fused_g_beta ->
    causal_conv_silu_varlen_parts -> chunk_gated_delta_rule_varlen (q/k L2
    norm on), bit for bit.

    mixed [N, C] bf16 raw q|k|v rows (C = 2*Hk*D + Hv*D, channel stride 1);
    conv_state [slots, C, 3] bf16 and state [slots, Hv, D, D] fp32 slot pools,
    both read and updated in place at rows state_ids (the sequence index if
    None); conv_weight [C, 4] (or [C, 1, 4]); b, a [N, Hv] bf16; a_log,
    dt_bias [Hv]; cu_seqlens [n+1] (device).  fresh: optional bool/uint8 [n]:
    those sequences start from zero recurrent and conv states and their pool
    rows are not read (the slot zeroing of a fresh prefill,
    model_runner.py:305-322, folded into the call).  cu_seqlens_cpu /
    max_segments: as chunk_gated_delta_rule_varlen.

    late / side_stream (split state pass): after the prep kernel on the
    current stream, the state pass of the sequences with late[r] runs on the
    current stream and that of the others on side_stream, concurrently.  The
    caller orders later work on side_stream's results itself (e.g. the current
    stream waits for side_stream) and keeps the tensors appended to `keep`
    alive until then.  Returns o [N, Hv, D] bf16, and with `late` also an
    event recorded on side_stream after its state pass."""
    dev = _check_cuda(mixed, conv_state, conv_weight, b, a, a_log, dt_bias, cu_seqlens, state, state_ids)
    _bf16(mixed, "mixed")
    _bf16(conv_state, "conv_state")
    _bf16(a, "a")
    _bf16(b, "b")
    Hk, Hv, D = num_k_heads, num_v_heads, head_dim
    N, C = mixed.shape
    assert C == 2 * Hk * D + Hv * D and Hv % Hk == 0
    w = conv_weight.reshape(C, -1)
    _bf16(w, "conv_weight")
    assert w.shape[1] == 4, "the fused path is built for conv width 4"
    w = w.contiguous()
    if mixed.stride(1) != 1 or mixed.stride(0) % 8 or mixed.data_ptr() % 16:
        mixed = mixed.contiguous()
    assert conv_state.stride(2) == 1 and tuple(conv_state.shape[1:]) == (C, 3)
    a = a.contiguous()
    b = b.contiguous()
    assert a.shape == (N, Hv) and b.shape == (N, Hv)
    if a_log.dtype != dt_bias.dtype or a_log.dtype not in (torch.bfloat16, torch.float32):
        a_log = a_log.float()
        dt_bias = dt_bias.float()
    a_log = a_log.contiguous()
    dt_bias = dt_bias.contiguous()
    assert _state_view_ok(state, Hv, D), "state must be an fp32 [slots, Hv, D, D] view"
    cu = cu_seqlens.to(torch.int64).contiguous()
    n = cu.shape[0] - 1
    ids = None
    if state_ids is not None:
        ids = state_ids.to(torch.int64).contiguous()
        assert ids.shape[0] == n
    fr = None
    if fresh is not None:
        fr = fresh.to(device=mixed.device, dtype=torch.uint8).contiguous()
        assert fr.shape == (n,)
    if range_check_enabled():
        rows_read = torch.arange(n, device=mixed.device) if ids is None else ids
        if fr is not None:
            rows_read = rows_read[fr == 0]
        _check_range(rows=mixed, conv_weight=w, states=state.index_select(0, rows_read))
    if scale is None:
        scale = D ** -0.5
    o = torch.empty(N, Hv, D, dtype=torch.bfloat16, device=mixed.device)
    ws_bytes = _lib.load().gdn_conv_chunk_prefill_workspace_size(N, n, Hv, D)
    if ws_bytes < 0:
        raise ValueError(f"unsupported chunk shape N={N} n_seqs={n} Hv={Hv} D={D}")
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=mixed.device)
    cu_host = _host_offsets(cu_seqlens_cpu, n)

    def launch(phase, select, stream):
        _lib.call("gdn_conv_chunk_prefill", _lib.ptr(mixed), mixed.stride(0), _lib.ptr(conv_state),
                  conv_state.stride(0), conv_state.stride(1), _lib.ptr(w), _lib.ptr(b), _lib.ptr(a),
                  _lib.ptr(a_log), _lib.ptr(dt_bias), int(a_log.dtype == torch.float32), _lib.ptr(state),
                  _lib.ptr(state), _lib.ptr(ids), _lib.ptr(fr), state.stride(0), _lib.ptr(cu),
                  _host_ptr(cu_host), int(max_segments), phase, _host_ptr(select), n, N, Hk, Hv, D, float(scale),
                  1, _lib.ptr(o), _lib.ptr(ws), ws_bytes, stream)

    if late is None:
        launch(3, None, _stream(dev))
        return o
    assert side_stream is not None and cu_host is not None and len(late) == n
    sel_late = torch.tensor([bool(x) for x in late], dtype=torch.uint8)
    sel_early = 1 - sel_late
    cur = torch.cuda.current_stream(dev)
    launch(1, None, cur.cuda_stream)                       # prep
    ev = torch.cuda.Event()
    ev.record(cur)
    side_stream.wait_event(ev)
    launch(2, sel_late, cur.cuda_stream)                   # the long sequences
    launch(2, sel_early, side_stream.cuda_stream)          # the others, concurrently
    side_done = torch.cuda.Event()
    side_done.record(side_stream)
    if keep is not None:
        keep.extend([mixed, w, a, b, a_log, dt_bias, cu, ids, fr, o, ws, conv_state, state])
    return o, side_done


def conv_chunk_prefill_varlen_noalloc(mixed: torch.Tensor, conv_state: torch.Tensor, conv_weight: torch.Tensor,
                                      b: torch.Tensor, a: torch.Tensor, a_log: torch.Tensor, dt_bias: torch.Tensor,
                                      cu_seqlens: torch.Tensor, state: torch.Tensor, state_ids: torch.Tensor | None,
                                      num_k_heads: int, num_v_heads: int, head_dim: int, out: torch.Tensor,
                                      scale: float | None = None, fresh: torch.Tensor | None = None,
                                      cu_seqlens_cpu: torch.Tensor | None = None, max_segments: int = 0) -> None:
    """conv_chunk_prefill_varlen through the allocation-free entry point: the
    records live in the library's fixed per-GPU scratch array (no workspace
    allocation), and the output goes to the caller's `out` [N, Hv, D] bf16.
    Nothing here allocates device memory or copies: the inputs must already
    have the layouts the kernels read (checked).  Calls that overlap on one
    GPU race on the shared array.  A call whose records do not fit the array
    runs in pieces (sequence groups, and long sequences as token ranges), the
    same bits as max_segments=1; that needs cu_seqlens_cpu, without which such
    a call raises GDNKernelError."""
    dev = _check_cuda(mixed, conv_state, conv_weight, b, a, a_log, dt_bias, cu_seqlens, state, state_ids, out, fresh)
    Hk, Hv, D = num_k_heads, num_v_heads, head_dim
    N, C = mixed.shape
    for t, nm in ((mixed, "mixed"), (conv_state, "conv_state"), (a, "a"), (b, "b"), (out, "out"),
                  (conv_weight, "conv_weight")):
        _bf16(t, nm)
    assert C == 2 * Hk * D + Hv * D and Hv % Hk == 0
    assert mixed.stride(1) == 1 and mixed.stride(0) % 8 == 0
    assert conv_weight.is_contiguous() and conv_weight.numel() == 4 * C
    assert conv_state.stride(2) == 1 and tuple(conv_state.shape[1:]) == (C, 3)
    assert a.is_contiguous() and b.is_contiguous() and a.shape == (N, Hv) and b.shape == (N, Hv)
    assert a_log.dtype == dt_bias.dtype and a_log.dtype in (torch.bfloat16, torch.float32)
    assert a_log.is_contiguous() and dt_bias.is_contiguous()
    assert _state_view_ok(state, Hv, D), "state must be an fp32 [slots, Hv, D, D] view"
    assert cu_seqlens.dtype == torch.int64 and cu_seqlens.is_contiguous()
    n = cu_seqlens.shape[0] - 1
    if state_ids is not None:
        assert state_ids.dtype == torch.int64 and state_ids.is_contiguous() and state_ids.shape == (n,)
    if fresh is not None:
        assert fresh.dtype == torch.uint8 and fresh.is_contiguous() and fresh.shape == (n,)
    assert out.shape == (N, Hv, D) and out.is_contiguous()
    cu_host = _host_offsets(cu_seqlens_cpu, n)
    if scale is None:
        scale = D ** -0.5
    _lib.call("gdn_conv_chunk_prefill_noalloc", _lib.ptr(mixed), mixed.stride(0), _lib.ptr(conv_state),
              conv_state.stride(0), conv_state.stride(1), _lib.ptr(conv_weight), _lib.ptr(b), _lib.ptr(a),
              _lib.ptr(a_log), _lib.ptr(dt_bias), int(a_log.dtype == torch.float32), _lib.ptr(state),
              _lib.ptr(state), _lib.ptr(state_ids), _lib.ptr(fresh), state.stride(0), _lib.ptr(cu_seqlens),
              _host_ptr(cu_host), int(max_segments), n, N, Hk, Hv, D, float(scale), 1, _lib.ptr(out), _stream(dev))


def chunk_gated_delta_rule(query, key, value, g=None, beta=None, scale=None, initial_state=None,
                           output_final_state=False, use_qk_l2norm_in_kernel=False,
                           cu_seqlens=None, cu_seqlens_cpu=None, chunk_size=64, **kwargs):
    """Drop-in for the chunk GDN entry point the reference calls.

    Covers both reference call forms:
      * chunk_gated_delta_rule(q, k, v, g, beta, chunk_size=64, initial_state=...)
        (nanovllm/models/qwen3_5.py:140-149): batched [B, T, H, D], always
        returns the final state, L2-norm in kernel;
      * the fla varlen call (qwen3_5.py:956-960): q[None] [1, N, H, D],
        cu_seqlens int64 [n+1], initial_state [n, H, D, D].
    Returns (o [B, T, Hv, D] bf16, final [B or n, Hv, D, D] fp32 or None)."""
    if chunk_size != 64:
        raise ValueError("only chunk_size=64 is built (the reference's value)")
    if "cu_seqlens" in kwargs:
        cu_seqlens = kwargs.pop("cu_seqlens")
    B, T, Hq, D = query.shape
    Hv = value.shape[2]
    if cu_seqlens is not None:
        assert B == 1, "varlen mode takes a single packed batch row"
        cu = cu_seqlens
        qf, kf, vf = query[0], key[0], value[0]
        gf, bf = g[0], beta[0]
    else:
        cu = torch.arange(B + 1, device=query.device, dtype=torch.int64) * T
        qf = query.reshape(B * T, Hq, D)
        kf = key.reshape(B * T, Hq, D)
        vf = value.reshape(B * T, Hv, D)
        gf = g.reshape(B * T, Hv)
        bf = beta.reshape(B * T, Hv)
    o, final = chunk_gated_delta_rule_varlen(qf, kf, vf, gf, bf, cu, initial_state,
                                             output_final_state=output_final_state,
                                             use_qk_l2norm_in_kernel=use_qk_l2norm_in_kernel,
                                             scale=scale, cu_seqlens_cpu=cu_seqlens_cpu)
    return o.view(B, T, Hv, D), final


def chunk_gated_delta_rule_ref_api(query, key, value, g, beta, chunk_size=64, initial_state=None):
    """The reference module's own signature (nanovllm/models/qwen3_5.py:140-149):
    final state always returned, q/k L2-normalised in kernel."""
    return chunk_gated_delta_rule(query, key, value, g=g, beta=beta, initial_state=initial_state,
                                  output_final_state=True, use_qk_l2norm_in_kernel=True,
                                  chunk_size=chunk_size)


# ---------------------------------------------------------- recurrent rule --
def _recurrent(q, k, v, g, beta, s_in, s_out, ids, inter, scale, l2norm, src_states=None, src_accepted=None):
    dev = _check_cuda(q, k, v, g, beta, s_in, s_out, ids, inter, src_states, src_accepted)
    for t, nm in ((q, "q"), (k, "k"), (v, "v"), (beta, "beta")):
        _bf16(t, nm)
    Bsz, T, Hk, D = k.shape
    Hv = v.shape[2]
    assert q.shape == k.shape and v.shape[:2] == (Bsz, T) and v.shape[3] == D and Hv % Hk == 0
    assert q.stride(2) == D and k.stride(2) == D and v.stride(2) == D
    assert q.stride(3) == 1 and k.stride(3) == 1 and v.stride(3) == 1
    g = g.float() if g.dtype != torch.float32 else g
    assert g.is_contiguous() and beta.is_contiguous()
    assert g.numel() == Bsz * T * Hv and beta.numel() == Bsz * T * Hv
    assert _state_view_ok(s_in, Hv, D)
    if s_out is not None:
        assert _state_view_ok(s_out, Hv, D)
    ids64 = None
    if ids is not None:
        ids64 = ids.to(torch.int64).contiguous()
        assert ids64.shape[0] == Bsz
    if inter is not None:
        assert inter.is_contiguous() and inter.dtype == torch.float32
        assert inter.shape == (Bsz, T, Hv, D, D)
    src_acc, src_T = None, 1
    if src_accepted is not None:
        assert src_states is not None and src_states.is_contiguous() and src_states.dtype == torch.float32
        assert src_states.dim() == 5 and src_states.shape[0] == Bsz and src_states.shape[2:] == (Hv, D, D)
        src_T = src_states.shape[1]
        src_acc = src_accepted if src_accepted.dtype == torch.int64 else src_accepted.to(torch.int64)
        assert src_acc.shape == (Bsz,) and src_acc.is_contiguous()
    out = torch.empty(Bsz, T, Hv, D, dtype=v.dtype, device=v.device)
    if scale is None:
        scale = D ** -0.5
    _lib.call("gdn_recurrent", _lib.ptr(q), q.stride(0), q.stride(1), _lib.ptr(k), k.stride(0),
              k.stride(1), _lib.ptr(v), v.stride(0), v.stride(1), _lib.ptr(g), _lib.ptr(beta),
              _lib.ptr(s_in), s_in.stride(0), _lib.ptr(s_out), s_out.stride(0) if s_out is not None else 0,
              _lib.ptr(ids64), _lib.ptr(inter), _lib.ptr(out), Bsz, T, Hk, Hv, D, float(scale),
              int(bool(l2norm)), _lib.ptr(src_states if src_acc is not None else None), _lib.ptr(src_acc),
              src_T, _stream(dev))
    return out


def recurrent_gdn_inplace(q, k, v, g, beta, s_pool, ids):
    """q/k/v [bs, 1, H, D] bf16, g/beta [bs, 1, H]; updates s_pool rows `ids`
    in place, returns out [bs, 1, H, DV] bf16.  q/k/v may be strided views
    of the conv output; s_pool a per-layer view of the state pool.
    Reference: recurrent_gdn_inplace, nanovllm/models/qwen3_5.py:597-613."""
    bs, _, H, DK = k.shape
    DV = v.shape[-1]
    assert q.stride(2) == DK and k.stride(2) == DK and v.stride(2) == DV
    assert g.is_contiguous() and beta.is_contiguous()
    assert s_pool.stride(1) == DK * DV and s_pool.stride(2) == DV and s_pool.stride(3) == 1
    return _recurrent(q, k, v, g, beta, s_pool, s_pool, ids, None, None, True)


# (sequence, head) tiles from which every recurrent kernel runs whole heads per
# workgroup.  With fewer the head's columns may be split over workgroups: in the
# multi-token kernel that changes the summation order of S^T k, so its
# whole-head and split runs differ in the last bits; one-token steps add in one
# order at every split.  (Also the line below which the one-launch step takes
# only the rows that the q/k conv's launch, which ran there before it, takes; the
# library's own line between its two one-launch kernels is a matter of speed.)
WHOLE_HEAD_TILES = 2048


# With two value heads per key head the one-launch step holds two state tiles per
# workgroup; from about this many tiles on, the q/k conv's own launch costs no
# more than the smaller workgroups of the two-launch form gain (32 value heads,
# graph-replayed core: 32 rows 37.2 us in two launches, 29.6 in one; 64 rows 58.4
# and 53.7; 150 rows 117.0 and 116.3; 200 rows 149.0 and 149.1; 256 rows 187.2
# and 189.0).
GROUPED_STEP_TILES = 5120


def one_launch_decode(B: int, num_k_heads: int, num_v_heads: int) -> bool:
    """Whether the whole decode step, q/k conv included, runs in one kernel:
    with one value head per key head always, with two at small batches."""
    return num_v_heads == num_k_heads or (num_v_heads == 2 * num_k_heads and B * num_v_heads < GROUPED_STEP_TILES)


def recurrent_decode_fused(qk, mixed, conv_pool, conv_weight, b, a, a_log, dt_bias, s_pool, ids, Hk, Hv, D,
                           scale=None, z=None, norm_weight=None, eps=1e-6, fuse_norm=None, grouped=False,
                           out=None, fp8=False):
    """The decode step after the q/k conv, in one kernel: the gates from a, b,
    the v channels' conv1d + SiLU (their conv state rolled in place at `ids`)
    and the in-place recurrent update.  qk [B, 2*Hk*D] is conv_decode_step's
    output for the q and k channels; mixed [B, C] the raw rows; conv_pool
    [slots, C, 3] and s_pool [slots, Hv, D, D] per-layer pool views; b, a
    [B, Hv] bf16.  Returns out [B, 1, Hv, D] bf16, the same bits as
    fused_g_beta -> conv_decode_step -> recurrent_gdn_inplace
    (nanovllm/models/qwen3_5.py:1008-1030).  With z ([B, Hv*D] bf16, head
    dim contiguous) and norm_weight ([D]) `out` is the layer's gated RMSNorm
    of it (qwen3_5.py:1083-1085), the same bits as rms_norm_gated on the core
    output, in the same kernel (fuse_norm=False: as a second launch).

    qk=None (Hk == Hv; with grouped also Hv == 2 * Hk): the q and k channels'
    decode conv runs in the kernel as well, their conv states rolled there
    (the whole step in one launch); the same bits as conv_decode_step on
    those channels followed by the call above with its output.  out: a
    contiguous bf16 tensor of B * Hv * D elements that takes the result.

    fp8 (with z, D == 128): the norm in e4m3 for an 8-bit out projection, the bits of
    rms_norm_gated_fp8 on the core output.  Returns (e4m3 [B, 1, Hv, D], scales [B, Hv])."""
    dev = _check_cuda(qk, mixed, conv_pool, conv_weight, b, a, a_log, dt_bias, s_pool, ids, z, norm_weight)
    for t, nm in ((qk, "qk"), (mixed, "mixed"), (conv_pool, "conv_pool"), (b, "b"), (a, "a")):
        if t is not None:
            _bf16(t, nm)
    B, C = mixed.shape
    kd = Hk * D
    assert C == 2 * kd + Hv * D
    if qk is None:
        assert Hk == Hv or (grouped and Hv == 2 * Hk), \
            "the q/k conv runs in the decode kernel only with one key head per value head (grouped: per two)"
        fuse_norm = True
    else:
        assert qk.shape == (B, 2 * kd) and qk.stride(1) == 1
    assert mixed.stride(1) == 1 and conv_pool.stride(2) == 1
    w = conv_weight.reshape(C, -1)
    assert w.shape[1] == 4
    w = w.contiguous()
    b, a = b.contiguous(), a.contiguous()
    assert b.shape == (B, Hv) and a.shape == (B, Hv)
    assert a_log.dtype == dt_bias.dtype and a_log.dtype in (torch.bfloat16, torch.float32)
    a_log, dt_bias = a_log.contiguous(), dt_bias.contiguous()
    assert a_log.numel() == Hv and dt_bias.numel() == Hv
    assert _state_view_ok(s_pool, Hv, D)
    ids64 = ids.to(torch.int64).contiguous()
    assert ids64.shape == (B,), "one slot id per row"
    if fp8 and (z is None or D != FP8_GROUP or out is not None or (fuse_norm is not None and not fuse_norm)):
        raise ValueError(f"fp8 outputs need z, a head dim of {FP8_GROUP} and the norm in the kernel, and take no out")
    if z is not None and fuse_norm is not None and not fuse_norm:
        core = recurrent_decode_fused(qk, mixed, conv_pool, conv_weight, b, a, a_log, dt_bias, s_pool, ids, Hk, Hv,
                                      D, scale)
        return rms_norm_gated(core, z.reshape(B, 1, Hv, D), norm_weight, eps, out)
    nw, sz = None, 0
    if z is not None:
        _bf16(z, "z")
        z = z.reshape(B, Hv * D)
        # (rows that overlap, as of one gate row expanded over the batch, are
        # copied too: the kernel takes whole rows)
        if z.stride(1) != 1 or (B > 1 and (z.stride(0) % 4 or z.stride(0) < Hv * D)):
            z = z.contiguous()
        sz = z.stride(0) if B > 1 else Hv * D
        assert norm_weight is not None and norm_weight.numel() == D
        nw = norm_weight.to(torch.bfloat16).contiguous()
    if scale is None:
        scale = D ** -0.5
    if fp8:
        y = torch.empty(B, 1, Hv, D, dtype=FP8, device=mixed.device)
        y_scale = _fp8_scales(B, Hv, mixed.device)
        if qk is not None:
            q_k = (_lib.ptr(qk), qk.stride(0), _lib.ptr(qk[:, kd:]), qk.stride(0))
        else:
            q_k = (None, 0, None, 0)
            if mixed.stride(0) % 8 or mixed.data_ptr() % 16:
                mixed = mixed.contiguous() if mixed.data_ptr() % 16 == 0 else mixed.clone()
        _lib.call("gdn_decode_fp8", *q_k, _lib.ptr(mixed), mixed.stride(0), _lib.ptr(conv_pool), conv_pool.stride(0),
                  conv_pool.stride(1), _lib.ptr(w), _lib.ptr(a), _lib.ptr(b), _lib.ptr(a_log), _lib.ptr(dt_bias),
                  int(a_log.dtype == torch.float32), _lib.ptr(s_pool), s_pool.stride(0), _lib.ptr(ids64), _lib.ptr(y),
                  _lib.ptr(y_scale), B, B, Hk, Hv, D, float(scale), 1, _lib.ptr(z), sz, _lib.ptr(nw), float(eps),
                  _stream(dev))
        return y, y_scale
    if out is None:
        out = torch.empty(B, 1, Hv, D, dtype=mixed.dtype, device=mixed.device)
    else:
        out = _out(out, B * Hv * D, dev).view(B, 1, Hv, D)
    entry, q_k = "gdn_recurrent_decode_fused", (None, 0, None, 0)
    if qk is not None:
        q_k = (_lib.ptr(qk), qk.stride(0), _lib.ptr(qk[:, kd:]), qk.stride(0))
    elif grouped and (Hk != Hv or B * Hv < WHOLE_HEAD_TILES):
        # (takes the rows that the q/k conv's own launch takes, and no others)
        entry, q_k = "gdn_decode_step", ()
    _lib.call(entry, *q_k, _lib.ptr(mixed), mixed.stride(0), _lib.ptr(conv_pool), conv_pool.stride(0),
              conv_pool.stride(1), _lib.ptr(w), _lib.ptr(a), _lib.ptr(b), _lib.ptr(a_log), _lib.ptr(dt_bias),
              int(a_log.dtype == torch.float32), _lib.ptr(s_pool), s_pool.stride(0), _lib.ptr(ids64),
              _lib.ptr(out), B, Hk, Hv, D, float(scale), 1, _lib.ptr(z), sz, _lib.ptr(nw), float(eps), _stream(dev))
    return out


def recurrent_gated_delta_rule(query, key, value, g=None, beta=None, initial_state=None, scale=None,
                               output_final_state=True, use_qk_l2norm_in_kernel=True, **kwargs):
    """Gathered-state recurrent rule (T >= 1 tokens per row).
    query/key [B, T, Hk, D], value [B, T, Hv, D], g/beta [B, T, Hv];
    initial_state [B, Hv, D, D] fp32 or None (zeros).  Returns
    (out [B, T, Hv, D], final [B, Hv, D, D] or None).
    Reference: recurrent_gated_delta_rule / _torch_recurrent_gated_delta_rule,
    nanovllm/models/qwen3_5.py:230-238, :616-651."""
    Bsz, T, Hk, D = key.shape
    Hv = value.shape[2]
    if initial_state is None:
        s_in = torch.zeros(Bsz, Hv, D, D, dtype=torch.float32, device=value.device)
    else:
        s_in = initial_state if _state_view_ok(initial_state, Hv, D) else initial_state.float().contiguous()
    s_out = torch.empty(Bsz, Hv, D, D, dtype=torch.float32, device=value.device) if output_final_state else None
    out = _recurrent(query, key, value, g.contiguous(), beta.contiguous(), s_in, s_out, None, None, scale,
                     use_qk_l2norm_in_kernel)
    return out, s_out


def recurrent_gdn_multitoken(q, k, v, g, beta, s_pool, ids, intermediate_states=None, src_states=None,
                             src_accepted=None):
    """Speculative-verify decode: T draft tokens per sequence against the
    slot pool.  q/k [B, T, Hk, D], v [B, T, Hv, D], g/beta [B, T, Hv].
    With intermediate_states ([B, T, Hv, D, D] fp32) the per-token states
    are written there and the pool is left untouched (commit_states picks
    the accepted prefix); without it the pool is advanced by all T tokens.
    src_states / src_accepted: row b starts from src_states[b,
    src_accepted[b] - 1] where src_accepted[b] >= 1 instead of its pool row
    (the previous verify's accepted state, not yet committed; see
    SpecVerify).
    Returns out [B, T, Hv, D].  (No reference counterpart: spec decode is
    disabled for qwen3_5, nanovllm/config.py:84.)"""
    s_out = None if intermediate_states is not None else s_pool
    return _recurrent(q, k, v, g, beta, s_pool, s_out, ids, intermediate_states, None, True, src_states,
                      src_accepted)


class SpecVerify:
    """Speculative-verify steps of one GDN layer with the rollback folded
    into the next step instead of a commit copy.

    verify() runs the T-token kernel and keeps every per-token state in an
    [B, T, Hv, D, D] buffer; accept(accepted) records how many of them each
    row keeps (device int64 tensor, values 1..T: the first token of a draft
    block is the target model's own and always kept).  The next verify()
    starts row b from state [b, accepted[b] - 1] directly (the kernel reads it
    where the pool row would be read, and each state is read before the step
    overwrites it in place), so nothing runs between steps.  commit() writes
    the accepted states into the pool, for any other user of the slots (a
    plain decode, a prefill, or a sequence that leaves the batch).  The rows
    keep their order across steps (ids the same); a different batch must
    commit() first.  (No reference counterpart: spec decode is disabled for
    qwen3_5, nanovllm/config.py:84.)"""

    def __init__(self, s_pool: torch.Tensor):
        self.s_pool = s_pool
        self.inter = None
        self.ids = None
        self.accepted = None      # [B] int64 of the last verify, until the next verify or commit()

    def verify(self, q, k, v, g, beta, ids):
        Bsz, T = k.shape[:2]
        Hv, D = v.shape[2], v.shape[3]
        if self.accepted is not None:
            assert self.ids is not None and torch.equal(self.ids, ids), "the batch changed: commit() first"
        if self.inter is None or self.inter.shape != (Bsz, T, Hv, D, D):
            assert self.accepted is None, "the draft length changed: commit() first"
            self.inter = torch.empty(Bsz, T, Hv, D, D, dtype=torch.float32, device=v.device)
        out = recurrent_gdn_multitoken(q, k, v, g, beta, self.s_pool, ids, self.inter,
                                       self.inter if self.accepted is not None else None, self.accepted)
        self.ids = ids
        self.accepted = None      # the pool plus this step's states, until accept()
        return out

    def accept(self, accepted: torch.Tensor) -> None:
        """accepted [B] int64 (device): tokens kept per row, 1..T.  A row
        whose count lies outside 1..T starts the next verify from its pool
        row (the last committed state), as commit() leaves it untouched."""
        assert self.inter is not None and self.accepted is None, "accept() follows one verify()"
        assert accepted.dtype == torch.int64 and accepted.shape == (self.inter.shape[0],)
        assert accepted.device == self.inter.device and accepted.is_contiguous()
        self.accepted = accepted

    def commit(self) -> None:
        """Write the accepted states into the pool rows (a no-op when
        nothing is pending)."""
        if self.accepted is None:
            return
        commit_states(self.s_pool, self.ids, self.inter, self.accepted)
        self.accepted = None


def commit_states(s_pool, ids, intermediate_states, accepted):
    """s_pool[ids[b]] <- intermediate_states[b, accepted[b] - 1]
    (accepted in [1, T]; 0 leaves the slot unchanged)."""
    dev = _check_cuda(s_pool, ids, intermediate_states, accepted)
    Bsz, T, Hv, D, _ = intermediate_states.shape
    assert _state_view_ok(s_pool, Hv, D) and intermediate_states.is_contiguous()
    ids64 = ids.to(torch.int64).contiguous()
    acc = accepted.to(torch.int32).contiguous()
    assert ids64.shape == (Bsz,) and acc.shape == (Bsz,), "one slot id and one accepted length per row"
    _lib.call("gdn_state_commit", _lib.ptr(s_pool), s_pool.stride(0), _lib.ptr(ids64),
              _lib.ptr(intermediate_states), _lib.ptr(acc), Bsz, T, Hv, D, _stream(dev))


def state_tile_pass(s_pool: torch.Tensor, ids: torch.Tensor) -> None:
    """Measurement pass (no reference counterpart): reads every state tile
    s_pool[ids[b], h] and writes it back unchanged, with the one-token decode
    kernel's tile layout and cache policy -- that step's state traffic without
    its arithmetic.  s_pool [slots, Hv, D, D] fp32 (any slot stride)."""
    dev = _check_cuda(s_pool, ids)
    assert _state_view_ok(s_pool, s_pool.shape[1], s_pool.shape[-1])
    ids64 = ids.to(torch.int64).contiguous()
    _lib.call("gdn_state_tile_pass", _lib.ptr(s_pool), s_pool.stride(0), _lib.ptr(ids64), ids64.numel(),
              s_pool.shape[1], s_pool.shape[-1], _stream(dev))


def state_tile_copy(src_pool: torch.Tensor, dst_pool: torch.Tensor, ids: torch.Tensor) -> None:
    """Measurement pass (no reference counterpart): state_tile_pass with each
    tile written to dst_pool[ids[b], h] instead of back in place (the same
    launch shape, layout and cache policy).  Both pools [slots, Hv, D, D]
    fp32 with the same slot stride, not overlapping."""
    dev = _check_cuda(src_pool, dst_pool, ids)
    assert src_pool.shape == dst_pool.shape and src_pool.stride(0) == dst_pool.stride(0)
    assert _state_view_ok(src_pool, src_pool.shape[1], src_pool.shape[-1])
    assert _state_view_ok(dst_pool, dst_pool.shape[1], dst_pool.shape[-1])
    ids64 = ids.to(torch.int64).contiguous()
    _lib.call("gdn_state_tile_copy", _lib.ptr(src_pool), _lib.ptr(dst_pool), src_pool.stride(0), _lib.ptr(ids64),
              ids64.numel(), src_pool.shape[1], src_pool.shape[-1], _stream(dev))


# --------------------------------------------- verify over a tree of drafts --
MAX_TREE_NODES = 64


def _tree_parents(parents: torch.Tensor, B: int, T: int):
    """(int32 parents, row stride) of a [B, T] or [T] (one tree for all) tensor."""
    if not 1 <= T <= MAX_TREE_NODES:
        raise ValueError(f"a tree has 1 to {MAX_TREE_NODES} nodes, got {T}")
    stride = T if parents.dim() == 2 else 0
    if parents.shape != ((B, T) if stride else (T,)) or parents.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"parents must be int32 or int64 [{B}, {T}] or [{T}], got {parents.dtype} "
                         f"{list(parents.shape)}")
    if parents.dtype == torch.int64:
        # (out of int32's range: not a node either way)
        parents = parents.clamp(-2, MAX_TREE_NODES).to(torch.int32)
    return parents if parents.is_contiguous() else parents.contiguous(), stride


def _tree_ids(ids: torch.Tensor, B: int, name: str = "ids") -> torch.Tensor:
    if ids.dtype == torch.int64 and ids.shape == (B,) and ids.is_contiguous():
        return ids
    if ids.shape != (B,) or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int64 (or int32) [{B}], got {ids.dtype} {list(ids.shape)}")
    return ids.to(torch.int64).contiguous()


def _tree_rows(t: torch.Tensor, name: str, shape: tuple):
    """bf16 [B, T, heads, D] or [B, T, C] with dense rows that the kernels read in
    16-byte pieces (else copied once), and its strides per sequence and node."""
    if t.shape != shape or t.dtype != torch.bfloat16:
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    width = shape[2] if len(shape) == 3 else shape[2] * shape[3]
    st = t.stride()
    dense = st[-1] == 1 and (len(shape) == 3 or st[2] == shape[3] or shape[2] == 1)
    if not dense or not width <= st[1] < 1 << 24 or st[0] % 8 or st[1] % 8 or t.data_ptr() % 16:
        t = t.contiguous() if not t.is_contiguous() else t.clone(memory_format=torch.contiguous_format)
        return t, shape[1] * width, width
    return t, st[0], st[1]


def _tree_f32(t: torch.Tensor, name: str, shape: tuple) -> torch.Tensor:
    if t.dtype != torch.float32 or t.shape != shape:
        raise ValueError(f"{name} must be float32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _conv_pool_ok(pool: torch.Tensor, C: int) -> tuple:
    _bf16(pool, "conv_pool")
    st = pool.stride()
    if pool.dim() != 3 or pool.shape[1] != C or pool.shape[2] != 3 or st[2] != 1:
        raise ValueError(f"conv_pool must be a [slots, {C}, 3] view with contiguous taps, got {list(pool.shape)}")
    return st


def _s_pool_ok(pool: torch.Tensor, Hv: int, D: int) -> None:
    if pool.shape[1:] != (Hv, D, D) or pool.stride()[1:] != (D * D, D, 1) or pool.dtype != torch.float32:
        raise ValueError(f"s_pool must be an fp32 [slots, {Hv}, {D}, {D}] view with dense slots")


def conv_tree_step(x: torch.Tensor, conv_pool: torch.Tensor, ids: torch.Tensor, weight: torch.Tensor,
                   parents: torch.Tensor, pending: tuple | None = None) -> torch.Tensor:
    """Causal conv + SiLU of a tree of T drafted tokens per sequence: the taps of a
    node are its ancestors' rows and, past the root, the sequence's taps in the
    pool, which stays as it is.  x [B, T, C] bf16; conv_pool [slots, C, 3]; ids
    [B]; weight [C, 4] (or [C, 1, 4]); parents [B, T] (or [T], one tree for all):
    the node before each node, -1 for the sequence's own state; a node whose
    parent is neither -1 nor an earlier used node (-2 for padding) is unused and
    its output 0.  A sequence whose id is no slot has zero outputs.

    pending = (x, parents, accepted) of the step before, for the same sequences in
    the same rows: the rows on the path to node accepted[b] of each sequence (-1:
    none) go into the pool first, so the slot of a row with an accepted node is in no
    other row (which would read it while it is written); a slot of which nothing is
    accepted may be in several (a padded batch's rows: the dummy slot, or id -1).  Along a
    path the results are conv_decode_step's, bit for bit.  Returns y [B, T, C].
    (No reference counterpart: spec decode is disabled for qwen3_5,
    nanovllm/config.py:84.)"""
    y = _lib.quick().conv_tree(x, conv_pool, ids, weight, parents, pending)
    return y if y is not None else _conv_tree_ready(x, conv_pool, ids, weight, parents, pending).launch()


def _conv_tree_ready(x, conv_pool, ids, weight, parents, pending, y=None) -> _Ready:
    """conv_tree_step's call, checked; y: a contiguous tensor that takes the result."""
    last_x, last_parents, accepted = pending if pending is not None else (None, None, None)
    idx = _device_of(x, conv_pool, ids, weight, parents, last_x, last_parents, accepted)
    if x.dim() != 3:
        raise ValueError(f"x must be [B, T, C], got {list(x.shape)}")
    shape = B, T, C = x.shape
    x, x_b, x_t = _tree_rows(x, "x", shape)
    pool_st = _conv_pool_ok(conv_pool, C)
    _bf16(weight, "weight")
    if weight.numel() != 4 * C or weight.shape[-1] != 4 or C % 8:
        raise ValueError(f"weight must be [{C}, 4] (conv width 4) and C a multiple of 8")
    w = weight
    if not w.is_contiguous() or w.data_ptr() % 16:
        w = w.clone(memory_format=torch.contiguous_format)
    ids = _tree_ids(ids, B)
    par, p_b = _tree_parents(parents, B, T)
    last = (0, 0, 0, 0, 0, 0, 0)
    if pending is not None:
        last_T = last_x.shape[1]
        last_x, lx_b, lx_t = _tree_rows(last_x, "pending x", (B, last_T, C))
        last_parents, lp_b = _tree_parents(last_parents, B, last_T)
        accepted = _tree_ids(accepted, B, "accepted")
        last = (last_x.data_ptr(), lx_b, lx_t, last_parents.data_ptr(), lp_b, accepted.data_ptr(), last_T)
    if y is None:
        y = x.new_empty(shape)
    args = (x.data_ptr(), x_b, x_t, conv_pool.data_ptr(), pool_st[0], pool_st[1], conv_pool.shape[0], ids.data_ptr(),
            w.data_ptr(), par.data_ptr(), p_b, *last, y.data_ptr(), B, T, C)
    return _Ready(idx, "gdn_conv_tree", args, y, (x, ids, w, par, last_x, last_parents, accepted))


def _rule_args(q, k, v, s_pool, ids, parents, pending):
    """The checked arguments of the rule over a tree: (B, T, Hk, Hv, D), those of the rows
    and those from the pool on, and the tensors that they point into."""
    if k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k, v must be [B, T, heads, D], got {list(k.shape)} and {list(v.shape)}")
    k_shape = B, T, Hk, D = k.shape
    Hv = v.shape[2]
    if Hk == 0 or Hv % Hk:
        raise ValueError(f"{Hv} value heads are no multiple of {Hk} key heads")
    q, q_b, q_t = _tree_rows(q, "q", k_shape)
    k, k_b, k_t = _tree_rows(k, "k", k_shape)
    v, v_b, v_t = _tree_rows(v, "v", (B, T, Hv, D))
    _s_pool_ok(s_pool, Hv, D)
    ids = _tree_ids(ids, B)
    par, p_b = _tree_parents(parents, B, T)
    last, keep = (0,) * 9, None
    if pending is not None:
        last_k, last_g, last_u, last_parents, accepted = pending
        last_T = last_k.shape[1]
        last_k, lk_b, lk_t = _tree_rows(last_k, "pending k", (B, last_T, Hk, D))
        last_g = _tree_f32(last_g, "pending g", (B, last_T, Hv))
        last_u = _tree_f32(last_u, "pending u", (B, last_T, Hv, D))
        last_parents, lp_b = _tree_parents(last_parents, B, last_T)
        accepted = _tree_ids(accepted, B, "accepted")
        last = (last_k.data_ptr(), lk_b, lk_t, last_g.data_ptr(), last_u.data_ptr(), last_parents.data_ptr(), lp_b,
                accepted.data_ptr(), last_T)
        keep = last_k, last_g, last_u, last_parents, accepted
    return ((B, T, Hk, Hv, D), (q.data_ptr(), q_b, q_t, k.data_ptr(), k_b, k_t, v.data_ptr(), v_b, v_t),
            (s_pool.data_ptr(), s_pool.stride(0), s_pool.shape[0], ids.data_ptr(), par.data_ptr(), p_b, *last),
            (q, k, v, ids, par, keep))


def recurrent_gdn_tree(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                       s_pool: torch.Tensor, ids: torch.Tensor, parents: torch.Tensor,
                       pending: tuple | None = None):
    """The gated delta rule over a tree of T drafted tokens per sequence: node t
    continues from its parent's state, a root from the sequence's state in the
    pool, which stays as it is.  q, k [B, T, Hk, D] and v [B, T, Hv, D] bf16 (after
    the conv; q and k are L2-normalised here), g [B, T, Hv] fp32, beta [B, T, Hv]
    bf16, s_pool [slots, Hv, D, D] fp32, ids [B], parents as conv_tree_step.

    Returns (o [B, T, Hv, D] bf16, u [B, T, Hv, D] fp32): the outputs, and the
    corrections from which, with k and g, the state after any node follows (no
    state of a node is stored).  pending = (k, g, u, parents, accepted) of the
    step before, for the same sequences in the same rows: the states after the
    accepted nodes go into the pool first, in the same pass over them, and the
    trees start from there (accepted[b] -1, or no used node: the row's state stays;
    slots as conv_tree_step's).  A decay of 0 (g = -inf) forgets what came before
    it, also what is not finite.
    (No reference counterpart: spec decode is disabled for qwen3_5,
    nanovllm/config.py:84; one token: qwen3_5.py:575-594.)"""
    out = _lib.quick().rule_tree(q, k, v, g, beta, s_pool, ids, parents, pending)
    return out if out is not None else _rule_tree_ready(q, k, v, g, beta, s_pool, ids, parents, pending).launch()


def _rule_tree_ready(q, k, v, g, beta, s_pool, ids, parents, pending) -> _Ready:
    """recurrent_gdn_tree's call, checked."""
    idx = _device_of(k, q, v, g, beta, s_pool, ids, parents, *(pending or ()))
    dims, rows, state, keep = _rule_args(q, k, v, s_pool, ids, parents, pending)
    B, T, Hk, Hv, D = dims
    g_shape, v_shape = (B, T, Hv), (B, T, Hv, D)
    g = _tree_f32(g, "g", g_shape)
    _bf16(beta, "beta")
    if beta.shape != g_shape:
        raise ValueError(f"beta must be {list(g_shape)}, got {list(beta.shape)}")
    if not beta.is_contiguous():
        beta = beta.contiguous()
    o, u = v.new_empty(v_shape), g.new_empty(v_shape)
    args = (*rows, g.data_ptr(), beta.data_ptr(), *state, o.data_ptr(), u.data_ptr(), *dims, D ** -0.5)
    return _Ready(idx, "gdn_rule_tree", args, (o, u), (g, beta, keep))


def recurrent_tree_fused(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, b: torch.Tensor, a: torch.Tensor,
                         a_log: torch.Tensor, dt_bias: torch.Tensor, z: torch.Tensor, norm_weight: torch.Tensor,
                         s_pool: torch.Tensor, ids: torch.Tensor, parents: torch.Tensor, eps: float = 1e-6,
                         pending: tuple | None = None, fp8: bool = False):
    """recurrent_gdn_tree with the layer's gates before it and its gated norm behind
    it in one launch: fused_g_beta(b, a) -> recurrent_gdn_tree -> rms_norm_gated (or
    with fp8, D = 128, rms_norm_gated_fp8), the same bits for every used node, and
    zeros for the others (rows of a slot that is none: g too).  b, a [B, T, Hv] bf16,
    a_log and dt_bias [Hv], z [B, T, Hv * D] bf16, norm_weight [D].  Returns (y [B, T,
    Hv, D] bf16, or its (e4m3, scales); u; g), g for the next step's pending."""
    out = _lib.quick().rule_tree_layer(q, k, v, b, a, a_log, dt_bias, z, norm_weight, s_pool, ids, parents, eps, pending,
                                       fp8)
    if out is not None:
        y, scale, u, g = out
        return (y, scale) if fp8 else y, u, g
    return _rule_tree_layer_ready(q, k, v, b, a, a_log, dt_bias, z, norm_weight, s_pool, ids, parents, eps, pending,
                                  fp8).launch()


def _rule_tree_layer_ready(q, k, v, b, a, a_log, dt_bias, z, norm_weight, s_pool, ids, parents, eps, pending,
                           fp8) -> _Ready:
    """recurrent_tree_fused's call, checked."""
    idx = _device_of(k, q, v, b, a, a_log, dt_bias, z, norm_weight, s_pool, ids, parents, *(pending or ()))
    dims, rows, state, keep = _rule_args(q, k, v, s_pool, ids, parents, pending)
    B, T, Hk, Hv, D = dims
    if fp8 and D != FP8_GROUP:
        raise ValueError(f"fp8 outputs have a scale for each head of {FP8_GROUP}, got head dim {D}")
    for t, name in ((b, "b"), (a, "a")):
        _bf16(t, name)
        if t.shape != (B, T, Hv):
            raise ValueError(f"{name} must be {[B, T, Hv]}, got {list(t.shape)}")
    b, a = b.contiguous(), a.contiguous()
    if a_log.dtype != dt_bias.dtype or a_log.dtype not in (torch.bfloat16, torch.float32):
        a_log, dt_bias = a_log.float(), dt_bias.float()
    a_log, dt_bias = a_log.contiguous(), dt_bias.contiguous()
    if a_log.numel() != Hv or dt_bias.numel() != Hv or norm_weight.numel() != D:
        raise ValueError(f"a_log and dt_bias must have {Hv} values, norm_weight {D}")
    z, z_b, z_t = _tree_rows(z, "z", (B, T, Hv * D))
    w = norm_weight
    if w.dtype != torch.bfloat16 or not w.is_contiguous() or w.data_ptr() % 16:
        w = w.to(torch.bfloat16).clone(memory_format=torch.contiguous_format)
    y = v.new_empty((B, T, Hv, D), dtype=FP8 if fp8 else torch.bfloat16)
    scale = _fp8_scales(B * T, Hv, v.device) if fp8 else None
    u = v.new_empty((B, T, Hv, D), dtype=torch.float32)
    g = v.new_empty((B, T, Hv), dtype=torch.float32)
    out = (0, y.data_ptr(), scale.data_ptr()) if fp8 else (y.data_ptr(), 0, 0)
    args = (*rows, b.data_ptr(), a.data_ptr(), a_log.data_ptr(), dt_bias.data_ptr(), int(a_log.dtype == torch.float32),
            *state, z.data_ptr(), z_b, z_t, w.data_ptr(), float(eps), *out, u.data_ptr(), g.data_ptr(), *dims, D ** -0.5)
    return _Ready(idx, "gdn_rule_tree_layer", args, ((y, scale) if fp8 else y, u, g), (b, a, a_log, dt_bias, z, w, keep))


def _verify_tree(x, conv_pool, weight, b, a, a_log, dt_bias, z, norm_weight, s_pool, ids, parents, Hk, Hv, D, eps,
                 last_conv, last_rule, fp8, gates, timed):
    """conv_tree_step and the rule with the layer's gates and norm (recurrent_tree_fused, or where heads
    of 64 share a scale its three calls, gates() giving g and beta), of which all are launched or none:
    each is checked, and all memory allocated, before the conv moves its pool on.  timed(name): a
    context around a launch, or None.  Returns (out, k, u, g)."""
    conv = (x, conv_pool, ids, weight, parents, last_conv)
    layer = (b, a, a_log, dt_bias, z, norm_weight, s_pool, ids, parents, eps, last_rule, fp8)
    fused = not fp8 or D == FP8_GROUP
    g = beta = None
    if not fused:
        g, beta = gates()
    if timed is None:
        quick = _lib.quick()
        if fused:
            out = quick.verify_tree(*conv, Hk, D, *layer)
            if out is not None:
                y, scale, k, u, g = out
                return (y, scale) if fp8 else y, k, u, g
        else:
            out = quick.verify_tree_norm(*conv, Hk, D, g, beta, s_pool, ids, parents, last_rule, z, norm_weight, eps)
            if out is not None:
                y, scale, k, u = out
                return (y, scale), k, u, g
    B, T, C = x.shape
    kd = Hk * D
    if C != 2 * kd + Hv * D:
        raise ValueError(f"x must have {2 * kd + Hv * D} channels, got {C}")
    y = x.new_empty(x.shape)
    q, k, v = (y[..., :kd].unflatten(-1, (Hk, D)), y[..., kd:2 * kd].unflatten(-1, (Hk, D)),
               y[..., 2 * kd:].unflatten(-1, (Hv, D)))
    if conv_pool.shape[0] != s_pool.shape[0]:     # (a slot of one of them alone)
        raise ValueError(f"the pools have {s_pool.shape[0]} and {conv_pool.shape[0]} slots")
    calls = [("conv_tree", _conv_tree_ready(*conv, y))]
    if fused:
        calls.append(("recurrent_tree", _rule_tree_layer_ready(q, k, v, *layer)))
        out, u, g = calls[1][1].out
    else:
        calls.append(("recurrent_tree", _rule_tree_ready(q, k, v, g, beta, s_pool, ids, parents, last_rule)))
        o, u = calls[1][1].out
        calls.append(("rmsnorm_gated", _norm_fp8_ready(o, z.reshape(B, T, Hv, D), norm_weight, eps)))
        out = calls[2][1].out
    for _, call in calls:
        call.check()
    for name, call in calls:
        with contextlib.nullcontext() if timed is None else timed(name):
            call.launch()
    return out, k, u, g


def commit_tree(s_pool: torch.Tensor, conv_pool: torch.Tensor, ids: torch.Tensor, parents: torch.Tensor,
                accepted: torch.Tensor, x: torch.Tensor, k: torch.Tensor, g: torch.Tensor, u: torch.Tensor) -> None:
    """The accepted path of a verified tree into both pools, for another user of the
    slots than the next verify (whose `pending` does the same): row ids[b] of
    s_pool becomes the state after node accepted[b], that of conv_pool the last
    three raw rows on its path; -1 (or no used node) leaves both as they are (slots
    as conv_tree_step's).
    x [B, T, C] the raw rows, k [B, T, Hk, D], g [B, T, Hv], u [B, T, Hv, D] and
    parents those of the verified step."""
    if _lib.quick().commit_tree(s_pool, conv_pool, ids, parents, accepted, x, k, g, u):
        return
    idx = _device_of(s_pool, conv_pool, ids, parents, accepted, x, k, g, u)
    if k.dim() != 4 or u.dim() != 4 or x.dim() != 3:
        raise ValueError(f"x, k, u must be [B, T, C], [B, T, Hk, D], [B, T, Hv, D], got {list(x.shape)}, "
                         f"{list(k.shape)}, {list(u.shape)}")
    k_shape = B, T, Hk, D = k.shape
    Hv, C = u.shape[2], x.shape[2]
    if Hk == 0 or Hv % Hk:
        raise ValueError(f"{Hv} value heads are no multiple of {Hk} key heads")
    x, x_b, x_t = _tree_rows(x, "x", (B, T, C))
    k, k_b, k_t = _tree_rows(k, "k", k_shape)
    g, u = _tree_f32(g, "g", (B, T, Hv)), _tree_f32(u, "u", (B, T, Hv, D))
    _s_pool_ok(s_pool, Hv, D)
    pool_st = _conv_pool_ok(conv_pool, C)
    slots = s_pool.shape[0]
    if conv_pool.shape[0] != slots:
        raise ValueError(f"the pools have {slots} and {conv_pool.shape[0]} slots")
    ids, accepted = _tree_ids(ids, B), _tree_ids(accepted, B, "accepted")
    par, p_b = _tree_parents(parents, B, T)
    _call_on(idx, "gdn_commit_tree", s_pool.data_ptr(), s_pool.stride(0), conv_pool.data_ptr(), pool_st[0], pool_st[1],
             slots, ids.data_ptr(), par.data_ptr(), p_b, accepted.data_ptr(), x.data_ptr(), x_b, x_t, k.data_ptr(), k_b,
             k_t, g.data_ptr(), u.data_ptr(), B, T, Hk, Hv, D, C)


# ------------------------------------------------------------- projections --
def linear(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor | None = None,
           gates: dict | None = None) -> torch.Tensor:
    """F.linear(x, weight) without bias on the bf16 matrix cores (fp32
    accumulation): x [..., K] bf16 (last dim contiguous), weight [N, K] bf16
    (nn.Linear layout).  Returns [..., N] bf16 (or writes `out`, a [M, N]
    view with contiguous rows).  gates: {"gate_col", "A_log", "dt_bias"}
    (and the Hv of A_log): the columns [gate_col, gate_col + Hv) are the b
    projection and the next Hv the a projection; beta (bf16) and g (fp32)
    [M, Hv] of them are also computed and returned as (y, g, beta), equal to
    fused_g_beta on those columns.
    Reference: ColumnParallelLinear / RowParallelLinear.forward,
    nanovllm/layers/linear.py:74-75, :154-158 (tp = 1)."""
    dev = _check_cuda(x, weight, out)
    _bf16(x, "x")
    _bf16(weight, "weight")
    K = x.shape[-1]
    N = weight.shape[0]
    assert weight.shape[1] == K
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    w = weight if (weight.stride(1) == 1 and weight.stride(0) % 8 == 0 and weight.data_ptr() % 16 == 0) \
        else weight.contiguous()
    M = x2.shape[0]
    if out is None:
        y = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
    else:
        _bf16(out, "out")
        assert out.shape == (M, N) and out.stride(1) == 1
        y = out
    g = beta = None
    a_log = dt_bias = None
    gate_col = Hv = 0
    if gates is not None:
        a_log, dt_bias = gates["A_log"], gates["dt_bias"]
        if a_log.dtype != dt_bias.dtype or a_log.dtype not in (torch.bfloat16, torch.float32):
            a_log, dt_bias = a_log.float(), dt_bias.float()
        a_log, dt_bias = a_log.contiguous(), dt_bias.contiguous()
        Hv = a_log.numel()
        gate_col = int(gates["gate_col"])
        g = torch.empty(M, Hv, dtype=torch.float32, device=x.device)
        beta = torch.empty(M, Hv, dtype=torch.bfloat16, device=x.device)
    _lib.call("gdn_gemm_bf16", _lib.ptr(x2), x2.stride(0), _lib.ptr(w), w.stride(0), _lib.ptr(y), y.stride(0),
              M, N, K, _lib.ptr(g), _lib.ptr(beta), _lib.ptr(a_log), _lib.ptr(dt_bias),
              int(a_log is not None and a_log.dtype == torch.float32), gate_col, Hv, _stream(dev))
    y = y.view(*x.shape[:-1], N) if out is None else y
    return y if gates is None else (y, g, beta)


def linear_cols(x: torch.Tensor, weight: torch.Tensor, widths: list[int],
                gates: dict | None = None):
    """linear(x, weight) with the output's columns split into len(widths)
    (1-4) contiguous tensors [M, widths[s]] (sum(widths) == weight rows;
    every boundary a multiple of 16): the same values as linear's columns.
    For the GDN layer's in_proj over its four concatenated weights, so that
    the qkv, z, b and a parts come out as tensors of their own, as the
    reference's separate projections produce them
    (nanovllm/models/qwen3_5.py:929-939).  gates: as in linear (gate_col
    counts the concatenated columns).  Returns the list of parts, and with
    gates (parts, g, beta)."""
    dev = _check_cuda(x, weight)
    _bf16(x, "x")
    _bf16(weight, "weight")
    K = x.shape[-1]
    N = weight.shape[0]
    assert weight.shape[1] == K and sum(widths) == N and 1 <= len(widths) <= 4
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    w = weight if (weight.stride(1) == 1 and weight.stride(0) % 8 == 0 and weight.data_ptr() % 16 == 0) \
        else weight.contiguous()
    M = x2.shape[0]
    parts = [torch.empty(M, wd, dtype=torch.bfloat16, device=x.device) for wd in widths]
    ends, e = [], 0
    for wd in widths:
        e += wd
        ends.append(e)
    n = len(widths)
    c_arr = (ctypes.c_void_p * n)(*[p.data_ptr() for p in parts])
    ld_arr = (ctypes.c_int64 * n)(*[p.stride(0) for p in parts])
    end_arr = (ctypes.c_int * n)(*ends)
    g = beta = None
    a_log = dt_bias = None
    gate_col = Hv = 0
    if gates is not None:
        a_log, dt_bias = gates["A_log"], gates["dt_bias"]
        if a_log.dtype != dt_bias.dtype or a_log.dtype not in (torch.bfloat16, torch.float32):
            a_log, dt_bias = a_log.float(), dt_bias.float()
        a_log, dt_bias = a_log.contiguous(), dt_bias.contiguous()
        Hv = a_log.numel()
        gate_col = int(gates["gate_col"])
        g = torch.empty(M, Hv, dtype=torch.float32, device=x.device)
        beta = torch.empty(M, Hv, dtype=torch.bfloat16, device=x.device)
    _lib.call("gdn_gemm_bf16_cols", _lib.ptr(x2), x2.stride(0), _lib.ptr(w), w.stride(0), M, N, K, n, c_arr,
              ld_arr, end_arr, _lib.ptr(g), _lib.ptr(beta), _lib.ptr(a_log), _lib.ptr(dt_bias),
              int(a_log is not None and a_log.dtype == torch.float32), gate_col, Hv, _stream(dev))
    parts = [p.view(*x.shape[:-1], p.shape[1]) for p in parts]
    return parts if gates is None else (parts, g, beta)


# ------------------------------------------------------- 8-bit projections --
FP8 = torch.float8_e4m3fn
FP8_GROUP = 128   # values with one scale
# Up to so many rows the bf16 columns beside an 8-bit product come with the launch that quantizes
# its rows (linear_fp8_cols' wide); past it they are a product of their own.
FP8_WIDE_ROWS = 1024


def _rows_of(x: torch.Tensor, align: int):
    """x [..., K] as [M, K] rows that the kernels read in 16-byte pieces, and their stride."""
    K = x.shape[-1]
    if x.is_contiguous():
        if x.data_ptr() % 16:
            x = x.clone(memory_format=torch.contiguous_format)
        return x, x.numel() // K, K
    x2 = x.reshape(-1, K)
    st = x2.stride()
    if st[1] != 1 or st[0] % align or st[0] < K or x2.data_ptr() % 16:
        x2 = x2.contiguous() if not x2.is_contiguous() else x2.clone(memory_format=torch.contiguous_format)
        return x2, x2.shape[0], K
    return x2, x2.shape[0], st[0]


def _fp8_scales(M: int, G: int, dev) -> torch.Tensor:
    """[M, G] fp32 with the rows of one group side by side (as the GEMM reads them)."""
    return torch.empty_strided((M, G), (1, M), dtype=torch.float32, device=dev)


def quantize_fp8(x: torch.Tensor):
    """x [..., K] bf16 or fp32 (K a multiple of 128) -> (e4m3 [..., K], scales [M, K /
    128] fp32): each row's groups of 128 columns have the scale max(amax * fp32(1 /
    448), 2^-126), and a value is x times the scale's fp32 reciprocal, rounded to
    nearest.  NaN stays NaN without counting in amax; an infinity makes its group's
    scale infinite.  (The scales' memory holds the rows of a group side by side.)"""
    idx = _device_of(x)
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"x must be bfloat16 or float32, got {x.dtype}")
    K = x.shape[-1]
    if K == 0 or K % FP8_GROUP:
        raise ValueError(f"the last dim must be a positive multiple of {FP8_GROUP}, got {K}")
    f32 = x.dtype == torch.float32
    rows, M, stride = _rows_of(x, 4 if f32 else 8)
    y = torch.empty(x.shape, dtype=FP8, device=x.device)
    scale = _fp8_scales(M, K // FP8_GROUP, x.device)
    _call_on(idx, "gdn_quantize_fp8", rows.data_ptr(), int(f32), stride, y.data_ptr(), K, scale.data_ptr(), 1, M, M, K,
             1)
    return y, scale


def quantize_weight_fp8(weight: torch.Tensor):
    """weight [N, K] bf16 or fp32 (nn.Linear layout, K a multiple of 128) -> (e4m3 [N,
    K], scales [ceil(N / 128), K / 128] fp32), a scale for each 128 x 128 block; once,
    when the weights are loaded.  The rounding is quantize_fp8's."""
    idx = _device_of(weight)
    if weight.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"weight must be bfloat16 or float32, got {weight.dtype}")
    if weight.dim() != 2 or weight.shape[1] == 0 or weight.shape[1] % FP8_GROUP:
        raise ValueError(f"weight must be [N, K] with K a positive multiple of {FP8_GROUP}, got {list(weight.shape)}")
    f32 = weight.dtype == torch.float32
    N, K = weight.shape
    rows, _, stride = _rows_of(weight, 4 if f32 else 8)
    y = torch.empty(N, K, dtype=FP8, device=weight.device)
    scale = torch.empty(-(-N // FP8_GROUP), K // FP8_GROUP, dtype=torch.float32, device=weight.device)
    _call_on(idx, "gdn_quantize_fp8", rows.data_ptr(), int(f32), stride, y.data_ptr(), K, scale.data_ptr(),
             K // FP8_GROUP, 1, N, K, FP8_GROUP)
    return y, scale


def _check_fp8(x, weight, weight_scale, x_scale):
    """The shapes of a product: (M, N, K)."""
    if weight.dtype != FP8 or weight.dim() != 2:
        raise TypeError(f"weight must be float8_e4m3fn [N, K], got {weight.dtype} {list(weight.shape)}")
    N, K = weight.shape
    if K == 0 or K % FP8_GROUP or x.shape[-1] != K:
        raise ValueError(f"x [..., {x.shape[-1]}] and weight [{N}, {K}]: equal last dims, a positive multiple of "
                         f"{FP8_GROUP}")
    G = K // FP8_GROUP
    if weight_scale.dtype != torch.float32 or weight_scale.shape != (-(-N // FP8_GROUP), G):
        raise ValueError(f"weight_scale must be float32 {[-(-N // FP8_GROUP), G]}, got {weight_scale.dtype} "
                         f"{list(weight_scale.shape)}")
    M = x.numel() // K
    if x.dtype == FP8:
        if x_scale is None or x_scale.dtype != torch.float32 or x_scale.shape != (M, G):
            raise ValueError(f"a float8_e4m3fn x needs x_scale float32 {[M, G]}")
    elif x.dtype != torch.bfloat16 or x_scale is not None:
        raise TypeError(f"x must be bfloat16, or float8_e4m3fn with x_scale, got {x.dtype}"
                        + ("" if x_scale is None else " with x_scale"))
    return M, N, K


@functools.lru_cache(maxsize=256)
def _fp8_workspace(M: int, N: int, K: int) -> int:
    return _lib.load().gdn_gemm_fp8_workspace_size(M, N, K, 1)


def _linear_fp8(x, weight, weight_scale, x_scale, M, N, K, outs, widths, wide=None):
    """The product into outs, [M, widths[s]] each; the columns past N from the bf16 weight
    `wide`."""
    idx = _device_of(x, weight, weight_scale, x_scale, wide, *outs)
    wide_args = (0, 0, 0)
    if wide is not None:
        if wide.stride(1) != 1 or wide.stride(0) % 8 or wide.stride(0) < K or wide.data_ptr() % 16:
            wide = wide.clone(memory_format=torch.contiguous_format)
        wide_args = (wide.data_ptr(), wide.stride(0), wide.shape[0])
    w, w_st = weight, weight.stride()
    if w_st[1] != 1 or w_st[0] % 16 or w_st[0] < K or w.data_ptr() % 16:
        w = w.contiguous() if not w.is_contiguous() else w.clone(memory_format=torch.contiguous_format)
        w_st = (K, 1)
    G = K // FP8_GROUP
    ws_st = weight_scale.stride()
    ws = weight_scale if (ws_st[1] == 1 or G == 1) and (ws_st[0] >= G or N <= FP8_GROUP) else weight_scale.contiguous()
    bf16 = x_scale is None
    x2, _, x_row = _rows_of(x, 8 if bf16 else 16)
    work, ws_bytes, xs = None, 0, (0, 0, 0)
    if bf16:
        ws_bytes = _fp8_workspace(M, N, K)
        if ws_bytes > 0:
            work = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
    else:
        xs = (x_scale.data_ptr(), *x_scale.stride())
    n = len(widths)
    if n == 1:
        y = outs[0]
        parts = (y.data_ptr(), max(y.stride(0), N), N)
    else:
        parts, end = [], 0
        for y, width in zip(outs, widths):
            end += width
            parts += (y.data_ptr(), width, end)
    pack, head = _lib.GEMM_FP8_WORDS[n]
    _launch_on(idx, "gdn_gemm_fp8", pack(head, x2.data_ptr(), bf16, x_row, *xs, w.data_ptr(), w_st[0], ws.data_ptr(),
                                         ws.stride(0) if N > FP8_GROUP else G, *wide_args, M, N, K, n,
                                         0 if work is None else work.data_ptr(), ws_bytes, _lib.stream_of(idx),
                                         *parts))


def linear_fp8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
               x_scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """linear(x, weight) with the weight in e4m3 [N, K] and weight_scale [ceil(N / 128),
    K / 128] fp32, one for each 128 x 128 block (quantize_weight_fp8's, or a
    checkpoint's).  x [..., K] bf16, quantized in the call (the bits of quantize_fp8 and
    a call with its result), or e4m3 with its x_scale [M, K / 128] (any strides).  K a
    multiple of 128; x and weight below 2 GiB each (more rows in several calls).  fp32
    accumulation; returns [..., N] bf16 (or writes `out`, a [M, N] view with contiguous
    rows of any alignment)."""
    if out is None:
        y = _lib.quick().linear_fp8(x, weight, weight_scale, x_scale)
        if y is not None:
            return y
    M, N, K = _check_fp8(x, weight, weight_scale, x_scale)
    if out is None:
        y = torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
    else:
        _bf16(out, "out")
        if out.shape != (M, N) or (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise ValueError(f"out must be a {[M, N]} view with contiguous rows that do not overlap")
        y = out
    _linear_fp8(x, weight, weight_scale, x_scale, M, N, K, (y,), (N,))
    return y if out is not None or x.dim() == 2 else y.view(*x.shape[:-1], N)


def linear_fp8_cols(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, widths: list[int],
                    x_scale: torch.Tensor | None = None, wide: torch.Tensor | None = None) -> list[torch.Tensor]:
    """linear_fp8 with the output's columns split into len(widths) (1-4) contiguous
    tensors [..., widths[s]], every boundary a multiple of 16 (as linear_cols).

    wide: a bf16 weight [N2, K] (N2 and N multiples of 16) whose product with the bf16 x
    follows as the last columns, N2 of the widths' sum, a boundary at N: the GDN layer's
    gate projections, which stay in bf16, without a launch of their own where x is
    quantized in the call's."""
    M, N, K = _check_fp8(x, weight, weight_scale, x_scale)
    total = N
    if wide is not None:
        if wide.dtype != torch.bfloat16 or x.dtype != torch.bfloat16:
            raise TypeError(f"wide and x must be bfloat16, got {wide.dtype} and {x.dtype}")
        if wide.dim() != 2 or wide.shape[1] != K or wide.shape[0] % 16 or wide.shape[0] == 0 or N % 16:
            raise ValueError(f"wide must be [N2, {K}] with N2 and N = {N} positive multiples of 16, got "
                             f"{list(wide.shape)}")
        total += wide.shape[0]
    ends = [sum(widths[:i + 1]) for i in range(len(widths))]
    if not 1 <= len(widths) <= 4 or ends[-1] != total or min(widths) <= 0 or any(w % 16 for w in widths[:-1]) \
            or N not in ends:
        raise ValueError(f"widths {widths}: 1 to 4 parts of {total} columns, boundaries at multiples of 16"
                         + (f" and at {N}" if wide is not None else ""))
    parts = [torch.empty(M, w, dtype=torch.bfloat16, device=x.device) for w in widths]
    _linear_fp8(x, weight, weight_scale, x_scale, M, N, K, parts, widths, wide)
    return parts if x.dim() == 2 else [p.view(*x.shape[:-1], p.shape[1]) for p in parts]


# ------------------------------------------------------ low-rank adapters --
LORA_MAX_RANK = 256
LORA_SORT = 256       # GDN_LORA_SORT


class LoraPool:
    """The low-rank adapters of one projection, or of several side by side, that are
    loaded together: slot s adds scale[s] * (x A_s^T) B_s^T to the rows that name it.

    widths: the columns of each projection (1 to 4 of them, boundaries at multiples of
    16), each with an A of its own.  a [slots, len(widths) * rank, in_features] bf16, b
    [slots, sum(widths), rank] bf16 and scale [slots] fp32 are laid out once and filled
    in place (captured graphs see an adapter that is loaded later); `rank` is brought up
    to a multiple of 8, and adapters of a smaller one are padded with zeros."""

    def __init__(self, slots: int, rank: int, in_features: int, widths: list[int], device="cuda"):
        self.widths, self.in_features = list(widths), in_features
        self.rank = -(-rank // 8) * 8
        if slots < 0 or not 1 <= rank <= LORA_MAX_RANK:
            raise ValueError(f"slots = {slots} (0 or more) and rank = {rank} (1 to {LORA_MAX_RANK})")
        if not 1 <= len(self.widths) <= 4 or min(self.widths) <= 0 or any(w % 16 for w in self.widths[:-1]):
            raise ValueError(f"widths {widths}: 1 to 4 projections, boundaries at multiples of 16")
        self.a = torch.zeros(slots, len(self.widths) * self.rank, in_features, dtype=torch.bfloat16, device=device)
        self.b = torch.zeros(slots, sum(self.widths), self.rank, dtype=torch.bfloat16, device=device)
        self.scale = torch.zeros(slots, dtype=torch.float32, device=device)

    def _slot(self, slot: int) -> None:
        if not 0 <= slot < self.a.shape[0]:
            raise ValueError(f"slot {slot} of {self.a.shape[0]}")

    def check(self, slot: int, parts) -> None:
        """Raises where load would."""
        self._slot(slot)
        if len(parts) != len(self.widths):
            raise ValueError(f"{len(parts)} parts for {len(self.widths)} projections")
        for part, width in zip(parts, self.widths):
            if part is not None:
                r = part[0].shape[0]
                if r > self.rank or part[0].shape != (r, self.in_features) or part[1].shape != (width, r):
                    raise ValueError(f"A must be [r, {self.in_features}] and B [{width}, r] with r <= {self.rank}, got "
                                     f"{list(part[0].shape)} and {list(part[1].shape)}")

    def load(self, slot: int, parts, scale: float) -> None:
        """An adapter into a slot: for each projection (A [r, in_features], B [width, r]),
        r at most the pool's rank, or None where the adapter has nothing for it; scale as
        the checkpoint defines it (alpha / r)."""
        self.check(slot, parts)
        self.clear(slot)
        col = 0
        for p, (part, width) in enumerate(zip(parts, self.widths)):
            if part is not None:
                r = part[0].shape[0]
                self.a[slot, p * self.rank:p * self.rank + r].copy_(part[0])
                self.b[slot, col:col + width, :r].copy_(part[1])
            col += width
        self.scale[slot] = scale

    def clear(self, slot: int) -> None:
        """An empty adapter (its rows get the projection alone)."""
        self._slot(slot)
        self.a[slot].zero_()
        self.b[slot].zero_()
        self.scale[slot] = 0.0


def adapter_rows(adapters: torch.Tensor, cu_seqlens: torch.Tensor, rows: int) -> torch.Tensor:
    """The adapter of each of `rows` rows, int32 [rows], from those of the sequences,
    adapters [n] (-1: none), and the sequences' offsets cu_seqlens [n + 1] on the same
    device: once per step, for all of its layers.  Rows behind the last sequence have none."""
    if adapters.dim() != 1 or cu_seqlens.shape != (adapters.shape[0] + 1,) or adapters.device != cu_seqlens.device:
        raise ValueError(f"adapters [n] and cu_seqlens [n + 1] on one device, got {list(adapters.shape)} on {adapters.device} "
                         f"and {list(cu_seqlens.shape)} on {cu_seqlens.device}")
    at = torch.searchsorted(cu_seqlens[1:].contiguous(), torch.arange(rows, dtype=cu_seqlens.dtype, device=adapters.device),
                            right=True)
    if adapters.dtype == torch.int64:   # (a number that 32 bits do not hold is no slot either)
        adapters = adapters.clamp(-1, 2**31 - 1)
    return torch.cat([adapters.to(torch.int32), adapters.new_full((1,), -1, dtype=torch.int32)])[at]


def _lora_check(x, N, K, widths, lora_a, lora_b, lora_scale, ids):
    """The adapters' shapes beside a product with N columns: (M, P, R)."""
    M = x.numel() // K
    P = len(widths)
    if not 1 <= P <= 4 or sum(widths) != N or min(widths) <= 0 or any(w % 16 for w in widths[:-1]):
        raise ValueError(f"widths {list(widths)}: 1 to 4 parts of {N} columns, boundaries at multiples of 16")
    for t, nm in ((lora_a, "lora_a"), (lora_b, "lora_b")):
        _bf16(t, nm)
        if t.dim() != 3:
            raise ValueError(f"{nm} must have 3 dims, got {list(t.shape)}")
    S, R = lora_b.shape[0], lora_b.shape[2]
    if R % 8 or not 8 <= R <= LORA_MAX_RANK:
        raise ValueError(f"the rank must be a multiple of 8 up to {LORA_MAX_RANK} (LoraPool pads), got {R}")
    if lora_a.shape != (S, P * R, K) or lora_b.shape[1] != N:
        raise ValueError(f"lora_a must be {[S, P * R, K]} and lora_b {[S, N, R]}, got {list(lora_a.shape)} and "
                         f"{list(lora_b.shape)}")
    for t, nm in ((lora_a, "lora_a"), (lora_b, "lora_b")):
        rows, cols = t.shape[1:]
        if S and (t.stride(2) != 1 or t.stride(1) != cols or t.data_ptr() % 16
                  or (S > 1 and (t.stride(0) % 8 or t.stride(0) < rows * cols))):
            raise ValueError(f"{nm}'s slots must be contiguous and 16-byte aligned (they are not copied)")
    if lora_scale.dtype != torch.float32 or lora_scale.shape != (S,) or not (lora_scale.is_contiguous() or S < 2):
        raise ValueError(f"lora_scale must be float32 {[S]} contiguous, got {lora_scale.dtype} {list(lora_scale.shape)}")
    if ids.dtype != torch.int32 or ids.numel() != M or ids.shape not in ((M,), x.shape[:-1]):
        raise ValueError(f"ids must be int32 {[M]}, got {ids.dtype} {list(ids.shape)}")
    return M, P, R


def _check_gates(gates, N):
    """gates' parameters beside a product with N columns."""
    a_log, dt_bias, col = gates["A_log"], gates["dt_bias"], int(gates["gate_col"])
    if not (a_log.dtype.is_floating_point and dt_bias.dtype.is_floating_point):
        raise TypeError(f"A_log and dt_bias must be floating point, got {a_log.dtype} and {dt_bias.dtype}")
    Hv = a_log.numel()
    if Hv < 1 or dt_bias.numel() != Hv or not 0 <= col <= N - 2 * Hv:
        raise ValueError(f"A_log and dt_bias must have as many values, their columns within the product's {N}, got {Hv} and "
                         f"{dt_bias.numel()} from column {col}")
    return a_log, dt_bias


def _lora_shrink(idx, rows, stride, x_scale, lora_a, lora_scale, ids, M, K, P, R, x8=None, x8_scale=None):
    """(v [M, P, 2, R] of the rows with an adapter, the adapters of their groups of 16 and, of few
    rows, their order); x8 and its scales [M, K / 128] take quantize_fp8 of the rows."""
    v = torch.empty(M, P * 2 * R, dtype=torch.bfloat16, device=rows.device)
    groups = torch.empty(-(-M // 16) + (2 * M if M <= LORA_SORT else 0), dtype=torch.int32, device=rows.device)
    xs = (0, 0, 0) if x_scale is None else (x_scale.data_ptr(), *x_scale.stride())
    to = (0, K, 0, 0, 0) if x8 is None else (x8.data_ptr(), K, x8_scale.data_ptr(), *x8_scale.stride())
    _call_on(idx, "gdn_lora_shrink", rows.data_ptr(), int(x_scale is None), stride, *xs, lora_a.data_ptr(),
             lora_a.stride(0), lora_scale.data_ptr(), ids.data_ptr(), lora_a.shape[0], P, R, M, K, v.data_ptr(), 2 * P * R,
             groups.data_ptr(), *to)
    return v, groups


def _tables(outs, widths, slices):
    """The GEMMs' part and slice tables."""
    n, ends = len(widths), [sum(widths[:i + 1]) for i in range(len(widths))]
    return ((ctypes.c_void_p * n)(*[t.data_ptr() for t in outs]),
            (ctypes.c_int64 * n)(*[max(t.stride(0), w) for t, w in zip(outs, widths)]), (ctypes.c_int * n)(*ends),
            (ctypes.c_int * len(slices))(*[sum(slices[:i + 1]) for i in range(len(slices))]))


def _gemm_bf16_lora(idx, rows, stride, weight, outs, widths, slices, first, col, shrunk, lora_b, ids, gates=None):
    """The bf16 product and the adapters' part into outs: its columns are lora_b's from `col` on, its
    slices v's from `first` on.  With gates, (g, beta)."""
    v, groups = shrunk
    M, (N, K) = v.shape[0], weight.shape
    R = lora_b.shape[2]
    c, ld, ends, slice_ends = _tables(outs, widths, slices)
    g = beta = a_log = dt_bias = None
    gate_col = Hv = 0
    if gates is not None:
        a_log, dt_bias = gates["A_log"], gates["dt_bias"]
        if a_log.dtype != dt_bias.dtype or a_log.dtype not in (torch.bfloat16, torch.float32):
            a_log, dt_bias = a_log.float(), dt_bias.float()
        a_log, dt_bias = a_log.contiguous(), dt_bias.contiguous()
        Hv, gate_col = a_log.numel(), int(gates["gate_col"])
        g = torch.empty(M, Hv, dtype=torch.float32, device=v.device)
        beta = torch.empty(M, Hv, dtype=torch.bfloat16, device=v.device)
    with torch.cuda.device(idx):
        _lib.call("gdn_gemm_bf16_lora", rows.data_ptr(), stride, weight.data_ptr(), weight.stride(0), M, N, K, len(widths),
                  c, ld, ends, _lib.ptr(g), _lib.ptr(beta), _lib.ptr(a_log), _lib.ptr(dt_bias),
                  int(a_log is not None and a_log.dtype == torch.float32), gate_col, Hv, v.data_ptr() + 4 * first * R,
                  v.stride(0), groups.data_ptr(), lora_b.data_ptr() + 2 * col * R, lora_b.stride(0), ids.data_ptr(), lora_b.shape[0], R,
                  len(slices), slice_ends, _lib.stream_of(idx))
    return g, beta


def _weight_rows(w: torch.Tensor, align: int) -> torch.Tensor:
    """A weight [N, K] whose rows the kernels read in 16-byte pieces."""
    if w.stride(1) != 1 or w.stride(0) % align or w.stride(0) < w.shape[1] or w.data_ptr() % 16:
        w = w.contiguous() if not w.is_contiguous() else w.clone(memory_format=torch.contiguous_format)
    return w


def linear_lora(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                lora_scale: torch.Tensor, ids: torch.Tensor, widths: list[int] | None = None,
                gates: dict | None = None):
    """linear(x, weight) with a low-rank adapter for each row beside the shared weight:
    y[m] = x[m] W^T + lora_scale[s] * (x[m] A_s^T) B_s^T, s = ids[m]; a row whose s is
    outside of 0 .. slots - 1 has no adapter.  x [..., K] bf16, weight [N, K] bf16 (K in
    steps of 64); ids int32, one per row, in any order.

    widths: y comes as len(widths) (1-4) contiguous tensors (as linear_cols), each part a
    projection of its own with an A of its own; None is one part.  lora_a [slots,
    parts * R, K] and lora_b [slots, N, R] bf16 (R a multiple of 8 up to 256), lora_scale
    [slots] fp32: a LoraPool's.  gates: as linear_cols; they are of the adapted columns.

    fp32 accumulation of both, one rounding; x A_s^T is held to 2^-16 in between.  A row's
    result does not depend on the adapters of the others, whatever these hold (an infinity in
    its own makes it infinite or NaN).  Two launches; x, weight, one slot of the adapters and the
    shrunk rows (4 parts R bytes each) below 2 GiB.  Returns [..., N], or the list of
    parts, with gates (that, g, beta)."""
    if gates is None:
        y = _lib.quick().linear_lora(x, weight, lora_a, lora_b, lora_scale, ids, widths)
        if y is not None:
            return y
    parts = [weight.shape[0]] if widths is None else list(widths)
    if weight.dim() != 2:
        raise ValueError(f"weight must be [N, K], got {list(weight.shape)}")
    N, K = weight.shape
    _bf16(x, "x")
    _bf16(weight, "weight")
    if K == 0 or K % 64 or x.shape[-1] != K:
        raise ValueError(f"x [..., {x.shape[-1]}] and weight [{N}, {K}]: equal last dims, a positive multiple of 64")
    M, P, R = _lora_check(x, N, K, parts, lora_a, lora_b, lora_scale, ids)
    idx = _device_of(x, weight, lora_a, lora_b, lora_scale, ids, *(() if gates is None else _check_gates(gates, N)))
    rows, _, stride = _rows_of(x, 8)
    weight, ids = _weight_rows(weight, 8), ids.contiguous()
    outs = [torch.empty(M, w, dtype=torch.bfloat16, device=x.device) for w in parts]
    shrunk = _lora_shrink(idx, rows, stride, None, lora_a, lora_scale, ids, M, K, P, R)
    g, beta = _gemm_bf16_lora(idx, rows, stride, weight, outs, parts, parts, 0, 0, shrunk, lora_b, ids, gates)
    y = [t.view(*x.shape[:-1], t.shape[1]) for t in outs]
    y = y[0] if widths is None else y
    return y if gates is None else (y, g, beta)


def linear_fp8_lora(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, lora_a: torch.Tensor,
                    lora_b: torch.Tensor, lora_scale: torch.Tensor, ids: torch.Tensor,
                    x_scale: torch.Tensor | None = None, widths: list[int] | None = None,
                    wide: torch.Tensor | None = None, gates: dict | None = None):
    """linear_fp8(x, weight, weight_scale) with a low-rank adapter for each row, as
    linear_lora: the shared weight in e4m3 with its block scales, the adapters in bf16.  x
    [..., K] bf16 is quantized for the shared weight (quantize_fp8) and read as it is by
    the adapters; e4m3 with its x_scale both read as the values it stands for.

    wide: a bf16 weight [N2, K] (N2 and N multiples of 16) whose product with the bf16 x
    follows as the last columns, a boundary of widths at N; the adapters' columns then go
    on over these (lora_b [slots, N + N2, R]).  gates: of the wide columns (gate_col
    counted from N).  Returns as linear_lora."""
    if wide is None and gates is None:
        y = _lib.quick().linear_fp8_lora(x, weight, weight_scale, lora_a, lora_b, lora_scale, ids, x_scale, widths)
        if y is not None:
            return y
    M, N, K = _check_fp8(x, weight, weight_scale, x_scale)
    total = N
    if wide is not None:
        if wide.dtype != torch.bfloat16 or x.dtype != torch.bfloat16:
            raise TypeError(f"wide and x must be bfloat16, got {wide.dtype} and {x.dtype}")
        if wide.dim() != 2 or wide.shape[1] != K or wide.shape[0] % 16 or wide.shape[0] == 0 or N % 16:
            raise ValueError(f"wide must be [N2, {K}] with N2 and N = {N} positive multiples of 16, got "
                             f"{list(wide.shape)}")
        total += wide.shape[0]
    elif gates is not None:
        raise ValueError("gates are of the wide columns")
    parts = [total] if widths is None else list(widths)
    M, P, R = _lora_check(x, total, K, parts, lora_a, lora_b, lora_scale, ids)
    narrow = [i for i in range(1, P + 1) if sum(parts[:i]) == N]
    if not narrow:
        raise ValueError(f"widths {parts}: a boundary at {N}")
    n = narrow[0]
    idx = _device_of(x, weight, weight_scale, x_scale, wide, lora_a, lora_b, lora_scale, ids,
                     *(() if gates is None else _check_gates(gates, total - N)))
    rows, _, stride = _rows_of(x, 8 if x_scale is None else 16)
    weight, ids = _weight_rows(weight, 16), ids.contiguous()
    G = K // FP8_GROUP
    if not weight_scale.is_contiguous():
        weight_scale = weight_scale.contiguous()
    outs = [torch.empty(M, w, dtype=torch.bfloat16, device=x.device) for w in parts]
    x8, x8_stride, xs = rows, stride, x_scale
    if x_scale is None:
        x8 = torch.empty(M, K, dtype=FP8, device=x.device)
        xs, x8_stride = _fp8_scales(M, G, x.device), K
        shrunk = _lora_shrink(idx, rows, stride, None, lora_a, lora_scale, ids, M, K, P, R, x8, xs)
    else:
        shrunk = _lora_shrink(idx, rows, stride, x_scale, lora_a, lora_scale, ids, M, K, P, R)
    v, groups = shrunk
    c, ld, ends, slice_ends = _tables(outs[:n], parts[:n], parts[:n])
    with torch.cuda.device(idx):
        _lib.call("gdn_gemm_fp8_lora", x8.data_ptr(), x8_stride, xs.data_ptr(), *xs.stride(), weight.data_ptr(),
                  weight.stride(0), weight_scale.data_ptr(), G, M, N, K, n, c, ld, ends, v.data_ptr(), v.stride(0),
                  groups.data_ptr(), lora_b.data_ptr(), lora_b.stride(0), ids.data_ptr(), lora_b.shape[0], R, n, slice_ends,
                  _lib.stream_of(idx))
    g = beta = None
    if wide is not None:
        g, beta = _gemm_bf16_lora(idx, rows, stride, _weight_rows(wide, 8), outs[n:], parts[n:], parts[n:], n, N, shrunk,
                                  lora_b, ids, gates)
    y = [t.view(*x.shape[:-1], t.shape[1]) for t in outs]
    y = y[0] if widths is None else y
    return y if gates is None else (y, g, beta)


# ----------------------------------------------------- norms around blocks --
NORM_MAX_COLUMNS = 16384


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float, *,
                 post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, gate_sigmoid: bool = False,
                 scale: float = 1.0, offset: float = 1.0, residual_out: torch.Tensor | None = None):
    """The seam between two blocks: the residual stream takes a block's output x, and the
    next block reads its RMSNorm.  Over the last dim, in fp32:

      h = x; with post_weight, the block's own norm: h rsqrt(mean(h^2) + eps) (offset +
      post_weight); with gate, h * gate (gate_sigmoid: h * sigmoid(gate));
      r = residual + scale * h;  y = r rsqrt(mean(r^2) + eps) (offset + weight)

    x [..., H] bf16; residual like x in bf16 or fp32, or None (the stream begins: r is
    scale * h); weight, post_weight [H] bf16 or fp32, held as their distance from 1 with
    offset = 1 (the reference's), as they are with offset = 0; gate bf16 or fp32: [..., 1]
    (per row), [H] (per column) or like x.  H up to 16384.

    Returns (y bf16, r in the residual's type, bf16 without one).  y is formed before r is
    rounded.  r goes into residual_out where that is given (contiguous, r's type; it may be
    an input of its shape and type, the residual as a rule, and overlaps none otherwise); where r is x (no residual, nothing else either), it is x that is
    returned.
    Reference: _gemma_rms_forward, _gemma_add_rms_forward,
    nanovllm/models/qwen3_5.py:99-118 (x and residual alone)."""
    if residual_out is None:
        out = _lib.quick().add_norm(x, residual, weight, eps, post_weight, gate, gate_sigmoid, scale, offset, True, False)
        if out is not None:
            return out[0], out[3]
    y, _, _, r = _add_rms_norm(x, residual, weight, eps, post_weight, gate, gate_sigmoid, scale, offset, residual_out,
                               True, False)
    return y, r


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float, *,
                     post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                     gate_sigmoid: bool = False, scale: float = 1.0, offset: float = 1.0,
                     residual_out: torch.Tensor | None = None, keep: bool = False):
    """add_rms_norm with y in e4m3 for an 8-bit projection: quantize_fp8's groups of 128
    of the fp32 values, rounded once (H a multiple of 128).  Returns (y8 [..., H], its
    scales [rows, H / 128], r), with keep also the bf16 y (for what reads the same rows in
    bf16: the layer's gate projections)."""
    out = None
    if residual_out is None:
        out = _lib.quick().add_norm(x, residual, weight, eps, post_weight, gate, gate_sigmoid, scale, offset, bool(keep), True)
    y, y8, y_scale, r = out or _add_rms_norm(x, residual, weight, eps, post_weight, gate, gate_sigmoid, scale, offset,
                                             residual_out, keep, True)
    return (y8, y_scale, r, y) if keep else (y8, y_scale, r)


def _add_rms_norm(x, residual, weight, eps, post_weight, gate, gate_sigmoid, scale, offset, residual_out, bf16, fp8):
    idx = _device_of(x, residual, weight, post_weight, gate, residual_out)
    _bf16(x, "x")
    if x.dim() < 1:
        raise ValueError("x must be [..., H]")
    H = x.shape[-1]
    if not 1 <= H <= NORM_MAX_COLUMNS or (fp8 and H % FP8_GROUP):
        raise ValueError(f"rows of 1 to {NORM_MAX_COLUMNS} columns" + (f" in multiples of {FP8_GROUP}" if fp8 else "")
                         + f", got {H}")
    floats = (torch.bfloat16, torch.float32)
    for t, nm in ((residual, "residual"), (weight, "weight"), (post_weight, "post_weight"), (gate, "gate")):
        if t is not None and t.dtype not in floats:
            raise TypeError(f"{nm} must be bfloat16 or float32, got {t.dtype}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual must be {list(x.shape)}, got {list(residual.shape)}")
    if post_weight is not None and post_weight.dtype != weight.dtype:
        weight, post_weight = weight.float(), post_weight.float()
    for t, nm in ((weight, "weight"), (post_weight, "post_weight")):
        if t is not None and t.shape != (H,):
            raise ValueError(f"{nm} must be [{H}], got {list(t.shape)}")
    weight = weight.contiguous()
    post_weight = None if post_weight is None else post_weight.contiguous()
    M = x.numel() // H

    def rows(t):
        """[..., H] as rows with dense columns, and their stride."""
        if t.is_contiguous():
            return t, H
        t = t.reshape(-1, H)
        return (t, t.stride(0)) if (t.stride(1) == 1 or H == 1) and (t.stride(0) >= H or M < 2) else (t.contiguous(), H)

    x2, sx = rows(x)
    r2, sr = (None, 0) if residual is None else rows(residual)
    g_row = g_col = 0
    if gate is not None:
        if gate.shape == (*x.shape[:-1], 1) and H > 1:
            gate = gate.reshape(-1)
            g_row = gate.stride(0) if gate.numel() > 1 else 0
        elif gate.shape == x.shape:
            gate, g_row = rows(gate)
            g_col = 1
        elif gate.shape == (H,):
            gate, g_col = gate.contiguous(), 1
        else:
            raise ValueError(f"gate must be {[*x.shape[:-1], 1]}, {[H]} or {list(x.shape)}, got {list(gate.shape)}")
    kind = torch.bfloat16 if residual is None else residual.dtype
    same = residual is None and post_weight is None and gate is None and scale == 1.0   # r is x
    if residual_out is not None:
        r = residual_out
        if r.dtype != kind or r.shape != x.shape or not r.is_contiguous():
            raise ValueError(f"residual_out must be {kind} {list(x.shape)} contiguous, got {r.dtype} {list(r.shape)}")
    else:
        r = x if same else torch.empty(x.shape, dtype=kind, device=x.device)
    written = residual_out is not None or not same
    y = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device) if bf16 else None
    y8 = y_scale = None
    if fp8:
        # (the rows that the kernel reads in whole pieces)
        x2, sx = _pieces(x2, sx, H, 8)
        if r2 is not None:
            r2, sr = _pieces(r2, sr, H, 8)
        if gate is not None and g_col:
            gate, g_row = _pieces(gate, g_row, H, 8)
        weight = weight if weight.data_ptr() % 16 == 0 else weight.clone()
        if post_weight is not None and post_weight.data_ptr() % 16:
            post_weight = post_weight.clone()
        if written and r.data_ptr() % 16:
            raise ValueError("residual_out must be 16-byte aligned")
        y8 = torch.empty(x.shape, dtype=FP8, device=x.device)
        y_scale = _fp8_scales(M, H // FP8_GROUP, x.device)
    if residual_out is not None and M:
        _check_in_place(r, M, H, (x2, sx, H, "x"), (r2, sr, H, "residual"), (gate, g_row, H if g_col else 1, "gate"),
                        (weight, None, H, "weight"), (post_weight, None, H, "post_weight"))
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    f32 = lambda t: int(t is not None and t.dtype == torch.float32)  # noqa: E731
    _call_on(idx, "gdn_add_rms_norm", x2.data_ptr(), sx, ptr(r2), sr, int(kind == torch.float32), weight.data_ptr(),
             ptr(post_weight), f32(weight), float(offset), ptr(gate), f32(gate), g_row, g_col, int(bool(gate_sigmoid)),
             float(scale), float(eps), r.data_ptr() if written else 0, ptr(y), ptr(y8), ptr(y_scale), 1, max(M, 1), M, H)
    return y, y8, y_scale, r


def _check_in_place(r, M, H, *read):
    """read: (tensor, stride of its M rows, their columns, name) of what a norm's call reads; stride None: one row for all,
    read behind the store.  A row is read and then written by the same threads: r may lie where rows like its own do, value
    for value, and apart from all else."""
    size, at = r.element_size(), r.data_ptr()
    for t, stride, cols, name in read:
        if t is None:
            continue
        begin, n = t.data_ptr(), t.element_size()
        if begin < at + M * H * size and at < begin + ((M - 1) * (stride or 0) + cols) * n:
            if begin != at or n != size or cols != H or stride is None or (M > 1 and stride != H):
                raise ValueError(f"residual_out overlaps {name} otherwise than value for value")


def _pieces(t, stride, H, align):
    """Rows that are read in 16-byte pieces (else copied), and their stride; stride 0: one row for all."""
    if t.data_ptr() % 16 or stride % align:
        t = t.contiguous() if not t.is_contiguous() else t.clone(memory_format=torch.contiguous_format)
        return t, H if stride else 0
    return t, stride


# -------------------------------------------------------------- gated norm --
def rms_norm_gated(hidden_states: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor,
                   eps: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """y = bf16(float(bf16(w * bf16(x * rsqrt(mean(x^2) + eps)))) * silu(float(z)))
    over the last dim.  hidden_states / gate [..., H, D] bf16 (head dim
    contiguous, rows of a token contiguous).  out: a contiguous bf16 tensor of as
    many elements that takes the result.
    Reference: _rms_gated_forward, nanovllm/models/qwen3_5.py:121-131."""
    dev = _check_cuda(hidden_states, gate, weight)
    _bf16(hidden_states, "hidden_states")
    _bf16(gate, "gate")
    D = hidden_states.shape[-1]
    assert hidden_states.dim() >= 2 and gate.shape == hidden_states.shape
    w = weight.to(torch.bfloat16).contiguous()
    assert w.numel() == D
    H = hidden_states.shape[-2]
    x2 = hidden_states.reshape(-1, H, D)
    z2 = gate.reshape(-1, H, D)
    if x2.stride(2) != 1 or x2.stride(1) != D:
        x2 = x2.contiguous()
    if z2.stride(2) != 1 or z2.stride(1) != D:
        z2 = z2.contiguous()
    n_tok, H, _ = x2.shape
    if out is None:
        y = torch.empty(n_tok, H, D, dtype=hidden_states.dtype, device=hidden_states.device)
    else:
        y = _out(out, n_tok * H * D, dev)
    _lib.call("gdn_rmsnorm_gated", _lib.ptr(x2), x2.stride(0), _lib.ptr(z2), z2.stride(0), _lib.ptr(w),
              _lib.ptr(y), n_tok, H, D, float(eps), _stream(dev))
    return y.view(hidden_states.shape)


def rms_norm_gated_ranges(hidden_states: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor, eps: float,
                          out: torch.Tensor, ranges: torch.Tensor, n_sel_tok: int) -> None:
    """rms_norm_gated on the tokens of some ranges only, into `out` (the same
    arithmetic, rows at the tokens' positions).  hidden_states / gate / out
    [N, H, D] bf16 with head-contiguous rows; ranges int64 [3 * n] on the
    device: (first token, token count, selected tokens before it)."""
    dev = _check_cuda(hidden_states, gate, weight, out, ranges)
    _bf16(hidden_states, "hidden_states")
    _bf16(gate, "gate")
    N, H, D = hidden_states.shape
    assert gate.shape == hidden_states.shape and out.shape == hidden_states.shape and out.is_contiguous()
    assert hidden_states.stride(2) == 1 and hidden_states.stride(1) == D
    assert gate.stride(2) == 1 and gate.stride(1) == D
    w = weight.to(torch.bfloat16).contiguous()
    _lib.call("gdn_rmsnorm_gated_ranges", _lib.ptr(hidden_states), hidden_states.stride(0), _lib.ptr(gate),
              gate.stride(0), _lib.ptr(w), _lib.ptr(out), N, _lib.ptr(ranges), ranges.numel() // 3, n_sel_tok, H,
              D, float(eps), _stream(dev))


def _token_heads(t: torch.Tensor, H: int, D: int):
    """[..., H, D] as tokens with dense heads that the kernel reads in 16-byte pieces
    (else copied once), and their stride."""
    if t.is_contiguous():
        return (t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)), H * D
    t = t.reshape(-1, H, D)
    st = t.stride()
    if st[2] != 1 or st[1] != D or st[0] % 8 or t.data_ptr() % 16:
        return t.contiguous() if not t.is_contiguous() else t.clone(memory_format=torch.contiguous_format), H * D
    return t, st[0]


def rms_norm_gated_fp8(hidden_states: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor, eps: float):
    """rms_norm_gated written in e4m3 for an 8-bit out projection: y = x * rsqrt(mean(x^2)
    + eps) * w * silu(z) in fp32 over the last dim, then quantize_fp8's groups of 128
    over a token's H * D columns (a multiple of 128), rounded once.  hidden_states / gate
    [..., H, D] bf16.  Returns (e4m3 [..., H, D], scales [tokens, H * D / 128] fp32)."""
    out = _lib.quick().norm_fp8(hidden_states, gate, weight, eps)
    return out if out is not None else _norm_fp8_ready(hidden_states, gate, weight, eps).launch()


def _norm_fp8_ready(hidden_states, gate, weight, eps) -> _Ready:
    """rms_norm_gated_fp8's call, checked."""
    idx = _device_of(hidden_states, gate, weight)
    _bf16(hidden_states, "hidden_states")
    _bf16(gate, "gate")
    if hidden_states.dim() < 2 or gate.shape != hidden_states.shape:
        raise ValueError(f"hidden_states and gate must be [..., H, D] alike, got {list(hidden_states.shape)} and "
                         f"{list(gate.shape)}")
    H, D = hidden_states.shape[-2:]
    if weight.dtype != torch.bfloat16 or not weight.is_contiguous() or weight.data_ptr() % 16:
        weight = weight.to(torch.bfloat16).clone(memory_format=torch.contiguous_format)
    if weight.numel() != D or H == 0 or H * D % FP8_GROUP:
        raise ValueError(f"weight must have {D} values and H * D = {H * D} be a multiple of {FP8_GROUP}")

    x, x_tok = _token_heads(hidden_states, H, D)
    z, z_tok = _token_heads(gate, H, D)
    n_tok = hidden_states.numel() // (H * D)
    y = x.new_empty(hidden_states.shape, dtype=FP8)
    scale = _fp8_scales(n_tok, H * D // FP8_GROUP, x.device)
    args = (x.data_ptr(), x_tok, z.data_ptr(), z_tok, weight.data_ptr(), y.data_ptr(), scale.data_ptr(), 1, n_tok, n_tok,
            H, D, float(eps))
    return _Ready(idx, "gdn_rmsnorm_gated_fp8", args, (y, scale), (x, z, weight))


class Qwen3_5RMSNormGated(torch.nn.Module):
    """Delta-net output norm on the value head dim, gated by silu(z).
    Reference: Qwen3_5RMSNormGated, nanovllm/models/qwen3_5.py:697-709."""

    def __init__(self, hidden_size: int, eps: float = 1e-6):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(hidden_size))
        self.eps = eps

    def forward(self, hidden_states: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
        return rms_norm_gated(hidden_states, gate, self.weight, self.eps)
