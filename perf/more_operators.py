"""Calls around the mixer's projections, each beside its plain form: the norms at a block's two ends, and low-rank
adapters of many requests beside the projections' shared weights.

  norm   the residual stream takes a block's output, scaled, gated and with a norm of its own where the model has
         them, and the next block's RMSNorm reads the sum: bf16 rows, or e4m3 rows with a scale for each 128 columns
         (and the bf16 rows beside them, for the gate projections)
  lora   y = x W^T + scale_s (x A_s^T) B_s^T with a bf16 W, s the adapter of the row; the columns are those of one
         projection or of several side by side, each with an A of its own
  lora8  the same with W in e4m3, one fp32 scale for each 128 x 128 block; x is bf16 (the product takes it in e4m3,
         quantized per row and 128 columns, the adapters as it is) or comes in e4m3 already

The geometries are those of perf/cases.py: hidden size 2048, 16 key heads and 16 or 32 value heads of 128.

  listed()               the cases by name
  draw(rng)              another case of the same ranges
  prepare(case, seed)    inputs, weights and adapters on the GPU
  run(state)             one call (own: the package's, else its plain form); returns its outputs
  work(case)             what the call cannot do without
  exact(case, seed)      the same outputs in 64 bits
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

HK = 16          # key heads
D = 128          # head dim
HIDDEN = 2048
EPS = 1e-6
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn
GROUP = 128      # values with one scale
TOP = 448.0      # largest e4m3 value
SMALLEST = 2.0 ** -126


# ------------------------------------------------------------------- cases --
# norm: M, H  rows and columns; form: what of the block's end there is
#         plain  x + residual, then the norm
#         first  no residual yet: the norm of x alone, which becomes the stream
#         post   the block's output has a norm of its own, then a scale
#         gate   a gate per row through a sigmoid, and a scale
#         layer  a gate per column
#         full   a gate per value, and the block's own norm
#       wide: the stream is fp32; e4m3: the rows are written in e4m3, and in bf16 beside them
# lora: M rows, side "in" (qkv, z, b and a side by side; qkv and z with 8-bit weights) or "out", Hv value heads,
#       R the adapters' rank, S of them loaded; seqs: the rows are so many sequences with an adapter each (0: each
#       row is a request of its own); bare: the share of requests without an adapter
# lora8: ready: x comes in e4m3 with its scales
def listed():
    return [
        # one user typing: the stream of a single decode row
        dict(name="norm_1", op="norm", M=1, H=HIDDEN, form="plain", wide=False, e4m3=False),
        # a decode batch of a model with norms at both ends of a block and a scaled branch
        dict(name="norm_201_post", op="norm", M=201, H=HIDDEN, form="post", wide=False, e4m3=False),
        # a 16,384-token prefill step
        dict(name="norm_16384", op="norm", M=16384, H=HIDDEN, form="plain", wide=False, e4m3=False),
        # the same in front of 8-bit projections, the stream kept in fp32, the branch behind a gate per row
        dict(name="norm_16384_e4m3", op="norm", M=16384, H=HIDDEN, form="gate", wide=True, e4m3=True),
        # one user's decode row through the in projection
        dict(name="lora_1", op="lora", M=1, side="in", Hv=32, R=16, S=8, seqs=0, bare=0.0),
        # a decode batch, nearly every request with an adapter of its own, through the in projection
        dict(name="lora_64", op="lora", M=64, side="in", Hv=32, R=16, S=64, seqs=0, bare=0.1),
        # a prefill step of eight prompts through the in projection
        dict(name="lora_16384", op="lora", M=16384, side="in", Hv=32, R=16, S=8, seqs=8, bare=0.1),
        # a ragged prefill step through the out projection, larger adapters
        dict(name="lora_17001_out", op="lora", M=17001, side="out", Hv=16, R=64, S=12, seqs=21, bare=0.2),
        # a lightly loaded server's out projection on what the gated norm wrote in 8 bits
        dict(name="lora8_37_out", op="lora8", M=37, side="out", Hv=32, R=16, S=16, seqs=0, bare=0.1, ready=True),
        # a decode batch through the 8-bit in projection, from bf16 rows
        dict(name="lora8_200", op="lora8", M=200, side="in", Hv=32, R=32, S=32, seqs=0, bare=0.1, ready=False),
        # a prefill step through the 8-bit in projection
        dict(name="lora8_16384", op="lora8", M=16384, side="in", Hv=32, R=32, S=8, seqs=8, bare=0.1, ready=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Norms of 1 to 16,384 rows of 64 to 8192 columns (odd widths among them) in every form; projections of 1 to
    16,384 rows with adapters of rank 8 to 128, 1 to 64 of them, by request and by sequence."""
    op = rng.choice(["norm", "norm", "lora", "lora", "lora8"])
    if op == "norm":
        e4m3 = rng.random() < 0.4
        H = rng.choice([HIDDEN, HIDDEN, 2 * HIDDEN, GROUP * _log_int(rng, 1, 64)] if e4m3 else
                       [HIDDEN, HIDDEN, 2 * HIDDEN, 8 * _log_int(rng, 8, 1024), _log_int(rng, 64, 4999)])
        return dict(op=op, M=_log_int(rng, 1, min(16384, (1 << 26) // H)), H=H,
                    form=rng.choice(["plain", "plain", "first", "post", "gate", "layer", "full"]),
                    wide=rng.random() < 0.4, e4m3=e4m3)
    case = dict(op=op, M=0, side=rng.choice(["in", "out"]), Hv=rng.choice([16, 32]),
                R=rng.choice([8, 16, 16, 24, 32, 64, 128]), S=_log_int(rng, 1, 64))
    N, K, P = sum(_widths(case)), _inner(case), len(_widths(case))
    # (the plain form multiplies with all adapters: no more than the largest listed case takes)
    most = 16384 * 12352 * HIDDEN // (N * K + case["S"] * case["R"] * (P * K + N))
    M = _log_int(rng, 1, min(16384, most))
    case.update(M=M, seqs=0 if M <= 256 and rng.random() < 0.7 else _log_int(rng, 1, max(1, min(64, M // 16))),
                bare=rng.choice([0.0, 0.1, 0.5]))
    return case if op == "lora" else dict(case, ready=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs --
class _Random:
    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.gen = torch.Generator(device=self.dev).manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=BF16):
        t = torch.randn(*shape, generator=self.gen, device=self.dev)
        return (t.mul_(std) if std != 1.0 else t).to(dtype)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=self.gen, device=self.dev).mul_(hi - lo).add_(lo)

    def below(self, n, *shape):
        return torch.randint(0, n, shape, generator=self.gen, device=self.dev)


def _stream(r, M, K):
    """Rows as a residual stream has them: a few columns are twenty times the others, and rows differ in size."""
    loud = torch.where(r.uniform(K) < 0.01, 20.0, 1.0)
    return r.normal(M, K, dtype=F32) * loud * r.uniform(M, 1, lo=-2.0, hi=2.0).exp()


def _norm_state(r, case):
    M, H, form = case["M"], case["H"], case["form"]
    st = {"op": "norm", "e4m3": case["e4m3"], "weight": r.normal(H, std=0.1), "x": r.normal(M, H), "residual": None,
          "post_weight": None, "gate": None, "gate_sigmoid": False, "scale": 1.0}
    stream = _stream(r, M, H).to(F32 if case["wide"] else BF16)
    if form == "first":
        st["x"] = stream.to(BF16)
        return st
    st["residual"] = stream
    if form in ("post", "full"):
        st["post_weight"] = r.normal(H, std=0.1)
    if form == "post":
        st["scale"] = 0.22
    if form == "gate":
        st.update(gate=r.normal(M, 1), gate_sigmoid=True, scale=0.5)
    if form == "layer":
        st["gate"] = r.normal(H, std=0.3)
    if form == "full":
        st["gate"] = r.normal(M, H)
    return st


def _widths(case):
    """The columns of the projections that lie side by side."""
    Hv = case["Hv"]
    if case["side"] == "out":
        return [HIDDEN]
    both = [(2 * HK + Hv) * D, Hv * D]
    return both if case["op"] == "lora8" else both + [Hv, Hv]


def _inner(case):
    return HIDDEN if case["side"] == "in" else case["Hv"] * D


def _requests(r, case):
    """The adapter of each row, -1 for none, int32 [M]."""
    M, S, seqs = case["M"], case["S"], case["seqs"]
    n = seqs or M
    ids = torch.where(r.uniform(n) < case["bare"], -1, r.below(S, n))
    if seqs:
        cuts = (r.uniform(M) * 1e6).argsort()[:seqs - 1]        # sequences of all lengths
        ids = ids[torch.zeros(M, dtype=torch.int64, device=r.dev).index_fill_(0, cuts, 1).cumsum(0).clamp(max=n - 1)]
    return ids.to(torch.int32).contiguous()


def _lora_state(r, case):
    M, R, S = case["M"], case["R"], case["S"]
    widths, K = _widths(case), _inner(case)
    N = sum(widths)
    st = {"op": case["op"], "widths": widths, "ids": _requests(r, case), "x_scale": None, "w_scale": None,
          "a": r.normal(S, len(widths) * R, K, std=K ** -0.5),      # every projection's A, one after the other
          "b": r.normal(S, N, R, std=0.5 * R ** -0.5),              # and the B of its columns
          "scale": r.uniform(S, lo=0.25, hi=2.0)}
    w = r.normal(N, K, std=K ** -0.5, dtype=F32) * r.uniform(N, 1, lo=-0.7, hi=0.7).exp()
    if case["op"] == "lora":
        return dict(st, x=r.normal(M, K), w=w.to(BF16))
    st["w"], st["w_scale"] = _to_e4m3_blocks(w)
    st["x"] = _stream(r, M, K).to(BF16)
    if case["ready"]:
        x8, xs = _to_e4m3_rows(st["x"].float())
        # the scales of one group of columns side by side, as the package's own calls write them
        st["x"], st["x_scale"] = x8, xs.t().contiguous().t()
    return st


def prepare(case, seed):
    r = _Random(seed)
    return _norm_state(r, case) if case["op"] == "norm" else _lora_state(r, case)


# -------------------------------------------------------------------- calls --
def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _ops():
    return importlib.import_module("nano-vllm-extend_amd").ops


def _own_norm(s):
    how = dict(post_weight=s["post_weight"], gate=s["gate"], gate_sigmoid=s["gate_sigmoid"], scale=s["scale"])
    if s["e4m3"]:
        return _ops().add_rms_norm_fp8(s["x"], s["residual"], s["weight"], EPS, keep=True, **how)
    return _ops().add_rms_norm(s["x"], s["residual"], s["weight"], EPS, **how)


def _own_lora(s):
    return _ops().linear_lora(s["x"], s["w"], s["a"], s["b"], s["scale"], s["ids"], widths=s["widths"])


def _own_lora8(s):
    return _ops().linear_fp8_lora(s["x"], s["w"], s["w_scale"], s["a"], s["b"], s["scale"], s["ids"],
                                  x_scale=s["x_scale"], widths=s["widths"])


# -------------------------------------------------------------- plain forms --
def _scales(top):
    """The scale of a group whose largest magnitude is `top`, and its reciprocal, both fp32."""
    scale = (top * (1.0 / TOP)).clamp(min=SMALLEST)
    return scale, torch.reciprocal(scale)


def _to_e4m3_rows(x):
    """x [M, K] fp32 -> e4m3 [M, K] and the scales [M, K / 128]."""
    groups = x.unflatten(-1, (-1, GROUP))
    scale, inv = _scales(groups.abs().amax(-1))
    return (groups * inv[..., None]).to(E4M3).flatten(-2), scale


def _to_e4m3_blocks(w):
    """w [N, K] fp32 -> e4m3 [N, K] and the scales [ceil(N / 128), K / 128]."""
    N, K = w.shape
    rows = -(-N // GROUP)
    padded = torch.nn.functional.pad(w, (0, 0, 0, rows * GROUP - N))
    scale, inv = _scales(padded.view(rows, GROUP, K // GROUP, GROUP).abs().amax((1, 3)))
    return (w * _spread(inv, N)).to(E4M3), scale


def _spread(scale, N):
    """Block scales [ceil(N / 128), K / 128] -> one for each weight, [N, K]."""
    return scale.repeat_interleave(GROUP, 0)[:N].repeat_interleave(GROUP, 1)


def _unit(t):
    return t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt()


def _plain_norm(s):
    h = s["x"].float()
    if s["post_weight"] is not None:
        h = _unit(h) * (1 + s["post_weight"].float())
    if s["gate"] is not None:
        g = s["gate"].float()
        h = h * (1 / (1 + (-g).exp()) if s["gate_sigmoid"] else g)
    if s["scale"] != 1.0:
        h = h * s["scale"]
    stream, kind = h, BF16
    if s["residual"] is not None:
        stream, kind = s["residual"].float() + h, s["residual"].dtype
    y = _unit(stream) * (1 + s["weight"].float())
    if not s["e4m3"]:
        return y.to(BF16), stream.to(kind)
    y8, scale = _to_e4m3_rows(y)
    return y8, scale, stream.to(kind), y.to(BF16)


def _plain_delta(x, s):
    """scale (x A^T) B^T of every row's adapter, x [M, K] fp32: all adapters' A at once, the others' values 0."""
    a, b, ids, widths = s["a"].float(), s["b"].float(), s["ids"], s["widths"]
    S, N, R = b.shape
    M = len(x)
    mine = (ids[:, None] == torch.arange(S, device=x.device)).float() * s["scale"]              # [M, S]
    v = (x @ a.flatten(0, 1).t()).view(M, S, len(widths), R) * mine[:, :, None, None]
    return torch.cat([v[:, :, p].reshape(M, S * R) @ bp.transpose(0, 1).reshape(-1, S * R).t()
                      for p, bp in enumerate(b.split(widths, 1))], 1)


def _plain_lora(s):
    x = s["x"].float()
    y = x @ s["w"].float().t() + _plain_delta(x, s)
    return [t.contiguous() for t in y.to(BF16).split(s["widths"], 1)]


def _plain_lora8(s):
    x, xs = s["x"], s["x_scale"]
    rows = x.float()
    if xs is None:
        x, xs = _to_e4m3_rows(rows)
        seen = rows
    quant = (x.float().unflatten(-1, (-1, GROUP)) * xs[..., None]).flatten(-2)
    if s["x_scale"] is not None:
        seen = quant
    y = quant @ (s["w"].float() * _spread(s["w_scale"], s["w"].shape[0])).t() + _plain_delta(seen, s)
    return [t.contiguous() for t in y.to(BF16).split(s["widths"], 1)]


_own = {"norm": _own_norm, "lora": _own_lora, "lora8": _own_lora8}
_plain = {"norm": _plain_norm, "lora": _plain_lora, "lora8": _plain_lora8}


# --------------------------------------------------------------- the yards --
def work(case):
    M = case["M"]
    if case["op"] == "norm":
        n = M * case["H"]
        held = 4 if case["wide"] else 2
        rows = 2 + (2 if case["form"] == "full" else 0) + 2 + (1 + 4 / GROUP if case["e4m3"] else 0)
        stream = 0 if case["form"] == "first" else 2 * held    # (the first row is the stream as it comes)
        return {"bytes": float(n * (rows + stream) + 2 * case["H"]), "flops": 12.0 * n}
    widths, K, R = _widths(case), _inner(case), case["R"]
    N, P = sum(widths), len(widths)
    # adapters that a call meets: of S, as many as its requests name
    n = case["seqs"] or M
    met = case["S"] * (1 - (1 - (1 - case["bare"]) / case["S"]) ** n)
    small = 2.0 * met * R * (P * K + N)
    flops = 2.0 * M * N * K + 2.0 * M * (1 - case["bare"]) * R * (P * K + N)
    if case["op"] == "lora":
        return {"bytes": 2.0 * (M * K + N * K + M * N) + small, "flops": flops}
    x = M * K + 4.0 * M * K / GROUP if case["ready"] else 2.0 * M * K
    return {"bytes": x + N * K + 4.0 * -(-N // GROUP) * K / GROUP + 2.0 * M * N + small, "flops": flops}


# ----------------------------------------------------------------- 64 bits --
def _round_e4m3(t):
    """The nearest e4m3 value, ties to the even one (4 significant bits, steps of 2^-9 at least)."""
    e = torch.frexp(t)[1].clamp(min=-5) - 4
    return torch.ldexp(torch.round(torch.ldexp(t, -e)), e)


def _exact_norm(s):
    def norm(t, w):
        return t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * (1.0 + w.double())

    h = s["x"].double()
    if s["post_weight"] is not None:
        h = norm(h, s["post_weight"])
    if s["gate"] is not None:
        g = s["gate"].double()
        h = h * (torch.sigmoid(g) if s["gate_sigmoid"] else g)
    h = h * s["scale"]
    if s["residual"] is not None:
        h = h + s["residual"].double()
    y = norm(h, s["weight"])
    if not s["e4m3"]:
        return y, h
    # (no values for the e4m3 rows: which of its two neighbours a value next to a tie falls to is decided by the last
    # bits of whatever computed it)
    return None, y.reshape(len(y), -1, GROUP).abs().amax(-1) / TOP, h, y


def _exact_lora(s):
    x = s["x"].double()
    M, K = x.shape
    seen = x
    if s["w_scale"] is None:
        w = s["w"].double()
    else:
        if s["x_scale"] is None:
            # scale and value of an e4m3 operand are defined in fp32, each rounded once
            x = x.view(M, K // GROUP, GROUP)
            f32 = lambda t: t.float().double()  # noqa: E731
            scale = f32(x.abs().amax(-1) * f32(torch.tensor(1 / TOP, dtype=F64))).clamp(min=SMALLEST)
            x = (_round_e4m3(f32(x * f32(1 / scale)[..., None])) * scale[..., None]).reshape(M, K)
        else:
            x = seen = (x.view(M, K // GROUP, GROUP) * s["x_scale"].double()[..., None]).reshape(M, K)
        w = torch.cat([block.double() * scale.double().repeat_interleave(GROUP)
                       for block, scale in zip(s["w"].split(GROUP), s["w_scale"])])
    y = x @ w.t()
    R = s["b"].shape[2]
    for slot in range(len(s["a"])):
        rows = (s["ids"] == slot).nonzero()[:, 0]
        if len(rows):
            v = float(s["scale"][slot]) * (seen[rows] @ s["a"][slot].double().t())
            parts = s["b"][slot].double().split(s["widths"])
            y[rows] += torch.cat([v[:, R * p:R * p + R] @ t.t() for p, t in enumerate(parts)], 1)
    return [t.contiguous() for t in y.split(s["widths"], 1)]


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if s["op"] == "norm" else _exact_lora(s)
