"""Calls of the mixer's 8-bit projections and of its verify step over a tree of drafted tokens, each beside its plain
form.

  linear   y = x W^T with W held in e4m3 and one fp32 scale for each 128 x 128 block; x is bf16 and is brought to
           e4m3 with one scale for each row and 128 columns inside of the call, or comes that way already
  norm     the gated RMSNorm of the delta rule's output, written in e4m3 with a scale for each 128 columns (what the
           out projection above reads)
  conv     the causal conv1d + SiLU of a tree of drafted tokens: a node's taps are its ancestors' rows, then the
           conv pool's; before it, where the case says so, the path that the last step accepted goes into the pool
  rule     the gated delta rule over the same tree against the state pool, with the same accepted path before it
  commit   the accepted paths into both pools, for sequences that go on without a tree

The geometries are those of perf/cases.py: head dim 128 (64 now and then), 16 key heads with 16 or 32 value heads,
hidden size 2048; the pools hold two layers and a call works on the strided view of one.

  listed()               the cases by name
  draw(rng)              another case of the same ranges
  prepare(case, seed)    inputs, weights and pools on the GPU
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
HIDDEN = 2048
LAYERS = 2       # layers in a pool; the calls use the last one
EPS = 1e-6
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn
GROUP = 128      # values with one scale
TOP = 448.0      # largest e4m3 value
SMALLEST = 2.0 ** -126


# ------------------------------------------------------------------- cases --
# M, N, K  rows of x, rows of W, columns of both; ready: x comes in e4m3 with its scales
# B, T     sequences and nodes of each one's tree (unused ones included)
# back     how far behind a node its parent can be: 1 is a chain, more is a bushier tree
# ragged   trees of different sizes: the nodes past a sequence's last one are unused (parent -2)
# pending  the call begins with the path that the step before accepted
def listed():
    return [
        # one user typing: the in projection of a single decode row, bound by the weights' way in
        dict(name="linear_1", op="linear", M=1, N=12288, K=2048, ready=False),
        # a lightly loaded server's out projection, an odd number of rows
        dict(name="linear_37", op="linear", M=37, N=2048, K=4096, ready=False),
        # an engine's 16,384-token prefill step: the in projection of the grouped geometry
        dict(name="linear_16384", op="linear", M=16384, N=12288, K=2048, ready=False),
        # the out projection of a varlen prefill step, on what the gated norm wrote in 8 bits
        dict(name="linear_17001", op="linear", M=17001, N=2048, K=2048, ready=True),
        # the norm before a decode batch's out projection
        dict(name="norm_201", op="norm", M=201, Hv=32, D=128),
        # the norm of a prefill step
        dict(name="norm_16384", op="norm", M=16384, Hv=32, D=128),
        # one user's drafted tree through the conv
        dict(name="conv_1x8", op="conv", B=1, T=8, Hv=32, D=128, back=3, ragged=False, pending=True),
        # a full batch of trees, each of its own size
        dict(name="conv_64x16", op="conv", B=64, T=16, Hv=32, D=128, back=4, ragged=True, pending=True),
        # one user's first drafted tree against the state
        dict(name="rule_1x8", op="rule", B=1, T=8, Hv=32, D=128, back=3, ragged=False, pending=False),
        # a full batch in the middle of its generation: the last step's accepted paths, then the new trees
        dict(name="rule_64x16", op="rule", B=64, T=16, Hv=32, D=128, back=4, ragged=True, pending=True),
        # one sequence leaves the batch
        dict(name="commit_1x8", op="commit", B=1, T=8, Hv=32, D=128, back=3, ragged=False),
        # the whole batch goes on with plain decode steps
        dict(name="commit_64x16", op="commit", B=64, T=16, Hv=32, D=128, back=4, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Products of 1 to 16,384 rows with the layer's weights and with others of odd heights, norms of 1 to 16,384
    rows, and trees of 1 to 48 nodes (chains among them) for 1 to 64 sequences."""
    op = rng.choice(["linear", "linear", "linear", "norm", "conv", "rule", "rule", "commit"])
    if op == "linear":
        N, K = rng.choice([(12288, 2048), (8192, 2048), (2048, 2048), (2048, 4096),
                           (rng.randint(40, 9000), 128 * rng.randint(1, 40))])
        most = min(16384, 16384 * 12288 * 2048 // (N * K))
        return dict(op=op, M=_log_int(rng, 1, most), N=N, K=K, ready=rng.random() < 0.4)
    Hv, D = rng.choice([16, 32]), rng.choice([128, 128, 128, 64])
    if op == "norm":
        return dict(op=op, M=_log_int(rng, 1, 16384), Hv=Hv, D=D)
    T = _log_int(rng, 1, 48)
    B = _log_int(rng, 1, max(1, min(64, 1024 // T)))
    case = dict(op=op, B=B, T=T, Hv=Hv, D=D, back=rng.choice([1, 2, 4, 8]), ragged=rng.random() < 0.5)
    return case if op == "commit" else dict(case, pending=rng.random() < 0.6)


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


def _activations(r, M, K):
    """Rows as a residual stream has them: a few columns are twenty times the others, and rows differ in size."""
    x = r.normal(M, K, dtype=F32)
    loud = torch.where(r.uniform(K) < 0.01, 20.0, 1.0)
    return (x * loud * r.uniform(M, 1, lo=-2.0, hi=2.0).exp()).to(BF16)


def _tree(r, case):
    """parents [B, T] int32: a node's parent is up to `back` nodes before it, -1 the sequence's own state, -2 unused;
    and an accepted node of each row (-1 now and then: nothing was accepted)."""
    B, T = case["B"], case["T"]
    t = torch.arange(T, device=r.dev)
    parents = (t - 1 - r.below(case["back"], B, T)).clamp(min=0)
    parents[:, 0] = -1
    size = torch.full((B,), T, device=r.dev)
    if case["ragged"]:
        size = 1 + (r.uniform(B) * T).long().clamp(max=T - 1)
        parents = torch.where(t < size[:, None], parents, -2)
    accepted = (r.uniform(B) * size).long().clamp(max=T - 1)
    accepted = torch.where(r.uniform(B) < 0.05, -1, accepted)
    return parents.to(torch.int32).contiguous(), accepted


def _gates(r, *shape):
    """g and beta of tokens, as the gate kernel gives them."""
    Hv = shape[-1]
    A = torch.exp(r.uniform(Hv, hi=math.log(16.0)))
    g = -A * torch.nn.functional.softplus(r.normal(*shape, dtype=F32) + r.uniform(Hv, lo=-1.0))
    return g, torch.sigmoid(r.normal(*shape, dtype=F32)).to(BF16)


def _pools(r, case, C):
    B, Hv, D = case["B"], case["Hv"], case["D"]
    slots = B + 3
    return {"ids": torch.randperm(slots, generator=r.gen, device=r.dev)[:B],
            "s_cache": r.normal(slots + 1, LAYERS, Hv, D, D, std=0.1, dtype=F32)[:, LAYERS - 1],
            "conv_cache": r.normal(slots + 1, LAYERS, C, 3)[:, LAYERS - 1]}


def prepare(case, seed):
    r = _Random(seed)
    op = case["op"]
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        w = r.normal(N, K, std=K ** -0.5, dtype=F32) * r.uniform(N, 1, lo=-0.7, hi=0.7).exp()
        w8, ws = _to_e4m3_blocks(w)
        st = {"x": _activations(r, M, K), "w8": w8, "w_scale": ws, "x_scale": None}
        if case["ready"]:
            x8, xs = _to_e4m3_rows(st["x"].float())
            # the scales of one group of columns side by side, as the package's own calls write them
            st["x"], st["x_scale"] = x8, xs.t().contiguous().t()
        return dict(st, op=op)
    Hv, D = case["Hv"], case["D"]
    if op == "norm":
        M = case["M"]
        # (the delta rule's outputs are small; their rows differ in size)
        core = (r.normal(M, Hv, D, dtype=F32) * r.uniform(M, Hv, 1, lo=-5.0, hi=-1.0).exp()).to(BF16)
        return {"op": op, "core": core, "z": r.normal(M, Hv, D),
                "weight": (1 + r.normal(D, std=0.02, dtype=F32)).to(BF16)}
    B, T = case["B"], case["T"]
    C = 2 * HK * D + Hv * D
    st = dict(_pools(r, case, C), op=op, weight=r.normal(C, 4, std=0.5))
    st["parents"], _ = _tree(r, case)
    st["last_parents"], st["accepted"] = _tree(r, case)
    st["pending"] = case.get("pending", True)
    # the step before: its raw rows, its keys after the conv, its gates and its corrections
    st["last_x"] = r.normal(B, T, C)
    st["last_k"] = r.normal(B, T, HK, D)
    st["last_g"], _ = _gates(r, B, T, Hv)
    st["last_u"] = r.normal(B, T, Hv, D, std=0.5, dtype=F32)
    if op == "conv":
        st["x"] = r.normal(B, T, C)
    if op == "rule":
        y = r.normal(B, T, C)  # the conv's output, whose parts the rule reads
        st["q"], st["k"], st["v"] = (y[..., a:b].unflatten(-1, (-1, D)) for a, b in
                                     ((0, HK * D), (HK * D, 2 * HK * D), (2 * HK * D, C)))
        st["g"], st["beta"] = _gates(r, B, T, Hv)
    return st


# -------------------------------------------------------------------- calls --
def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _ops():
    return importlib.import_module("nano-vllm-extend_amd").ops


def _own_linear(s):
    return _ops().linear_fp8(s["x"], s["w8"], s["w_scale"], x_scale=s["x_scale"])


def _own_norm(s):
    return _ops().rms_norm_gated_fp8(s["core"], s["z"], s["weight"], EPS)


def _own_conv(s):
    pending = (s["last_x"], s["last_parents"], s["accepted"]) if s["pending"] else None
    y = _ops().conv_tree_step(s["x"], s["conv_cache"], s["ids"], s["weight"], s["parents"], pending=pending)
    return y, s["conv_cache"]


def _own_rule(s):
    pending = (s["last_k"], s["last_g"], s["last_u"], s["last_parents"], s["accepted"]) if s["pending"] else None
    o, u = _ops().recurrent_gdn_tree(s["q"], s["k"], s["v"], s["g"], s["beta"], s["s_cache"], s["ids"], s["parents"],
                                     pending=pending)
    return o, u, s["s_cache"]


def _own_commit(s):
    _ops().commit_tree(s["s_cache"], s["conv_cache"], s["ids"], s["last_parents"], s["accepted"], s["last_x"],
                       s["last_k"], s["last_g"], s["last_u"])
    return s["s_cache"], s["conv_cache"]


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


def _plain_linear(s):
    x, xs = s["x"], s["x_scale"]
    if xs is None:
        x, xs = _to_e4m3_rows(x.float())
    a = (x.float().unflatten(-1, (-1, GROUP)) * xs[..., None]).flatten(-2)
    w = s["w8"].float() * _spread(s["w_scale"], s["w8"].shape[0])
    return (a @ w.t()).to(BF16)


def _plain_norm(s):
    x, z = s["core"].float(), s["z"].float()
    y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["weight"].float()
    y = y * (z / (1 + (-z).exp()))
    y8, scale = _to_e4m3_rows(y.flatten(-2))
    return y8.view(x.shape), scale


def _lines(parents, dtype):
    """[B, T, T]: 1 where column s is node t or one of its ancestors; rows and columns of unused nodes are 0."""
    T = parents.shape[1]
    at = torch.arange(T, device=parents.device)
    used = parents >= -1
    eye = (at[:, None] == at) & used[:, :, None]
    line = (eye | (parents[:, :, None] == at)).to(dtype)
    for _ in range(max(1, (T - 1).bit_length())):
        line = (line @ line).clamp(max=1)
    return line


def _decay(line, g):
    """exp of the sum of g over the nodes after s down to t, [B, H, T, T], and from the start down to t, [B, H, T].
    The sums in 64 bits: they reach hundreds, and their differences matter."""
    G = (line.double() @ g.double()).transpose(1, 2)
    d = torch.where(line[:, None] > 0, (G[..., :, None] - G[..., None, :]), -math.inf)
    return d.exp().float(), G.exp().float()


def _unit(t):
    return t * (t.square().sum(-1, keepdim=True) + EPS).rsqrt()


def _heads(t, Hv):
    """[B, T, Hk, D] -> [B, Hv, T, D]"""
    return t.repeat_interleave(Hv // t.shape[2], 2).transpose(1, 2)


def _plain_advance(S, k, g, u, parents, accepted):
    """The states S [B, Hv, D, D] after the accepted nodes (S where nothing was accepted)."""
    Hv = u.shape[2]
    row = accepted.clamp(min=0)[:, None]
    line = _lines(parents, F64)
    line = line.gather(1, row[..., None].expand(-1, -1, line.shape[2]))
    total = line @ g.double()                                        # [B, 1, Hv]
    each = total - _lines(parents, F64) @ g.double()                 # [B, T, Hv]
    weight = torch.where(line.transpose(1, 2) > 0, each, -math.inf).exp().float()
    keys = _heads(_unit(k.float()), Hv) * weight.transpose(1, 2)[..., None]
    new = S * total[:, 0].exp().float()[..., None, None] + keys.transpose(-1, -2) @ u.transpose(1, 2)
    return torch.where((accepted >= 0)[:, None, None, None], new, S)


def _plain_taps(taps, x, parents, accepted):
    """The taps [B, C, 3] after the accepted nodes."""
    rows = torch.cat([taps.transpose(1, 2), x], 1)                   # a path goes back into the taps
    up = torch.cat([torch.arange(-1, 2, device=x.device).expand(len(x), 3), torch.where(parents < 0, 2, parents + 3)], 1)
    at = torch.where(accepted < 0, 2, accepted + 3)
    first = up.gather(1, at[:, None])[:, 0]
    second = up.gather(1, first[:, None])[:, 0]
    at = torch.stack([second, first, at], 1)
    return rows.gather(1, at[..., None].expand(-1, -1, rows.shape[2])).transpose(1, 2)


def _plain_conv(s):
    ids, x, parents = s["ids"], s["x"], s["parents"].long()
    taps = s["conv_cache"][ids]
    if s["pending"]:
        taps = _plain_taps(taps, s["last_x"], s["last_parents"].long(), s["accepted"])
        s["conv_cache"][ids] = taps
    B, T, C = x.shape
    rows = torch.cat([taps.transpose(1, 2), x], 1).float()
    up = torch.cat([torch.arange(-1, 2, device=x.device).expand(B, 3), torch.where(parents < 0, 2, parents + 3)], 1)
    at = torch.arange(3, T + 3, device=x.device).expand(B, T)
    w = s["weight"].float()
    y = rows.gather(1, at[..., None].expand(B, T, C)) * w[:, 3]
    for tap in (2, 1, 0):
        at = up.gather(1, at)
        y = y + rows.gather(1, at[..., None].expand(B, T, C)) * w[:, tap]
    y = y / (1 + (-y).exp())
    return torch.where((parents >= -1)[..., None], y, 0).to(BF16), s["conv_cache"]


def _plain_rule(s):
    ids, Hv, D = s["ids"], s["v"].shape[2], s["v"].shape[3]
    S = s["s_cache"][ids]
    if s["pending"]:
        S = _plain_advance(S, s["last_k"], s["last_g"], s["last_u"], s["last_parents"].long(), s["accepted"])
        s["s_cache"][ids] = S
    parents = s["parents"].long()
    T = parents.shape[1]
    line = _lines(parents, F32)
    decay, start = _decay(line, s["g"])
    q, k = (_heads(_unit(s[n].float()), Hv) for n in ("q", "k"))
    v, beta = s["v"].float().transpose(1, 2), s["beta"].float().transpose(1, 2)[..., None]
    eye = torch.eye(T, dtype=F32, device=S.device)
    kT = k.transpose(-1, -2)
    L = beta * (k @ kT) * decay * (1 - eye)
    # (1 + L)^-1 = (1 - L) (1 + L^2) (1 + L^4) ...: L is strictly lower triangular
    inverse, power = eye - L, L
    for _ in range(max(0, (T - 1).bit_length() - 1)):
        power = power @ power
        inverse = inverse @ (eye + power)
    u = inverse @ (beta * (v - start[..., None] * (k @ S)))
    o = D ** -0.5 * (start[..., None] * (q @ S) + ((q @ kT) * decay) @ u)
    used = (parents >= -1)[:, None, :, None]
    o, u = (torch.where(used, t, 0).transpose(1, 2).contiguous() for t in (o, u))
    return o.to(BF16), u, s["s_cache"]


def _plain_commit(s):
    ids, parents, accepted = s["ids"], s["last_parents"].long(), s["accepted"]
    s["s_cache"][ids] = _plain_advance(s["s_cache"][ids], s["last_k"], s["last_g"], s["last_u"], parents, accepted)
    s["conv_cache"][ids] = _plain_taps(s["conv_cache"][ids], s["last_x"], parents, accepted)
    return s["s_cache"], s["conv_cache"]


_own = {"linear": _own_linear, "norm": _own_norm, "conv": _own_conv, "rule": _own_rule, "commit": _own_commit}
_plain = {"linear": _plain_linear, "norm": _plain_norm, "conv": _plain_conv, "rule": _plain_rule,
          "commit": _plain_commit}


# --------------------------------------------------------------- the yards --
def work(case):
    op = case["op"]
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x = M * K + M * (K // GROUP) * 4 if case["ready"] else 2 * M * K
        return {"bytes": float(x + N * K + -(-N // GROUP) * (K // GROUP) * 4 + 2 * M * N), "flops": 2.0 * M * N * K}
    Hv, D = case["Hv"], case["D"]
    if op == "norm":
        n = case["M"] * Hv * D
        return {"bytes": 5.0 * n + 4 * n / GROUP, "flops": 14.0 * n}
    B, T = case["B"], case["T"]
    C = 2 * HK * D + Hv * D
    depth = -(-T // (2 * case["back"])) + 1      # of an accepted path: about half of the tree's nodes, `back` a level
    state, taps = 4.0 * B * Hv * D * D, 6.0 * B * C
    path = B * depth * (2 * HK * D + 4 * Hv * D + 4 * Hv)
    if op == "commit":
        return {"bytes": 2 * state + 2 * taps + path + 6.0 * B * C, "flops": B * Hv * D * D * (1.0 + 2 * depth)}
    if op == "conv":
        more = taps + 6.0 * B * C if case["pending"] else 0.0
        return {"bytes": 4.0 * B * T * C + 8 * C + taps + more, "flops": 12.0 * B * T * C}
    rows = B * T * (2 * C + 6 * Hv + 2 * Hv * D + 4 * Hv * D)
    flops = B * Hv * (4.0 * T * D * D + 8.0 * T * depth * D)
    if not case["pending"]:
        return {"bytes": state + rows, "flops": flops}
    return {"bytes": 2 * state + rows + path, "flops": flops + B * Hv * D * D * (1.0 + 2 * depth)}


# ----------------------------------------------------------------- 64 bits --
def _round_e4m3(t):
    """The nearest e4m3 value, ties to the even one (4 significant bits, steps of 2^-9 at least)."""
    e = torch.frexp(t)[1].clamp(min=-5) - 4
    return torch.ldexp(torch.round(torch.ldexp(t, -e)), e)


def _exact_linear(s):
    x = s["x"].double()
    M, K = x.shape
    if s["x_scale"] is None:
        # scale and value of an e4m3 operand are defined in fp32, each rounded once
        x = x.view(M, K // GROUP, GROUP)
        f32 = lambda t: t.float().double()  # noqa: E731
        scale = f32(x.abs().amax(-1) * f32(torch.tensor(1 / TOP, dtype=F64))).clamp(min=SMALLEST)
        x = _round_e4m3(f32(x * f32(1 / scale)[..., None])) * scale[..., None]
    else:
        x = x.view(M, K // GROUP, GROUP) * s["x_scale"].double()[..., None]
    y = torch.zeros(M, s["w8"].shape[0], dtype=F64, device=x.device)
    for n in range(0, y.shape[1], GROUP):
        w = s["w8"][n:n + GROUP].double().view(-1, K // GROUP, GROUP) * s["w_scale"][n // GROUP].double()[None, :, None]
        y[:, n:n + GROUP] = x.reshape(M, K) @ w.reshape(-1, K).t().contiguous()
    return y


def _exact_norm(s):
    x, z = s["core"].double(), s["z"].double()
    y = s["weight"].double() * x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * z * torch.sigmoid(z)
    # (no values for the e4m3 outputs: which of its two neighbours a value next to a tie falls to is decided by the
    # last bits of whatever computed it)
    return None, y.reshape(len(y), -1, GROUP).abs().amax(-1) / TOP


def _exact_path(parents, node):
    """The nodes from the root down to `node`."""
    path = []
    while node >= 0:
        path.insert(0, node)
        node = parents[node]
    return path


def _exact_norms(t):
    return t / (t.square().sum(-1, keepdim=True) + EPS).sqrt()


def _exact_step(S, k, v, g, beta):
    """One token: S [H, D, D] (rows: keys) -> the new state and the correction."""
    S = S * g.exp()[:, None, None]
    u = beta[:, None] * (v - (S * k[:, :, None]).sum(1))
    return S + k[:, :, None] * u[:, None, :], u


def _exact_advanced(s, pool, taps):
    """Both pools' rows after the accepted paths."""
    rep = s["last_u"].shape[2] // HK
    parents, accepted = s["last_parents"].tolist(), s["accepted"].tolist()
    for b, slot in enumerate(s["ids"].tolist()):
        path = _exact_path(parents[b], accepted[b])
        for t in path:
            k = _exact_norms(s["last_k"][b, t].double()).repeat_interleave(rep, 0)
            pool[slot] = pool[slot] * s["last_g"][b, t].double().exp()[:, None, None]
            pool[slot] += k[:, :, None] * s["last_u"][b, t].double()[:, None, :]
            taps[slot] = torch.cat([taps[slot][:, 1:], s["last_x"][b, t].double()[:, None]], 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "linear":
        return _exact_linear(s)
    if op == "norm":
        return _exact_norm(s)
    pool, taps = s["s_cache"].double(), s["conv_cache"].double()
    if s["pending"]:
        _exact_advanced(s, pool, taps)
    if op == "commit":
        return pool, taps
    parents, ids = s["parents"].tolist(), s["ids"].tolist()
    if op == "conv":
        y = torch.zeros(s["x"].shape, dtype=F64, device=pool.device)
        w = s["weight"].double()
        for b, line in enumerate(parents):
            for t, up in enumerate(line):
                if up >= -1:
                    rows = [taps[ids[b]][:, j] for j in range(3)] + [s["x"][b, n].double() for n in _exact_path(line, t)]
                    y[b, t] = sum(row * w[:, j] for j, row in enumerate(rows[-4:]))
        return y * torch.sigmoid(y), taps
    B, T, Hv, D = s["v"].shape
    o, u = (torch.zeros(B, T, Hv, D, dtype=F64, device=pool.device) for _ in range(2))
    q, k = (_exact_norms(s[n].double()).repeat_interleave(Hv // HK, 2) for n in ("q", "k"))
    for b, line in enumerate(parents):
        states = {-1: pool[ids[b]]}
        for t, up in enumerate(line):
            if up >= -1:
                states[t], u[b, t] = _exact_step(states[up], k[b, t], s["v"][b, t].double(), s["g"][b, t].double(),
                                                 s["beta"][b, t].double())
                o[b, t] = D ** -0.5 * (states[t] * q[b, t][:, :, None]).sum(1)
    return o, u, pool
