"""64-bit CPU forms of the tree verify and of the 8-bit operands, with bounds on how
far fp32 arithmetic may be from them (shared by the GPU tests)."""
from __future__ import annotations

import torch

F64 = torch.float64
U32 = 2.0 ** -24      # half a step of fp32, relative
HALF_BF16 = 2.0 ** -8
EPS = 1e-6


def tree(gen, B, T, back=4, ragged=False):
    """parents int32 [B, T] and an accepted node per row (-1 where a row keeps nothing)."""
    parents = torch.full((B, T), -1, dtype=torch.int32)
    accepted = torch.empty(B, dtype=torch.int64)
    for b in range(B):
        size = int(torch.randint(1, T + 1, (1,), generator=gen)) if ragged else T
        for t in range(1, T):
            parents[b, t] = max(0, t - 1 - int(torch.randint(0, back, (1,), generator=gen))) if t < size else -2
        accepted[b] = int(torch.randint(-1, size, (1,), generator=gen))
    return parents, accepted


def used(parents):
    """Which nodes count: the walk to the root meets valid links only."""
    ok = []
    for t, p in enumerate(parents):
        ok.append(p == -1 or (0 <= p < t and ok[p]))
    return ok


def path(parents, node):
    out = []
    while node >= 0:
        out.insert(0, node)
        node = parents[node]
    return out


def unit(t):
    t = t.to(F64)
    return t / (t.square().sum(-1, keepdim=True) + EPS).sqrt()


def rule(q, k, v, g, beta, S, parents):
    """One sequence: q, k [T, Hk, D], v [T, Hv, D], g, beta [T, Hv], S [Hv, D, D] ->
    (o, u, states by node, bound on o before its rounding, bound on u).

    The bounds: with A the same recurrence on magnitudes (every product and sum of the
    formula with absolute values), one evaluation of u_t makes a relative error of at
    most c = (2 D + T + 32) 2^-24 of A_t (a dot of D terms twice over, for operands
    in parts; T weighted terms; the norms, the exponentials and their products), and an
    ancestor's own error is in A_t once per level."""
    T, Hk, D = k.shape
    Hv = v.shape[1]
    rep = Hv // Hk
    q, k = unit(q).repeat_interleave(rep, 1) * D ** -0.5, unit(k).repeat_interleave(rep, 1)
    v, g, beta, S = v.to(F64), g.to(F64), beta.to(F64), S.to(F64)
    ok, line = used(parents.tolist()), parents.tolist()
    o, u, eo, eu = (torch.zeros(T, Hv, D, dtype=F64) for _ in range(4))
    states = {-1: (S, S.abs(), 0)}
    c = (2 * D + T + 32) * U32
    for t in range(T):
        if not ok[t]:
            continue
        P, A, depth = states[line[t]]
        decay = g[t].exp()[:, None, None]
        P, A = P * decay, A * decay
        u[t] = beta[t][:, None] * (v[t] - (P * k[t][:, :, None]).sum(1))
        a = beta[t].abs()[:, None] * (v[t].abs() + (A * k[t].abs()[:, :, None]).sum(1))
        P, A = P + k[t][:, :, None] * u[t][:, None], A + k[t].abs()[:, :, None] * a[:, None]
        o[t] = (P * q[t][:, :, None]).sum(1)
        eu[t] = c * (depth + 1) * a
        eo[t] = c * (depth + 2) * (A * q[t].abs()[:, :, None]).sum(1)
        states[t] = (P, A, depth + 1)
    return o, u, states, eo, eu


def advanced(S, k, g, u, parents, node):
    """The state after `node` from the step's k, g, u, and a bound on its fp32 form."""
    Hv = u.shape[1]
    k = unit(k).repeat_interleave(Hv // k.shape[1], 1)
    S = S.to(F64)
    A = S.abs()
    for t in path(parents.tolist(), node):
        decay = g[t].to(F64).exp()[:, None, None]
        new = k[t][:, :, None] * u[t].to(F64)[:, None]
        S, A = S * decay + new, A * decay + new.abs()
    return S, (2 * len(parents) + 32) * U32 * A


def taps_after(taps, x, parents, node):
    """[C, 3] after the path to `node` (bit copies)."""
    for t in path(parents.tolist(), node):
        taps = torch.cat([taps[:, 1:], x[t][:, None]], 1)
    return taps


def conv(x, taps, w, parents):
    """One sequence x [T, C], taps [C, 3] -> (y, bound on y): fp32's error on the sum of
    four products, through a SiLU whose slope is at most 1.1, and bf16's half step."""
    ok, line = used(parents.tolist()), parents.tolist()
    x, taps, w = x.to(F64), taps.to(F64), w.to(F64)
    y, e = torch.zeros(x.shape, dtype=F64), torch.zeros(x.shape, dtype=F64)
    for t in range(len(x)):
        if ok[t]:
            rows = torch.stack(([taps[:, j] for j in range(3)] + [x[n] for n in path(line, t)])[-4:], 1)
            s = (rows * w).sum(1)
            y[t] = s * torch.sigmoid(s)
            e[t] = 1.1 * 16 * U32 * (rows * w).abs().sum(1) + 1e-6 * y[t].abs() + 4e-7 * s.abs()
            e[t] += HALF_BF16 * (y[t].abs() + e[t])
    return y, e


# ---------------------------------------------------------------- 8 bits --
def to_e4m3(x, rows):
    """x [M, K] fp32 on the CPU -> (e4m3, scales), one scale per `rows` x 128 values."""
    M, K = x.shape
    n = -(-M // rows)
    p = torch.nn.functional.pad(x, (0, 0, 0, n * rows - M)).view(n, rows, K // 128, 128)
    top = torch.where(p.isnan(), torch.zeros_like(p), p.abs()).amax((1, 3))
    scale = (top * torch.tensor(1 / 448.0, dtype=torch.float32)).clamp(min=2.0 ** -126)
    q = (p * (1.0 / scale)[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).reshape(n * rows, K)[:M].contiguous().view(torch.float8_e4m3fn), scale


def from_e4m3(q, scale, rows):
    """The values in 64 bits."""
    s = scale.to(F64).repeat_interleave(rows, 0)[: q.shape[0]].repeat_interleave(128, 1)
    return q.to(torch.float32).to(F64) * s


def linear(x8, xs, w8, ws):
    """(y, bound before the bf16 rounding, for every element).

    The matrix cores add the 128 products of a block after shifting them to the exponent of
    the largest one, and what lies below 2^-13 of that one is lost (two large products that
    cancel leave a third one of 2^-13 of them whole and lose one of 2^-14): each product is
    off by at most 2^-13 of the block's largest product, and by no more than itself.  To that
    comes fp32's error of the scales' product and of the sum over the blocks.  Here a block's
    largest product is taken as that of the operands' largest values; see linear_tight."""
    a, w = from_e4m3(x8, xs, 1), from_e4m3(w8, ws, 128)
    y = a @ w.t()
    n = x8.shape[1] // 128
    top = lambda t: t.abs().view(len(t), n, 128).amax(-1)  # noqa: E731
    lost = (top(a) @ top(w).t()) * 2.0 ** -13 * 128
    return y, lost + (a.abs() @ w.abs().t()) * ((n + 4) * 2 * U32)


def linear_tight(x8, xs, w8, ws, rows, cols):
    """linear's y and bound at some rows and columns, product by product."""
    a = from_e4m3(x8, xs, 1)[rows]
    w = from_e4m3(w8, ws, 128)[cols]
    n = a.shape[1] // 128
    y, e = torch.zeros(len(a), len(w), dtype=F64), torch.zeros(len(a), len(w), dtype=F64)
    for i in range(n):
        p = (a[:, None, 128 * i:128 * i + 128] * w[None, :, 128 * i:128 * i + 128]).abs()
        e += torch.minimum(p, 2.0 ** -13 * p.amax(-1, keepdim=True)).sum(-1) + p.sum(-1) * ((n + 4) * 2 * U32)
    y = a @ w.t()
    return y, e
