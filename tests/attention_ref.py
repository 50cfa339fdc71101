"""Block-sparse attention in 64 bits on the CPU, straight from its formulas, with bounds of what 16-bit operands of the
matrix products may cost.  Test infrastructure only.

u is half a unit in the last place of the element type.  The kernels hold sums and softmax statistics in fp32 and round
the softmax weights (and in the backward pass the score gradients) once to the element type:
  scores   |ds| <= dim * 2^-23 * |scale| * sum_d |q_d k_d|, a relative error of the weights (and twice that with their sum)
  out      u |out| + sum_j p_j |v_j| (u + 2 |ds| + 2^-19); weights below the type's smallest normal number keep 2^-24 of it
  a float16 result below 2^-14 is rounded to a multiple of 2^-24, whatever its size
and likewise for the gradients, with the error of dout . v and of the row sums in the score gradients."""
import math

import torch

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24}
HALF_STEP = {torch.float16: 2.0 ** -25}  # half the distance of neighbouring subnormal numbers: what rounding a result may cost there


def times_listed(pos, crd, lists, rows, columns):
    """How often each row of each list names each column; entries outside the structure are absent."""
    t = torch.zeros((lists * rows, columns), dtype=torch.float64)
    p = pos.clamp(0, crd.numel()).tolist()
    for r in range(lists * rows):
        for c in crd[p[r]:max(p[r], p[r + 1])].tolist():
            if 0 <= c < columns:
                t[r, c] += 1
    return t.reshape(lists, rows, columns)


def pair_weights(pos, crd, batch, kv_heads, queries, keys, block_m, block_n, causal):
    """batch x kv_heads x queries x keys: how often a pair takes part."""
    rows, columns = -(-queries // block_m), -(-keys // block_n)
    t = times_listed(pos.cpu(), crd.cpu(), batch * kv_heads, rows, columns).reshape(batch, kv_heads, rows, columns)
    i, j = torch.arange(queries), torch.arange(keys)
    w = t[:, :, i // block_m][:, :, :, j // block_n] if queries and keys else torch.zeros((batch, kv_heads, queries, keys), dtype=torch.float64)
    if causal:
        w = w * (j <= i[:, None] + keys - queries)
    return w


def _heads_first(x):
    return x.detach().cpu().double().transpose(1, 2)


def _expand(x, group):
    return x.repeat_interleave(group, 1)


def _product(a, b, keep):
    """a @ b where rows of a that are nowhere kept (weight 0) do not bring a NaN of b in."""
    return torch.where(keep, a, 0.0) @ torch.nan_to_num(b, nan=0.0, posinf=0.0, neginf=0.0)


def forward(q, k, v, w, scale):
    """(out, lse, bound of out, bound of lse); q: batch x queries x heads x dim."""
    dtype = q.dtype
    u, tiny = HALF_ULP[dtype], TINY[dtype]
    group = q.shape[2] // k.shape[2]
    Q, K, V = _heads_first(q), _expand(_heads_first(k), group), _expand(_heads_first(v), group)
    W = _expand(w, group)
    keep = W > 0
    S = torch.where(keep, scale * (Q @ K.transpose(2, 3)), -math.inf)
    ds = torch.where(keep, q.shape[3] * 2.0 ** -23 * abs(scale) * (Q.abs() @ K.abs().transpose(2, 3)), 0.0).amax(-1, keepdim=True) if K.shape[2] else torch.zeros_like(S).sum(-1, keepdim=True)
    top = S.amax(-1, keepdim=True) if K.shape[2] else torch.full_like(ds, -math.inf)
    P = torch.where(keep, W * torch.exp(S - torch.where(torch.isinf(top), 0.0, top)), 0.0)
    total = P.sum(-1, keepdim=True)
    empty = total == 0
    P = torch.where(empty, 0.0, P / torch.where(empty, 1.0, total))
    out = _product(P, V, keep)
    lse = torch.where(empty, -math.inf, top + torch.log(torch.where(empty, 1.0, total)))[..., 0]
    spread = _product(P, V.abs(), keep)
    bound = u * out.abs() + spread * (u + 2 * ds + 2.0 ** -19) + tiny * _product(keep.double(), V.abs(), keep)
    lse_bound = (2 * ds[..., 0] + 2.0 ** -19 + u / 4) + 2.0 ** -22 * torch.where(torch.isinf(lse), 0.0, lse.abs())
    back = lambda x: x.transpose(1, 2)  # noqa: E731
    return back(out), lse, back(bound), lse_bound


def backward(dout, q, k, v, out, lse, w, scale):
    """((dq, dk, dv), their bounds) from the forward pass's own results."""
    dtype = q.dtype
    u, tiny = HALF_ULP[dtype], TINY[dtype]
    group, dim = q.shape[2] // k.shape[2], q.shape[3]
    Q, DO, O = _heads_first(q), _heads_first(dout), _heads_first(out)
    K, V = _expand(_heads_first(k), group), _expand(_heads_first(v), group)
    W = _expand(w, group)
    keep = W > 0
    L = lse.detach().cpu().double()[..., None]
    P = torch.where(keep, W * torch.exp(scale * (Q @ K.transpose(2, 3)) - torch.where(torch.isinf(L), 0.0, L)), 0.0)
    P = torch.where(torch.isinf(L), 0.0, P)
    delta = (DO * O).sum(-1, keepdim=True)
    G = torch.where(keep, DO @ V.transpose(2, 3) - delta, 0.0)
    DS = P * G * scale
    es = torch.where(keep, dim * 2.0 ** -23 * abs(scale) * (Q.abs() @ K.abs().transpose(2, 3)) + 2.0 ** -20 * (1 + torch.where(torch.isinf(L), 0.0, L.abs())), 0.0)
    eg = torch.where(keep, dim * 2.0 ** -23 * (DO.abs() @ V.abs().transpose(2, 3) + (DO * O).abs().sum(-1, keepdim=True)), 0.0)
    EDS = DS.abs() * (u + 2 * es) + P * abs(scale) * eg + tiny * keep
    EP = P * (u + 2 * es) + tiny * keep
    t = lambda x: x.transpose(2, 3)  # noqa: E731
    dq = _product(DS, K, keep)
    edq = u * dq.abs() + _product(EDS + 2.0 ** -19 * DS.abs(), K.abs(), keep)
    fold = lambda x: x.reshape(x.shape[0], -1, group, *x.shape[2:]).sum(2).transpose(1, 2)  # noqa: E731
    dk, dv = fold(_product(t(DS), Q, t(keep))), fold(_product(t(P), DO, t(keep)))
    edk = u * dk.abs() + fold(_product(t(EDS + 2.0 ** -19 * DS.abs()), Q.abs(), t(keep)))
    edv = u * dv.abs() + fold(_product(t(EP + 2.0 ** -19 * P), DO.abs(), t(keep)))
    return (dq.transpose(1, 2), dk, dv), (edq.transpose(1, 2), edk, edv)


def assert_within(got, want, bound, what):
    dtype, got = got.dtype, got.detach().cpu().double()
    assert got.shape == want.shape, what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what + ": infinities"
    err = torch.where(inf, 0.0, (got - torch.where(inf, 0.0, want)).abs())
    bad = ~(err <= bound + HALF_STEP.get(dtype, 1e-30)) & ~inf
    assert not bool(bad.any()), "%s: %d of %d outside the bound; worst error %.3g where %.3g is allowed (value %.4g)" % (
        what, int(bad.sum()), bad.numel(), float(err[bad].nan_to_num(nan=math.inf).max()),
        float(bound[bad][err[bad].nan_to_num(nan=math.inf).argmax()]), float(want[bad][err[bad].nan_to_num(nan=math.inf).argmax()]))
