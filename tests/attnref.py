"""64-bit restatements of cross attention, the bucketed position bias and group norm, each with elementwise bounds on what rounding may
do to a kernel that keeps sums in fp32 and rounds probabilities, dS and results to the element type.

A rounding to type T is off by at most h(T) = finfo(T).eps / 2 of the value, or by half the smallest subnormal; an fp32 operation by
u = 2^-24, a sum of n terms by (n - 1) u of the sum of magnitudes.  The bounds below add these up term by term."""
import math

import torch

U = 2.0 ** -24
SUBNORMAL = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bucket(offset, buckets, bidirectional, max_distance):
    """The definition in whole numbers, one offset at a time."""
    side = buckets // 2 if bidirectional else buckets
    e = side // 2
    d = abs(offset) if bidirectional else max(-offset, 0)
    j = d
    if d >= e:
        j = e
        while j + 1 < side and d ** (side - e) >= max_distance ** (j + 1 - e) * e ** (side - j - 1):
            j += 1
    return j + (side if bidirectional and offset > 0 else 0)


def buckets_of(q_pos, k_pos, buckets, bidirectional, max_distance):
    """q_pos, k_pos [B, L, axes] (any batch of 1) -> int64 [axes, B, Lq, Lk]"""
    lut = torch.tensor([bucket(o, buckets, bidirectional, max_distance) for o in range(-max_distance, max_distance + 1)])
    off = k_pos.long()[:, None, :, :] - q_pos.long()[:, :, None, :]
    return lut[off.clamp(-max_distance, max_distance) + max_distance].permute(3, 0, 1, 2)


def attention(q, k, v, scale, keep, table=None, idx=None, gout=None):
    """CPU tensors of the operator's type; keep bool [B, Lk]; idx from buckets_of (batch 1 or B).  -> dict name -> (value, bound)."""
    dtype = q.dtype
    hT, sub = half_step(dtype), SUBNORMAL[dtype]
    b, lq, h, dim = q.shape
    lk, hk = k.shape[1:3]
    g = h // hk
    Q = q.double().permute(0, 2, 1, 3)
    rows = keep[:, None, :, None]
    K, V = (torch.where(rows, t.double().permute(0, 2, 1, 3), torch.zeros(()).double()).repeat_interleave(g, 1) for t in (k, v))
    s = Q @ K.transpose(2, 3) * scale
    bias = torch.zeros(1, 1, 1, 1, dtype=torch.float64)
    if table is not None:
        t64 = table.double()
        bias = sum(t64[a][idx[a]] for a in range(table.shape[0])).permute(0, 3, 1, 2)      # [B|1, H, Lq, Lk]
        s = s + bias
    finite_bias = torch.where(torch.isfinite(bias), bias.abs(), torch.zeros(()).double())
    # scores: a dot of dim terms, scale, log2(e), bias, the subtraction of the maximum; exp2 within 2 u of its argument's result
    s_err = (U * ((dim + 6) * scale * (Q.abs() @ K.abs().transpose(2, 3)) + 6 * finite_bias)).amax(dim=-1, keepdim=True) + 4 * U
    s = torch.where(keep[:, None, None, :], s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    p_rel = 2 * s_err + (lk + 16) * U + 4 * U * (s - top).abs().nan_to_num(0, 0, 0).clamp(max=200)
    o = p @ V
    o_err = (p * (p_rel + hT)) @ V.abs() + sub * 512 * V.abs().sum(2, keepdim=True) * (total > 0) + (lk + 4) * U * (p @ V.abs())
    perm = (0, 2, 1, 3)
    out = {'out': (o.permute(perm), (o_err + hT * (o.abs() + o_err) + sub).permute(perm))}
    if gout is None:
        return out
    G = gout.double().permute(0, 2, 1, 3)
    dv = p.transpose(2, 3) @ G
    dv_err = (p * (p_rel + hT + (lq * g + 4) * U)).transpose(2, 3) @ G.abs() + sub * G.abs().sum(2, keepdim=True)
    dp = G @ V.transpose(2, 3)
    D = (G * o).sum(-1, keepdim=True)
    d_err = (G.abs() * (o_err + hT * (o.abs() + o_err) + sub)).sum(-1, keepdim=True) + (dim + 2) * U * (G.abs() * o.abs()).sum(-1, keepdim=True)
    ds = p * (dp - D)
    ds_err32 = p * ((p_rel + 3 * U) * (dp - D).abs() + (dim + 2) * U * (G.abs() @ V.abs().transpose(2, 3)) + d_err) * (1 + 2 * s_err)
    ds_err = ds_err32 + hT * (ds.abs() + ds_err32) + sub
    dq = scale * ds @ K
    dq_err = scale * (ds_err @ K.abs() + (lk + 4) * U * (ds.abs() @ K.abs()))
    dk = scale * ds.transpose(2, 3) @ Q
    dk_err = scale * (ds_err.transpose(2, 3) @ Q.abs() + (lq * g + 4) * U * (ds.abs().transpose(2, 3) @ Q.abs()))
    zero = torch.zeros(()).double()

    def group(t):       # query heads of a kv head, masked rows exactly zero
        return torch.where(rows, t.reshape(b, hk, g, lk, dim).sum(2), zero).permute(perm)
    out['dq'] = (dq.permute(perm), (dq_err + hT * (dq.abs() + dq_err) + sub).permute(perm))
    for name, val, err in (('dk', dk, dk_err), ('dv', dv, dv_err)):
        val, err = group(val), group(err)
        out[name] = (val, err + hT * (val.abs() + err) + torch.where(rows, torch.full((), sub).double(), zero).permute(perm))
    if table is not None:
        dt, dt_err = torch.zeros_like(t64), torch.zeros_like(t64)
        for a in range(table.shape[0]):
            ia = idx[a].expand(b, lq, lk)
            for hh in range(h):
                for acc, w in ((dt, ds[:, hh]), (dt_err, ds_err32[:, hh] + 700 * U * ds[:, hh].abs())):
                    acc[a, :, hh] = torch.bincount(ia.reshape(-1), weights=w.reshape(-1), minlength=table.shape[1])
        out['dtable'] = (dt, dt_err + hT * (dt.abs() + dt_err) + sub)
    return out


def group_norm(x, groups, weight, bias, eps, act, gout=None):
    """x [B, C, ...] on the CPU, weight / bias [C] or None -> dict name -> (value, bound)."""
    dtype = x.dtype
    hT, sub = half_step(dtype), SUBNORMAL[dtype]
    b, c = x.shape[:2]
    shape = (b, groups, c // groups, x[0, 0].numel())
    X = x.double().reshape(shape)
    W = (weight if weight is not None else torch.ones(c)).double().view(1, groups, -1, 1)
    Bs = (bias if bias is not None else torch.zeros(c)).double().view(1, groups, -1, 1)
    n = X[0, 0].numel()
    mean = X.mean((2, 3), keepdim=True)
    var = ((X - mean) ** 2).mean((2, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = (X - mean) * rstd
    z = xhat * W + Bs
    # a thread adds a few terms, a workgroup at most 256 threads, a wave 64 chunks: no chain of sums is longer than K
    K = 400
    spread = X.amax((2, 3), keepdim=True) - X.amin((2, 3), keepdim=True)
    m_err = K * U * spread + 2 * U * mean.abs()
    r_rel = 0.5 * (K * U * spread ** 2 + m_err ** 2) / (var + eps) + 6 * U
    h_err = rstd * (m_err + U * (X - mean).abs()) + xhat.abs() * (r_rel + 2 * U)
    z_err = W.abs() * h_err + 3 * U * ((xhat * W).abs() + Bs.abs())
    sig = torch.sigmoid(z)
    one = torch.ones_like(z)
    value, slope, lip, curve = {
        None: (z, one, 1.0, 0.0), 'relu': (z.clamp_min(0), (z > 0).double(), 1.0, 0.0),
        'leaky_relu': (torch.where(z > 0, z, 0.1 * z), torch.where(z > 0, one, 0.1 * one), 1.0, 0.0),
        'sigmoid': (sig, sig * (1 - sig), 0.25, 0.1), 'silu': (z * sig, sig * (1 + z * (1 - sig)), 1.1, 0.5)}[act]
    trans = (8 + 2 * z.abs()) * U               # exp of an argument rounded to fp32, one division
    y_err = lip * z_err + trans * value.abs()
    out = {'y': (value.reshape(x.shape), (y_err + hT * (value.abs() + y_err) + sub).reshape(x.shape)), 'z': (z.reshape(x.shape), z_err.reshape(x.shape))}
    if gout is None:
        return out
    G = gout.double().reshape(shape)
    dz = G * slope
    dz_err = G.abs() * (curve * z_err + trans * (slope.abs() + z.abs() * (curve > 0)) + 4 * U)
    dxh = dz * W
    dxh_err = dz_err * W.abs() + U * dxh.abs()
    m0, m1 = dxh.sum((2, 3), keepdim=True) / n, (dxh * xhat).sum((2, 3), keepdim=True) / n
    m0_err = (dxh_err + K * U * dxh.abs()).sum((2, 3), keepdim=True) / n
    m1_err = (dxh_err * xhat.abs() + dxh.abs() * h_err + K * U * (dxh * xhat).abs()).sum((2, 3), keepdim=True) / n
    dx = rstd * (dxh - m0 - xhat * m1)
    dx_err = rstd * (dxh_err + m0_err + xhat.abs() * m1_err + h_err * m1.abs() + (4 * U + r_rel) * (dxh.abs() + m0.abs() + (xhat * m1).abs()))
    out['dx'] = (dx.reshape(x.shape), (dx_err + hT * (dx.abs() + dx_err) + sub).reshape(x.shape))
    for name, val, err, p in (('dw', dz * xhat, dz_err * xhat.abs() + dz.abs() * h_err, weight), ('db', dz, dz_err, bias)):
        if p is not None:
            tot = val.sum((0, 3)).reshape(c)
            e = (err + (K + b) * U * val.abs()).sum((0, 3)).reshape(c)
            hp = half_step(p.dtype)
            out[name] = (tot, e + hp * (tot.abs() + e) + SUBNORMAL[p.dtype])
    return out


def assert_within(got, want_bound, what):
    want, bound = want_bound
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    excess = (got - want).abs() - bound
    bad = ~(excess <= 0)
    assert not bad.any(), '%s: %d of %d outside the bound, worst |diff| %.3g against %.3g' % (
        what, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].nan_to_num(math.inf).max()), float(bound[bad].min()))
