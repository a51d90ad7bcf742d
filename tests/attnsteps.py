"""Cross attention in 64 bits from given probabilities, with elementwise bounds that follow the kernels step by step, narrower than those
of attnref.py where the kernels keep more than one term:

* a training forward of a 16-bit type takes P as two terms and keeps `out` in fp32 for D = do . o;
* fp16 takes dS times a power of two that brings its bound to 2^14 .. 2^15 before rounding it, so that only what is below 2^-38 of that bound is lost.

h = finfo.eps / 2 is the half step of the type, u = 2^-24 that of an fp32 operation."""
import math

import torch

import attnref
from attnref import SUBNORMAL, U, half_step

NO = torch.zeros((), dtype=torch.float64)


def _heads(c):
    g = c['q'].shape[2] // c['k'].shape[2]
    rows = c['keep'][:, None, :, None]
    Q = c['q'].double().permute(0, 2, 1, 3)
    K, V = (torch.where(rows, c[n].double().permute(0, 2, 1, 3), NO).repeat_interleave(g, 1) for n in 'kv')
    return Q, K, V, g


def softmax(c, bias, scale=None, rounded_at=0.0, roundings=1):
    """c: q, k, v, keep; bias [B|1, H|1, Lq, Lk] in 64 bits, -inf takes a pair out -> (p, relative error of p).
    rounded_at [Lq] or number: what the scores were added to in fp32 before they were compared (a constant of the row, left out of `bias`).
    roundings: sums in fp32 at that size, each off by half a step there: that of the axes' entries (two axes), and that with the product."""
    Q, K, _, _ = _heads(c)
    scale = c['q'].shape[-1] ** -0.5 if scale is None else scale
    s = scale * Q @ K.transpose(2, 3)
    mags = scale * (Q.abs() @ K.abs().transpose(2, 3))
    out = torch.isneginf(bias) | ~c['keep'][:, None, None, :]
    base = torch.as_tensor(rounded_at, dtype=torch.float64).abs().reshape(1, 1, -1, 1)
    step = torch.where(base > 0, 2.0 ** (torch.floor(torch.log2(base.clamp(min=1e-300) / math.log(2))) - 23), NO)      # of fp32 there, log2 units
    swallowed = (s.abs() + bias.nan_to_num(0, 0, 0).abs()).amax(-1, keepdim=True) / math.log(2) < 0.45 * step
    s = torch.where(swallowed, NO, s + bias)
    s = torch.where(out, torch.full_like(s, -math.inf), s)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isneginf(top), NO, top))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    lk, dim = K.shape[2], Q.shape[3]
    # a dot of dim terms, scale, log2(e), the bias; the reference, of the size of the highest score, in every step of a product that starts there
    err = torch.where(out, NO, U * ((dim + 6) * mags + 6 * bias.nan_to_num(0, 0, 0).abs() + 10 * top.nan_to_num(0, 0, 0).abs())).amax(-1, keepdim=True) + 4 * U
    err = torch.where(swallowed, 4 * U, err + torch.expm1(roundings * step * math.log(2)) / 2)
    return p, 2 * err + (lk + 16) * U + 4 * U * torch.where(out, NO, s - top).abs().clamp(max=200)


def attention(c, p, p_rel, training=True, scale=None, idx=None, buckets=0):
    """-> dict name -> (value, bound); gradients of c['go'] where training"""
    dtype = c['q'].dtype
    h, sub = half_step(dtype), SUBNORMAL[dtype]
    Q, K, V, g = _heads(c)
    b, heads, lq, dim = Q.shape
    lk, hk = K.shape[2], heads // g
    scale = dim ** -0.5 if scale is None else scale
    perm = (0, 2, 1, 3)
    o = p @ V
    # P is rounded next to a sum of 1 or more: once, or to what two terms leave of it
    p_step = 0.0 if dtype == torch.float32 else h * h if training else h
    o_err = (p * (p_rel + p_step + (lk + 4) * U)) @ V.abs() + sub * V.abs().sum(2, keepdim=True) * (p.sum(-1, keepdim=True) > 0)
    out = {'out': (o.permute(perm), (o_err + h * (o.abs() + o_err) + sub).permute(perm))}
    if not training:
        return out
    G = c['go'].double().permute(perm)
    l1 = G.abs().sum(-1, keepdim=True)
    reach = 2 * V.abs().amax((2, 3), keepdim=True)          # |dp - D| <= reach * l1
    lost_q = 2.0 ** -38 * reach * l1 if dtype == torch.float16 else NO
    lost_k = 2.0 ** -38 * reach * l1.reshape(b, hk, -1).amax(-1).repeat_interleave(g, 1)[..., None, None] if dtype == torch.float16 else NO
    D = (G * o).sum(-1, keepdim=True)
    d_err = (G.abs() * o_err).sum(-1, keepdim=True) + (dim + 2) * U * (G.abs() * o.abs()).sum(-1, keepdim=True)
    dp = G @ V.transpose(2, 3)
    ds = p * (dp - D)
    ds32 = p * ((p_rel + 3 * U) * (dp - D).abs() + (dim + 2) * U * (G.abs() @ V.abs().transpose(2, 3)) + 10 * U * D.abs() + d_err) * (1 + p_rel)
    hs = 0.0 if dtype == torch.float32 else h
    dq = scale * ds @ K
    dq_err = scale * (ds32 + hs * (ds.abs() + ds32) + lost_q + (lk + 4) * U * ds.abs()) @ K.abs()
    dk = scale * ds.transpose(2, 3) @ Q
    dk_err = scale * (ds32 + hs * (ds.abs() + ds32) + lost_k + (lq * g + 4) * U * ds.abs()).transpose(2, 3) @ Q.abs()
    dv = p.transpose(2, 3) @ G
    # dv's P is taken times 2^10 in fp16
    dv_err = (p * (p_rel + hs + (lq * g + 4) * U)).transpose(2, 3) @ G.abs() + sub / 1024 * G.abs().sum(2, keepdim=True)
    rows = c['keep'][:, None, :, None]
    out['dq'] = (dq.permute(perm), (dq_err + h * (dq.abs() + dq_err) + sub).permute(perm))
    for name, val, err in (('dk', dk, dk_err), ('dv', dv, dv_err)):
        val, err = (torch.where(rows, t.reshape(b, hk, g, lk, dim).sum(2), NO) for t in (val, err))
        out[name] = (val.permute(perm), (err + h * (val.abs() + err) + torch.where(rows, torch.full((), sub).double(), NO)).permute(perm))
    if idx is not None:
        val, err = torch.zeros(2, idx.shape[0], buckets, heads, dtype=torch.float64)
        for a in range(idx.shape[0]):
            flat = idx[a].expand(b, lq, lk).reshape(-1)
            for i in range(heads):
                val[a, :, i] = torch.bincount(flat, weights=ds[:, i].reshape(-1), minlength=buckets)
                err[a, :, i] = torch.bincount(flat, weights=(ds32[:, i] + 700 * U * ds[:, i].abs()).reshape(-1), minlength=buckets)
        out['dtable'] = (val, err + h * (val.abs() + err) + sub)
    return out


def assert_within(got, want_bound, name):
    """attnref.assert_within; a value beyond the type's largest number has to come out as infinity"""
    want, bound = want_bound
    largest = torch.finfo(got.dtype).max * (1 + half_step(got.dtype))
    over = want.abs() - bound > largest
    assert torch.equal(got.detach().cpu().double()[over], torch.copysign(torch.full_like(want, math.inf), want)[over]), name
    bound = torch.where(want.abs() + bound > largest, math.inf, bound)      # within the bound of the border: either
    attnref.assert_within(torch.where(over, NO, got.detach().cpu().double().clamp(-1e300, 1e300)), (torch.where(over, NO, want), torch.where(over, NO, bound)), name)
