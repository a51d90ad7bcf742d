"""Cross attention and the bucketed relative position bias (camli_cross_attention_*, camli_rel_bias_*: csrc/hip/xattn.h, relbias.hip).

What an attentive camera-LiDAR fusion needs where the reference gathers one nearest point per pixel (models/clfm.py:7-60): every
pixel may attend every point and the other way round, with a learned bias by the offset of the two in the image.  Keys and values are
never expanded over query heads and no score matrix is stored; the backward recomputes the probabilities from each row's log-sum.
"""
import ctypes
import functools
import math

import torch

from . import _lib
from .norm import TYPE_CODES, address, first_order, needs_node, same_device
from .wrapper import _on_device, _require_cuda, _stream_ptr

MAX_HEAD_DIM = 128
MAX_BIAS_ROWS = 128
MAX_BIAS_DISTANCE = 1023
MAX_BIAS_HEADS = 65535
MAX_POSITION = 2 ** 26
MAX_ENTRY = 2.0 ** 125 * math.log(2)


# ------------------------------------------------------------------------------------------------
# the bias: checks, buckets, stand-alone operator
# ------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=64)
def _bucket_of_offsets(buckets, bidirectional, max_distance):
    """Bucket of every offset -max_distance .. max_distance, in exact integer arithmetic (the composed formulation's table)."""
    side = buckets // 2 if bidirectional else buckets
    exact = side // 2
    steps = side - exact
    out = []
    for offset in range(-max_distance, max_distance + 1):
        d = abs(offset) if bidirectional else max(-offset, 0)
        if d < exact:
            n = d
        else:
            n = exact + sum(1 for j in range(1, steps) if d ** steps >= max_distance ** j * exact ** (steps - j))
        out.append(n + (side if bidirectional and offset > 0 else 0))
    return out


def _check_bias(name, table, q_pos, k_pos, bidirectional, max_distance, dtype, heads=None, batch=None, lq=None, lk=None):
    """-> (table, q_pos, k_pos, batch of the bias or None, axes); positions [B or none, L, axes] int32 contiguous."""
    if table is None or q_pos is None or k_pos is None:
        raise ValueError('%s: a position bias needs the table and both positions' % name)
    if table.dim() != 3 or table.dtype != dtype or dtype not in TYPE_CODES:
        raise ValueError('%s: the table must be [axes, buckets, heads] of type %s, got %s %s' % (name, dtype, tuple(table.shape), table.dtype))
    axes, buckets, h = table.shape
    if axes not in (1, 2) or axes * buckets > MAX_BIAS_ROWS or not 1 <= h <= MAX_BIAS_HEADS or (heads is not None and h != heads):
        raise ValueError('%s: the table needs 1 or 2 axes, axes * buckets <= %d and %s heads, got %s' % (
            name, MAX_BIAS_ROWS, heads if heads is not None and heads <= MAX_BIAS_HEADS else '1 .. %d' % MAX_BIAS_HEADS, tuple(table.shape)))
    side = buckets // 2 if bidirectional else buckets
    if side < 2 or (bidirectional and buckets % 2) or not side // 2 < max_distance <= MAX_BIAS_DISTANCE or int(max_distance) != max_distance:
        raise ValueError('%s: need at least two buckets a side (an even number when bidirectional) and %d < max_distance <= %d, got %d buckets and %r'
                         % (name, side // 2, MAX_BIAS_DISTANCE, buckets, max_distance))
    leads = []
    for what, pos, n in (('q_pos', q_pos, lq), ('k_pos', k_pos, lk)):
        shape = pos.shape
        if pos.dtype != torch.int32 or len(shape) not in (2, 3) or shape[-1] != axes or (n is not None and shape[-2] != n) or (
                len(shape) == 3 and batch is not None and shape[0] != batch) or pos.device != table.device:
            raise ValueError('%s: %s must be int32 [L, %d] or [B, L, %d] for the operands\' B and L, beside the table on %s; got %s %s on %s' % (
                name, what, axes, axes, table.device, tuple(shape), pos.dtype, pos.device))
        if len(shape) == 3:
            leads.append(shape[0])
    if len(leads) == 2 and leads[0] != leads[1]:
        raise ValueError('%s: q_pos and k_pos of different batches: %s' % (name, leads))
    return table.contiguous(), q_pos.contiguous(), k_pos.contiguous(), (leads[0] if leads else None), axes


def _pos_stride(pos):
    return pos.shape[1] * pos.shape[2] if pos.dim() == 3 else 0


def _composed_bias(table, q_pos, k_pos, bidirectional, max_distance):
    axes, buckets, _ = table.shape
    lut = torch.tensor(_bucket_of_offsets(buckets, bool(bidirectional), int(max_distance)), device=table.device)
    total = 0
    for a in range(axes):
        offset = (k_pos[..., None, :, a].clamp(-MAX_POSITION, MAX_POSITION).long()
                  - q_pos[..., :, None, a].clamp(-MAX_POSITION, MAX_POSITION).long())
        total = total + table[a].float()[lut[offset.clamp(-max_distance, max_distance) + max_distance]]
    return total.movedim(-1, -3)            # [(B,) H, Lq, Lk]


def _within_range(table):
    """Finite entries beyond +-MAX_ENTRY count as that (sums of two and their distances are finite then); the gradient is the entry's own."""
    x = table.float()
    return x + torch.where(torch.isfinite(x), x.clamp(-MAX_ENTRY, MAX_ENTRY) - x, torch.zeros_like(x)).detach()


@functools.lru_cache(maxsize=1024)
def _bias_workspace_bytes(b, h, lq, lk, axes, buckets, code):
    return int(_lib.load().camli_rel_bias_bwd_workspace_bytes(b, h, lq, lk, axes, buckets, code))


def _run_bias(table, q_pos, k_pos, batch, bidirectional, max_distance):
    axes, buckets, h = table.shape
    lq, lk = q_pos.shape[-2], k_pos.shape[-2]
    out = torch.empty((h, lq, lk) if batch is None else (batch, h, lq, lk), dtype=table.dtype, device=table.device)
    n = out.numel()
    if n:
        with _on_device(table):
            _lib.launch('camli_rel_bias_fwd', _lib.load().camli_rel_bias_fwd, table.data_ptr(), q_pos.data_ptr(), _pos_stride(q_pos),
                        k_pos.data_ptr(), _pos_stride(k_pos), out.data_ptr(), batch or 1, h, lq, lk, axes, buckets, int(bidirectional),
                        max_distance, TYPE_CODES[table.dtype], _stream_ptr(table), work=(float(n * out.element_size()), 'B'))
    return out


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, q_pos, k_pos, batch, bidirectional, max_distance):
        ctx.save_for_backward(q_pos, k_pos)
        ctx.args = (tuple(table.shape), batch, bidirectional, max_distance, table.dtype)
        return _run_bias(table, q_pos, k_pos, batch, bidirectional, max_distance)

    @first_order
    def backward(ctx, gout):
        q_pos, k_pos = ctx.saved_tensors
        shape, batch, bidirectional, max_distance, dtype = ctx.args
        axes, buckets, h = shape
        lq, lk = q_pos.shape[-2], k_pos.shape[-2]
        n = gout.numel()
        if not n:
            return torch.zeros(shape, dtype=dtype, device=gout.device), None, None, None, None, None
        gout = gout.contiguous()
        gtable = torch.empty(shape, dtype=dtype, device=gout.device)
        code, b = TYPE_CODES[dtype], batch or 1
        ws_bytes = _bias_workspace_bytes(b, h, lq, lk, axes, buckets, code)
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=gout.device)
        with _on_device(gout):
            _lib.launch('camli_rel_bias_bwd', _lib.load().camli_rel_bias_bwd, gout.data_ptr(), q_pos.data_ptr(), _pos_stride(q_pos),
                        k_pos.data_ptr(), _pos_stride(k_pos), gtable.data_ptr(), ws.data_ptr(), ws_bytes, b, h, lq, lk, axes, buckets,
                        int(bidirectional), max_distance, code, _stream_ptr(gout), work=(float(n * gout.element_size()), 'B'))
        return gtable, None, None, None, None, None


def relative_position_bias(table: torch.Tensor, q_pos: torch.Tensor, k_pos: torch.Tensor, bidirectional=True, max_distance=128,
                           cpp_impl=True):
    """The learned bias of every query and key by their bucketed offset, [H, Lq, Lk] ([B, H, Lq, Lk] where a position tensor has a
    batch): sum over axes a of table[a, bucket(k_pos[j, a] - q_pos[i, a]), h].

    ``table`` [axes, buckets, H] (fp32, bf16 or fp16; the result has its type); ``q_pos`` / ``k_pos`` int32 [L, axes] or [B, L, axes], whole
    numbers (the running index of a sequence, pixel coordinates); beyond -2^26 .. 2^26 they count as that bound.  ``bidirectional``: half the buckets for each sign, the upper half
    for keys after the query; otherwise all buckets for keys before the query, and keys after it share bucket 0.  Of the s buckets of a
    side, e = s // 2 hold one distance each; bucket e + j begins at the first distance >= e (max_distance / e)^(j / (s - e)), and the last
    one holds everything from there on.  1 or 2 axes, axes * buckets <= 128, max_distance <= 1023; at most 65535 samples x heads, 2000000 queries, 16000000 keys.
    Differentiable in the table (once, in reverse mode; a workgroup's elements are added in fp32, the workgroups' sums in 64 bits); the same
    bits on every run.  ``cpp_impl=False``: the same from torch primitives, on any device."""
    name = 'relative_position_bias'
    table, q_pos, k_pos, batch, _ = _check_bias(name, table, q_pos, k_pos, bidirectional, max_distance, table.dtype if table is not None else None)
    if (batch or 1) * table.shape[2] > 65535 or q_pos.shape[-2] > 2000000 or k_pos.shape[-2] > 16000000:
        raise ValueError('%s: more than 65535 samples x heads, 2000000 queries or 16000000 keys' % name)
    if not cpp_impl:
        return _composed_bias(table, q_pos, k_pos, bidirectional, int(max_distance)).to(table.dtype)
    _require_cuda(name, table)
    run = _RelativeBias.apply if needs_node(table) else _run_bias
    return run(table, q_pos, k_pos, batch, bool(bidirectional), int(max_distance))


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
def _rows16(t):
    """t itself if its elements are adjacent, rows start on 16 bytes and are less than 2^23 elements apart, else a dense copy."""
    size = t.element_size()
    if t.stride(3) == 1 and t.data_ptr() % 16 == 0 and t.stride(1) < 2 ** 23 and all(s * size % 16 == 0 for n, s in zip(t.shape[:3], t.stride()[:3]) if n > 1):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strides(t):
    return [s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3])]


def _descriptor(q, k, v, kv_lengths, key_mask, table, q_pos, k_pos, scale, bidirectional, max_distance):
    """the bytes of a camli_attention (include/camli_hip.h)"""
    b, lq, h, dim = q.shape
    lk, hk = k.shape[1:3]
    bias = (0, 0, 0, 0, 0, 0, 0, 0, 0)
    if table is not None:
        axes, buckets, _ = table.shape
        bias = (table.data_ptr(), q_pos.data_ptr(), k_pos.data_ptr(), _pos_stride(q_pos), _pos_stride(k_pos), axes, buckets, bidirectional,
                max_distance)
    return _lib.ATTENTION_PACK(TYPE_CODES[q.dtype], b, h, hk, lq, lk, dim, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                               *_strides(q), *_strides(k), *_strides(v), 0 if kv_lengths is None else kv_lengths.data_ptr(),
                               0 if key_mask is None else key_mask.data_ptr(), lk, *bias)


@functools.lru_cache(maxsize=1024)
def _attention_workspace_bytes(backward, flag, head, bias):
    """by sizes alone; flag: training (forward), a table gradient (backward); head = (type, B, H, Hk, Lq, Lk, D), bias = (axes, buckets, bidirectional, max_distance)"""
    lib = _lib.load()
    d = _lib.AttentionDesc(*head)
    d.scale = 1.0
    d.q = d.k = d.v = 16
    if bias[0]:
        d.bias_table = d.q_pos = d.k_pos = 16
        d.bias_axes, d.bias_buckets, d.bias_two_sided, d.bias_max_distance = bias
    n = (lib.camli_cross_attention_bwd_workspace_bytes if backward else lib.camli_cross_attention_fwd_workspace_bytes)(ctypes.byref(d), int(flag))
    if n < 0:
        _lib.check(int(n), 'camli_cross_attention_%s_workspace_bytes' % ('bwd' if backward else 'fwd'))
    return int(n)


def _sizes(q, k, table, bidirectional, max_distance):
    b, lq, h, dim = q.shape
    lk, hk = k.shape[1:3]
    return ((TYPE_CODES[q.dtype], b, h, hk, lq, lk, dim),
            (0, 0, 0, 0) if table is None else (table.shape[0], table.shape[1], int(bidirectional), max_distance))


def _run_attention(q, k, v, table, kv_lengths, key_mask, q_pos, k_pos, scale, bidirectional, max_distance, train):
    """-> (out, operands as the kernels read them, 16-bit types' out before its rounding, row log-sums)"""
    b, lq, h, dim = q.shape
    lk, hk = k.shape[1:3]
    if q.numel() == 0 or lk == 0:
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device), (q, k, v), None, None
    lib = _lib.load()
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    out = torch.empty((b, lq, h, dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((2, b, h, lq), dtype=torch.float32, device=q.device) if train else None      # two terms
    out_f32 = torch.empty(out.shape, dtype=torch.float32, device=q.device) if train and q.dtype != torch.float32 else None
    desc = _descriptor(q, k, v, kv_lengths, key_mask, table, q_pos, k_pos, scale, bidirectional, max_distance)
    n = _attention_workspace_bytes(False, train, *_sizes(q, k, table, bidirectional, max_distance))
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    with _on_device(q):
        _lib.launch('camli_cross_attention_fwd', lib.camli_cross_attention_fwd, desc, out.data_ptr(), address(out_f32), address(lse), address(ws), n,
                    _stream_ptr(q), work=(2.0 * q.element_size() * dim * b * (lq * h + lk * hk), 'B'), flop=4.0 * b * h * lq * lk * dim)
    return out, (q, k, v), out_f32, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, kv_lengths, key_mask, q_pos, k_pos, scale, bidirectional, max_distance):
        ctx.args = (scale, bidirectional, max_distance)
        out, operands, out_f32, lse = _run_attention(q, k, v, table, kv_lengths, key_mask, q_pos, k_pos, scale, bidirectional, max_distance, True)
        ctx.save_for_backward(*operands, table, kv_lengths, key_mask, q_pos, k_pos, out if out_f32 is None and lse is not None else out_f32, lse)
        return out

    @first_order
    def backward(ctx, gout):
        q, k, v, table, kv_lengths, key_mask, q_pos, k_pos, out_f32, lse = ctx.saved_tensors
        need_q, need_k, need_v, need_t = ctx.needs_input_grad[:4]
        nothing = (None,) * 7
        if lse is None:
            return (torch.zeros_like(q) if need_q else None, torch.zeros_like(k) if need_k else None,
                    torch.zeros_like(v) if need_v else None, torch.zeros_like(table) if need_t else None) + nothing
        lib = _lib.load()
        b, lq, h, dim = q.shape
        lk, hk = k.shape[1:3]
        gout = gout.contiguous()
        if gout.data_ptr() % 16:
            gout = gout.clone()
        gq = torch.empty((b, lq, h, dim), dtype=q.dtype, device=q.device) if need_q else None
        gk = gv = None
        if need_k or need_v:
            gk = torch.empty((b, lk, hk, dim), dtype=q.dtype, device=q.device)
            gv = torch.empty_like(gk)
        gt = torch.empty(table.shape, dtype=table.dtype, device=q.device) if need_t else None
        desc = _descriptor(q, k, v, kv_lengths, key_mask, table, q_pos, k_pos, *ctx.args)
        n = _attention_workspace_bytes(True, need_t, *_sizes(q, k, table, *ctx.args[1:]))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        with _on_device(q):
            _lib.launch('camli_cross_attention_bwd', lib.camli_cross_attention_bwd, desc, out_f32.data_ptr(), gout.data_ptr(),
                        lse.data_ptr(), address(gq), address(gk), address(gv), address(gt), ws.data_ptr(), n, _stream_ptr(q),
                        work=(4.0 * q.element_size() * dim * b * (lq * h + lk * hk), 'B'), flop=10.0 * b * h * lq * lk * dim)
        return (gq, gk if need_k else None, gv if need_v else None, gt) + nothing


def _composed_attention(q, k, v, scale, kv_lengths, key_mask, bias):
    b, lq, h, dim = q.shape
    lk, hk = k.shape[1:3]
    qh = q.float().permute(0, 2, 1, 3)
    kh, vh = (t.float().permute(0, 2, 1, 3).repeat_interleave(h // hk, dim=1) for t in (k, v))
    keep = torch.ones(b, lk, dtype=torch.bool, device=q.device)
    if kv_lengths is not None:
        keep &= torch.arange(lk, device=q.device) < kv_lengths[:, None]
    if key_mask is not None:
        keep &= key_mask
    rows = keep[:, None, :, None]
    kh, vh = torch.where(rows, kh, torch.zeros_like(kh)), torch.where(rows, vh, torch.zeros_like(vh))
    with torch.autocast(q.device.type, enabled=False):      # 32 bits, like the kernels' sums: autocast would take the products in 16
        scores = torch.matmul(qh, kh.transpose(2, 3).contiguous()) * scale
        if bias is not None:
            scores = scores + bias
        scores = torch.where(keep[:, None, None, :], scores, torch.full_like(scores, -math.inf))
        if lk == 0:         # zeros, in the graph of q, k and v
            return torch.matmul(scores, vh).permute(0, 2, 1, 3).to(q.dtype)
        top = scores.amax(dim=-1, keepdim=True).detach()
        weights = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = weights.sum(dim=-1, keepdim=True)
        return torch.matmul(weights / torch.where(total == 0, torch.ones_like(total), total), vh).permute(0, 2, 1, 3).to(q.dtype)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale=None, kv_lengths=None, key_mask=None, bias_table=None,
                    q_pos=None, k_pos=None, bidirectional=True, max_distance=128, cpp_impl=True):
    """softmax(scale q k^T + bias) v of queries q [B, Lq, H, D] over keys and values k, v [B, Lk, Hk, D] of another length -> [B, Lq, H, D].

    fp32, bf16 or fp16 (one type for all; sums and softmax in fp32).  16-bit types: the probabilities are rounded to the type for the product
    with v (where a gradient is wanted they enter as two terms of it), and they and the gradients of the scores once each for the products
    that give the gradients of v, q and k.  fp32 factors go through the matrix unit as three bf16 parts each, exact to 2^-25, so an infinity
    or a value beyond 3.38e38 among kept fp32 operands gives NaN.  Scores that are all as low as a finite mask entry differ by what fp32 holds
    next to it.  D a multiple of 8 up to 128; H a multiple of Hk (query heads
    h share key / value head h // (H / Hk)).  Any strides: rows that are not adjacent or 16-byte aligned are copied first.  ``scale``:
    from 1e-15 to 1e15, default D ** -0.5.  One token (Lq = 1) and other short queries are split over the keys.

    ``kv_lengths`` int32 [B]: keys from there on are padding (values outside 0 .. Lk are clamped); ``key_mask`` bool [B, Lk]: False masks a
    key; a key is kept if both keep it.  Masked keys and values may hold anything, NaN included, and get zero gradients.  A query that
    keeps no key gives zeros and takes no part in any gradient.

    ``bias_table`` [axes, buckets, H] of q's type with int32 ``q_pos`` [Lq, axes] or [B, Lq, axes] and ``k_pos`` likewise adds the bias
    that :func:`relative_position_bias` describes, without storing it.  Entries may be as low as the type goes, or -inf, which takes their
    pairs out (finite ones beyond +-2.9e37 count as that).  Differentiable in q, k, v and bias_table (once, in reverse mode); the same
    bits on every run.  ``cpp_impl=False``: the same from torch primitives, on any device."""
    name = 'cross_attention'
    if any(t.dim() != 4 for t in (q, k, v)) or q.dtype not in TYPE_CODES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError('%s: q, k, v must be [B, L, H, D] of one type (fp32, bf16, fp16), got %s' % (
            name, ', '.join('%s %s' % (tuple(t.shape), t.dtype) for t in (q, k, v))))
    b, lq, h, dim = q.shape
    lk, hk = k.shape[1:3]
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != dim or hk < 1 or h < 1 or h % hk:
        raise ValueError('%s: shapes do not belong together: q %s, k %s, v %s' % (name, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if dim % 8 or not 8 <= dim <= MAX_HEAD_DIM:
        raise ValueError('%s: the head width must be a multiple of 8 up to %d, got %d' % (name, MAX_HEAD_DIM, dim))
    scale = float(dim) ** -0.5 if scale is None else float(scale)
    if not 1e-15 <= scale <= 1e15:
        raise ValueError('%s: scale must be positive, from 1e-15 to 1e15, got %r' % (name, scale))
    if b * h * ((lq + 31) // 32) >= 2 ** 24 or b * hk * ((lk + 127) // 128) >= 2 ** 24 or h * dim >= 2 ** 23:
        raise ValueError('%s: too many samples x heads x rows for one launch: q %s, k %s' % (name, tuple(q.shape), tuple(k.shape)))
    if kv_lengths is not None and (kv_lengths.shape != (b,) or kv_lengths.dtype != torch.int32):
        raise ValueError('%s: kv_lengths must be int32 [%d], got %s %s' % (name, b, tuple(kv_lengths.shape), kv_lengths.dtype))
    if key_mask is not None and (key_mask.shape != (b, lk) or key_mask.dtype != torch.bool):
        raise ValueError('%s: key_mask must be bool [%d, %d], got %s %s' % (name, b, lk, tuple(key_mask.shape), key_mask.dtype))
    if bias_table is not None or q_pos is not None or k_pos is not None:
        bias_table, q_pos, k_pos, _, _ = _check_bias(name, bias_table, q_pos, k_pos, bidirectional, max_distance, q.dtype, h, b, lq, lk)
    same_device(name, q, k, v, kv_lengths, key_mask, bias_table)
    if not cpp_impl:
        bias = _composed_bias(_within_range(bias_table), q_pos, k_pos, bidirectional, int(max_distance)) if bias_table is not None else None
        return _composed_attention(q, k, v, scale, kv_lengths, key_mask, bias)
    _require_cuda(name, q)
    args = (q, k, v, bias_table, kv_lengths.contiguous() if kv_lengths is not None else None,
            key_mask.contiguous() if key_mask is not None else None, q_pos, k_pos, scale, bool(bidirectional), int(max_distance))
    if needs_node(q, k, v, bias_table):
        return _CrossAttention.apply(*args)
    return _run_attention(*args, False)[0]
