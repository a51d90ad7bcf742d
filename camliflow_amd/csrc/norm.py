"""Group normalisation with an activation on channels-last maps (camli_group_norm_*, csrc/hip/groupnorm.hip).

Stands beside the batch / instance / layer norms of ``cores/blocks.py`` (models/mlp.py:43-100 has no group norm): one pass for
the statistics and one for normalisation, scale, shift and activation together, on the layout the library's NHWC convolutions and
the ``nn.Linear`` layers of the attention modules produce.
"""
import functools
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .wrapper import _on_device, _require_cuda, _stream_ptr

TYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
NORM_ACTS = {None: 0, 'relu': 1, 'leaky_relu': 2, 'sigmoid': 3, 'silu': 6}
MAX_CHANNELS = 4096


def same_device(name, first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError('%s: tensors on %s and %s' % (name, first.device, t.device))


def first_order(backward):
    """A node's backward that refuses to be differentiated again.  Without create_graph there is nothing to refuse, and the
    decorator's bookkeeping (a tenth of a small step's host time) is left out."""
    guarded = once_differentiable(backward)

    def wrapper(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)
    return staticmethod(wrapper)


def needs_node(*tensors):
    """Does a call have to go through its autograd node: a gradient is wanted, or an input carries a forward-mode tangent (which the node
    refuses; the kernels alone would drop it)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    # no level, no tangents: unpacking each tensor to find that out takes a quarter of a small call's host time
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def address(t):
    return t.data_ptr() if t is not None else None


def _dense_strides(b, c, spatial):
    """strides of a dense channels-last map of logical shape [b, c, *spatial]"""
    out, n = [], c
    for size in reversed(spatial):
        out.append(n)
        n *= size
    return (n, 1) + tuple(reversed(out))


def _pitch(shape, stride):
    """(batch stride, pixel pitch) of a [B, C, *spatial] tensor whose channels are adjacent and whose pixels are evenly spaced, or None"""
    if stride[1] != 1 and shape[1] != 1:
        return None
    pitch, span = None, 0
    for n, s in zip(shape[:1:-1], stride[:1:-1]):
        if n > 1:
            if pitch is None:
                pitch, span = s, s * n
            elif s == span:
                span *= n
            else:
                return None
    if pitch is None:
        pitch = span = shape[1]
    return (stride[0] if shape[0] > 1 else span), pitch


def _channel_rows(x):
    """x -> (tensor, batch stride, pixel pitch): x itself where its memory allows (channels-last maps, transposed rows, channel slices
    of wider ones), else a channels-last copy."""
    found = _pitch(x.shape, x.stride())
    if found is not None:
        return x, found[0], found[1]
    x = x.movedim(1, -1).contiguous().movedim(-1, 1)
    return x, x[0].numel(), x.shape[1]


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(b, c, groups, p, code):
    lib = _lib.load()
    return (int(lib.camli_group_norm_fwd_workspace_bytes(b, c, groups, p, code)),
            int(lib.camli_group_norm_bwd_workspace_bytes(b, c, groups, p, code)))


def _run_forward(x, weight, bias, groups, eps, act, keep_stat):
    """-> (y, x as the kernels read it, its pitches, [b, c, groups, positions, act, type, parameter type], stat)"""
    shape = x.shape
    b, c = shape[:2]
    y = torch.empty_strided(shape, _dense_strides(b, c, shape[2:]), dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return y, x, (0, 0), None, None
    p = x.numel() // (b * c)
    code = TYPE_CODES[x.dtype]
    wtype = TYPE_CODES[(weight if weight is not None else bias if bias is not None else x).dtype]
    rows, x_bs, x_ld = _channel_rows(x)
    # one allocation: the statistics (kept for the backward), then the chunks' moments
    head = 2 * b * groups if keep_stat else 0
    n = _workspace_bytes(b, c, groups, p, code)[0]
    buf = torch.empty(head + n // 4, dtype=torch.float32, device=x.device)
    at = buf.data_ptr()
    with _on_device(x):
        _lib.launch('camli_group_norm_fwd', _lib.load().camli_group_norm_fwd, rows.data_ptr(), x_bs, x_ld, address(weight), address(bias),
                    wtype, y.data_ptr(), at if keep_stat else None, at + 4 * head, n, b, c, groups, p, eps, act, code, _stream_ptr(x),
                    work=(2.0 * x.numel() * x.element_size(), 'B'))
    return y, rows, (x_bs, x_ld), (b, c, groups, p, act, code, wtype), buf


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y, rows, ctx.pitch, ctx.args, stat = _run_forward(x, weight, bias, groups, eps, act, True)
        ctx.save_for_backward(rows, weight, bias, stat)
        return y

    @first_order
    def backward(ctx, gy):
        x, weight, bias, stat = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        if ctx.args is None:
            return (torch.zeros_like(x) if need_x else None, torch.zeros_like(weight) if need_w else None,
                    torch.zeros_like(bias) if need_b else None, None, None, None)
        b, c, groups, p, act, code, wtype = ctx.args
        x_bs, x_ld = ctx.pitch
        dense = _dense_strides(b, c, x.shape[2:])
        if gy.stride() != dense:
            gy = gy.movedim(1, -1).contiguous()
        gx = torch.empty_strided(x.shape, dense, dtype=x.dtype, device=x.device) if need_x else None
        gw = torch.empty(c, dtype=torch.float32, device=x.device) if need_w else None
        gb = torch.empty(c, dtype=torch.float32, device=x.device) if need_b else None
        n = _workspace_bytes(b, c, groups, p, code)[1]
        ws = torch.empty(n, dtype=torch.uint8, device=x.device)
        with _on_device(x):
            _lib.launch('camli_group_norm_bwd', _lib.load().camli_group_norm_bwd, gy.data_ptr(), x.data_ptr(), x_bs, x_ld, address(weight),
                        address(bias), wtype, stat.data_ptr(), address(gx), address(gw), address(gb), ws.data_ptr(), n, b, c, groups, p, act,
                        code, _stream_ptr(x), work=(3.0 * x.numel() * x.element_size(), 'B'))
        if wtype:
            gw, gb = gw.to(weight.dtype) if need_w else None, gb.to(bias.dtype) if need_b else None
        return gx, gw, gb, None, None, None


def _composed(x, groups, weight, bias, eps, act):
    shape = x.shape
    grouped = x.float().reshape(shape[0], groups, shape[1] // groups * math.prod(shape[2:]))
    centred = grouped - grouped.mean(dim=2, keepdim=True)
    z = (centred * torch.rsqrt((centred * centred).mean(dim=2, keepdim=True) + eps)).reshape(shape)
    per_channel = (1, -1) + (1,) * (x.dim() - 2)
    if weight is not None:
        z = z * weight.float().view(per_channel)
    if bias is not None:
        z = z + bias.float().view(per_channel)
    if act == 'relu':
        z = torch.relu(z)
    elif act == 'leaky_relu':
        z = torch.nn.functional.leaky_relu(z, 0.1)
    elif act == 'sigmoid':
        z = torch.sigmoid(z)
    elif act == 'silu':
        z = z * torch.sigmoid(z)
    return z.to(x.dtype)


def group_norm_act(x: torch.Tensor, num_groups: int, weight=None, bias=None, eps=1e-5, act=None, cpp_impl=True):
    """act(group_norm(x) * weight + bias) of a map x [B, C, *spatial] (fp32, bf16 or fp16), statistics over each sample's group of
    C / num_groups channels and all positions, in fp32.  ``act``: None, 'relu', 'leaky_relu' (0.1), 'sigmoid' or 'silu'.

    The kernels work on channels-last memory: x may be a channels-last map, rows [B, N, C] seen as x.transpose(1, 2), or a channel slice
    of a wider one; anything else is copied to that layout first.  The result is [B, C, *spatial] on dense channels-last memory, of
    x's type.  ``weight`` and ``bias`` [C] (either may be None) are fp32 or of x's type.  Differentiable in x, weight and bias
    (once, in reverse mode); no float atomics, the same bits on every run.  ``cpp_impl=False``: the same formula from torch primitives, on any device."""
    name = 'group_norm_act'
    shape = x.shape
    if len(shape) < 2 or x.dtype not in TYPE_CODES:
        raise ValueError('%s: x must be [B, C, ...] of type fp32, bf16 or fp16, got %s %s' % (name, tuple(shape), x.dtype))
    c = shape[1]
    if not 1 <= num_groups <= c or c % num_groups or c > MAX_CHANNELS:
        raise ValueError('%s: %d channels (at most %d) do not split into %d groups' % (name, c, MAX_CHANNELS, num_groups))
    if act not in NORM_ACTS:
        raise ValueError('%s: unknown activation %r' % (name, act))
    if not eps >= 0:
        raise ValueError('%s: eps must not be negative, got %r' % (name, eps))
    for t in (weight, bias):
        if t is not None and (t.shape != (c,) or t.dtype not in (torch.float32, x.dtype)):
            raise ValueError('%s: weight and bias must be [%d], fp32 or of the type of x, got %s %s' % (name, c, tuple(t.shape), t.dtype))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError('%s: weight and bias of different types (%s, %s)' % (name, weight.dtype, bias.dtype))
    if shape[0] > 65535 or x.numel() // max(1, shape[0] * c) >= 2 ** 31 - 2 ** 16:
        raise ValueError('%s: more than 65535 samples or 2^31 positions: %s' % (name, tuple(shape)))
    same_device(name, x, weight, bias)
    if not cpp_impl:
        return _composed(x, num_groups, weight, bias, eps, act)
    _require_cuda(name, x)
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if needs_node(x, weight, bias):
        return _GroupNormAct.apply(x, weight, bias, num_groups, eps, NORM_ACTS[act])
    return _run_forward(x, weight, bias, num_groups, eps, NORM_ACTS[act], False)[0]
