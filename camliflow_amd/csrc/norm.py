"""Group normalisation with an activation on channels-last maps (camli_group_norm_*, csrc/hip/groupnorm.hip).

Stands beside the batch / instance / layer norms of ``cores/blocks.py`` (models/mlp.py:43-100 has no group norm): one pass for
the statistics and one for normalisation, scale, shift and activation together, on the layout the library's NHWC convolutions and
the ``nn.Linear`` layers of the attention modules produce.
"""
import torch
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


def _channel_rows(x):
    """x [B, C, *spatial] -> (tensor, batch stride, pixel pitch) with adjacent channels and evenly spaced pixels: x itself where its
    memory is that (channels-last maps, transposed rows, channel slices of wider ones), else a channels-last copy."""
    c = x.shape[1]
    if c == 1 or x.stride(1) == 1:
        dims = [(n, s) for n, s in zip(x.shape[2:], x.stride()[2:]) if n > 1]
        if all(s0 == n1 * s1 for (_, s0), (n1, s1) in zip(dims[:-1], dims[1:])):
            pitch = dims[-1][1] if dims else c
            return x, (x.stride(0) if x.shape[0] > 1 else pitch * x[0, 0].numel()), pitch
    x = x.movedim(1, -1).contiguous().movedim(-1, 1)
    return x, x[0].numel(), c


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    @torch.amp.custom_fwd(device_type='cuda')
    def forward(ctx, x, weight, bias, groups, eps, act):
        lib = _lib.load()
        b, c = x.shape[:2]
        spatial = tuple(x.shape[2:])
        y = torch.empty((b,) + spatial + (c,), dtype=x.dtype, device=x.device).movedim(-1, 1)
        ctx.dims = (b, c, spatial, groups, act)
        if x.numel() == 0:
            ctx.save_for_backward(x, weight, bias, None)
            return y
        p = x[0, 0].numel()
        code = TYPE_CODES[x.dtype]
        rows, x_bs, x_ld = _channel_rows(x)
        stat = torch.empty((b, groups, 2), dtype=torch.float32, device=x.device) if any(ctx.needs_input_grad[:3]) else None
        ws_bytes = int(lib.camli_group_norm_fwd_workspace_bytes(b, c, groups, p, code))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=x.device)
        wtype = TYPE_CODES[(weight if weight is not None else bias if bias is not None else x).dtype]
        with _on_device(x):
            _lib.launch('camli_group_norm_fwd', lib.camli_group_norm_fwd, rows.data_ptr(), x_bs, x_ld,
                        weight.data_ptr() if weight is not None else None, bias.data_ptr() if bias is not None else None, wtype,
                        y.data_ptr(), stat.data_ptr() if stat is not None else None, ws.data_ptr(), ws_bytes, b, c, groups, p, eps, act,
                        code, _stream_ptr(x), work=(2.0 * x.numel() * x.element_size(), 'B'))
        ctx.save_for_backward(rows, weight, bias, stat)
        return y

    @staticmethod
    @torch.amp.custom_bwd(device_type='cuda')
    @once_differentiable
    def backward(ctx, gy):
        lib = _lib.load()
        x, weight, bias, stat = ctx.saved_tensors
        b, c, spatial, groups, act = ctx.dims
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        if x.numel() == 0:
            return (torch.zeros_like(x) if need_x else None, torch.zeros_like(weight) if need_w else None,
                    torch.zeros_like(bias) if need_b else None, None, None, None)
        p = x[0, 0].numel()
        code = TYPE_CODES[x.dtype]
        x, x_bs, x_ld = _channel_rows(x)
        gy = gy.movedim(1, -1).contiguous()
        gx = torch.empty((b,) + spatial + (c,), dtype=x.dtype, device=x.device).movedim(-1, 1) if need_x else None
        gw = torch.empty(c, dtype=torch.float32, device=x.device) if need_w else None
        gb = torch.empty(c, dtype=torch.float32, device=x.device) if need_b else None
        ws_bytes = int(lib.camli_group_norm_bwd_workspace_bytes(b, c, groups, p, code))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
        wtype = TYPE_CODES[(weight if weight is not None else bias if bias is not None else x).dtype]

        def ptr(t):
            return t.data_ptr() if t is not None else None
        with _on_device(x):
            _lib.launch('camli_group_norm_bwd', lib.camli_group_norm_bwd, gy.data_ptr(), x.data_ptr(), x_bs, x_ld, ptr(weight), ptr(bias),
                        wtype, stat.data_ptr(), ptr(gx), ptr(gw), ptr(gb), ws.data_ptr(), ws_bytes, b, c, groups, p, act, code,
                        _stream_ptr(x), work=(3.0 * x.numel() * x.element_size(), 'B'))
        return (gx, gw.to(weight.dtype) if need_w else None, gb.to(bias.dtype) if need_b else None, None, None, None)


def _composed(x, groups, weight, bias, eps, act):
    shape = x.shape
    grouped = x.float().reshape(shape[0], groups, -1)
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
    (once); no float atomics, the same bits on every run.  ``cpp_impl=False``: the same formula from torch primitives, on any device."""
    name = 'group_norm_act'
    if x.dim() < 2 or x.dtype not in TYPE_CODES:
        raise ValueError('%s: x must be [B, C, ...] of type fp32, bf16 or fp16, got %s %s' % (name, tuple(x.shape), x.dtype))
    c = x.shape[1]
    if not (1 <= num_groups <= c) or c % num_groups or c > MAX_CHANNELS:
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
    if x.shape[0] > 65535 or x[:1, :1].numel() >= 2 ** 31 - 2 ** 16:
        raise ValueError('%s: more than 65535 samples or 2^31 positions: %s' % (name, tuple(x.shape)))
    same_device(name, x, weight, bias)
    if not cpp_impl:
        return _composed(x, num_groups, weight, bias, eps, act)
    _require_cuda(name, x)
    return _GroupNormAct.apply(x, weight.contiguous() if weight is not None else None, bias.contiguous() if bias is not None else None,
                               int(num_groups), float(eps), NORM_ACTS[act])
