"""Bidirectional camera-LiDAR fusion module, CLFM (counterpart of models/clfm.py).

2D<-3D: ``FusionAwareInterp`` -- every pixel takes its nearest projected point (2-D KNN, k=1), a
score MLP on the pixel offset gates the point feature, then a 1x1 conv.
3D<-2D: bilinear sample of the image feature at the projected points.
Both directions are merged by selective-kernel fusion (``SKFusion``, the default) or the add /
concat / gated variants.  ``fusion_fn='attn'`` (not in the reference) replaces nearest point, sample and merge by cross attention: every
pixel attends every point and the other way round (``CrossAttend``).  Inputs to the cross paths are detached exactly where the reference
detaches them (clfm.py:34,37-38).
"""
import torch
import torch.nn as nn
from torch.nn.functional import softmax

from ..csrc import attention as _attention
from ..csrc import wrapper as _ops
from . import runtime
from .blocks import Conv1dNormRelu, Conv2dNormRelu, GroupNormAct
from .geometry import batch_indexing, grid_sample_wrapper, mesh_grid


def _aligner(feat_format):
    if feat_format == 'nchw':
        return Conv2dNormRelu
    if feat_format == 'ncm':
        return Conv1dNormRelu
    raise ValueError(feat_format)


class FusionAwareInterp(nn.Module):
    def __init__(self, n_channels_3d, k=1, norm=None):
        super().__init__()
        self.k = k
        self.out_conv = Conv2dNormRelu(n_channels_3d, n_channels_3d, norm=norm)
        self.score_net = nn.Sequential(
            Conv2dNormRelu(3, 16),
            Conv2dNormRelu(16, n_channels_3d, act='sigmoid'),
        )

    def _geometry(self, uv, grid, image_h, image_w):
        """(knn_indices, score) for this module.  The reference recomputes the 2-D KNN of every pixel
        and ``score_net(offset, |offset|)`` in every CLFM call although (uv, grid) never change across
        GRU iterations (11 calls per 4-iteration forward).  Inside a ``pass_cache()`` the
        index tensor is shared by every CLFM that sees the same ``uv`` and the score is evaluated once
        per module; its gradient is accumulated by autograd over the iterations.  Same values."""
        from . import setconv
        cache = setconv._pass_cache
        base = (uv.data_ptr(), tuple(uv.shape), image_h, image_w, self.k, torch.is_grad_enabled())
        knn_key, score_key = ('knn2d',) + base, ('score2d', id(self)) + base
        if cache is not None and score_key in cache:
            return cache[knn_key][0], cache[score_key][0]
        knn_indices = cache[knn_key][0] if cache is not None and knn_key in cache else None
        if knn_indices is None:
            knn_indices = _ops.k_nearest_neighbor(uv, grid, self.k)
        knn_offset = batch_indexing(uv, knn_indices) - grid[..., None]
        knn_offset_norm = torch.linalg.norm(knn_offset, dim=1, keepdim=True)
        score = self.score_net(torch.cat([knn_offset, knn_offset_norm], dim=1))
        if cache is not None:   # entries keep `uv` alive: the key is its address
            cache[knn_key], cache[score_key] = (knn_indices, uv), (score, uv)
        return knn_indices, score

    def forward(self, uv, feat_2d, feat_3d):
        bs, _, image_h, image_w = feat_2d.shape
        n_channels_3d = feat_3d.shape[1]
        grid = mesh_grid(bs, image_h, image_w, uv.device).reshape(bs, 2, -1)       # [B,2,HW]
        if runtime.fused():
            # the pixel -> nearest-point assignment and the score it induces depend only on
            # (uv, grid size), not on the features: one evaluation per pass (see _geometry)
            knn_indices, score = self._geometry(uv, grid, image_h, image_w)
            if self.k == 1 and feat_3d.is_cuda and not feat_3d.requires_grad:
                from ..csrc import fused          # gather * score in one launch (its own adjoint wrt the score)
                # squeeze, not [..., 0]: a view's adjoint is free, a select's is a zero fill + a copy of the [B,C,HW] score
                final = fused.gather_scale(feat_3d, score.squeeze(-1), knn_indices[..., 0])
                return self.out_conv(final.reshape(bs, -1, image_h, image_w))
            knn_feat3d = batch_indexing(feat_3d, knn_indices)                       # [B,C,HW,k]
        else:
            knn_indices = _ops.k_nearest_neighbor(uv, grid, self.k)                 # [B,HW,k]
            gathered = batch_indexing(torch.cat([uv, feat_3d], dim=1), knn_indices)    # [B,2+C,HW,k]
            knn_uv, knn_feat3d = torch.split(gathered, [2, n_channels_3d], dim=1)
            knn_offset = knn_uv - grid[..., None]
            knn_offset_norm = torch.linalg.norm(knn_offset, dim=1, keepdim=True)
            score = self.score_net(torch.cat([knn_offset, knn_offset_norm], dim=1))    # [B,C,HW,k]
        final = (score * knn_feat3d).sum(dim=-1).reshape(bs, -1, image_h, image_w)
        return self.out_conv(final)


class AddFusion(nn.Module):
    def __init__(self, in_channels_2d, in_channels_3d, out_channels, feat_format, norm=None):
        super().__init__()
        conv = _aligner(feat_format)
        self.align1 = conv(in_channels_2d, out_channels, norm=norm)
        self.align2 = conv(in_channels_3d, out_channels, norm=norm)
        self.relu = nn.LeakyReLU(negative_slope=0.1, inplace=True)

    def forward(self, feat_2d, feat_3d):
        return self.relu(self.align1(feat_2d) + self.align2(feat_3d))


class ConcatFusion(nn.Module):
    def __init__(self, in_channels_2d, in_channels_3d, out_channels, feat_format, norm=None):
        super().__init__()
        self.mlp = _aligner(feat_format)(in_channels_2d + in_channels_3d, out_channels, norm=norm)

    def forward(self, feat_2d, feat_3d):
        return self.mlp(torch.cat([feat_2d, feat_3d], dim=1))


class GatedFusion(nn.Module):
    def __init__(self, in_channels_2d, in_channels_3d, out_channels, feat_format, norm=None):
        super().__init__()
        conv = _aligner(feat_format)
        self.align1 = conv(in_channels_2d, out_channels, norm=norm)
        self.align2 = conv(in_channels_3d, out_channels, norm=norm)
        self.mlp1 = conv(out_channels, 2, norm=None, act='sigmoid')
        self.mlp2 = conv(out_channels, 2, norm=None, act='sigmoid')

    def forward(self, feat_2d, feat_3d):
        feat_2d, feat_3d = self.align1(feat_2d), self.align2(feat_3d)
        weight = softmax(self.mlp1(feat_2d) + self.mlp2(feat_3d), dim=1)
        return feat_2d * weight[:, 0:1] + feat_3d * weight[:, 1:2]


class SKFusion(nn.Module):
    """Selective-kernel fusion (clfm.py:170-213): channel attention from the pooled sum decides,
    per channel, the mix between the two aligned branches."""

    def __init__(self, in_channels_2d, in_channels_3d, out_channels, feat_format, norm=None, reduction=1):
        super().__init__()
        conv = _aligner(feat_format)
        self.align1 = conv(in_channels_2d, out_channels, norm=norm)
        self.align2 = conv(in_channels_3d, out_channels, norm=norm)
        self.avg_pool = nn.AdaptiveAvgPool2d(1) if feat_format == 'nchw' else nn.AdaptiveAvgPool1d(1)
        self.fc_mid = nn.Sequential(nn.Linear(out_channels, out_channels // reduction, bias=False), nn.ReLU(inplace=True))
        self.fc_out = nn.Sequential(nn.Linear(out_channels // reduction, out_channels * 2, bias=False), nn.Sigmoid())

    def forward(self, feat_2d, feat_3d):
        bs = feat_2d.shape[0]
        feat_2d, feat_3d = self.align1(feat_2d), self.align2(feat_3d)
        if runtime.fused() and feat_2d.is_cuda and bs * feat_2d.shape[1] > 65535:
            runtime.fallback('SKFusion', 'B*C = %d exceeds the kernels\' grid limit 65535' % (bs * feat_2d.shape[1]))
        if runtime.fused() and feat_2d.is_cuda and bs * feat_2d.shape[1] <= 65535:
            # pooled sum, mix and both adjoints as four streaming kernels (camli_sk_*); the gate stays in torch
            from ..csrc import fused
            state = fused.SkState()
            squeezed = fused.sk_pool(feat_2d, feat_3d, state)
            w_mid, w_out = self.fc_mid[0].weight, self.fc_out[0].weight
            if w_mid.shape[1] <= 1024 and w_mid.shape[0] <= 512:
                weight = fused.sk_gate(squeezed, w_mid, w_out)           # the whole gate: one launch forward, two backward (no atomics)
            else:
                runtime.fallback('sk_gate', 'C=%d R=%d outside the gate kernel (C<=1024, R<=512)' % (w_mid.shape[1], w_mid.shape[0]))
                weight = softmax(self.fc_out(self.fc_mid(squeezed)).reshape(bs, -1, 2), dim=-1)
            return fused.sk_mix(feat_2d, feat_3d, weight, state)
        squeezed = self.avg_pool(feat_2d + feat_3d).reshape(bs, -1)
        weight = softmax(self.fc_out(self.fc_mid(squeezed)).reshape(bs, -1, 2), dim=-1)
        bshape = [bs, -1] + [1] * (feat_2d.dim() - 2)
        return feat_2d * weight[..., 0].reshape(bshape) + feat_3d * weight[..., 1].reshape(bshape)


class CrossAttend(nn.Module):
    """x + out(attention(q(norm(x)), kv(norm(context)))) with a learned bias by the bucketed image offset of query and key, per axis.

    x [B, Cx, ...] and context [B, Cc, ...] are maps of any spatial shape (pixels or points); positions are int32 [L, 2] or [B, L, 2] pixel
    coordinates.  Heads are 32 wide.  The output projection starts at zero: a fresh module passes x through."""
    HEAD = 32

    def __init__(self, channels, context_channels, buckets=32, max_distance=64):
        super().__init__()
        self.heads = max(1, channels // self.HEAD)
        self.max_distance = max_distance
        inner = self.heads * self.HEAD
        self.norm_x, self.norm_context = GroupNormAct(channels), GroupNormAct(context_channels)
        self.to_q = nn.Linear(channels, inner, bias=False)
        self.to_kv = nn.Linear(context_channels, 2 * inner, bias=False)
        self.out = nn.Linear(inner, channels)
        nn.init.zeros_(self.out.weight)
        nn.init.zeros_(self.out.bias)
        self.bias_table = nn.Parameter(torch.zeros(2, buckets, self.heads))

    def forward(self, x, context, x_pos, context_pos):
        rows = self.norm_x(x).movedim(1, -1).flatten(1, -2)                         # [B, L, C], a view: the norm's memory is that
        context_rows = self.norm_context(context).movedim(1, -1).flatten(1, -2)
        q = self.to_q(rows).unflatten(-1, (self.heads, self.HEAD))
        k, v = self.to_kv(context_rows).unflatten(-1, (2, self.heads, self.HEAD)).unbind(2)
        att = _attention.cross_attention(q, k, v, bias_table=self.bias_table.to(q.dtype), q_pos=x_pos, k_pos=context_pos,
                                         max_distance=self.max_distance, cpp_impl=runtime.fused())
        return x + self.out(att.flatten(2)).transpose(1, 2).reshape(x.shape)


_FUSIONS = {'add': (AddFusion, {}), 'concat': (ConcatFusion, {}), 'gated': (GatedFusion, {}),
            'sk': (SKFusion, {'reduction': 2})}


class CLFM(nn.Module):
    """``norm`` is that of the interpolation's and the merge's layers; ``fusion_fn='attn'`` has neither, and group norms of its own."""

    def __init__(self, in_channels_2d, in_channels_3d, fusion_fn='sk', norm=None):
        super().__init__()
        self.attends = fusion_fn == 'attn'
        if self.attends:
            self.attend2d = CrossAttend(in_channels_2d, in_channels_3d)
            self.attend3d = CrossAttend(in_channels_3d, in_channels_2d)
            return
        self.interp = FusionAwareInterp(in_channels_3d, k=1, norm=norm)
        self.mlps3d = Conv1dNormRelu(in_channels_2d, in_channels_2d, norm=norm)
        if fusion_fn not in _FUSIONS:
            raise ValueError(fusion_fn)
        cls, extra = _FUSIONS[fusion_fn]
        self.fuse2d = cls(in_channels_2d, in_channels_3d, in_channels_2d, 'nchw', norm, **extra)
        self.fuse3d = cls(in_channels_2d, in_channels_3d, in_channels_3d, 'ncm', norm, **extra)

    def _attend(self, uv, feat_2d, feat_3d):
        bs, _, image_h, image_w = feat_2d.shape
        pixels = mesh_grid(1, image_h, image_w, uv.device).reshape(2, -1).t().to(torch.int32).contiguous()            # [HW, 2]
        # projections far outside the image share the last bucket anyway
        points = uv.detach().nan_to_num().clamp(-2.0 ** 20, 2.0 ** 20).round().to(torch.int32).transpose(1, 2).contiguous()
        branch = runtime.Branch(feat_2d, feat_3d, points, pixels, slot=2)
        with branch:
            out3d = self.attend3d(feat_3d, feat_2d.detach(), points, pixels)
        out2d = self.attend2d(feat_2d, feat_3d.detach(), pixels, points)
        branch.join(out3d)
        return out2d, out3d

    def forward(self, uv, feat_2d, feat_3d):
        feat_2d, feat_3d = feat_2d.float(), feat_3d.float()
        if self.attends:
            return self._attend(uv, feat_2d, feat_3d)
        # the two directions are independent chains: 3D<-2D (a dozen kernels on [B,C,2048] tensors, latency-sized) goes to
        # an auxiliary stream next to 2D<-3D (runtime.Branch; one stream when the lanes are off)
        branch = runtime.Branch(feat_2d, feat_3d, uv, slot=2)
        with branch:
            feat_2d_sampled = grid_sample_wrapper(feat_2d.detach(), uv)
            out3d = self.fuse3d(self.mlps3d(feat_2d_sampled.detach()), feat_3d)
        feat_3d_interp = self.interp(uv, feat_2d.detach(), feat_3d.detach())
        out2d = self.fuse2d(feat_2d, feat_3d_interp)
        branch.join(out3d)
        return out2d, out3d
