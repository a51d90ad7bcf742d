"""Cross attention, position bias and group norm without a GPU: refusals, the composed formulations against 64-bit restatements, the bucket
borders of the library, the modules built on the operators."""
import ctypes

import pytest
import torch

import attnref
from camliflow_amd import csrc
from camliflow_amd.csrc import _lib


def _qkv(b=2, lq=5, lk=7, h=4, hk=2, d=16, dtype=torch.float32):
    g = torch.Generator().manual_seed(0)
    return tuple(torch.randn(b, n, m, d, generator=g).to(dtype) for n, m in ((lq, h), (lk, hk), (lk, hk)))


def _pos(n, axes=1):
    return torch.zeros(n, axes, dtype=torch.int32)


@pytest.mark.parametrize('change', [
    dict(q=torch.zeros(2, 5, 4)), dict(q=torch.zeros(2, 5, 4, 16, dtype=torch.float64)), dict(k=torch.zeros(2, 7, 2, 16, dtype=torch.bfloat16)),
    dict(v=torch.zeros(2, 8, 2, 16)), dict(k=torch.zeros(3, 7, 2, 16), v=torch.zeros(3, 7, 2, 16)), dict(k=torch.zeros(2, 7, 3, 16), v=torch.zeros(2, 7, 3, 16)),
    dict(k=torch.zeros(2, 7, 0, 16), v=torch.zeros(2, 7, 0, 16)), dict(scale=0.0), dict(scale=-1.0), dict(scale=float('inf')), dict(scale=float('nan')), dict(scale=1e-16), dict(scale=1e16),
    dict(kv_lengths=torch.zeros(2, dtype=torch.int64)), dict(kv_lengths=torch.zeros(3, dtype=torch.int32)), dict(key_mask=torch.ones(2, 7)),
    dict(key_mask=torch.ones(7, dtype=torch.bool)), dict(bias_table=torch.zeros(1, 8, 4)), dict(q_pos=_pos(5)),
    dict(bias_table=torch.zeros(1, 8, 3), q_pos=_pos(5), k_pos=_pos(7)), dict(bias_table=torch.zeros(8, 4), q_pos=_pos(5), k_pos=_pos(7)),
    dict(bias_table=torch.zeros(1, 8, 4).half(), q_pos=_pos(5), k_pos=_pos(7)), dict(bias_table=torch.zeros(3, 8, 4), q_pos=_pos(5, 3), k_pos=_pos(7, 3)),
    dict(bias_table=torch.zeros(1, 130, 4), q_pos=_pos(5), k_pos=_pos(7)), dict(bias_table=torch.zeros(1, 7, 4), q_pos=_pos(5), k_pos=_pos(7)),
    dict(bias_table=torch.zeros(1, 8, 4), q_pos=_pos(6), k_pos=_pos(7)), dict(bias_table=torch.zeros(1, 8, 4), q_pos=_pos(5), k_pos=_pos(7).long()),
    dict(bias_table=torch.zeros(1, 8, 4), q_pos=_pos(5)[None].expand(3, -1, -1), k_pos=_pos(7)),
    dict(bias_table=torch.zeros(1, 8, 4), q_pos=_pos(5), k_pos=_pos(7), max_distance=2),
    dict(bias_table=torch.zeros(1, 8, 4), q_pos=_pos(5), k_pos=_pos(7), max_distance=1024),
    dict(bias_table=torch.zeros(1, 8, 4), q_pos=_pos(5), k_pos=_pos(7), max_distance=16.5)])
def test_attention_refuses(change):
    q, k, v = _qkv()
    args = dict(dict(q=q, k=k, v=v), **change)
    with pytest.raises(ValueError, match='cross_attention'):
        csrc.cross_attention(args.pop('q'), args.pop('k'), args.pop('v'), cpp_impl=False, **args)


@pytest.mark.parametrize('d', [4, 12, 136, 256])
def test_attention_refuses_head_widths(d):
    with pytest.raises(ValueError, match='head width'):
        csrc.cross_attention(*_qkv(d=d), cpp_impl=False)


@pytest.mark.parametrize('args', [
    dict(num_groups=0), dict(num_groups=3), dict(num_groups=16), dict(act='gelu'), dict(eps=-1e-5), dict(eps=float('nan')), dict(weight=torch.ones(7)),
    dict(weight=torch.ones(8).half()), dict(weight=torch.ones(8, dtype=torch.float64)), dict(x=torch.zeros(8)), dict(x=torch.zeros(2, 8, 3, dtype=torch.int32)),
    dict(x=torch.zeros(2, 8, 3, dtype=torch.float64)), dict(x=torch.zeros(1, 8192, 1)),
    dict(x=torch.zeros(2, 8, 3).half(), weight=torch.ones(8).half(), bias=torch.ones(8))])
def test_group_norm_refuses(args):
    args = dict(dict(x=torch.zeros(2, 8, 3), num_groups=2), **args)
    with pytest.raises(ValueError, match='group_norm_act'):
        csrc.group_norm_act(args.pop('x'), args.pop('num_groups'), cpp_impl=False, **args)


def test_bias_refuses():
    for table, q, k, kw in ((torch.zeros(1, 8, 2, dtype=torch.float64), _pos(3), _pos(3), {}), (torch.zeros(1, 8, 2), _pos(3), _pos(3, 2), {}),
                            (torch.zeros(1, 8, 2), _pos(3)[None].expand(2, -1, -1), _pos(3)[None].expand(3, -1, -1), {}),
                            (torch.zeros(1, 2, 2), _pos(3), _pos(3), {}), (torch.zeros(1, 1, 2), _pos(3), _pos(3), dict(bidirectional=False)),
                            (torch.zeros(1, 8, 2), None, _pos(3), {})):
        with pytest.raises(ValueError, match='relative_position_bias'):
            csrc.relative_position_bias(table, q, k, cpp_impl=False, **kw)


def test_bias_refuses_more_heads_than_a_launch_holds():
    wide = torch.zeros(1).expand(1, 8, 65536)
    with pytest.raises(ValueError, match='65535'):
        csrc.relative_position_bias(wide, _pos(3), _pos(3), cpp_impl=False)
    with pytest.raises(ValueError, match='65535'):
        csrc.cross_attention(torch.zeros(1).expand(1, 3, 65536, 8), *[torch.zeros(1, 3, 1, 8)] * 2, bias_table=wide, q_pos=_pos(3), k_pos=_pos(3), cpp_impl=False)


def test_bias_positions_count_as_their_bound():
    table = torch.arange(8, dtype=torch.float32).view(1, 8, 1)
    far = torch.tensor([[2 ** 31 - 1], [2 ** 26], [2 ** 26 - 1], [-2 ** 31]], dtype=torch.int32)
    got = csrc.relative_position_bias(table, far, far, max_distance=8, cpp_impl=False)[0]
    assert got.tolist() == [[0, 0, 1, 3], [0, 0, 1, 3], [5, 5, 0, 3], [7, 7, 7, 0]]


@pytest.mark.skipif(torch.cuda.is_available(), reason='CPU-only behaviour')
def test_operators_refuse_cpu_tensors():
    with pytest.raises(_lib.CamliHipError):
        csrc.cross_attention(*_qkv())
    with pytest.raises(_lib.CamliHipError):
        csrc.group_norm_act(torch.zeros(2, 8, 3), 2)
    with pytest.raises(_lib.CamliHipError):
        csrc.relative_position_bias(torch.zeros(1, 8, 2), _pos(3), _pos(3))


def test_attention_refuses_what_one_launch_cannot_hold():
    one = torch.zeros(1)
    for q, k in (((2 ** 24, 1, 1, 8), (2 ** 24, 1, 1, 8)), ((1, 1, 2 ** 20, 8), (1, 1, 1, 8)), ((1, 2 ** 29, 1, 8), (1, 1, 1, 8))):
        with pytest.raises(ValueError, match='too many'):
            csrc.cross_attention(one.expand(q), one.expand(k), one.expand(k))


def test_c_entries_refuse_and_report():
    """the C boundary checks for itself: nothing is launched and no exception crosses it"""
    lib = _lib.load()
    null = None
    assert lib.camli_group_norm_fwd(null, 0, 0, null, null, 0, null, null, null, 0, 1, 8, 2, 3, 1e-5, 0, 0, null) == -22
    assert b'null' in lib.camli_last_error_string()
    assert lib.camli_group_norm_fwd(1, 0, 0, null, null, 0, 1, null, 1, 1 << 30, 1, 8, 3, 3, 1e-5, 0, 0, null) == -22
    assert lib.camli_group_norm_bwd(1, 1, 0, 0, null, null, 0, 1, 1, null, null, 1, 0, 1, 8, 2, 3, 0, 0, null) == -22
    assert lib.camli_group_norm_fwd_workspace_bytes(1, 8192, 2, 3, 0) == 0
    assert lib.camli_rel_bias_fwd(1, 1, 0, 1, 0, 1, 1, 1, 3, 3, 1, 300, 1, 128, 0, null) == -22
    assert lib.camli_rel_bias_bwd(1, 1, 0, 1, 0, 1, 1, 0, 1, 1, 3, 3, 1, 32, 1, 128, 0, null) == -22
    d = _lib.AttentionDesc()
    assert lib.camli_cross_attention_fwd_workspace_bytes(null, 0) == -22
    assert lib.camli_cross_attention_fwd(ctypes.byref(d), 16, null, null, null, 0, null) == -22
    for name, value in (('type', 0), ('B', 1), ('H', 2), ('Hk', 1), ('Lq', 3), ('Lk', 4), ('D', 32), ('scale', 0.2)):
        setattr(d, name, value)
    d.q, d.k, d.v = 4096, 8192, 12288
    for s in (d.q_stride, d.k_stride, d.v_stride):
        s[0], s[1], s[2] = 0, 64, 32
    assert lib.camli_cross_attention_fwd_workspace_bytes(ctypes.byref(d), 0) >= 0
    assert lib.camli_cross_attention_bwd_workspace_bytes(ctypes.byref(d), 0) > 0
    for name, bad in (('D', 36), ('D', 0), ('H', 3), ('Lk', 0), ('B', 0), ('type', 3), ('scale', 0.0), ('scale', 1e-16), ('k', 8200), ('bias_axes', 1), ('Lq', 2 ** 31 - 1)):
        keep = getattr(d, name)
        d.Hk = 2 if name == 'H' else 1
        setattr(d, name, bad)
        assert lib.camli_cross_attention_fwd_workspace_bytes(ctypes.byref(d), 0) == -22, name
        assert lib.camli_cross_attention_bwd(ctypes.byref(d), 16, 16, 16, 16, 16, 16, null, 16, 1 << 30, null) == -22, name
        setattr(d, name, keep)
    for row in (-64, 2 ** 23, 66):
        d.k_stride[1] = row
        assert lib.camli_cross_attention_fwd(ctypes.byref(d), 16, null, null, 16, 1 << 30, null) == -22
    d.k_stride[1] = 64
    assert lib.camli_cross_attention_fwd(ctypes.byref(d), 24, null, null, 16, 1 << 30, null) == -22       # unaligned output
    assert lib.camli_cross_attention_bwd(ctypes.byref(d), 16, 16, 16, 16, 16, null, null, 16, 1 << 30, null) == -22     # one of gk, gv
    assert lib.camli_cross_attention_bwd(ctypes.byref(d), 16, 16, 16, 16, 16, 16, null, 16, 0, null) == -22            # no workspace


@pytest.mark.parametrize('buckets,two_sided,limit', [(32, 1, 128), (32, 0, 128), (8, 1, 48), (64, 0, 100), (64, 1, 1023), (128, 0, 1023), (4, 1, 2), (2, 0, 2),
                                                     (128, 0, 65), (6, 1, 3), (7, 0, 4)])
def test_library_borders_equal_whole_number_definition(buckets, two_sided, limit):
    lib = _lib.load()
    border = (ctypes.c_int * 64)()
    n = lib.camli_rel_bias_borders(buckets, two_sided, limit, border)
    side = buckets // 2 if two_sided else buckets
    e = side // 2
    assert n == side - e - 1
    for o in range(-limit - 3, limit + 4):
        d = abs(o) if two_sided else max(-o, 0)
        mine = d if d < e else e + sum(border[j] <= d for j in range(n))
        assert mine + (side if two_sided and o > 0 else 0) == attnref.bucket(o, buckets, bool(two_sided), limit)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_composed_attention(dtype):
    q, k, v = _qkv(b=3, dtype=dtype)
    g = torch.Generator().manual_seed(1)
    table = torch.randn(2, 8, 4, generator=g).to(dtype)
    qp, kp = (torch.randint(-60, 60, (3, n, 2), generator=g, dtype=torch.int32) for n in (5, 7))
    lengths = torch.tensor([0, 4, 7], dtype=torch.int32)
    mask = torch.rand(3, 7, generator=g) < 0.7
    keep = mask & (torch.arange(7) < lengths[:, None])
    k[~keep] = float('nan')
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    out = csrc.cross_attention(q, k, v, kv_lengths=lengths, key_mask=mask, bias_table=table, q_pos=qp, k_pos=kp, max_distance=48, cpp_impl=False)
    go = torch.randn(out.shape, generator=g).to(dtype)
    grads = torch.autograd.grad(out, leaves, go)
    idx = attnref.buckets_of(qp, kp, 8, True, 48)
    want = attnref.attention(q.detach(), k.detach(), v.detach(), 0.25, keep, table.detach(), idx, go)
    for name, t in zip(('out', 'dq', 'dk', 'dv', 'dtable'), (out,) + grads):
        attnref.assert_within(t, want[name], name)


@pytest.mark.parametrize('act', [None, 'sigmoid', 'silu'])
def test_composed_group_norm(act):
    g = torch.Generator().manual_seed(2)
    x, go = torch.randn(2, 24, 5, 7, generator=g) + 3, torch.randn(2, 24, 5, 7, generator=g)
    w, b = torch.randn(24, generator=g), torch.randn(24, generator=g)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = csrc.group_norm_act(x, 3, w, b, act=act, cpp_impl=False)
    want = attnref.group_norm(x.detach(), 3, w.detach(), b.detach(), 1e-5, act, go)
    for name, t in zip(('y', 'dx', 'dw', 'db'), (y,) + torch.autograd.grad(y, leaves, go)):
        attnref.assert_within(t, want[name], name)


def test_oracle_notices_a_planted_mistake():
    """the bounds are not so wide that a wrong bucket, a lost key or a wrong gradient factor would pass"""
    q, k, v = _qkv(b=1, lq=9, lk=40, h=1, hk=1)
    g = torch.Generator().manual_seed(3)
    table, go = torch.randn(1, 8, 1, generator=g), torch.randn(9 * 16, generator=g).view(1, 9, 1, 16)
    qp, kp = torch.arange(9, dtype=torch.int32)[None, :, None], torch.arange(40, dtype=torch.int32)[None, :, None]
    idx = attnref.buckets_of(qp, kp, 8, True, 48)
    keep = torch.ones(1, 40, dtype=torch.bool)
    want = attnref.attention(q, k, v, 0.25, keep, table, idx, go)
    wrong = idx.clone()
    wrong[0, 0, 3, 30] = (wrong[0, 0, 3, 30] + 1) % 8
    lost = keep.clone()
    lost[0, 39] = False
    for bad in (attnref.attention(q, k, v, 0.25, keep, table, wrong, go), attnref.attention(q, k, v, 0.25, lost, table, idx, go),
                attnref.attention(q, k, v, 0.2501, keep, table, idx, go)):
        with pytest.raises(AssertionError):
            for name in want:
                attnref.assert_within(bad[name][0], want[name], name)


# ------------------------------------------------------------------------------------------------ modules
def test_group_norm_is_a_norm_of_the_blocks():
    from camliflow_amd.cores import runtime
    from camliflow_amd.cores.blocks import Conv1dNormRelu, Conv2dNormRelu
    with runtime.use_backend('composed'):
        for layer, x in ((Conv2dNormRelu(12, 24, kernel_size=3, padding=1, norm='group_norm'), torch.randn(2, 12, 5, 6)),
                         (Conv1dNormRelu(12, 20, norm='group_norm', act='sigmoid'), torch.randn(2, 12, 9))):
            want = torch.nn.functional.group_norm(layer.conv_fn(x), layer.norm_fn.num_groups, layer.norm_fn.weight, layer.norm_fn.bias)
            want = torch.sigmoid(want) if layer.norm_fn.act == 'sigmoid' else torch.nn.functional.leaky_relu(want, 0.1)
            torch.testing.assert_close(layer(x), want, rtol=1e-5, atol=1e-5)
            assert {'norm_fn.weight', 'norm_fn.bias'} <= set(dict(layer.named_parameters()))


def test_attentive_fusion_module():
    from camliflow_amd.cores import runtime
    from camliflow_amd.cores.fusion import CLFM
    torch.manual_seed(0)
    mod = CLFM(64, 32, fusion_fn='attn')
    uv = torch.rand(2, 2, 11) * 8
    f2, f3 = torch.randn(2, 64, 6, 8, requires_grad=True), torch.randn(2, 32, 11, requires_grad=True)
    with runtime.use_backend('composed'):
        a, b = mod(uv, f2, f3)
        assert torch.equal(a, f2) and torch.equal(b, f3)            # a fresh module passes its inputs through
        for m in (mod.attend2d, mod.attend3d):
            torch.nn.init.normal_(m.out.weight, std=0.1)
            torch.nn.init.normal_(m.bias_table, std=0.3)
        a, b = mod(uv, f2, f3)
        assert a.shape == f2.shape and b.shape == f3.shape
        (a.square().sum() + b.square().sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in mod.parameters())
    with pytest.raises(ValueError):
        CLFM(8, 8, fusion_fn='attention')
