"""Cross attention and group norm at the ends of their ranges, without a GPU: the composed formulations, refusals and host arithmetic."""
import pytest
import torch

import attnref
import attnsteps
from camliflow_amd import csrc
from camliflow_amd.csrc import _lib
from test_attention_range_gpu import _common_value_case, _lowest_twice, _sized_case, _sized_reference


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_composed_attention_with_entries_of_the_lowest_value_on_both_axes(dtype):
    c, p = _lowest_twice(dtype, 12, 50)
    leaves = [c[n].requires_grad_(True) for n in ('q', 'k', 'v', 'table')]
    out = csrc.cross_attention(*leaves[:3], bias_table=leaves[3], q_pos=c['qp'], k_pos=c['kp'], max_distance=64, cpp_impl=False)
    got = dict(zip(('out', 'dq', 'dk', 'dv'), (out,) + torch.autograd.grad(out, leaves[:3], c['go'])))
    want = attnsteps.attention({n: t.detach() if isinstance(t, torch.Tensor) else t for n, t in c.items()}, p, torch.full((1, 1, 1, 1), 70 * attnref.U).double())
    for name in want:
        attnsteps.assert_within(got[name], want[name], name)


def _rounded_steps(c, round_ds=True, p_terms=2, keep_out=True):
    """the adjoints of c in 64 bits but for roundings to its type: of dS without any scaling, of P to one or two terms, of out before D"""
    dtype = c['q'].dtype
    r = lambda t: t.to(dtype).double()          # noqa: E731
    Q, K, V, g = attnsteps._heads(c)
    idx, bias = None, torch.zeros(1, 1, 1, 1, dtype=torch.float64)
    if c['table'] is not None:
        idx = attnref.buckets_of(c['qp'][None], c['kp'][None], c['buckets'], True, c['max_distance'])
        bias = sum(c['table'][a].double()[idx[a]] for a in range(idx.shape[0])).permute(0, 3, 1, 2)
    p, _ = attnsteps.softmax(c, bias)
    first = r(p)
    o = (first if p_terms == 1 else first + r(p - first)) @ V
    G = c['go'].double().permute(0, 2, 1, 3)
    ds = p * (G @ V.transpose(2, 3) - (G * (o if keep_out else r(o))).sum(-1, keepdim=True))
    dsr, scale = r(ds) if round_ds else ds, Q.shape[-1] ** -0.5
    b, h, lq, d = Q.shape
    out = {'dq': (scale * dsr @ K).permute(0, 2, 1, 3), 'dk': (scale * dsr.transpose(2, 3) @ Q).reshape(b, h // g, g, -1, d).sum(2).permute(0, 2, 1, 3)}
    if idx is not None:
        out['dtable'] = torch.stack([torch.stack([torch.bincount(idx[a].expand(b, -1, -1).reshape(-1), weights=ds[:, i].reshape(-1), minlength=c['buckets'])
                                                  for i in range(h)], -1) for a in range(idx.shape[0])])
    return {n: t.to(dtype) for n, t in out.items()}



def test_bounds_reject_half_gradients_without_a_scale():
    """dS rounded to fp16 as it is: subnormal for small gradients, infinite for large values; and no gradient at all"""
    for v, go, lq, lk, d, seed in ((1.0, 2.0 ** -16, 16, 3000, 32, 1), (2e4, 1.0, 16, 16, 128, 2), (2.0 ** -12, 2.0 ** -6, 16, 2000, 32, 3)):
        for qk, name in ((2.0 ** -5, 'dq'), (2.0 ** 5, 'dk')):
            c = _sized_case(torch.float16, lq, lk, d, v, go, qk, seed=seed)
            want = _sized_reference(c)
            attnsteps.assert_within(_rounded_steps(c, round_ds=False)[name], want[name], name)
            for bad in (_rounded_steps(c)[name], torch.zeros_like(c[name[1]])):
                with pytest.raises(AssertionError):
                    attnsteps.assert_within(bad, want[name], name)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=['bf16', 'f16'])
def test_bounds_reject_a_table_gradient_from_a_rounded_out(dtype):
    """D from out as it is returned, or from P of one term: what the second term and the fp32 copy of out are for"""
    c = _common_value_case(dtype)
    want = _sized_reference(c)
    attnsteps.assert_within(_rounded_steps(c)['dtable'], want['dtable'], 'dtable')
    for bad in (_rounded_steps(c, keep_out=False), _rounded_steps(c, p_terms=1)):
        with pytest.raises(AssertionError):
            attnsteps.assert_within(bad['dtable'], want['dtable'], 'dtable')


def test_composed_attention_is_fp32_under_autocast():
    """as the kernels, whose inputs decide the type; the backward's products too"""
    g = torch.Generator().manual_seed(0)
    leaves = [torch.randn(2, n, 2, 16, generator=g).requires_grad_(True) for n in (5, 7, 7)]
    go = torch.randn(2, 5, 2, 16, generator=g)
    results = []
    for enabled in (False, True):
        with torch.autocast('cpu', torch.bfloat16, enabled=enabled):
            out = csrc.cross_attention(*leaves, cpp_impl=False)
        results.append((out,) + torch.autograd.grad(out, leaves, go))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize('b,lq,lk', [(0, 3, 4), (2, 0, 4), (2, 3, 0)])
def test_composed_attention_of_nothing(b, lq, lk):
    q, k, v = (torch.randn(b, n, 2, 32, requires_grad=True) for n in (lq, lk, lk))
    out = csrc.cross_attention(q, k, v, cpp_impl=False)
    assert out.shape == q.shape and not out.any()
    for t, grad in zip((q, k, v), torch.autograd.grad(out.sum(), (q, k, v))):
        assert grad.shape == t.shape and not grad.any()


@pytest.mark.parametrize('shape', [(0, 8, 3, 4), (2, 8, 0, 4), (0, 8)])
def test_composed_group_norm_of_nothing(shape):
    x, w = torch.randn(shape, requires_grad=True), torch.ones(8, requires_grad=True)
    y = csrc.group_norm_act(x, 2, w, None, act='silu', cpp_impl=False)
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == x.shape and gx.shape == x.shape and not gw.any()


def test_a_tangent_goes_through_the_autograd_node():
    from torch.autograd import forward_ad
    from camliflow_amd.csrc.norm import needs_node
    x, leaf = torch.ones(3), torch.ones(3, requires_grad=True)
    assert not needs_node(x, None) and needs_node(None, leaf)
    with torch.no_grad():
        assert not needs_node(leaf)
        with forward_ad.dual_level():
            assert not needs_node(x, leaf, None) and needs_node(None, x, forward_ad.make_dual(x, torch.ones(3)))


@pytest.mark.parametrize('positions', [1, 4096, 4097, 2 ** 31 - 2 ** 23 - 1, 2 ** 31 - 2 ** 23 + 1, 2 ** 31 - 2 ** 16 - 1, 2 ** 31 - 1])
@pytest.mark.parametrize('b,c,groups,code', [(1, 1, 1, 2), (1, 1, 1, 0), (3, 8, 2, 1), (65535, 4, 4, 0)])
def test_group_norm_workspace_sizes(positions, b, c, groups, code):
    """one pair of floats a chunk and group (forward), and channel (backward): from 1 to 256 chunks a sample, never a negative number"""
    lib = _lib.load()
    size = lib.camli_group_norm_fwd_workspace_bytes(b, c, groups, positions, code)
    chunks, rest = divmod(size, 8 * b * groups)
    assert rest == 0 and 1 <= chunks <= min(256, positions)
    assert lib.camli_group_norm_bwd_workspace_bytes(b, c, groups, positions, code) == 8 * b * (chunks * c + c + groups)
