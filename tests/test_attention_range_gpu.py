"""Cross attention over the range of its types: finite table entries down to the lowest (the usual mask of a bucket), rows that keep nothing
else, scores whose neighbours in fp32 are far apart.  Against 64-bit restatements (attnsteps.py)."""
import math

import pytest
import torch

import attnref
import attnsteps
from test_attention_gpu import IDS, TYPES, _case, _run

pytestmark = pytest.mark.gpu

# what the two outermost buckets (keys far before the query, far behind it) hold
LEVELS = {
    torch.float32: [(-1e9, -1e9), (-1e6, -1e9), (-1e9, -1e6), (1e6, -1e30), (-1e30, -1e9)],
    torch.bfloat16: [(-1e9, -1e9), (-1e6, -1e9), (-1e9, -1e6), (1e6, -1e30), (-1e30, -1e9)],
    torch.float16: [(-6e4, -6e4), (-3e4, -6e4), (-6e4, -3e4), (3e4, -6e4), (-300.0, -6e4)],
}
LEVEL_CASES = [pytest.param(t, n, id='%s-%d' % (i, n)) for t, i in zip(TYPES, IDS) for n in range(5)]
BEFORE, BEHIND = 15, 31         # of 32 buckets, 64 positions


def _level_case(dtype, levels, b=2, lq=40, lk=700, h=2, hk=1, d=32, seed=0, axes=1):
    """on the first axis: 300 keys far before nearly every query, then 100 far behind, then the near ones; the last six queries are far
    from all keys"""
    c = _case(b, lq, lk, h, hk, d, dtype, axes=axes, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    c['table'][0, BEFORE], c['table'][0, BEHIND] = levels
    c['kp'] = torch.randint(-40, 41, (lk, axes), generator=g, dtype=torch.int32)
    c['kp'][:3 * lk // 7, 0], c['kp'][3 * lk // 7:4 * lk // 7, 0] = -2000, 2000
    c['qp'] = torch.randint(-20, 21, (lq, axes), generator=g, dtype=torch.int32)
    c['qp'][-6:-1, 0], c['qp'][-1, 0] = 900, 5000
    return c


def _level_reference(c, training):
    """Levels are so far apart that only the pairs of a row's highest count, at scores that differ by what fp32 holds beside that level."""
    idx = attnref.buckets_of(c['qp'][None], c['kp'][None], 32, True, 64)
    level = torch.zeros(32, dtype=torch.float64)
    level[BEFORE], level[BEHIND] = c['table'][0, BEFORE, 0].double(), c['table'][0, BEHIND, 0].double()
    pair = level[idx[0, 0]]                                  # [Lq, Lk]
    row = pair.amax(dim=1, keepdim=True)
    entry = torch.where((level == 0)[:, None], c['table'][0].double(), attnsteps.NO)
    bias = torch.where((pair == row)[..., None], entry[idx[0, 0]], torch.full((), -math.inf).double())
    for a in range(1, idx.shape[0]):
        bias = bias + c['table'][a].double()[idx[a, 0]]
    bias = bias.permute(2, 0, 1)[None]
    p, p_rel = attnsteps.softmax(c, bias, rounded_at=row[:, 0], roundings=idx.shape[0])
    return attnsteps.attention(c, p, p_rel, training, idx=idx, buckets=32)


@pytest.mark.parametrize('dtype,n', LEVEL_CASES)
@pytest.mark.parametrize('d', [32, 64, 128])
def test_attention_low_entries_forward(dtype, n, d):
    """whole tiles of one level before the next: the digits of later scores survive, also of rows that have nothing but a low entry"""
    c = _level_case(dtype, LEVELS[dtype][n], d=d, seed=d)
    for training in (False, True):
        attnsteps.assert_within(_run(c, grad=training)['out'], _level_reference(c, training)['out'], 'out, training %s' % training)


@pytest.mark.parametrize('dtype,n', LEVEL_CASES)
def test_attention_low_entries_few_queries_and_splits(dtype, n):
    """few queries, most of them far from everything, and long rows split over workgroups, some of which see one level only"""
    for lq, lk, d in ((7, 2500, 64), (7, 2500, 32), (7, 900, 128)):
        c = _level_case(dtype, LEVELS[dtype][n], b=1, lq=lq, lk=lk, h=4, hk=2, d=d, seed=lq)
        for training in (False, True):
            attnsteps.assert_within(_run(c, grad=training)['out'], _level_reference(c, training)['out'], 'out, training %s' % training)


def _tied_case(dtype, lq, lk, seed):
    """scores of 2^30 and beyond, exact in fp32, the highest one held by two keys of different tiles: each has half of the weight"""
    c = _case(2, lq, lk, 2, 2, 32, dtype, seed=seed)
    big = 2.0 ** (15 if dtype == torch.float16 else 20)
    q, k = torch.zeros_like(c['q']), torch.zeros_like(c['k'])
    q[..., 3] = big
    k[..., 3] = -big / 2
    k[:, 5, :, 3] = k[:, lk - 4, :, 3] = big
    k[:, lk // 2, :, 3] = 0.875 * big
    return dict(c, q=q, k=k)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('lq,lk', [(3, 600), (50, 333)])
def test_attention_huge_tied_scores(dtype, lq, lk):
    c = _tied_case(dtype, lq, lk, seed=40)
    pair = c['v'][:, [5, lk - 4]].double()                                     # [B, 2, H, D]
    want = (pair.sum(1) / 2)[:, None].expand(c['q'].shape)
    # the weights are exact in every type; a sum of two products, a reciprocal, the result's own rounding
    bound = 6 * attnref.U * pair.abs().sum(1)[:, None] + attnref.half_step(dtype) * want.abs() + attnref.SUBNORMAL[dtype]
    for grad in (False, True):
        attnsteps.assert_within(_run(c, grad=grad)['out'], (want, bound), 'out')


@pytest.mark.parametrize('dtype,n', LEVEL_CASES)
@pytest.mark.parametrize('d,axes', [(32, 1), (32, 2), (64, 1), (64, 2), (128, 2)])
def test_attention_low_entries_gradients(dtype, n, d, axes):
    """a row that has nothing but a low entry weighs its keys by the same probabilities in both directions, and the rows beside it are right"""
    for shape in (dict(), dict(b=1, lq=8, lk=1500, h=4, hk=2), dict(b=1, lq=900, lk=40)):       # the latter two split over keys, over queries
        c = _level_case(dtype, LEVELS[dtype][n], d=d, axes=axes, seed=d + axes, **shape)
        want, got = _level_reference(c, True), _run(c)
        assert set(want) == set(got)
        for name in want:
            attnsteps.assert_within(got[name], want[name], name)


def test_attention_low_entries_gradients_without_the_table():
    """a frozen table: the same gradients of the other operands"""
    from camliflow_amd import csrc
    for dtype in TYPES:
        c = _level_case(dtype, LEVELS[dtype][0], axes=2, seed=5)
        want = _level_reference(c, True)
        leaves = [c[n].cuda().requires_grad_(True) for n in 'qkv']
        out = csrc.cross_attention(*leaves, bias_table=c['table'].cuda(), q_pos=c['qp'].cuda(), k_pos=c['kp'].cuda(), max_distance=64)
        for name, grad in zip(('dq', 'dk', 'dv'), torch.autograd.grad(out, leaves, c['go'].cuda())):
            attnsteps.assert_within(grad, want[name], name)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('lq,lk', [(3, 600), (50, 333)])
def test_attention_huge_tied_scores_gradients(dtype, lq, lk):
    c = _tied_case(dtype, lq, lk, seed=41)
    p = torch.zeros(2, 2, lq, lk, dtype=torch.float64)
    p[..., 5] = p[..., lk - 4] = 0.5
    want, got = attnsteps.attention(c, p, torch.full((1, 1, 1, 1), 8 * attnref.U).double()), _run(c)
    for name in want:
        attnsteps.assert_within(got[name], want[name], name)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('other', ['lowest', -1e9])
@pytest.mark.parametrize('d,axes', [(32, 1), (64, 2)])
def test_attention_entries_of_the_lowest_value(dtype, other, d, axes):
    """the type's lowest number is finite: a row of nothing else weighs its keys like any other (log2 e times it is not)"""
    low = torch.finfo(dtype).min
    for shape in (dict(), dict(b=1, lq=8, lk=1500, h=4, hk=2)):
        c = _level_case(dtype, (low, low if other == 'lowest' else other), d=d, axes=axes, seed=d, **shape)
        want, got = _level_reference(c, True), _run(c)
        for name in want:
            attnsteps.assert_within(got[name], want[name], name)
        attnsteps.assert_within(_run(c, grad=False)['out'], _level_reference(c, False)['out'], 'out')


def _lowest_twice(dtype, lq, lk):
    """the second axis adds the lowest number to every pair, the first one adds it again to some: -> (case, probabilities)"""
    c = _level_case(dtype, (torch.finfo(dtype).min,) * 2, b=1, lq=lq, lk=lk, axes=2, seed=43)
    c['table'][1] = torch.finfo(dtype).min
    idx = attnref.buckets_of(c['qp'][None], c['kp'][None], 32, True, 64)[0, 0]
    once = (idx != BEFORE) & (idx != BEHIND)
    kept = torch.where(once.any(1, keepdim=True), once, torch.ones_like(once)).double()
    return c, (kept / kept.sum(1, keepdim=True)).expand(1, 2, -1, -1)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('lq,lk', [(40, 300), (8, 1500)])
def test_attention_entries_of_the_lowest_value_on_both_axes(dtype, lq, lk):
    """their sum is no number of the type, but lower than one of them"""
    c, p = _lowest_twice(dtype, lq, lk)
    for training in (False, True):
        want = attnsteps.attention(c, p, torch.full((1, 1, 1, 1), (lk + 16) * attnref.U).double(), training)
        got = _run(c, grad=training)
        for name in want:
            attnsteps.assert_within(got[name], want[name], name)


def _sized_case(dtype, lq, lk, d, v, go, qk=1.0, axes=0, h=2, hk=1, seed=0, **kw):
    """values and incoming gradients of given sizes; q times qk and k / qk (powers of two: the same scores)"""
    c = _case(1, lq, lk, h, hk, d, dtype, axes=axes, seed=seed, **kw)
    return dict(c, q=c['q'] * qk, k=c['k'] / qk, v=(c['v'].float() * v).clamp(-6e4, 6e4).to(dtype), go=c['go'] * go)


def _sized_reference(c):
    idx, bias = None, torch.zeros(1, 1, 1, 1, dtype=torch.float64)
    if c['table'] is not None:
        idx = attnref.buckets_of(c['qp'][None], c['kp'][None], c['buckets'], True, c['max_distance'])
        bias = sum(c['table'][a].double()[idx[a]] for a in range(idx.shape[0])).permute(0, 3, 1, 2)
    return attnsteps.attention(c, *attnsteps.softmax(c, bias), idx=idx, buckets=c['buckets'])


SIZES = [(3e4, 2.0 ** -10), (3e4, 1.0), (1e3, 1.0), (1.0, 2.0 ** -12), (1.0, 2.0 ** -16), (1e-3, 1.0), (2.0 ** -12, 2.0 ** -6), (1e-3, 256.0)]


@pytest.mark.parametrize('v,go', SIZES)
@pytest.mark.parametrize('qk', [2.0 ** -5, 2.0 ** 5], ids=['k', 'q'])
@pytest.mark.parametrize('lq,lk,d,axes', [(40, 16, 128, 0), (64, 5000, 32, 1), (70, 333, 64, 2)])
def test_attention_half_gradients_of_any_size(v, go, qk, lq, lk, d, axes):
    """fp16 has 30 powers of two: neither large values nor long rows of small ones may take dS out of them, while dq (large keys) or dk (large
    queries) is well inside"""
    c = _sized_case(torch.float16, lq, lk, d, v, go, qk, axes=axes, seed=lk)
    want, got = _sized_reference(c), _run(c)
    for name in want:
        attnsteps.assert_within(got[name], want[name], name)


def test_attention_half_gradients_of_masked_large_values():
    """what is masked does not count as large"""
    c = _sized_case(torch.float16, 60, 900, 32, 1e-3, 2.0 ** -6, 32.0, axes=1, lengths=[700], masked=0.2, seed=3)
    want = _run(c)
    c['v'] = torch.where(c['keep'][:, :, None, None], c['v'], torch.full_like(c['v'], 6e4))
    for name, t in _run(c).items():
        assert torch.equal(t, want[name]), name
    for name, pair in _sized_reference(c).items():
        attnsteps.assert_within(want[name], pair, name)


def _common_value_case(dtype, seed=4):
    """values near a common one, gradients of one sign: dp and D nearly cancel, and what D loses is the table's gradient's error.  Few rows and flat scores keep the
    bound narrow."""
    c = _case(1, 4, 40, 2, 1, 32, dtype, axes=2, buckets=8, max_distance=48, seed=seed)
    c['table'] = (c['table'].float() / 4).to(dtype)
    return dict(c, q=c['q'] / 16, v=(4 + c['v'].float() / 4).to(dtype), go=c['go'].abs())


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_attention_table_gradient_of_a_common_value(dtype):
    for seed in range(4):
        c = _common_value_case(dtype, seed)
        want, got = _sized_reference(c), _run(c)
        for name in want:
            attnsteps.assert_within(got[name], want[name], name)


# ------------------------------------------------------------------------------------------------ forward mode
@pytest.mark.parametrize('which', ['q', 'v', 'table', 'bias table', 'x', 'weight', 'shift'])
def test_forward_mode_is_refused(which):
    """a tangent is not dropped: the kernels have no forward-mode derivative"""
    from torch.autograd import forward_ad
    from camliflow_amd import csrc
    c = _case(1, 5, 9, 2, 2, 32, torch.float32, axes=1, seed=1)
    c['x'], c['weight'], c['shift'], c['bias table'] = torch.randn(2, 8, 3, 4), torch.ones(8), torch.zeros(8), c['table']
    t = {n: c[n].cuda() for n in ('q', 'k', 'v', 'table', 'qp', 'kp', 'x', 'weight', 'shift', 'bias table')}

    def call():
        if which in ('q', 'v', 'table'):
            return csrc.cross_attention(t['q'], t['k'], t['v'], bias_table=t['table'], q_pos=t['qp'], k_pos=t['kp'])
        if which == 'bias table':
            return csrc.relative_position_bias(t['bias table'], t['qp'], t['kp'])
        return csrc.group_norm_act(t['x'], 2, t['weight'], t['shift'], act='silu')
    want = call()
    with forward_ad.dual_level(), torch.no_grad():
        assert torch.equal(call(), want)                # without a tangent nothing changes
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError):
            call()


# ------------------------------------------------------------------------------------------------ group norm
def test_norm_of_nearly_two_to_the_31_positions():
    """the largest map that is taken, forward and backward: its last positions as the first ones"""
    from camliflow_amd import csrc
    n = 2 ** 31 - 2 ** 16 - 1
    x = torch.empty(1, 1, n, dtype=torch.bfloat16, device='cuda')
    x.view(-1)[:] = 1.0
    x.view(-1)[::2] = 3.0           # exact: mean 2 and variance 1 but for 2^-31
    leaf = x.requires_grad_(True)
    y = csrc.group_norm_act(leaf, 1, eps=0.0)
    gx, = torch.autograd.grad(y, leaf, y.detach())          # of a group's own values: zero
    for part in (slice(0, 1000), slice(n // 2, n // 2 + 1000), slice(n - 1000, n)):
        assert torch.equal(y[0, 0, part], x.detach()[0, 0, part] - 2)
        assert gx[0, 0, part].abs().max() <= 2.0 ** -7      # a mean and a sum of 2^31 terms in fp32, rounded to bf16 once
    del x, leaf, y, gx
    torch.cuda.empty_cache()
