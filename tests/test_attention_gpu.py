"""Cross attention, the bucketed position bias and channels-last group norm on the GPU against 64-bit restatements (attnref.py)."""
import pytest
import torch

import attnref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ['f32', 'bf16', 'f16']


def _cuda(t):
    return t.cuda() if isinstance(t, torch.Tensor) else t


# ------------------------------------------------------------------------------------------------ attention
def _case(b, lq, lk, h, hk, d, dtype, axes=0, buckets=32, max_distance=64, lengths=None, masked=0.0, batched_pos=False, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, go = (torch.randn(b, n, m, d, generator=g).to(dtype) for n, m in ((lq, h), (lk, hk), (lk, hk), (lq, h)))
    q = q * gain
    keep = torch.ones(b, lk, dtype=torch.bool)
    kvl = None
    if lengths is not None:
        kvl = torch.tensor(lengths, dtype=torch.int32)
        keep &= torch.arange(lk) < kvl[:, None]
    mask = None
    if masked:
        mask = torch.rand(b, lk, generator=g) >= masked
        keep &= mask
    table = qp = kp = None
    if axes:
        table = (torch.randn(axes, buckets, h, generator=g) * 0.7).to(dtype)
        lead = (b,) if batched_pos else ()
        qp = torch.randint(-90, 90, lead + (lq, axes), generator=g, dtype=torch.int32)
        kp = torch.randint(-90, 90, lead + (lk, axes), generator=g, dtype=torch.int32)
    return dict(q=q, k=k, v=v, go=go, keep=keep, kvl=kvl, mask=mask, table=table, qp=qp, kp=kp, buckets=buckets, max_distance=max_distance)


def _reference(c, bidirectional=True, scale=None, grad=True):
    idx = None
    if c['table'] is not None:
        lead = lambda t: t if t.dim() == 3 else t[None]     # noqa: E731
        idx = attnref.buckets_of(lead(c['qp']), lead(c['kp']), c['buckets'], bidirectional, c['max_distance'])
    scale = c['q'].shape[-1] ** -0.5 if scale is None else scale
    return attnref.attention(c['q'], c['k'], c['v'], scale, c['keep'], c['table'], idx, c['go'] if grad else None)


def _run(c, bidirectional=True, scale=None, grad=True):
    from camliflow_amd import csrc
    leaves = {n: c[n].cuda().requires_grad_(grad) for n in ('q', 'k', 'v', 'table') if c[n] is not None}
    out = csrc.cross_attention(leaves['q'], leaves['k'], leaves['v'], scale=scale, kv_lengths=_cuda(c['kvl']), key_mask=_cuda(c['mask']),
                               bias_table=leaves.get('table'), q_pos=_cuda(c['qp']), k_pos=_cuda(c['kp']), bidirectional=bidirectional,
                               max_distance=c['max_distance'])
    got = {'out': out}
    if grad:
        got.update(zip(['d' + n for n in leaves], torch.autograd.grad(out, list(leaves.values()), c['go'].cuda())))
    return got


def _check(c, **kw):
    want, got = _reference(c, **kw), _run(c, **kw)
    assert set(want) == set(got)
    for name in want:
        attnref.assert_within(got[name], want[name], name)
    return got


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('dim', [8, 32, 40, 64, 96, 128])
@pytest.mark.parametrize('lq,lk', [(1, 1), (7, 3), (33, 65), (130, 129)])
def test_attention_sizes(dtype, dim, lq, lk):
    _check(_case(2, lq, lk, 2, 2, dim, dtype, seed=dim + lq))


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('axes,bidirectional,buckets,max_distance', [(1, True, 32, 64), (2, True, 32, 64), (2, False, 64, 100), (1, False, 7, 1023), (1, True, 128, 300)])
def test_attention_bias(dtype, axes, bidirectional, buckets, max_distance):
    c = _case(2, 70, 150, 3, 3, 32, dtype, axes=axes, buckets=buckets, max_distance=max_distance, seed=axes)
    _check(c, bidirectional=bidirectional)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('dim', [32, 64, 128])
def test_attention_bias_batched_positions_ragged_shared_heads(dtype, dim):
    _check(_case(4, 37, 203, 6, 2, dim, dtype, axes=2, batched_pos=True, lengths=[0, 1, 150, 203], masked=0.3, seed=dim))


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_attention_split_over_keys_and_queries(dtype):
    """few rows and a long other side: the forward and both adjoints run split and joined"""
    _check(_case(1, 2, 1500, 2, 1, 64, dtype, axes=1, lengths=[1411], seed=3))
    _check(_case(1, 1300, 5, 2, 1, 32, dtype, axes=1, seed=4))


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_attention_single_token_packs_shared_heads(dtype):
    _check(_case(3, 1, 700, 8, 2, 64, dtype, axes=2, lengths=[700, 0, 33], masked=0.1, seed=5))


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_attention_large_scores(dtype):
    """one key takes nearly all of the weight; the running maximum rises over many tiles"""
    c = _case(1, 40, 600, 1, 1, 32, dtype, seed=6, gain=4.0)
    c['k'] = c['k'] * torch.linspace(0.1, 3.0, 600)[None, :, None, None].to(dtype)
    _check(c)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('poison', [float('nan'), float('inf'), -float('inf'), 'lowest'])
def test_attention_masked_places_may_hold_anything(dtype, poison):
    c = _case(3, 20, 140, 4, 2, 40, dtype, axes=1, lengths=[0, 77, 140], masked=0.4, seed=7)
    clean = _run(c)
    value = torch.finfo(dtype).min if poison == 'lowest' else poison
    hidden = ~c['keep'][:, :, None, None]
    for n in ('k', 'v'):
        c[n] = torch.where(hidden, torch.full_like(c[n], value), c[n])
    dirty = _run(c)
    for name in clean:
        assert torch.equal(clean[name], dirty[name]), name
    assert not clean['out'][0].any() and not clean['dq'][0].any()
    assert not clean['dk'][hidden.expand_as(c['k']).cuda()].any() and not clean['dv'][hidden.expand_as(c['v']).cuda()].any()


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('dim', [8, 32, 40, 64, 96, 128])
@pytest.mark.parametrize('lq,lk,h,hk', [(1, 1, 1, 1), (1, 31, 4, 1), (1, 700, 8, 2), (5, 129, 6, 2), (32, 40, 2, 2), (8, 1100, 4, 1)])
def test_attention_few_queries(dtype, dim, lq, lk, h, hk):
    """without a gradient: at most 32 rows to a kv head, every wave on its own keys"""
    _check(_case(2, lq, lk, h, hk, dim, dtype, seed=24), grad=False)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('axes,bidirectional,buckets,max_distance', [(1, True, 32, 64), (2, False, 64, 100), (2, True, 64, 1023)])
def test_attention_few_queries_bias_lengths_masks(dtype, axes, bidirectional, buckets, max_distance):
    c = _case(5, 3, 1700, 4, 2, 64, dtype, axes=axes, buckets=buckets, max_distance=max_distance, lengths=[1700, 0, 1, 33, 901], masked=0.3,
              batched_pos=True, seed=25)
    c['mask'][3] = False        # a sample that keeps nothing, and one with its first tiles masked
    c['mask'][4, :500] = False
    c['keep'] = c['mask'] & (torch.arange(1700) < c['kvl'][:, None])
    got = _check(c, bidirectional=bidirectional, grad=False)
    assert not got['out'][1].any() and not got['out'][3].any()


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_attention_few_queries_masked_places_and_rising_scores(dtype):
    """poison in masked places; keys that grow along the row move the softmax reference tile after tile"""
    c = _case(2, 2, 900, 4, 1, 40, dtype, lengths=[900, 610], masked=0.2, seed=26)
    c['k'] = (c['k'].float() * torch.linspace(0, 12, 900)[:, None, None]).to(dtype)
    want = _check(c, grad=False)['out']
    hidden = ~c['keep'][:, :, None, None].expand_as(c['k'])
    for poison in (float('nan'), float('inf'), torch.finfo(dtype).min):
        p = dict(c, k=torch.where(hidden, torch.full_like(c['k'], poison), c['k']), v=torch.where(hidden, torch.full_like(c['v'], poison), c['v']))
        assert torch.equal(_run(p, grad=False)['out'], want)
    p = dict(c, q=c['q'].clone())
    p['q'][1, 0, 2] = float('nan')      # one head's query: its row alone
    out = _run(p, grad=False)['out']
    assert out[1, 0, 2].isnan().all()
    out[1, 0, 2] = want[1, 0, 2]
    assert torch.equal(out, want)


def test_attention_few_queries_in_a_graph_and_past_32_bits():
    from camliflow_amd import csrc
    c = _case(3, 1, 2500, 8, 2, 64, torch.bfloat16, axes=1, lengths=[2500, 7, 0], seed=27)
    cuda = {n: _cuda(c[n]) for n in ('q', 'k', 'v', 'table', 'kvl', 'qp', 'kp')}

    def run():
        with torch.no_grad():
            return csrc.cross_attention(cuda['q'], cuda['k'], cuda['v'], kv_lengths=cuda['kvl'], bias_table=cuda['table'], q_pos=cuda['qp'], k_pos=cuda['kp'])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for step in range(3):
        cuda['q'].add_(0.25)
        cuda['kvl'].copy_(torch.tensor([2500 - 600 * step, 7 + step, 900 * step], dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, run())
    pitch = 2 ** 30 + 2 ** 20
    store = torch.empty(2 * pitch + 90 * 64, dtype=torch.bfloat16, device='cuda')
    k = torch.as_strided(store, (3, 90, 1, 32), (pitch, 64, 64, 1))
    v = torch.as_strided(store, (3, 90, 1, 32), (pitch, 64, 64, 1), 32)
    k.normal_()
    v.normal_()
    q = torch.randn(3, 1, 4, 32, device='cuda').bfloat16()
    assert torch.equal(csrc.cross_attention(q, k, v), csrc.cross_attention(q, k.contiguous(), v.contiguous()))


@pytest.mark.parametrize('scale', [1e-15, 1e-4, 3.0])
def test_attention_scales(scale):
    _check(_case(1, 20, 90, 2, 2, 32, torch.float32, axes=1, seed=16), scale=scale)


def test_attention_lengths_are_clamped():
    c = _case(3, 9, 50, 2, 2, 32, torch.float32, lengths=[50, 0, 50], seed=8)
    got = _run(c)
    c['kvl'] = torch.tensor([1000, -5, 50], dtype=torch.int32)
    for name, t in _run(c).items():
        assert torch.equal(t, got[name])


def test_attention_table_of_minus_infinity_masks():
    """a bucket of -inf takes its pairs out; a row whose every pair has it gives zeros"""
    c = _case(1, 12, 80, 2, 2, 32, torch.float32, axes=1, buckets=8, max_distance=48, seed=9)
    c['table'][0, 4:, :] = -float('inf')           # keys behind the query
    c['qp'][0] = -200                              # every key is behind this one
    got = _check(c)
    assert not got['out'][0, 0].any() and not got['dq'][0, 0].any()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_attention_strides(dtype):
    """[B, H, L, D] operands, halves of one projection, a shared (expanded) encoder state, unaligned rows, rows of stride 2"""
    from camliflow_amd import csrc
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 4, 30, 32, generator=g).to(dtype).cuda().transpose(1, 2)
    kv = torch.randn(2, 90, 2, 4, 32, generator=g).to(dtype).cuda()
    want = csrc.cross_attention(q.contiguous(), kv[:, :, 0].contiguous(), kv[:, :, 1].contiguous())
    assert torch.equal(csrc.cross_attention(q, kv[:, :, 0], kv[:, :, 1]), want)
    shifted = torch.empty(kv.numel() + 1, dtype=dtype, device='cuda')[1:].view(kv.shape).copy_(kv)
    assert shifted.data_ptr() % 16
    assert torch.equal(csrc.cross_attention(q, shifted[:, :, 0], shifted[:, :, 1]), want)
    wide = torch.empty(2, 90, 2, 4, 64, dtype=dtype, device='cuda')
    wide[..., ::2] = kv
    assert torch.equal(csrc.cross_attention(q, wide[:, :, 0, :, ::2], wide[:, :, 1, :, ::2]), want)
    # one encoder state for the whole batch: gradients of the broadcast input are summed over it
    one = kv[:1].detach().requires_grad_(True)
    shared = one.expand(2, -1, -1, -1, -1)
    out = csrc.cross_attention(q, shared[:, :, 0], shared[:, :, 1])
    go = torch.randn(out.shape, generator=g).to(dtype).cuda()
    got, = torch.autograd.grad(out, one, go)
    both = kv[:1].repeat(2, 1, 1, 1, 1).requires_grad_(True)
    parts, = torch.autograd.grad(csrc.cross_attention(q, both[:, :, 0], both[:, :, 1]), both, go)
    assert torch.equal(out, csrc.cross_attention(q, both[:, :, 0], both[:, :, 1]))
    torch.testing.assert_close(got[0].float(), parts.float().sum(0), rtol=2 * torch.finfo(dtype).eps, atol=2 * torch.finfo(dtype).eps)


def test_attention_empty():
    from camliflow_amd import csrc
    for b, lq, lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = (torch.randn(b, n, 2, 32, device='cuda', requires_grad=True) for n in (lq, lk, lk))
        out = csrc.cross_attention(q, k, v)
        assert out.shape == q.shape and not out.any()
        for t, grad in zip((q, k, v), torch.autograd.grad(out.sum(), (q, k, v))):
            assert grad.shape == t.shape and not grad.any()


def test_attention_gradient_subsets():
    """each gradient alone equals the one computed with all others"""
    c = _case(2, 40, 70, 4, 2, 32, torch.float32, axes=2, lengths=[70, 31], seed=10)
    full = _run(c)
    from camliflow_amd import csrc
    for name in ('q', 'k', 'v', 'table'):
        leaves = {n: c[n].cuda().requires_grad_(n == name) for n in ('q', 'k', 'v', 'table')}
        out = csrc.cross_attention(leaves['q'], leaves['k'], leaves['v'], kv_lengths=c['kvl'].cuda(), bias_table=leaves['table'],
                                   q_pos=c['qp'].cuda(), k_pos=c['kp'].cuda(), max_distance=c['max_distance'])
        grad, = torch.autograd.grad(out, leaves[name], c['go'].cuda())
        assert torch.equal(grad, full['d' + name])


def test_attention_gradients_against_differences():
    """directional derivative of <out, go> in 64 bits around the fp32 inputs against the kernels' gradients"""
    c = _case(1, 9, 21, 2, 1, 16, torch.float32, axes=1, lengths=[17], seed=11)
    got = _run(c)
    g = torch.Generator().manual_seed(1)
    step = 1e-4
    for name in ('q', 'k', 'v', 'table'):
        direction = torch.randn(c[name].shape, generator=g).double()
        ends = []
        for sign in (1, -1):
            moved = dict(c, **{n: c[n].double() for n in ('q', 'k', 'v', 'table')})
            moved[name] = moved[name] + sign * step * direction
            idx = attnref.buckets_of(c['qp'][None], c['kp'][None], c['buckets'], True, c['max_distance'])
            attnref.SUBNORMAL[torch.float64] = 0.0
            ends.append(float((attnref.attention(moved['q'], moved['k'], moved['v'], 0.25, c['keep'], moved['table'], idx)['out'][0] * c['go'].double()).sum()))
        slope = (ends[0] - ends[1]) / (2 * step)
        mine = float((got['d' + name].cpu().double() * direction).sum())
        # differences: step^2 times a third derivative of order 10^2; gradients: fp32
        assert abs(slope - mine) < 1e-5 * max(1.0, float((got['d' + name].cpu().double().abs() * direction.abs()).sum()))


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('factor', [2.0 ** -12, 2.0 ** 8])
def test_attention_gradients_scale_with_the_incoming_gradient(dtype, factor):
    """a long row's dS is 1 / Lk of the gradient: it must not sink into fp16's subnormal numbers, nor a large gradient overflow them"""
    c = _case(1, 64, 5000, 2, 1, 32, dtype, axes=1, seed=15)
    c['go'] = (c['go'] / 64).to(dtype)
    base = _run(c)
    c['go'] = c['go'] * factor          # exact: a power of two, and no element of this go is below 2^-13 / 64 but by chance
    scaled = _run(c)
    for name in ('dq', 'dk', 'dv', 'dtable'):
        a, b = scaled[name].double() / factor, base[name].double()
        # both are roundings of the same numbers: a step of the larger one's type, or of the subnormal numbers it was written as
        step = torch.finfo(dtype).eps * b.abs() + 2 * attnref.SUBNORMAL[dtype] * max(1.0, 1.0 / factor)
        # elements of go that became subnormal: each off by half a step of 2^-24, through sums of at most 5000 weights that add up to 1
        lost = 2 ** -24 * 64 / factor if dtype == torch.float16 and factor < 1 else 0.0
        assert ((a - b).abs() <= 2 * step + lost + 1e-6 * b.abs().max()).all(), name


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('exponent', [-90, 60])
def test_attention_gradients_keep_their_bits_under_powers_of_two(dtype, exponent):
    """every step is linear in the incoming gradient and these types have range to spare: the same bits, shifted"""
    c = _case(1, 70, 150, 2, 1, 40, dtype, axes=2, seed=17)
    base = _run(c)
    c['go'] = c['go'] * 2.0 ** exponent
    for name, t in _run(c).items():
        assert torch.equal(t.double(), base[name].double() * (1.0 if name == 'out' else 2.0 ** exponent)), name


@pytest.mark.parametrize('magnitude', [1e-30, 1e30])
def test_attention_fp32_products_over_the_range(magnitude):
    """values and keys far from 1: an fp32 factor's three parts still hold all of its bits"""
    c = _case(1, 33, 130, 2, 1, 32, torch.float32, seed=18)
    c['v'], c['k'], c['q'] = c['v'] * magnitude, c['k'] * magnitude, c['q'] / magnitude
    c['go'] = c['go'] / magnitude
    _check(c)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('dim,axes,buckets,bidirectional', [(128, 2, 64, True), (64, 1, 128, False), (32, 2, 64, False)])
def test_attention_largest_tables(dtype, dim, axes, buckets, bidirectional):
    """what takes the most shared memory: two columns of 2047 offsets and 128 histogram rows beside the widest tiles"""
    c = _case(1, 140, 200, 2, 1, dim, dtype, axes=axes, buckets=buckets, max_distance=1023, seed=19)
    c['qp'], c['kp'] = c['qp'] * 12, c['kp'] * 12
    _check(c, bidirectional=bidirectional)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_attention_rows_without_keys_take_no_part(dtype):
    """a sample without keys, by length or by mask: its gradient may be anything and reaches nothing"""
    c = _case(3, 37, 65, 2, 2, 32, dtype, axes=2, lengths=[65, 0, 65], masked=0.2, seed=20)
    c['mask'][2] = False
    c['keep'][2] = False
    c['go'][1:] = 0
    want = _run(c)
    c['go'][1] = float('nan')
    c['go'][2] = float('inf')
    for name, t in _run(c).items():
        assert torch.equal(t, want[name]), name
    assert not want['dq'][1:].any() and not want['dk'][1:].any() and not want['dv'][1:].any()


def test_attention_broadcast_gradient_and_strided_masks():
    from camliflow_amd import csrc
    c = _case(2, 50, 90, 4, 2, 64, torch.bfloat16, axes=1, lengths=[90, 41], masked=0.3, seed=21)
    c['go'] = torch.ones_like(c['go'])
    want = _run(c)
    kvl = torch.stack([c['kvl'], c['kvl']], dim=1).cuda()[:, 0]
    mask = c['mask'].t().contiguous().cuda().t()
    pos = torch.cat([c['qp'], c['qp']], dim=1).cuda()[:, :1]
    assert not kvl.is_contiguous() and not mask.is_contiguous() and not pos.is_contiguous()
    leaves = {n: c[n].cuda().requires_grad_(True) for n in ('q', 'k', 'v', 'table')}
    out = csrc.cross_attention(leaves['q'], leaves['k'], leaves['v'], kv_lengths=kvl, key_mask=mask, bias_table=leaves['table'], q_pos=pos,
                               k_pos=c['kp'].cuda(), max_distance=c['max_distance'])
    out.sum().backward()            # an expanded gradient
    for name, leaf in leaves.items():
        assert torch.equal(leaf.grad, want['d' + name])


def test_attention_two_streams_at_once():
    """calls of different sizes in flight on two streams do not touch each other's workspaces"""
    cases = [_case(2, 300, 700, 4, 2, 32, torch.bfloat16, axes=2, seed=22), _case(1, 1, 3000, 4, 1, 64, torch.float32, seed=23)]
    want = [_run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        for c, stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                got.append(_run(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for name, t in g.items():
            assert torch.equal(t, want[i % 2][name]), name


def test_attention_same_bits_every_run_and_refuses_double_backward():
    c = _case(2, 150, 333, 4, 2, 64, torch.bfloat16, axes=2, lengths=[333, 100], seed=12)
    first = _run(c)
    for _ in range(3):
        for name, t in _run(c).items():
            assert torch.equal(t, first[name])
    from camliflow_amd import csrc
    q = torch.randn(1, 4, 1, 8, device='cuda', requires_grad=True)
    grad, = torch.autograd.grad(csrc.cross_attention(q, q, q).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_attention_offsets_past_32_bits():
    """keys and values whose last sample starts more than 2^31 elements in"""
    from camliflow_amd import csrc
    b, lk = 5, 600
    pitch = 2 ** 29 + 2 ** 20
    store = torch.empty((b - 1) * pitch + lk * 2 * 32, dtype=torch.bfloat16, device='cuda')
    k = torch.as_strided(store, (b, lk, 1, 32), (pitch, 64, 64, 1))
    v = torch.as_strided(store, (b, lk, 1, 32), (pitch, 64, 64, 1), 32)
    g = torch.Generator(device='cuda').manual_seed(0)
    k.copy_(torch.randn(k.shape, generator=g, device='cuda'))
    v.copy_(torch.randn(v.shape, generator=g, device='cuda'))
    q = torch.randn(b, 9, 1, 32, generator=g, device='cuda').bfloat16()
    assert torch.equal(csrc.cross_attention(q, k, v), csrc.cross_attention(q, k.contiguous(), v.contiguous()))


# ------------------------------------------------------------------------------------------------ position bias
@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('lq,lk', [(1, 1), (5, 9), (64, 256), (70, 333)])
@pytest.mark.parametrize('axes,bidirectional,buckets,max_distance', [(1, True, 32, 128), (2, False, 16, 48), (2, True, 64, 256), (1, False, 128, 1023)])
def test_bias(dtype, lq, lk, axes, bidirectional, buckets, max_distance):
    from camliflow_amd import csrc
    g = torch.Generator().manual_seed(lq)
    for batch in (None, 3):
        lead = () if batch is None else (batch,)
        table = torch.randn(axes, buckets, 3, generator=g).to(dtype)
        qp = torch.randint(-1500, 1500, lead + (lq, axes), generator=g, dtype=torch.int32)
        kp = torch.randint(-1500, 1500, (lk, axes), generator=g, dtype=torch.int32)
        idx = attnref.buckets_of(qp if batch else qp[None], kp[None], buckets, bidirectional, max_distance)     # [axes, B, Lq, Lk]
        want = sum(table[a].float()[idx[a]] for a in range(axes)).permute(0, 3, 1, 2).to(dtype)
        leaf = table.cuda().requires_grad_(True)
        out = csrc.relative_position_bias(leaf, qp.cuda(), kp.cuda(), bidirectional=bidirectional, max_distance=max_distance)
        assert torch.equal(out.cpu(), want if batch else want[0])
        go = torch.randn(out.shape, generator=g).to(dtype)
        grad, = torch.autograd.grad(out, leaf, go.cuda())
        g64 = go.double().reshape((-1,) + go.shape[-3:])
        val, mag = torch.zeros(2, axes, buckets, 3, dtype=torch.float64)
        for a in range(axes):
            for h in range(3):
                flat = idx[a].reshape(-1)
                val[a, :, h] = torch.bincount(flat, weights=g64[:, h].reshape(-1), minlength=buckets)
                mag[a, :, h] = torch.bincount(flat, weights=g64[:, h].abs().reshape(-1), minlength=buckets)
        # no thread adds more than 300 values here, and the columns are joined in 10 steps
        err = 310 * attnref.U * mag
        attnref.assert_within(grad, (val, err + attnref.half_step(dtype) * (val.abs() + err) + attnref.SUBNORMAL[dtype]), 'dtable')


def test_bias_extreme_positions():
    """offsets that do not fit 32 bits saturate: the last buckets"""
    from camliflow_amd import csrc
    table = torch.arange(64, dtype=torch.float32).view(1, 32, 2).cuda()
    lo, hi = -2 ** 31, 2 ** 31 - 1
    qp = torch.tensor([[lo], [0], [hi]], dtype=torch.int32).cuda()
    kp = torch.tensor([[hi], [1], [lo]], dtype=torch.int32).cuda()
    got = csrc.relative_position_bias(table, qp, kp)[0].cpu() / 2
    assert got.tolist() == [[31, 31, 0], [31, 17, 15], [0, 15, 15]]


def test_bias_many_short_samples():
    """one query a sample: the backward's rows walk over many samples at a step"""
    from camliflow_amd import csrc
    g = torch.Generator().manual_seed(0)
    table = torch.zeros(1, 8, 2).cuda().requires_grad_(True)
    qp = torch.randint(-9, 9, (9000, 1, 1), generator=g, dtype=torch.int32).cuda()
    kp = torch.randint(-9, 9, (9000, 3, 1), generator=g, dtype=torch.int32).cuda()
    out = csrc.relative_position_bias(table, qp, kp, max_distance=8)
    go = torch.randint(-4, 5, out.shape, generator=g).float().cuda()        # whole numbers: every sum is exact
    grad, = torch.autograd.grad(out, table, go)
    plain, = torch.autograd.grad(csrc.relative_position_bias(table, qp, kp, max_distance=8, cpp_impl=False), table, go)
    assert torch.equal(grad, plain)


# ------------------------------------------------------------------------------------------------ group norm
def _norm_case(b, c, spatial, dtype, ptype, seed=0, offset=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(b, *spatial, c, generator=g) * 1.5 + offset).to(dtype).movedim(-1, 1)
    w = (1 + 0.2 * torch.randn(c, generator=g)).to(ptype)
    bs = (0.2 * torch.randn(c, generator=g)).to(ptype)
    go = torch.randn(b, *spatial, c, generator=g).to(dtype).movedim(-1, 1)
    return x, w, bs, go


def _norm_check(x, w, bs, go, groups, act, eps=1e-5, run_x=None):
    from camliflow_amd import csrc
    want = attnref.group_norm(x, groups, w, bs, eps, act, go)
    if act in ('relu', 'leaky_relu'):       # the slope within rounding of the kink is undefined: move such elements away
        z, z_err = want['z']
        for _ in range(8):
            near = z.abs() <= 4 * z_err
            if not near.any():
                break
            x = torch.where(near, x + 0.125, x)
            want = attnref.group_norm(x, groups, w, bs, eps, act, go)
            z, z_err = want['z']
    leaf = (run_x(x) if run_x else x.cuda()).detach().requires_grad_(True)
    params = [t.cuda().requires_grad_(True) if t is not None else None for t in (w, bs)]
    y = csrc.group_norm_act(leaf, groups, *params, eps=eps, act=act)
    assert y.movedim(1, -1).is_contiguous() and y.dtype == x.dtype
    attnref.assert_within(y, want['y'], 'y')
    live = [leaf] + [p for p in params if p is not None]
    names = ['dx'] + [n for n, p in zip(('dw', 'db'), params) if p is not None]
    for name, grad in zip(names, torch.autograd.grad(y, live, go.cuda())):
        attnref.assert_within(grad, want[name], name)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('c,groups', [(8, 1), (8, 8), (33, 3), (96, 12), (128, 8), (520, 4)])
@pytest.mark.parametrize('spatial', [(3, 1), (17, 30), (611,)])
def test_norm_sizes(dtype, c, groups, spatial):
    _norm_check(*_norm_case(2, c, spatial, dtype, torch.float32, seed=c), groups, 'silu')


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
@pytest.mark.parametrize('act', [None, 'relu', 'leaky_relu', 'sigmoid', 'silu'])
def test_norm_activations(dtype, act):
    x, w, bs, go = _norm_case(3, 32, (9, 13), dtype, dtype, seed=1)
    _norm_check(x, w, bs, go, 4, act)
    _norm_check(x, None, bs, go, 4, act)
    _norm_check(x, w, None, go, 4, act)
    _norm_check(x, None, None, go, 4, act)


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_norm_far_mean_and_many_chunks(dtype):
    """a mean far from zero costs no digits; a long map goes through many chunks"""
    _norm_check(*_norm_case(1, 16, (40, 501), dtype, torch.float32, seed=2, offset=50.0), 2, 'silu')


@pytest.mark.parametrize('dtype', TYPES, ids=IDS)
def test_norm_layouts(dtype):
    """channel-first memory, channel slices of a wider map, a crop, an expanded batch"""
    x, w, bs, go = _norm_case(2, 24, (6, 10), dtype, torch.float32, seed=3)
    _norm_check(x, w, bs, go, 3, 'silu', run_x=lambda t: t.contiguous().cuda())

    def sliced(t):
        wide = torch.zeros(2, 6, 10, 40, dtype=dtype, device='cuda')
        wide[..., 8:32] = t.movedim(1, -1).cuda()
        return wide.movedim(-1, 1)[:, 8:32]

    def odd_slice(t):
        wide = torch.zeros(2, 6, 10, 31, dtype=dtype, device='cuda')
        wide[..., 5:29] = t.movedim(1, -1).cuda()
        return wide.movedim(-1, 1)[:, 5:29]

    def crop(t):
        wide = torch.zeros(2, 9, 14, 24, dtype=dtype, device='cuda')
        wide[:, 1:7, 2:12] = t.movedim(1, -1).cuda()
        return wide.movedim(-1, 1)[:, :, 1:7, 2:12]
    for f in (sliced, odd_slice, crop):
        _norm_check(x, w, bs, go, 3, 'silu', run_x=f)
    one = x[:1].expand(2, -1, -1, -1)
    _norm_check(one, w, bs, go, 3, 'silu', run_x=lambda t: t[:1].cuda().expand(2, -1, -1, -1))


def test_norm_empty_and_constant():
    from camliflow_amd import csrc
    w = torch.ones(8, device='cuda', requires_grad=True)
    for shape in ((0, 8, 3, 4), (2, 8, 0, 4)):
        x = torch.randn(shape, device='cuda', requires_grad=True)
        y = csrc.group_norm_act(x, 2, w, None)
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == x.shape and gx.shape == x.shape and not gw.any()
    x = torch.full((2, 8, 5, 5), 3.0, device='cuda')        # no spread: the bias alone
    assert not csrc.group_norm_act(x, 2, w, None).any()
    assert not csrc.group_norm_act(x[:, :, :1, :1], 8).any()


def test_norm_nan_stays_in_its_group():
    from camliflow_amd import csrc
    x = torch.randn(2, 16, 7, 9, device='cuda')
    want = csrc.group_norm_act(x, 4, act='relu')
    x[0, 5, 2, 2] = float('nan')
    got = csrc.group_norm_act(x, 4, act='relu')
    assert got[0, 4:8].isnan().all()
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[0, 4:8] = True
    assert torch.equal(got[~hit], want[~hit])


# ------------------------------------------------------------------------------------------------ streams, graphs
def _chain(x, wn, bn, wq, wkv, wo, points, table, qp, kp, lengths):
    """group norm -> projections -> attention with the bias -> projection, residual: how the operators are used together"""
    from camliflow_amd import csrc
    b, c, h, w = x.shape
    rows = csrc.group_norm_act(x, 4, wn, bn, act='silu').movedim(1, -1).reshape(b, h * w, c)
    q = (rows @ wq).view(b, h * w, 2, -1)
    k, v = (points @ wkv).view(b, points.shape[1], 2, 2, -1).unbind(2)
    att = csrc.cross_attention(q, k, v, kv_lengths=lengths, bias_table=table, q_pos=qp, k_pos=kp, max_distance=64)
    return rows + att.reshape(b, h * w, -1) @ wo


def _chain_inputs(seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device='cuda')      # noqa: E731
    x = n(2, 9, 12, 64).movedim(-1, 1)
    qp = torch.stack(torch.meshgrid(torch.arange(9), torch.arange(12), indexing='ij'), -1).reshape(-1, 2).int().cuda()
    kp = torch.randint(0, 12, (2, 50, 2), generator=g, device='cuda', dtype=torch.int32)
    leaves = [x, 1 + 0.1 * n(64), 0.1 * n(64), n(64, 64) / 8, n(64, 128) / 8, n(64, 64) / 8, n(2, 50, 64), n(2, 16, 2)]
    return [t.requires_grad_(True) for t in leaves], qp, kp, torch.tensor([50, 20], dtype=torch.int32, device='cuda')


def test_chain_matches_composed_formulation():
    import camliflow_amd.csrc as csrc
    leaves, qp, kp, lengths = _chain_inputs()
    out = _chain(*leaves, qp, kp, lengths)
    go = torch.randn_like(out)
    grads = torch.autograd.grad(out, leaves, go)
    real = csrc.group_norm_act, csrc.cross_attention
    try:
        csrc.group_norm_act = lambda *a, **k: real[0](*a, cpp_impl=False, **k)
        csrc.cross_attention = lambda *a, **k: real[1](*a, cpp_impl=False, **k)
        out2 = _chain(*leaves, qp, kp, lengths)
        grads2 = torch.autograd.grad(out2, leaves, go)
    finally:
        csrc.group_norm_act, csrc.cross_attention = real
    # both sides are fp32 chains of sums of a few hundred terms: 2^-24 * 1000 of the largest value
    for a, b in zip((out,) + grads, (out2,) + grads2):
        assert float((a - b).abs().max()) <= 6e-5 * float(b.abs().max())


def test_chain_on_a_side_stream():
    leaves, qp, kp, lengths = _chain_inputs(1)
    go = torch.randn(2, 108, 64, device='cuda')
    want = [_chain(*leaves, qp, kp, lengths)]
    want += torch.autograd.grad(want[0], leaves, go)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_chain(*leaves, qp, kp, lengths)]
        got += torch.autograd.grad(got[0], leaves, go)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_chain_forward_in_a_graph():
    """captured forward passes replay on new inputs, interleaved with eager work; two graphs do not disturb each other"""
    cases = [_chain_inputs(s) for s in (2, 3)]
    with torch.no_grad():
        for leaves, qp, kp, lengths in cases:
            _chain(*leaves, qp, kp, lengths)
        torch.cuda.synchronize()
        graphs = []
        for leaves, qp, kp, lengths in cases:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = _chain(*leaves, qp, kp, lengths)
            graphs.append((graph, out))
        for i in range(4):
            for (leaves, qp, kp, lengths) in cases:
                leaves[0].copy_(torch.randn_like(leaves[0]))
                lengths.copy_(torch.tensor([50 - 7 * i, 11 * i], dtype=torch.int32))
            for graph, _ in graphs:
                graph.replay()
            for (leaves, qp, kp, lengths), (_, out) in zip(cases, graphs):
                assert torch.equal(out, _chain(*leaves, qp, kp, lengths))
            torch.cuda.synchronize()


def test_training_step_in_a_graph():
    """forward and backward of the operators captured together and replayed with new inputs"""
    from camliflow_amd import csrc
    c = _case(2, 33, 90, 4, 2, 32, torch.float32, axes=1, lengths=[90, 40], seed=13)
    static = {n: c[n].cuda().requires_grad_(True) for n in ('q', 'k', 'v', 'table')}
    x = torch.randn(2, 32, 5, 7, device='cuda').to(memory_format=torch.channels_last).requires_grad_(True)
    qp, kp, kvl, go = (c[n].cuda() for n in ('qp', 'kp', 'kvl', 'go'))

    def step(t, xx):
        out = csrc.cross_attention(t['q'], t['k'], t['v'], kv_lengths=kvl, bias_table=t['table'], q_pos=qp, k_pos=kp, max_distance=64)
        y = csrc.group_norm_act(xx, 4, act='silu')
        bias = csrc.relative_position_bias(t['table'], qp, kp, max_distance=64)
        return torch.autograd.grad([out, y, bias], list(t.values()) + [xx], [go, torch.ones_like(y), torch.ones_like(bias)])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step(static, x)
    for i in range(4):
        with torch.no_grad():
            for t in list(static.values()) + [x]:
                t.copy_(torch.randn_like(t))
        graph.replay()
        fresh = {n: t.detach().clone().requires_grad_(True) for n, t in static.items()}
        want = step(fresh, x.detach().clone(memory_format=torch.preserve_format).requires_grad_(True))
        for a, b in zip(grads, want):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ modules
def _randomised(mod):
    from modelutils import hashed_fill_
    hashed_fill_(mod)
    return mod


@pytest.mark.parametrize('autocast', [False, True], ids=['fp32', 'bf16'])
def test_attentive_fusion_module_matches_composed(autocast):
    from camliflow_amd.cores import runtime
    from camliflow_amd.cores.fusion import CLFM
    mod = _randomised(CLFM(96, 64, fusion_fn='attn')).cuda()
    g = torch.Generator().manual_seed(0)
    uv = torch.rand(2, 2, 301, generator=g) * torch.tensor([40.0, 30.0])[:, None]
    uv[0, 0, 3], uv[1, 1, 7] = 1e12, float('nan')           # a point behind the camera projects anywhere
    f2, f3 = torch.randn(2, 96, 30, 40, generator=g), torch.randn(2, 64, 301, generator=g)
    go2, go3 = torch.randn(f2.shape, generator=g).cuda(), torch.randn(f3.shape, generator=g).cuda()
    results = []
    for backend in ('hip', 'composed'):
        leaves = [f2.cuda().requires_grad_(True), f3.cuda().requires_grad_(True)]
        mod.zero_grad()
        with runtime.use_backend(backend), torch.autocast('cuda', torch.bfloat16, enabled=autocast):
            a, b = mod(uv.cuda(), *leaves)
        torch.autograd.backward([a, b], [go2, go3])
        results.append([a.detach(), b.detach()] + [t.grad for t in leaves] + [p.grad.clone() for _, p in sorted(mod.named_parameters())])
    # fp32: chains of sums of at most 1200 terms, 2^-24 * 1200 * a few; bf16: the same roundings of q, k, v, table and out on both sides, P and
    # dS rounded on one only: a few half steps (2^-8) of the largest value
    tol = 3e-2 if autocast else 3e-4
    for x, y in zip(*results):
        assert float((x.double() - y.double()).abs().max()) <= tol * float(y.abs().max().clamp(min=1e-3))


def test_group_norm_layers_match_composed():
    from camliflow_amd.cores import runtime
    from camliflow_amd.cores.blocks import Conv1dNormRelu, Conv2dNormRelu
    g = torch.Generator().manual_seed(0)
    for layer, shape in ((Conv2dNormRelu(32, 64, kernel_size=3, padding=1, norm='group_norm', act='sigmoid'), (2, 32, 17, 19)),
                         (Conv1dNormRelu(32, 40, norm='group_norm', act=None), (3, 32, 77))):
        layer = _randomised(layer).cuda()
        x, out = torch.randn(shape, generator=g).cuda(), []
        for backend in ('hip', 'composed'):
            leaf = x.clone().requires_grad_(True)
            layer.zero_grad()
            with runtime.use_backend(backend):
                y = layer(leaf)
            y.square().sum().backward()
            out.append([y.detach(), leaf.grad] + [p.grad.clone() for _, p in sorted(layer.named_parameters())])
        for a, b in zip(*out):
            assert float((a - b).abs().max()) <= 3e-4 * float(b.abs().max().clamp(min=1e-3))


def test_camliraft_with_attentive_fusion():
    """the flagship model with cross attention in all of its fusion modules: forward and backward on the kernels, strict mode"""
    from modelutils import camliraft_cfg, hashed_fill_, synthetic_inputs
    from camliflow_amd.cores import CamLiRAFT, runtime
    from camliflow_amd.csrc import _lib
    torch.manual_seed(0)
    model = CamLiRAFT(camliraft_cfg(n_iters=2, fusion_fn='attn')).cuda().train()
    for name, mod in model.named_modules():
        if type(mod).__name__ == 'CrossAttend':
            hashed_fill_(mod)
    batch = {k: v.cuda() for k, v in synthetic_inputs(1, 128, 160, 4608).items()}
    runtime.set_strict(True)
    _lib.TIMER.reset()
    _lib.TIMER.enabled = True
    try:
        out = model(batch)
        model.get_loss().backward()
        torch.cuda.synchronize()
        ran = _lib.TIMER.summary()
    finally:
        _lib.TIMER.enabled = False
        _lib.TIMER.reset()
        runtime.set_strict(False)
    assert {'camli_cross_attention_fwd', 'camli_cross_attention_bwd', 'camli_group_norm_fwd', 'camli_group_norm_bwd'} <= set(ran)
    assert torch.isfinite(out['flow_2d']).all() and torch.isfinite(out['flow_3d']).all()
    grads = [p.grad for n, p in model.named_parameters() if 'attend' in n]
    assert len(grads) > 20 and all(g is not None and torch.isfinite(g).all() for g in grads)
