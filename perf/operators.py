"""What is measured of the attention, position-bias and normalisation operators of ``camliflow_amd.csrc``.

``own = False`` computes every case in its plain form (elementary torch operations in 32 bits); ``own = True`` makes the
calls a user of the package makes.  Sizes are those of the flow models: 960 x 540 frames give 68 x 120 = 8160 pixels at
stride 8, KITTI frames 47 x 156 = 7332; 8192 points become 2048 after sampling; features have 64, 96, 128 or 256 channels.
"""
import math
from fractions import Fraction

import torch

own = False

_DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
_BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}


# ------------------------------------------------------------------------------------------------ the cases
def _gn(name, b, c, h, w, groups, act, dtype, train):
    return dict(name=name, op='group_norm', b=b, c=c, h=h, w=w, groups=groups, act=act, dtype=dtype, train=train)


def _attn(name, b, lq, lk, heads, kv_heads, dim, dtype, train, axes=0, buckets=32, max_distance=64, bidirectional=True,
          lengths='full', masked=False):
    return dict(name=name, op='attention', b=b, lq=lq, lk=lk, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, train=train,
                axes=axes, buckets=buckets, max_distance=max_distance, bidirectional=bidirectional, lengths=lengths, masked=masked)


def _bias(name, lq, lk, heads, axes, buckets, max_distance, bidirectional, dtype, train):
    return dict(name=name, op='bias', lq=lq, lk=lk, heads=heads, axes=axes, buckets=buckets, max_distance=max_distance,
                bidirectional=bidirectional, dtype=dtype, train=train)


def listed():
    return [
        # the coarsest map of one frame pair at inference: a few microseconds, nothing but latency
        _gn('norm_small_f32', 1, 128, 17, 30, 8, 'leaky_relu', 'f32', False),
        # an fp32 training step on the stride-8 feature maps of a batch of 8 pairs
        _gn('norm_train_f32', 8, 128, 68, 120, 8, 'leaky_relu', 'f32', True),
        # mixed-precision training on the stride-2 maps of both images of 8 pairs: pure bandwidth
        _gn('norm_train_bf16', 16, 64, 272, 480, 8, 'silu', 'bf16', True),
        # point features of a ragged number of points and an uncommon channel count
        _gn('norm_points_f16', 3, 96, 1, 2047, 12, 'relu', 'f16', True),
        # fp32 training of the fusion module: sampled points attend the pixels, offsets in the image bucketed along u and v
        _attn('points_to_pixels_f32', 2, 2048, 8160, 4, 4, 32, 'f32', True, axes=2),
        # mixed-precision training of the other direction at the full batch: pixels attend the points
        _attn('pixels_to_points_bf16', 8, 8160, 2048, 4, 4, 32, 'bf16', True, axes=2),
        # inference: every pixel of one image attends the other image, two wide heads
        _attn('image_to_image_bf16', 4, 8160, 8160, 2, 2, 128, 'bf16', False),
        # clouds of differing sizes with dropped points, shared key-value heads, odd lengths and an uncommon head width
        _attn('ragged_f16', 3, 501, 1237, 6, 2, 40, 'f16', True, axes=1, max_distance=128, lengths='ragged', masked=True),
        # one token per sample attends a dense cloud's features: bound by reading keys and values
        _attn('token_bf16', 16, 1, 16384, 8, 2, 64, 'bf16', False, lengths='ragged'),
        # one token against a small map: latency
        _attn('token_small_f32', 1, 1, 510, 4, 4, 32, 'f32', False),
        # the bias itself, as a tensor, for an odd number of queries and keys, with its gradient
        _bias('bias_f32', 501, 1237, 4, 1, 32, 128, True, 'f32', True),
        # the bias of all points against all pixels of a frame, with its gradient
        _bias('bias_bf16', 2048, 8160, 4, 2, 32, 64, True, 'bf16', True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case.  Sizes are log-uniform; the limits keep every draw below the largest listed case of its operator."""
    op = rng.choice(['group_norm', 'attention', 'attention', 'bias'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    train = rng.random() < 0.6
    if op == 'group_norm':
        groups = rng.choice([1, 2, 4, 8, 12, 16, 32])
        c = groups * rng.choice([1, 2, 3, 4, 5, 8, 16])
        b = _log_int(rng, 1, 16)
        limit = 130_000_000 // (2 if dtype == 'f32' else 1)
        pixels = _log_int(rng, 1, max(1, min(130_560, limit // (b * c))))
        # a group has 16 elements at least: with fewer the input gradient is a difference of equal numbers
        pixels = max(pixels, -(-16 * groups // c))
        h = min(rng.choice([1, 1, 2, 3, 7, 17, 68]), pixels)
        case = _gn('', b, c, h, max(1, pixels // h), groups, rng.choice([None, 'relu', 'leaky_relu', 'sigmoid', 'silu']), dtype, train)
    elif op == 'attention':
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        dim = rng.choice([8, 16, 32, 40, 64, 96, 128])
        b = _log_int(rng, 1, 16)
        lq = 1 if rng.random() < 0.25 else _log_int(rng, 1, 8160)
        lk = _log_int(rng, 8 if train else 1, 16384)      # over one key the gradients of the scores are differences of equal numbers
        limit = 270_000_000 // (4 if dtype == 'f32' else 1) // (3 if train else 1)
        size = 2 * _BYTES[dtype]
        while b * heads * lq * lk * max(1, dim // 32) > limit or b * (heads * lq + kv_heads * lk) * dim * size > (45_000_000 if train else 130_000_000):
            if b > 1:
                b = (b + 1) // 2
            elif lk > lq:
                lk = (lk + 1) // 2
            else:
                lq = (lq + 1) // 2
        axes = rng.choice([0, 0, 1, 2])
        case = _attn('', b, lq, lk, heads, kv_heads, dim, dtype, train, axes=axes, buckets=rng.choice([8, 16, 32, 64]),
                     max_distance=rng.choice([48, 64, 100, 128, 256]), bidirectional=rng.random() < 0.7,
                     lengths=rng.choice(['full', 'ragged']), masked=rng.random() < 0.3)
    else:
        heads = rng.choice([1, 2, 3, 4, 8])
        lq, lk = _log_int(rng, 1, 8160), _log_int(rng, 1, 8160)
        while heads * lq * lk > 66_000_000 // (2 if dtype == 'f32' else 1):
            lq, lk = (lq + 1) // 2, (lk + 1) // 2
        case = _bias('', lq, lk, heads, rng.choice([1, 2]), rng.choice([8, 16, 32, 64]), rng.choice([48, 64, 100, 128, 256]),
                     rng.random() < 0.7, dtype, train)
    del case['name']
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Valid keys per sample: all of them, or spread from none (where there are three samples or more) to all."""
    b, lk = case['b'], case['lk']
    if case['lengths'] == 'full':
        return [lk] * b
    if b == 1:
        return [(2 * lk + 2) // 3]
    return [lk * i // (b - 1) if b >= 3 else lk * (i + 1) // 2 for i in range(b)]


def _positions(case, n, axes, gen):
    """One axis: the running index, as in a sequence.  Two: rounded coordinates in a 120 x 68 map."""
    if axes == 1:
        return torch.arange(n, dtype=torch.int32, device='cuda').view(n, 1)
    u = torch.randint(0, 120, (n,), generator=gen, device='cuda', dtype=torch.int32)
    v = torch.randint(0, 68, (n,), generator=gen, device='cuda', dtype=torch.int32)
    return torch.stack([u, v], dim=1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype = _DTYPES[case['dtype']]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device='cuda') * scale + shift).to(to)

    state = {'case': case}
    grad = case['train']
    if case['op'] == 'group_norm':
        b, c, h, w = case['b'], case['c'], case['h'], case['w']
        x = normal(b, h, w, c, scale=1.5, shift=0.3)
        weight = normal(c, scale=0.2, shift=1.0, to=torch.float32)
        bias = normal(c, scale=0.2, to=torch.float32)
        if grad and case['act'] in ('relu', 'leaky_relu'):
            # within rounding of the kink the slope is a toss of the coin: such elements (one in a thousand) are moved away from it
            grouped = x.float().view(b, h * w, case['groups'], -1)
            var, mean = torch.var_mean(grouped, dim=(1, 3), correction=0, keepdim=True)
            z = ((grouped - mean) * torch.rsqrt(var + 1e-5)).view(b, h, w, c) * weight + bias
            x = torch.where(z.abs() < 1e-3, x + 0.05, x)
        state['x'] = x.permute(0, 3, 1, 2).requires_grad_(grad)
        state['weight'], state['bias'] = weight.requires_grad_(grad), bias.requires_grad_(grad)
        if grad:
            state['gout'] = normal(b, h, w, c).permute(0, 3, 1, 2)
        return state
    heads, axes = case['heads'], case['axes']
    if axes:
        state['table'] = normal(axes, case['buckets'], heads, scale=0.5).requires_grad_(grad)
        state['q_pos'] = _positions(case, case['lq'], axes, gen)
        state['k_pos'] = _positions(case, case['lk'], axes, gen)
        state['lut'] = torch.tensor(_bucket_lut(case), device='cuda')
    if case['op'] == 'bias':
        if grad:
            state['gout'] = normal(heads, case['lq'], case['lk'])
        return state
    b, lq, lk, dim = case['b'], case['lq'], case['lk'], case['dim']
    state['q'] = normal(b, lq, heads, dim).requires_grad_(grad)
    # keys and values are the halves of one projection, as an encoder's states give them
    kv = normal(b, lk, 2, case['kv_heads'], dim)
    state['k'] = kv[:, :, 0].detach().requires_grad_(grad)
    state['v'] = kv[:, :, 1].detach().requires_grad_(grad)
    lengths = _lengths(case)
    state['kv_lengths'] = None if case['lengths'] == 'full' else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    state['key_mask'] = (torch.rand(b, lk, generator=gen, device='cuda') < 0.9) if case['masked'] else None
    if grad:
        state['gout'] = normal(b, lq, heads, dim)
    return state


# ------------------------------------------------------------------------------------------------ one pass
_LEAVES = {'group_norm': ('x', 'weight', 'bias'), 'attention': ('q', 'k', 'v', 'table'), 'bias': ('table',)}


def run(state):
    case = state['case']
    if not case['train']:
        with torch.no_grad():
            return [_own_forward(state, case) if own else _plain_forward(state, case)]
    names = [n for n in _LEAVES[case['op']] if n in state]
    if own:
        out = _own_forward(state, case)
        return [out.detach(), *torch.autograd.grad(out, [state[n] for n in names], state['gout'])]
    if 'table' not in names:
        out = _plain_forward(state, case)
        return [out.detach(), *torch.autograd.grad(out, [state[n] for n in names], state['gout'])]
    # the table's gradient adds millions of terms into one place: a row's in 32 bits, the rows' sums in 64
    with torch.no_grad():
        bias = _bias_sum(state, case)
    out = _plain_forward(state, case, bias.requires_grad_(True))
    *grads, gbias = torch.autograd.grad(out, [state[n] for n in names[:-1]] + [bias], state['gout'])
    return [out.detach(), *grads, _plain_table_grad(state, case, gbias)]


def _own_forward(state, case):
    from camliflow_amd import csrc
    if case['op'] == 'group_norm':
        return csrc.group_norm_act(state['x'], case['groups'], state['weight'], state['bias'], eps=1e-5, act=case['act'])
    if case['op'] == 'bias':
        return csrc.relative_position_bias(state['table'], state['q_pos'], state['k_pos'], bidirectional=case['bidirectional'],
                                           max_distance=case['max_distance'])
    return csrc.cross_attention(state['q'], state['k'], state['v'], kv_lengths=state['kv_lengths'], key_mask=state['key_mask'],
                                bias_table=state.get('table'), q_pos=state.get('q_pos'), k_pos=state.get('k_pos'),
                                bidirectional=case['bidirectional'], max_distance=case['max_distance'])


# ------------------------------------------------------------------------------------------------ plain forms, 32 bits
def _plain_forward(state, case, bias=None):
    if case['op'] == 'group_norm':
        return _plain_group_norm(state, case)
    if bias is None and case['axes']:
        bias = _bias_sum(state, case)
    return bias.to(state['table'].dtype) if case['op'] == 'bias' else _plain_attention(state, case, bias)


def _plain_group_norm(state, case):
    x = state['x'].float().permute(0, 2, 3, 1)
    b, h, w, c = x.shape
    xg = x.reshape(b, h * w, case['groups'], c // case['groups'])
    mean = xg.mean(dim=(1, 3), keepdim=True)
    centred = xg - mean
    var = (centred * centred).mean(dim=(1, 3), keepdim=True)
    y = (centred * torch.rsqrt(var + 1e-5)).reshape(b, h, w, c) * state['weight'] + state['bias']
    if case['act'] == 'relu':
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif case['act'] == 'leaky_relu':
        y = torch.where(y > 0, y, 0.1 * y)
    elif case['act'] == 'sigmoid':
        y = 1 / (1 + torch.exp(-y))
    elif case['act'] == 'silu':
        y = y / (1 + torch.exp(-y))
    return y.to(state['x'].dtype).permute(0, 3, 1, 2)


def _bucket_lut(case):
    """Bucket of every offset -max_distance .. max_distance (key minus query).  Half the buckets of a side hold one distance
    each, the rest are equal steps of the logarithm up to max_distance; the borders are compared as exact fractions."""
    limit = case['max_distance']
    side = case['buckets'] // 2 if case['bidirectional'] else case['buckets']
    exact_to = side // 2
    steps = side - exact_to
    ratio = Fraction(limit, exact_to)
    powers = [ratio ** j for j in range(steps)]
    lut = []
    for offset in range(-limit, limit + 1):
        distance = abs(offset) if case['bidirectional'] else max(-offset, 0)
        if distance < exact_to:
            bucket = distance
        else:
            reach = Fraction(distance, exact_to) ** steps
            bucket = exact_to + sum(1 for p in powers[1:] if reach >= p)
        lut.append(bucket + (side if case['bidirectional'] and offset > 0 else 0))
    return lut


def _buckets(state, case):
    """Per axis the bucket of every query (row) and key (column)."""
    limit = case['max_distance']
    offsets = [state['k_pos'][None, :, a].long() - state['q_pos'][:, None, a].long() for a in range(case['axes'])]
    return [state['lut'][o.clamp(-limit, limit) + limit] for o in offsets]


def _bias_sum(state, case):
    parts = [state['table'][a].float().t()[:, bucket.reshape(-1)].view(-1, *bucket.shape) for a, bucket in enumerate(_buckets(state, case))]
    return parts[0] if len(parts) == 1 else parts[0] + parts[1]


def _plain_table_grad(state, case, gbias):
    zero = gbias.new_zeros(())
    sums = [torch.stack([torch.where(bucket == n, gbias, zero).sum(dim=2).sum(dim=1, dtype=torch.float64) for n in range(case['buckets'])])
            for bucket in _buckets(state, case)]
    return torch.stack(sums).to(state['table'].dtype)


def _plain_attention(state, case, bias):
    b, lk, group = case['b'], case['lk'], case['heads'] // case['kv_heads']
    q = state['q'].float().permute(0, 2, 1, 3).contiguous()
    k = state['k'].float().permute(0, 2, 1, 3).repeat_interleave(group, dim=1)
    v = state['v'].float().permute(0, 2, 1, 3).repeat_interleave(group, dim=1)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(case['dim'])
    if bias is not None:
        scores = scores + bias
    if state['kv_lengths'] is not None or state['key_mask'] is not None:
        keep = torch.ones(b, lk, dtype=torch.bool, device=q.device)
        if state['kv_lengths'] is not None:
            keep &= torch.arange(lk, device=q.device) < state['kv_lengths'][:, None]
        if state['key_mask'] is not None:
            keep &= state['key_mask']
        keep = keep[:, None, None, :]
        top = torch.where(keep, scores, torch.full_like(scores, -1e30)).amax(dim=-1, keepdim=True).detach()
        weights = torch.where(keep, torch.exp(torch.where(keep, scores - top, torch.zeros_like(scores))), torch.zeros_like(scores))
    else:
        weights = torch.exp(scores - scores.amax(dim=-1, keepdim=True).detach())
    total = weights.sum(dim=-1, keepdim=True)
    weights = weights / torch.where(total > 0, total, torch.ones_like(total))
    return torch.matmul(weights, v).permute(0, 2, 1, 3).to(state['q'].dtype)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = _BYTES[case['dtype']]
    if case['op'] == 'group_norm':
        n = case['b'] * case['c'] * case['h'] * case['w']
        # forward: x in, y out; a step also reads the gradient and x again and writes the input gradient
        return {'bytes': n * size * (5 if case['train'] else 2) + 16 * case['c'], 'flops': n * (30 if case['train'] else 10)}
    pos = 4 * case['axes'] * (case['lq'] + case['lk'])
    if case['op'] == 'bias':
        n = case['heads'] * case['lq'] * case['lk']
        return {'bytes': n * size * (2 if case['train'] else 1) + pos, 'flops': n * case['axes'] * (2 if case['train'] else 1)}
    pairs = case['heads'] * case['lq'] * sum(_lengths(case))
    q = case['b'] * case['lq'] * case['heads'] * case['dim'] * size
    kv = 2 * sum(_lengths(case)) * case['kv_heads'] * case['dim'] * size
    # a step: q, k, v in, output out; then all of these and the gradient in, three gradients out
    moved = (2 * q + kv) + ((3 * q + kv + q + kv) if case['train'] else 0)
    return {'bytes': moved + pos, 'flops': pairs * case['dim'] * (14 if case['train'] else 4)}


# ------------------------------------------------------------------------------------------------ the definition, 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {'group_norm': _exact_group_norm, 'attention': _exact_attention, 'bias': _exact_bias}[case['op']](state, case)


def _exact_group_norm(state, case):
    x = state['x'].detach().double()
    b, c, h, w = x.shape
    g, n = case['groups'], (c // case['groups']) * h * w
    shape = (b, g, c // g, h * w)
    wt, bs = (state[k].detach().double().view(1, g, c // g, 1) for k in ('weight', 'bias'))
    var, mean = torch.var_mean(x.reshape(shape), dim=(2, 3), correction=0, keepdim=True)
    rstd = 1 / torch.sqrt(var + 1e-5)
    xhat = (x.reshape(shape) - mean) * rstd
    z = xhat * wt + bs
    sig = torch.sigmoid(z)
    value, slope = {None: (z, torch.ones_like(z)), 'relu': (z.clamp_min(0), (z > 0).double()),
                    'leaky_relu': (torch.maximum(z, 0.1 * z), torch.where(z > 0, 1.0, 0.1).double()),
                    'sigmoid': (sig, sig * (1 - sig)), 'silu': (z * sig, sig * (1 + z * (1 - sig)))}[case['act']]
    out = [value.reshape(b, c, h, w)]
    if case['train']:
        dz = state['gout'].double().reshape(shape) * slope
        dxhat = dz * wt
        m1 = dxhat.sum(dim=(2, 3), keepdim=True) / n
        m2 = (dxhat * xhat).sum(dim=(2, 3), keepdim=True) / n
        out += [((dxhat - m1 - xhat * m2) * rstd).reshape(b, c, h, w), (dz * xhat).sum(dim=(0, 3)).reshape(c), dz.sum(dim=(0, 3)).reshape(c)]
    return out


def _exact_bucket(case, offset):
    """The same definition in whole numbers: the j-th step begins where d^steps >= limit^j e^(steps - j)."""
    two, limit = case['bidirectional'], case['max_distance']
    side = case['buckets'] // (2 if two else 1)
    e = side // 2
    steps = side - e
    d = abs(offset) if two else (-offset if offset < 0 else 0)
    if d < e:
        j = d
    else:
        j = 0
        while j + 1 < steps and d ** steps >= limit ** (j + 1) * e ** (steps - j - 1):
            j += 1
        j += e
    return j + (side if two and offset > 0 else 0)


def _exact_buckets(state, case):
    lim = case['max_distance']
    table = torch.tensor([_exact_bucket(case, o) for o in range(-lim, lim + 1)], dtype=torch.int64, device='cuda')
    q, k = state['q_pos'].long(), state['k_pos'].long()
    return [table[(k[:, a].unsqueeze(0) - q[:, a].unsqueeze(1)).clamp(-lim, lim) + lim] for a in range(case['axes'])]


def _exact_bias(state, case):
    buckets = _exact_buckets(state, case)
    tab = state['table'].detach().double()
    out = torch.zeros(case['heads'], case['lq'], case['lk'], dtype=torch.float64, device='cuda')
    grad = torch.zeros_like(tab)
    for h in range(case['heads']):
        for a, idx in enumerate(buckets):
            out[h] += tab[a, :, h][idx]
            if case['train']:
                grad[a, :, h] = torch.bincount(idx.reshape(-1), weights=state['gout'][h].double().reshape(-1), minlength=case['buckets'])
    return [out, grad] if case['train'] else [out]


def _exact_attention(state, case):
    heads, group, dim = case['heads'], case['heads'] // case['kv_heads'], case['dim']
    q, k, v = (state[n].detach().double() for n in 'qkv')
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    if case['axes']:
        buckets, tab = _exact_buckets(state, case), state['table'].detach().double()
        dtab = torch.zeros_like(tab)
    lengths = _lengths(case)
    for h in range(heads):
        bias = sum(tab[a, :, h][idx] for a, idx in enumerate(buckets)) if case['axes'] else None
        dbias = torch.zeros(case['lq'], case['lk'], dtype=torch.float64, device='cuda')
        for i in range(case['b']):
            valid = torch.arange(lengths[i], device='cuda')
            if state['key_mask'] is not None:
                valid = valid[state['key_mask'][i, :lengths[i]]]
            if valid.numel() == 0:
                continue
            qh, kh, vh = q[i, :, h], k[i, valid, h // group], v[i, valid, h // group]
            s = (qh @ kh.t()) / math.sqrt(dim)
            if bias is not None:
                s = s + bias[:, valid]
            p = torch.softmax(s, dim=1)
            out[i, :, h] = p @ vh
            if case['train']:
                do = state['gout'][i, :, h].double()
                dv[i, valid, h // group] += p.t() @ do
                ds = do @ vh.t()
                ds -= (do * out[i, :, h]).sum(dim=1, keepdim=True)
                ds *= p
                dq[i, :, h] = (ds @ kh) / math.sqrt(dim)
                dk[i, valid, h // group] += (ds.t() @ qh) / math.sqrt(dim)
                if bias is not None:
                    dbias[:, valid] += ds
        if case['train'] and bias is not None:
            for a, idx in enumerate(buckets):
                dtab[a, :, h] = torch.bincount(idx.reshape(-1), weights=dbias.reshape(-1), minlength=case['buckets'])
    if not case['train']:
        return [out]
    return [out, dq, dk, dv] + ([dtab] if case['axes'] else [])
