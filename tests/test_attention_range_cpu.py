"""Cross attention and group norm at the ends of their ranges, without a GPU: the composed formulations, refusals and host arithmetic."""
import pytest
import torch

import attnref
import attnsteps
from camliflow_amd import csrc
from test_attention_range_gpu import _lowest_twice


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_composed_attention_with_entries_of_the_lowest_value_on_both_axes(dtype):
    c, p = _lowest_twice(dtype, 12, 50)
    leaves = [c[n].requires_grad_(True) for n in ('q', 'k', 'v', 'table')]
    out = csrc.cross_attention(*leaves[:3], bias_table=leaves[3], q_pos=c['qp'], k_pos=c['kp'], max_distance=64, cpp_impl=False)
    got = dict(zip(('out', 'dq', 'dk', 'dv'), (out,) + torch.autograd.grad(out, leaves[:3], c['go'])))
    want = attnsteps.attention({n: t.detach() if isinstance(t, torch.Tensor) else t for n, t in c.items()}, p, torch.full((1, 1, 1, 1), 70 * attnref.U).double())
    for name in want:
        attnsteps.assert_within(got[name], want[name], name)
