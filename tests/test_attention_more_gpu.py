"""packed_attention's gradients one at a time, its scales, and the shapes at which another
kernel or another way to a workgroup's sequence is taken."""
import pytest
import torch

from tests import nn64
from tests.test_attention_gpu import DTYPES, _check, _dev, _offsets, _qkv

pytestmark = pytest.mark.gpu


# few rows and many, groups whose heads are shared by workgroups, more sequences than lanes
@pytest.mark.parametrize("lens_q,lens_k,Hq,Hk", [
    ([40, 1, 130], [40, 1, 130], 4, 2), ([5, 0, 3], [700, 9, 0], 16, 1),
    ([300, 64], [300, 64], 12, 3), ([b % 4 for b in range(70)], [b % 7 for b in range(70)], 2, 2),
])
@pytest.mark.parametrize("D", [40, 63])
@pytest.mark.parametrize("dtype", DTYPES)
def test_each_gradient_alone(tpo, dev, lens_q, lens_k, Hq, Hk, D, dtype):
    oq, ok = _offsets(lens_q), _offsets(lens_k)
    *qkv, go = _qkv(oq[-1], ok[-1], Hq, Hk, D, dtype, D)
    idx, go = _dev(dev, oq, ok), go.to(dev)
    ins = [t.to(dev).requires_grad_(True) for t in qkv]
    full = torch.autograd.grad(tpo.packed_attention(*ins, *idx), ins, go)
    for some in ((0,), (1,), (2,), (0, 2), (1, 2)):
        part = [t.detach().requires_grad_(i in some) for i, t in enumerate(ins)]
        got = torch.autograd.grad(tpo.packed_attention(*part, *idx), [part[i] for i in some], go)
        assert all(torch.equal(g, full[i]) for g, i in zip(got, some))
