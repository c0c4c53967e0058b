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


# Workgroups of 128 rows: groups of heads over several tiles in every type, with rooms in
# part used, scales and gradients.  (tests/test_nn_rules_cpu.py checks that these sizes, and
# the others here, take the kernel that they are meant for.)
PROMPT = [600, 1, 0, 437, 130, 64, 65]
PROMPT_HEADS = [(64, 32), (64, 16)]
ROOMS_Q, ROOMS_K = [300, 200, 0, 140, 500], [500, 20, 40, 140, 130]


@pytest.mark.parametrize("heads", PROMPT_HEADS)
@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_of_grouped_heads(tpo, dev, heads, D, dtype, causal):
    _check(tpo, dev, PROMPT, PROMPT, *heads, D, dtype, causal, seed=D, grad=D != 128)


@pytest.mark.parametrize("heads", PROMPT_HEADS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_of_grouped_heads_in_rooms(tpo, dev, heads, dtype, causal):
    _check(tpo, dev, ROOMS_Q, ROOMS_K, *heads, 32, dtype, causal, lq=[290, 129, 0, 0, 499],
           lk=[333, 20, 1, 140, 127], before=(3, 5), after=(7, 2), seed=33)


# a negative scale turns one operand's sign, 0 leaves every key alike; by 32 rows and by 128
SCALED = [([50, 1, 0, 90], 4, 2, 16), ([50, 1, 0, 90], 4, 2, 40), (PROMPT, 64, 16, 16)]


@pytest.mark.parametrize("lens,Hq,Hk,D", SCALED, ids=lambda v: str(v))
@pytest.mark.parametrize("scale", [-0.3, 0.0, 0.5])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_scales(tpo, dev, lens, Hq, Hk, D, scale, dtype, causal):
    _check(tpo, dev, lens, lens, Hq, Hk, D, dtype, causal, scale=scale, seed=Hq)


def _mixed(B, longest):
    return [0 if b % 9 == 4 else 1 + 37 * b % longest for b in range(B)]


# a lane has one sequence each up to 62, with the rows before and after; a search beyond
@pytest.mark.parametrize("B", [61, 62, 63, 64, 65])
@pytest.mark.parametrize("longest,Hq,Hk", [(40, 4, 2), (150, 16, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_numbers_of_sequences(tpo, dev, B, longest, Hq, Hk, dtype):
    lens = _mixed(B, longest)
    _check(tpo, dev, lens, lens, Hq, Hk, 32, dtype, True, seed=B, before=(2, 3), after=(1, 0))
    _check(tpo, dev, lens, lens[::-1], Hq, Hk, 32, dtype, False, lk=[n // 2 for n in lens],
           seed=B + 1, grad=B == 64)
