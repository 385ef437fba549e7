"""Shaped attention with a bias by places where rows see keys behind themselves: slope * (row's place - key's) is taken off whatever
the sign of the difference is, so a key behind the row gains what one in front loses. The formula in 64 bits decides."""
import math

import pytest
import torch

import attention_reference as ref
from test_gpu_attention import gen, paged
from test_gpu_shaped_attention import BF16, E4M3, F16, INT8, firsts, ints, ops, run, slopes_of  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dtype,dim", [(INT8, BF16, 128), (E4M3, F16, 64), (INT8, F16, 192), (E4M3, BF16, 256)])
@pytest.mark.parametrize("prefix", [[0, 0, 0], [40, 1, 150], [45, 400, 90], [-3, 2 ** 31 - 1, 47], [240, 3, 151]])
@pytest.mark.parametrize("sign", [1.0, -1.0, 0.0])
def test_prefixes_and_slopes(ops, device, kind, dtype, dim, prefix, sign):  # noqa: F811
    """Slopes of one sign, of the other, and of both in turn; with windows and a cap too."""
    context, new = [40, 3, 0], [200, 1, 150]
    slopes = slopes_of(4) * (torch.tensor([1.0, -1.0, 1.0, -1.0]) if sign == 0.0 else sign)
    more = dict(context=context, new=new, hq=4, dim=dim, kind=kind, dtype=dtype, prefix=ints(prefix), slopes=slopes, seed=3)
    run(ops, device, **more)
    run(ops, device, first=firsts(context, new, 61), cap=10.0, **more)


@pytest.mark.parametrize("kind", [INT8, E4M3])
def test_a_bias_that_a_prefix_makes_large(ops, device, kind):  # noqa: F811
    """1700 places ahead and slopes up to 1: the row's best key is the prefix's last by far."""
    run(ops, device, context=[9], new=[1750], hq=8, hkv=2, dim=64, page=64, kind=kind, dtype=F16, prefix=ints([1700]), slopes=torch.tensor([2.0 ** -i for i in range(8)]), seed=1)


@pytest.mark.parametrize("new,hq,hkv", [([1100], 16, 8), ([2100], 8, 2), ([600, 500], 8, 8)])
def test_prompts_in_whole_blocks_and_shares(ops, device, new, hq, hkv):  # noqa: F811
    context = [90 + 7 * b for b in range(len(new))]
    positions = ints([c + 2 * t for c, n in zip(context, new) for t in range(n)])
    for more in ({}, {"positions": positions}):
        run(ops, device, context=context, new=new, hq=hq, hkv=hkv, dim=64, page=64, kind=E4M3, prefix=ints([310] * len(new)), slopes=slopes_of(hq), seed=new[0], **more)


def test_a_bias_by_the_key_alone_is_the_same(ops, device):  # noqa: F811
    """A softmax does not see what all of a row's scores have in common: the signed bias is slope * (place of the key)."""
    g = gen(4)
    table, pages = paged([120], 16, g)
    slots = ref.Slots(pages * 16, 2, 64, INT8, g)
    q = torch.randn((60, 4, 64), generator=g).to(F16)
    slopes = slopes_of(4)
    out = ops.tree_attention(q.to(device), ops.KvCache(*slots.tensors(16, device)), table.to(device), ints([60]).to(device), ints([0, 60]).to(device), max_new=60, max_context=60,
                             slopes=slopes.to(device), prefix=ints([110]).to(device)).cpu().double()
    j = torch.arange(120)
    at = table[0].long()[j // 16] * 16 + j % 16
    k, v = slots.keys(at), slots.values(at)
    for h in range(4):
        s = q[:, h].double() @ k[:, h // 2].t() / 8 + float(slopes[h]) * j
        s = torch.where((j[None] < torch.maximum(torch.tensor(110), 61 + torch.arange(60))[:, None]), s, -math.inf)
        w = torch.softmax(s, -1)
        mean = w @ v[:, h // 2].abs()
        # Weights' rounding to half precision, the result's own, and the scores': sums of 64 products in 32 bits of up to |q||k| / 8, and
        # three roundings of a bias of up to 60 and of scores below 100; queries held to 2^-16 of their largest (see attention_reference.py)
        size = (q[:, h].double().abs() @ k[:, h // 2].abs().t() / 8).amax(-1, keepdim=True)
        fixed = 2.0 ** -17 * q[:, h].double().abs().amax(-1, keepdim=True) * k[:, h // 2].abs().sum(-1).max() / 8
        off = 2 * 72 * 2.0 ** -24 * size + 2.0 ** -22 * 160 + 2 * fixed
        ref.check(out[:, h], w @ v[:, h // 2], 2.0 ** -11 * (w @ v[:, h // 2]).abs() + (2.0 ** -11 + 2.0 ** -18 + 2 * off) * mean + 2.0 ** -31 * 120 * v.abs().max() + ref.LEAST[F16])
