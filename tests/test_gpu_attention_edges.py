"""Calls of the attention operators at the edges of what they accept, on the GPU: page tables without columns."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from fusedkernellibrary_amd import attention
    return attention


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(device, *values):
    return torch.tensor(values, dtype=torch.int32, device=device)


# every form without shares: one tile with eight waves and with four, two tiles, four
@pytest.mark.parametrize("batch,new,hq,hkv,dim", [(1, 1, 8, 2, 64), (3, 5, 6, 2, 96), (150, 2, 4, 2, 128), (130, 9, 6, 2, 128), (65, 64, 8, 8, 64), (150, 20, 2, 2, 192), (2, 3, 4, 1, 256)])
@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, F16)])
def test_page_tables_without_columns(ops, device, batch, new, hq, hkv, dim, kind, dtype):
    """No token of a sequence has a page, so nobody sees anything, whatever the contexts are said to be: zeros and -inf."""
    cache = ops.KvCache.allocate(1, hkv, 16, dim, codes=kind, device=device)
    tokens = batch * new
    q = torch.randn((tokens, hq, dim), generator=gen(batch)).to(dtype).to(device)
    start = ints(device, *range(0, tokens + 1, new))
    for context in (0, 700):
        for mask in (None, torch.full((tokens, 1), -1, dtype=torch.int64, device=device)):
            lse = torch.full((tokens, hq), 5.0, device=device)
            out = ops.tree_attention(q, cache, torch.zeros((batch, 0), dtype=torch.int32, device=device), ints(device, *[context] * batch), start, max_new=new, max_context=context, mask=mask,
                                     out=torch.full_like(q, 3.0), lse=lse)
            assert (out == 0).all() and (lse == -math.inf).all()
