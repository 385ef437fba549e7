"""How far a capped score is off, measured where it can be seen alone: with one key the logarithm of the sum of exponentials is its score."""
import pytest
import torch

from fusedkernellibrary_amd import attention as ops

pytestmark = pytest.mark.gpu
ROWS = 2001


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cap", [2.0 ** -6, 1.0, 30.0, 512.0])
def test_the_tanh(device, codes, dtype, cap):
    """Scores from -9 to 9 times the cap. The key has one element, so that the product has no sum, and codes hold it exactly.

    Score s, cap c, x = s / c, r = 1 / (1 + e^2x), result c - 2 c r. Roundings, in units of 2^-24 of the result or of what is named:
      s in units of log2: the key's scale, log2(e), its product with the scale and two more, 5 of s; 2 / c and the product with it, 2 more.
      They shift x by 7 |x|, and d tanh = sech^2(x) dx: at most 7 * max |x| sech^2 x = 7 * 0.448 = 3.2 of c.
      the exponential (to a unit in the last place, 2 of e): dr = r (1 - r) de / e, at most 2 / 4 = 0.5 of 1, so 1 of c.
      1 + e, 1 of it; its reciprocal, to a unit in the last place, 2: 3 r <= 3, so 6 of c.
      the last sum, 1 of c; c log2(e), 2 of c.
    Less than 14 * 2^-24 of c, 2^-20.2. (From the finished product on, 10.9: 2^-20.5.)
    The logarithm of the sum: the reference's and the sum's, 2 roundings of what is below c log2(e) + 64, the conversion from log2, 2 more, and
    log2 of a weight of 2^6, to 2^-20."""
    g = torch.Generator().manual_seed(1)
    x = torch.linspace(-9.0, 9.0, ROWS)
    page, dim = 16, 64
    cache = ops.KvCache.allocate(ROWS, 1, page, dim, codes=codes, device=device)
    for t in (cache.k, cache.v):
        t.view(torch.int8).zero_()
    one = torch.zeros(ROWS, 1, dim)
    one[:, 0, 5] = 1.0
    slots = (torch.randperm(ROWS, generator=g) * page).to(torch.int32).to(device)
    ops.kv_write(cache, one.to(dtype).to(device), one.to(dtype).to(device), slots)
    q = torch.zeros(ROWS, 1, dim)
    q[:, 0, 5] = x
    q = q.to(dtype)
    lse = torch.empty((ROWS, 1), dtype=torch.float32, device=device)
    at = torch.arange(ROWS + 1, dtype=torch.int32, device=device)
    ops.tree_attention(q.to(device), cache, (slots // page).view(ROWS, 1), torch.zeros(ROWS, dtype=torch.int32, device=device), at, max_new=1, max_context=0, scale=cap, lse=lse, cap=cap)
    s = q[:, 0, 5].double()
    want = cap * torch.tanh(s)
    off = (lse[:, 0].cpu().double() - want).abs()
    bound = cap * 14 * 2.0 ** -24 + 2 * 2.0 ** -24 * want.abs() + 2 * 2.0 ** -24 * (cap + 64) + 2.0 ** -20
    assert (off <= bound).all()
