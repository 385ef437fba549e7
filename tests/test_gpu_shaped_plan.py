"""How shaped attention of many sequences is dealt out: single tokens and trees whose rows see all of what is in front are in shares, like
those of scores as they are, unless none can be long; with windows a workgroup takes a whole block of rows."""
import pytest
import torch

import fusedkernellibrary_amd as fkl
from test_gpu_attention import ragged
from test_gpu_shaped_attention import BF16, E4M3, INT8, firsts, gen, ops, run, slopes_of  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dim,batch,new,hq,hkv,shares", [(INT8, 128, 64, 1, 20, 20, 768), (E4M3, 128, 72, 1, 32, 16, 768), (INT8, 256, 48, 1, 16, 8, 256), (E4M3, 192, 24, 1, 16, 16, 256),
                                                             (INT8, 128, 48, 30, 32, 8, 512), (E4M3, 64, 96, 16, 32, 8, 768), (E4M3, 256, 32, 20, 16, 8, 256)])
@pytest.mark.parametrize("said", [30000, 1500])
@pytest.mark.parametrize("window", [None, 20])
def test_many_heads_and_one_long_sequence(ops, device, kind, dim, batch, new, hq, hkv, shares, said, window):  # noqa: F811
    g = gen(batch)
    context, news = ragged(batch, 40, g), [max(1, n) for n in ragged(batch, new + 1, g)]
    context[batch // 3], news[0] = 1400, new
    more = {} if window is None else {"first": firsts(context, news, window)}
    run(ops, device, context=context, new=news, hq=hq, hkv=hkv, dim=dim, kind=kind, dtype=BF16, seed=batch, said=said, cap=8.0, **more)
    grid = fkl.last_launch()["grid"]
    if said == 30000 and window is None:
        assert grid == [shares, 1, 1]
    else:
        assert grid[2] == batch
