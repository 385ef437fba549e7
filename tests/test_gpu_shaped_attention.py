"""Attention whose scores are capped or biased by distance, or whose rows see a window, their document or a prefix, against its
formula in 64 bits."""
import math
import random

import pytest
import torch

import attention_reference as ref
import shaped_reference as shaped
from test_gpu_attention import gen, paged, ragged, tree_mask

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from fusedkernellibrary_amd import attention
    return attention


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def slopes_of(heads):
    return torch.tensor([2.0 ** (-6.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32)


def firsts(context, new, window):
    return ints([max(0, c + t + 1 - window) for c, n in zip(context, new) for t in range(n)])


def run(ops, device, *, context, new, hq=4, hkv=2, dim=64, page=16, kind=INT8, dtype=BF16, seed=0, said=None, q=None, scale=None, size=1.5, **more):
    """One call against the formula. What no row sees, and what belongs to nobody, holds NaN."""
    g = gen(seed)
    lengths = [c + n for c, n in zip(context, new)]
    table, pages = paged(lengths, page, g)
    slots = ref.Slots(pages * page, hkv, dim, kind, g)
    start = [sum(new[:b]) for b in range(len(new) + 1)]
    used = torch.zeros(pages * page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        if more.get("first") is not None and new[b]:
            j = j[max(0, int(more["first"][start[b]])):]
        used[table[b].long()[j // page] * page + j % page] = True
    for codes, s in ((slots.k, slots.ks), (slots.v, slots.vs)):
        codes[~used], s[~used] = 0x7f, math.nan
    if q is None:
        q = (size * torch.randn((sum(new), hq, dim), generator=g)).to(dtype)
    cache = ops.KvCache(*slots.tensors(page, device))
    lse = torch.full((sum(new), hq), 5.0, dtype=torch.float32, device=device)
    given = table
    if said is not None:
        given = torch.nn.functional.pad(table, (0, -(-(said + max(new)) // page) - table.shape[1]), value=-1)
    on = {n: x.to(device) if isinstance(x, torch.Tensor) else x for n, x in more.items()}
    out = ops.tree_attention(q.to(device), cache, given.to(device), ints(context).to(device), ints(start).to(device), max_new=max(new), max_context=max(context) if said is None else said,
                             scale=scale, lse=lse, **on)
    want, bound, want_lse, lse_bound = shaped.attention(q, slots, page, table, ints(context), ints(start), dim ** -0.5 if scale is None else scale, dtype, **more)
    ref.check(out, want, bound, "out")
    finite = want_lse.isfinite()
    assert torch.equal(lse.cpu().isfinite(), finite) and (lse.cpu()[~finite] == -math.inf).all()
    assert ((lse.cpu().double() - want_lse).abs()[finite] <= lse_bound[finite]).all()
    return out


CONTEXTS = [0, 1, 15, 16, 17, 31, 32, 33, 64, 95, 127, 128, 129, 255, 300]


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("what", ["cap", "bias", "window", "all"])
def test_single_tokens(ops, device, kind, dim, what):
    new = [1] * len(CONTEXTS)
    more = {}
    if what in ("cap", "all"):
        more["cap"] = 2.0
    if what in ("bias", "all"):
        more["slopes"] = slopes_of(8)
    if what in ("window", "all"):
        more["first"] = firsts(CONTEXTS, new, 33)
    run(ops, device, context=CONTEXTS, new=new, hq=8, dim=dim, kind=kind, seed=dim, **more)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("cap", [2.0 ** -6, 0.5, 30.0, 50.0, 512.0])
@pytest.mark.parametrize("kind,size", [(INT8, 1.5), (E4M3, 40.0)])
def test_caps(ops, device, dtype, cap, kind, size):
    """Caps that are far above the scores, and caps that nearly all scores reach."""
    run(ops, device, context=[70, 3, 300], new=[5, 1, 2], dim=128, kind=kind, dtype=dtype, cap=cap, size=size, seed=int(cap) + 1)
    run(ops, device, context=[70, 3, 300], new=[5, 1, 2], dim=128, kind=kind, dtype=dtype, cap=cap, size=size, scale=-0.3, seed=int(cap) + 2)


def test_a_cap_holds_queries_of_any_size(ops, device):
    """Scores far beyond the cap are the cap, of either sign."""
    g = gen(2)
    for big in (1e30, 1e38):
        q = (torch.randn((3, 4, 64), generator=g) * big).to(BF16)
        table, pages = paged([50], 16, g)
        slots = ref.Slots(pages * 16, 2, 64, INT8, g)
        out = ops.tree_attention(q.to(device), ops.KvCache(*slots.tensors(16, device)), table.to(device), ints([47]).to(device), ints([0, 3]).to(device), max_new=3, max_context=47, cap=4.0)
        j = torch.arange(50)
        at = table[0].long()[j // 16] * 16 + j % 16
        k, v = slots.keys(at), slots.values(at)
        for r in range(3):
            for h in range(4):
                s = 4.0 * torch.sign(k[: 48 + r, h // 2] @ q[r, h].double() / big)
                want = torch.softmax(s, -1) @ v[: 48 + r, h // 2]
                # the weights' rounding, and the result's
                assert ((out[r, h].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -17) * (torch.softmax(s, -1) @ v[: 48 + r, h // 2].abs()) + 1e-6).all()


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (14, 2), (20, 20), (64, 1), (33, 11)])
@pytest.mark.parametrize("page,kind,dtype", [(16, INT8, F16), (64, E4M3, BF16), (256, INT8, BF16)])
def test_shared_heads_and_pages(ops, device, hq, hkv, page, kind, dtype):
    """Every query head has a slope of its own."""
    context, new = [5, 130, 277], [3, 1, 9]
    run(ops, device, context=context, new=new, hq=hq, hkv=hkv, page=page, kind=kind, dtype=dtype, slopes=slopes_of(hq) * torch.tensor([(-1.0) ** h for h in range(hq)]), cap=20.0,
        first=firsts(context, new, 100), seed=hq)


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, F16)])
@pytest.mark.parametrize("new", [[1, 2, 5, 16], [17, 31, 3], [64, 63, 33, 1], [70, 128, 100]])
@pytest.mark.parametrize("window", [None, 1, 40])
def test_trees(ops, device, kind, dtype, new, window):
    """Positions of drafted tokens are their depths behind the context, and windows go by them."""
    g = gen(len(new))
    mask = tree_mask(new, -(-max(new) // 64), g)
    context = [(b * 37) % 101 for b in range(len(new))]
    depth = torch.stack([sum((w >> i) & 1 for i in range(64)) for w in mask.unbind(1)]).sum(0) - 1
    positions = (depth + torch.repeat_interleave(torch.tensor(context), torch.tensor(new))).to(torch.int32)
    more = {} if window is None else {"first": (positions + 1 - window).to(torch.int32)}
    run(ops, device, context=context, new=new, hq=8, dim=128, page=32, kind=kind, dtype=dtype, mask=mask, slopes=slopes_of(8), positions=positions, seed=7, **more)


@pytest.mark.parametrize("kind,dtype,dim", [(INT8, BF16, 128), (E4M3, F16, 64), (INT8, F16, 192)])
@pytest.mark.parametrize("prefix", [[0, 0, 0], [40, 1, 150], [45, 400, 90], [-3, 2 ** 31 - 1, 47], [240, 3, 151]])
def test_prefixes(ops, device, kind, dtype, dim, prefix):
    """None, one that ends in the context, one inside of the new tokens, all and more."""
    context, new = [40, 3, 0], [200, 1, 150]
    run(ops, device, context=context, new=new, hq=4, dim=dim, kind=kind, dtype=dtype, prefix=ints(prefix), seed=3)
    run(ops, device, context=context, new=new, hq=4, dim=dim, kind=kind, dtype=dtype, prefix=ints(prefix), first=firsts(context, new, 61), cap=10.0, seed=3)


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("window", [1, 2, 16, 31, 32, 33, 100, 10000])
def test_windows_of_prompts(ops, device, kind, window):
    context, new = [500, 0, 129], [300, 65, 1]
    run(ops, device, context=context, new=new, hq=8, dim=128, page=16, kind=kind, first=firsts(context, new, window), slopes=slopes_of(8), seed=window)


@pytest.mark.parametrize("documents", [[0, 7, 64], [0, 130, 131, 132, 200], [90]])
def test_documents_one_behind_the_other(ops, device, documents):
    context, new = [60, 0], [200, 260]
    first = ints([max([s for s in documents if s <= c + t], default=0) for c, n in zip(context, new) for t in range(n)])
    for kind in (INT8, E4M3):
        run(ops, device, context=context, new=new, hq=4, dim=64, kind=kind, dtype=F16, first=first, seed=len(documents))


def test_rows_that_see_nothing(ops, device):
    """Behind everything, behind the row's own place; in front of everything; not in order."""
    context, new = [40, 9, 0, 300, 17], [4, 3, 2, 2, 4]
    first = ints([0, 44, 43, 2 ** 31 - 1, 100, 0, -5, 0, 1, 299, 303, 20, 3, -2 ** 31, 21])
    for kind in (INT8, E4M3):
        out = run(ops, device, context=context, new=new, hq=4, dim=128, kind=kind, first=first, seed=2)
        assert (out[1] == 0).all() and (out[3] == 0).all() and (out[4:7] == 0).all() and (out[8] != 0).any() and (out[10] == 0).all()


def test_masks_without_a_bit(ops, device):
    mask = torch.zeros((6, 1), dtype=torch.int64)
    mask[3, 0], mask[5, 0] = 0b010, 0b101
    out = run(ops, device, context=[0, 9, 0, 40], new=[2, 1, 3, 0], hq=4, hkv=1, kind=E4M3, mask=mask, cap=5.0, slopes=slopes_of(4), seed=2)
    assert (out[:2] == 0).all() and (out[4] == 0).all() and (out[2] != 0).any() and (out[3] != 0).any()


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_queries_that_are_not_finite(ops, device, kind, bad):
    """A row that sees a key and has one is NaN, others are not, and a row that sees nothing is zero."""
    g = gen(5)
    q = torch.randn((4, 4, 64), generator=g).to(BF16)
    q[1, :, 3], q[2, 0, 5] = bad, bad
    table, pages = paged([204], 16, g)
    slots = ref.Slots(pages * 16, 2, 64, kind, g)
    cache = ops.KvCache(*slots.tensors(16, device))
    out = ops.tree_attention(q.to(device), cache, table.to(device), ints([200]).to(device), ints([0, 4]).to(device), max_new=4, max_context=200, cap=5.0, slopes=slopes_of(4).to(device),
                             first=ints([0, 0, 9999, 150]).to(device)).cpu()
    assert out[1].isnan().all() and (out[2] == 0).all() and out[0].isfinite().all() and out[3].isfinite().all()


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, BF16), (INT8, F16), (E4M3, F16)])
@pytest.mark.parametrize("form,dim,batch,new,hq,hkv,said,shared", [
    ("1x8", 128, 7, 3, 4, 2, None, False), ("1x4", 64, 150, 2, 4, 2, None, False), ("2x4", 128, 130, 9, 6, 2, None, False), ("4x4", 64, 65, 64, 8, 8, None, False),
    ("4x4", 128, 33, 64, 16, 16, None, False), ("1x4", 128, 40, 5, 2, 1, 20000, True), ("1x4", 256, 30, 4, 6, 2, 30000, True), ("2x4", 64, 19, 9, 6, 2, 9000, True),
    ("2x4", 256, 9, 8, 8, 2, 70000, True), ("2x4", 192, 150, 20, 2, 2, None, False), ("4x4", 128, 11, 33, 6, 3, 20000, True), ("4x4", 96, 9, 50, 4, 2, 70000, True),
    ("4x4", 64, 70, 40, 8, 4, 4000, True)])
def test_every_form(ops, device, kind, dtype, form, dim, batch, new, hq, hkv, said, shared):
    """The tiles and waves of a workgroup, and shares or none, that sizes lead to: everything at once, some sequences without new tokens."""
    import fusedkernellibrary_amd as fkl
    g = gen(batch)
    some = ragged(batch, new + 1, g)
    some[batch // 2] = new
    context = ragged(batch, 400, g)
    mask = tree_mask(some, 1, g) if new > 1 else None
    run(ops, device, context=context, new=some, hq=hq, hkv=hkv, dim=dim, kind=kind, dtype=dtype, seed=batch, said=said, mask=mask, cap=8.0, slopes=slopes_of(hq),
        positions=ints([c + t // 2 for c, n in zip(context, some) for t in range(n)]), first=firsts(context, some, 150))
    last = fkl.last_launch()
    if shared and form == "4x4" and (dim <= 96 or kind == E4M3):                   # (three workgroups of two tiles fit a compute unit)
        form = "2x4"
    assert last["form"] == "shaped_attention_" + form
    assert (last["grid"][1:] == [1, 1] and last["grid"][0] >= 64) if shared else last["grid"][2] == batch


@pytest.mark.parametrize("kind,dim,new", [(INT8, 128, 1), (E4M3, 64, 5), (INT8, 256, 3), (E4M3, 96, 2)])
@pytest.mark.parametrize("window", [None, 100, 3000])
def test_long_contexts_are_shared_out(ops, device, kind, dim, new, window):
    """One long and some short sequences, whole or in windows: the shares are of what is seen."""
    context, news = [5003, 0, 40, 1999], [new, 1, new, 1]
    more = {} if window is None else {"first": firsts(context, news, window)}
    run(ops, device, context=context, new=news, hq=6, hkv=2, dim=dim, page=64, kind=kind, dtype=F16, seed=dim + new, cap=30.0, slopes=slopes_of(6), **more)


def test_prompts_in_whole_blocks_and_shares(ops, device):
    rng = random.Random(1)
    for new, hq, hkv in (([1100], 16, 8), ([600, 500], 8, 8), ([2100], 8, 2)):
        context = [rng.randint(0, 300) for _ in new]
        run(ops, device, context=context, new=new, hq=hq, hkv=hkv, dim=64, page=64, kind=E4M3, first=firsts(context, new, 257), prefix=ints([310] * len(new)), cap=50.0, seed=new[0])


def test_nothing_of_what_is_in_front_is_read(ops, device):
    """Page table entries in front of the window may be anything."""
    g = gen(6)
    context, new, page = [1000, 700], [2, 1], 16
    table, pages = paged([1002, 701], page, g)
    slots = ref.Slots(pages * page, 2, 64, INT8, g)
    cache = ops.KvCache(*slots.tensors(page, device))
    q = torch.randn((3, 4, 64), generator=g).to(BF16)
    first = firsts(context, new, 50)
    call = lambda t: ops.tree_attention(q.to(device), cache, t.to(device), ints(context).to(device), ints([0, 2, 3]).to(device), max_new=2, max_context=1000, first=first.to(device))      # noqa: E731
    want = call(table)
    for value in (-1, 2 ** 31 - 1, -2 ** 31):
        stale = table.clone()
        stale[0, :951 // page], stale[1, :651 // page] = value, value
        assert torch.equal(call(stale), want)


def test_results_do_not_change_from_call_to_call(ops, device):
    g = gen(21)
    table, pages = paged([4000, 3000], 16, g)
    cache = ops.KvCache(*ref.Slots(pages * 16, 2, 128, INT8, g).tensors(16, device))
    q = torch.randn((6, 8, 128), generator=g).to(BF16).to(device)
    args = dict(max_new=4, max_context=3998, cap=20.0, slopes=slopes_of(8).to(device), first=firsts([3996, 2998], [4, 2], 1500).to(device))
    call = lambda: ops.tree_attention(q, cache, table.to(device), ints([3996, 2998]).to(device), ints([0, 4, 6]).to(device), **args)      # noqa: E731
    first = call()
    for _ in range(3):
        assert torch.equal(call(), first)


def test_a_captured_call(ops, device):
    g = gen(31)
    table, pages = paged([2100, 900], 32, g)
    cache = ops.KvCache(*ref.Slots(pages * 32, 2, 128, INT8, g).tensors(32, device))
    q = torch.randn((5, 8, 128), generator=g).to(BF16).to(device)
    slopes, first, prefix = slopes_of(8).to(device), ints([0] * 5).to(device), ints([0, 0]).to(device)
    context, start, table = ints([2097, 898]).to(device), ints([0, 3, 5]).to(device), table.to(device)
    call = lambda: ops.tree_attention(q, cache, table, context, start, max_new=3, max_context=2097, cap=20.0, slopes=slopes, first=first, prefix=prefix)      # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = call()
    for i in range(4):
        first.copy_(ints([1000 * (i % 3), 1900, 5, 3 * i, 400 * i]))
        prefix.copy_(ints([700 * i, 899]))
        slopes.copy_(slopes_of(8) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, call())


def test_rows_of_no_sequence(ops, device):
    g = gen(3)
    table, pages = paged([60, 700], 16, g)
    cache = ops.KvCache(*ref.Slots(pages * 16, 2, 64, INT8, g).tensors(16, device))
    q = torch.randn((9, 4, 64), generator=g).to(BF16).to(device)
    for said in (700, 30000):
        wide = torch.nn.functional.pad(table, (0, -(-(said + 3) // 16) - table.shape[1]), value=-1).to(device)
        out = ops.tree_attention(q, cache, wide, ints([58, 697]).to(device), ints([1, 3, 6]).to(device), max_new=3, max_context=said, cap=3.0, first=ints([0] * 9).to(device))
        assert (out[0] == 0).all() and (out[6:] == 0).all() and all((out[r] != 0).any() for r in range(1, 6))


def test_what_does_not_fit_is_refused(ops, device):
    cache = ops.KvCache.allocate(4, 2, 16, 64, device=device)
    q = torch.zeros((2, 4, 64), dtype=BF16, device=device)
    i = lambda *v: ints(v).to(device)      # noqa: E731
    call = lambda **more: ops.tree_attention(q, cache, i(0, 1, 2, 3).view(1, 4), i(3), i(0, 2), max_new=2, max_context=3, **more)      # noqa: E731
    mask = torch.ones((2, 1), dtype=torch.int64, device=device)
    for more, word in ((dict(cap=0.0), "cap"), (dict(cap=-1.0), "cap"), (dict(cap=math.nan), "cap"), (dict(cap=513.0), "cap"), (dict(cap=0.01), "cap"), (dict(slopes=torch.ones(3, device=device)), "slopes"),
                       (dict(slopes=torch.ones(4, device=device, dtype=BF16)), "slopes"), (dict(slopes=torch.ones(4)), "slopes"), (dict(first=i(0)), "first"), (dict(first=i(0, 0).long()), "first"),
                       (dict(prefix=i(0, 0)), "prefix"), (dict(prefix=i(0), mask=mask), "prefix and a mask"), (dict(positions=i(0), slopes=torch.ones(4, device=device)), "positions"),
                       (dict(slopes=torch.ones(4, device=device, requires_grad=True)), "gradient")):
        with pytest.raises(ValueError, match=word):
            call(**more)


CHUNKS = [
    # context, new tokens, options
    ([0, 5, 31, 32, 33, 64, 100, 260], [65, 128, 64, 90, 1, 0, 127, 129], dict(cap=30.0)),
    ([0, 5, 31, 32, 33, 64, 100, 260], [65, 128, 64, 90, 1, 0, 127, 129], dict(slopes=True, window=40)),
    ([300, 0, 77, 16, 15, 0, 1, 500], [64, 200, 3, 64, 66, 17, 140, 100], dict(prefix=[310, 0, 2 ** 31 - 1, 60, 17, -1, 90, 555], window=123, cap=9.0)),
    ([40, 41, 42, 43, 44, 45, 46, 47], [70, 71, 64, 5, 64, 66, 80, 0], dict(mask=True, positions=True, slopes=True, cap=20.0)),
    ([200, 0, 0, 3, 90, 0, 7, 0], [64, 64, 90, 100, 101, 102, 1, 64], dict(first="any", slopes=True)),
]


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, F16), (INT8, F16), (E4M3, BF16)])
@pytest.mark.parametrize("dim,page", [(64, 16), (96, 64), (128, 32), (192, 16), (256, 256)])
@pytest.mark.parametrize("case", range(len(CHUNKS)))
def test_chunks_of_prompts(ops, device, kind, dtype, dim, page, case):
    """Many rows to a sequence: lengths around every edge of a tile, a step and a block of rows."""
    context, new, options = CHUNKS[case]
    g, options = gen(case), dict(options)
    hq, hkv = (32, 16) if dim != 96 else (60, 20)
    more = {n: options[n] for n in ("cap",) if n in options}
    if "slopes" in options:
        more["slopes"] = slopes_of(hq)
    if "window" in options:
        more["first"] = firsts(context, new, options["window"])
    if "prefix" in options:
        more["prefix"] = ints(options["prefix"])
    if "mask" in options:
        more["mask"] = tree_mask(new, 2, g)
    if "positions" in options:
        more["positions"] = ints([c + t // 3 for c, n in zip(context, new) for t in range(n)])
    if "first" in options:
        rng = random.Random(case)
        more["first"] = ints([rng.choice([0, c, c + t, c + t + 1, c - 40, c + n, 2 ** 31 - 1, -1, 32, 33]) if t else min(c, 20) for c, n in zip(context, new) for t in range(n)])
    run(ops, device, context=context, new=new, hq=hq, hkv=hkv, dim=dim, page=page, kind=kind, dtype=dtype, seed=case, **more)


@pytest.mark.parametrize("kind", [INT8, E4M3])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_chunks_with_queries_that_are_not_finite(ops, device, kind, bad):
    g = gen(5)
    q = torch.randn((300, 32, 64), generator=g).to(BF16)
    q[7, :, 3], q[200, 5, 9], q[150, 1, 1] = bad, bad, bad
    first = torch.zeros(300, dtype=torch.int32)
    first[150] = 10 ** 9
    table, pages = paged([400], 16, g)
    slots = ref.Slots(pages * 16, 16, 64, kind, g)
    out = ops.tree_attention(q.to(device), ops.KvCache(*slots.tensors(16, device)), table.to(device).expand(4, -1).contiguous(), ints([100, 100, 0, 0]).to(device), ints([0, 300, 300, 300, 300]).to(device),
                             max_new=300, max_context=100, first=first.to(device)).cpu()
    want = torch.zeros((300, 32), dtype=torch.bool)
    want[7], want[200, 5] = True, True
    assert torch.equal(out.isnan().all(-1), want) and torch.equal(out.isnan().any(-1), want) and (out[150] == 0).all()


def test_chunks_whose_scores_rise_and_scales_of_all_sizes(ops, device):
    """The reference has to move, up and down the keys, over many orders of magnitude of values."""
    for kind in (INT8, E4M3):
        g = gen(9)
        n, page = 700, 32
        table, pages = paged([n], page, g)
        slots = ref.Slots(pages * page, 16, 64, kind, g)
        j = torch.arange(n)
        at = table[0].long()[j // page] * page + j % page
        slots.ks[at] *= (0.2 + (n - j) / 100.0).unsqueeze(1)
        slots.vs[at] *= (10.0 ** ((j * 7 % 13) - 9.0)).unsqueeze(1)
        slots.vs[at[::11]] = 0.0
        q = (1.5 * torch.randn((600, 32, 64), generator=g)).to(BF16)
        start, context = ints([0, 600]), ints([100])
        out = ops.tree_attention(q.to(device), ops.KvCache(*slots.tensors(page, device)), table.to(device), context.to(device), start.to(device), max_new=600, max_context=100, cap=40.0)
        want, bound, _, _ = shaped.attention(q, slots, page, table, context, start, 0.125, BF16, cap=40.0)
        ref.check(out, want, bound, "out")


def test_chunks_of_pages_that_are_no_pages_and_a_captured_call(ops, device):
    g = gen(6)
    table, pages = paged([900], 16, g)
    cache = ops.KvCache(*ref.Slots(pages * 16, 16, 128, E4M3, g).tensors(16, device))
    q = torch.randn((300, 32, 128), generator=g).to(BF16).to(device)
    first = firsts([600], [300], 100).to(device)
    call = lambda t: ops.tree_attention(q, cache, t, ints([600]).to(device), ints([0, 300]).to(device), max_new=300, max_context=600, first=first)      # noqa: E731
    want = call(table.to(device))
    for value in (-1, 2 ** 31 - 1):
        stale = table.clone()
        stale[0, :501 // 16] = value
        assert torch.equal(call(stale.to(device)), want)
    on, context, start = table.to(device), ints([600]).to(device), ints([0, 300]).to(device)
    prefix = ints([0]).to(device)
    again = lambda: ops.tree_attention(q, cache, on, context, start, max_new=300, max_context=600, first=first, prefix=prefix, cap=25.0)      # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        again()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = again()
    for i in range(3):
        prefix.fill_(300 * i)
        first.copy_(firsts([600], [300], 50 + 300 * i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, again())
