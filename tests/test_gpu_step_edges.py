"""Where the operators of a step could go wrong without being asked: places beyond what a float holds, lengths at the ends of their
type, limits larger than the step, gradients, tracers, inference mode, streams, results that share an allocation."""
import pytest
import torch

import attention_reference as ref
import shaped_reference as shaped
import step_reference
from test_gpu_shaped_attention import run, slopes_of

pytestmark = pytest.mark.gpu

BF16, F16, INT8, E4M3 = torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from fusedkernellibrary_amd import attention
    return attention


def ints(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


# ---- scores -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind,dtype,dim", [(INT8, BF16, 128), (E4M3, F16, 64), (INT8, F16, 256)])
@pytest.mark.parametrize("new", [1, 5, 40])
@pytest.mark.parametrize("placed", [False, True])
def test_distances_at_places_beyond_2_to_24(ops, device, kind, dtype, dim, new, placed):
    """A window behind 2^25 + 1 tokens, whose pages are a few over and over: distances are small, and as exact as at place 0."""
    g, page, context, hq, hkv = torch.Generator().manual_seed(dim + new), 256, 2 ** 25 + 1, 4, 2
    entries = (context + new) // page + 1
    table = torch.randint(0, 8, (1, entries), generator=g).to(torch.int32)
    table[0, -2:] = ints([8, 9])
    slots = ref.Slots(10 * page, hkv, dim, kind, g)
    cache = ops.KvCache(*slots.tensors(page, device))
    q = torch.randn((new, hq, dim), generator=g).to(dtype)
    first = ints([context + t - 100 for t in range(new)])
    more = dict(first=first, slopes=torch.tensor([1.0, 0.5, 0.25, 0.125]))
    if placed:
        more |= dict(positions=ints([context + t // 2 for t in range(new)]))
    out = ops.tree_attention(q.to(device), cache, table.to(device), ints([context], device), ints([0, new], device), max_new=new, max_context=context, **{n: x.to(device) for n, x in more.items()})
    # the reference from 512 tokens in front: the same keys, at places that are less by a multiple of a page
    skip = (context - 512) // page * page
    near = dict(first=first - skip, slopes=more["slopes"])
    if placed:
        near |= dict(positions=more["positions"] - skip)
    want, bound, _, _ = shaped.attention(q, slots, page, table[:, skip // page:], ints([context - skip]), ints([0, new]), dim ** -0.5, dtype, **near)
    ref.check(out, want, bound)


@pytest.mark.parametrize("kind,dtype,dim", [(INT8, BF16, 128), (E4M3, F16, 64), (E4M3, BF16, 256)])
@pytest.mark.parametrize("far", [5_000_001, 2 ** 30 - 100])
def test_positions_that_are_far_from_places(ops, device, kind, dtype, dim, far):
    """New tokens that are said to be far away of the context see each other as near as they are."""
    g = torch.Generator().manual_seed(far % 1000)
    new = [5, 1, 33]
    positions = ints([far + int(x) for n in new for x in torch.randint(0, 6, (n,), generator=g)])
    for slopes in (0.5 * slopes_of(4), torch.full((4,), 2.0 ** -30)):
        run(ops, device, context=[70, 3, 0], new=new, hq=4, dim=dim, kind=kind, dtype=dtype, slopes=slopes, positions=positions, seed=4)


@pytest.mark.parametrize("kind,dtype,dim", [(INT8, BF16, 128), (E4M3, F16, 64)])
def test_prefixes_and_first_places_at_the_ends_of_their_type(ops, device, kind, dtype, dim):
    low, high = -2 ** 31, 2 ** 31 - 1
    context, new = [40, 3, 0, 100], [70, 1, 90, 3]
    run(ops, device, context=context, new=new, hq=4, dim=dim, kind=kind, dtype=dtype, prefix=ints([low, low + 1, low, high]), seed=3)
    first = ints(sum(([low] * (n - 1) + [high if n > 1 else low] for n in new), []))
    run(ops, device, context=context, new=new, hq=4, dim=dim, kind=kind, dtype=dtype, first=first, prefix=ints([high, low, low, low]), seed=3)


@pytest.mark.parametrize("kind,dtype", [(INT8, BF16), (E4M3, F16)])
@pytest.mark.parametrize("forms,new,context,what", [
    ("2x4-512 2x4-768", [3, 13, 5, 8, 1, 13, 4, 9], [3000, 100, 4000, 7, 2500, 40, 0, 900], "window"),   # up to 52 rows, 28 in the mean
    ("4x4-512 2x4-768", [16, 13, 16, 15, 16, 16, 14, 16], [3000, 100, 4000, 7, 2500, 40, 0, 900], "window"),
    ("2x4-0 2x4-0", [290], [2900], "window"), ("4x4-0 2x4-0", [1100], [130], "cap"), ("4x4-0 2x4-0", [330, 500, 471], [1500, 1000, 1300], "cap"), ("4x4-512 2x4-768", [700], [2900], "cap"),
    ("4x4-0 2x4-0", [700], [2900], "window"), ("4x4-0 2x4-0", [700], [2900], "prefix")])
def test_forms_that_shaped_scores_choose(ops, device, kind, dtype, forms, new, context, what):
    """Fewer tiles where most would be empty, whole blocks where shares end within them; of int8 and of e4m3, with the shares, or 0 for whole blocks."""
    import fusedkernellibrary_amd as fkl
    hq, hkv = 32, 8
    form, grid = forms.split()[kind == E4M3].split("-")
    first = ints([max(0, c + t + 1 - 200) for c, n in zip(context, new) for t in range(n)])
    more = dict(window=dict(first=first, slopes=slopes_of(hq)), cap=dict(cap=30.0), prefix=dict(first=first // 500 * 500, prefix=ints([c + n // 2 for c, n in zip(context, new)]), cap=10.0))[what]
    run(ops, device, context=context, new=new, hq=hq, hkv=hkv, dim=128, page=32, kind=kind, dtype=dtype, seed=len(new), said=20000 if len(new) == 8 else None, **more)
    last = fkl.last_launch()
    assert last["form"] == "shaped_attention_" + form and (last["grid"][0] == int(grid) if int(grid) else last["grid"][0] == hkv and last["grid"][2] == len(new))


# ---- tables -----------------------------------------------------------------------------------------------------------

def tables(ops, device, new, context, page, tokens, max_new, width=4, parents=None):
    batch = len(new)
    table, free = [[-1] * width for _ in new], list(range(batch * width))
    on = [ints(x, device) for x in (table, [0] * batch, context, new, free, [len(free)])]
    got = ops.step_tables(*on, page_tokens=page, tokens=tokens, max_new=max_new, parents=None if parents is None else ints(parents, device))
    want = step_reference.step_tables(table, [0] * batch, context, new, free, len(free), page, tokens, min(max_new, tokens), parents)
    assert on[0].tolist() == want[0]
    for x, y in zip(got[:5], want[1:6]):
        assert x.tolist() == (y if isinstance(y, list) else [y])
    return got


@pytest.mark.parametrize("max_new", [4096, 1 << 27, (1 << 30) // 2 - 1])
def test_tables_of_a_step_that_could_be_larger(ops, device, max_new):
    """Rows are cut off by the step's, however many a request might have."""
    tables(ops, device, [700, 1500], [0, 0], 256, 2300, max_new, width=8)


@pytest.mark.parametrize("tokens,max_new", [(70000, 70000), (1500, 1200)])
def test_tables_of_long_prompts(ops, device, tokens, max_new):
    tables(ops, device, [max_new, 3], [5, 0], 256, tokens, max_new, width=300)


# ---- all --------------------------------------------------------------------------------------------------------------

def a_step(ops, device, **change):
    """The calls around attention by name, of one small step."""
    i = lambda *v: ints(v, device)      # noqa: E731
    q = torch.ones((3, 2, 64), dtype=BF16, device=device)
    cos = torch.ones((4, 32), device=device)
    cache = ops.KvCache.allocate(2, 2, 16, 64, device=device)
    ops.kv_write(cache, torch.zeros((32, 2, 64), dtype=BF16, device=device), torch.zeros((32, 2, 64), dtype=BF16, device=device), torch.arange(32, dtype=torch.int32, device=device))
    target = torch.full((3, 10), 0.1, device=device)
    shaping = dict(slopes=torch.ones(2, device=device))
    calls = dict(
        tables=(ops.step_tables, dict(page_table=i(0, -1).view(1, 2), held=i(1), context=i(15), new=i(3), free=i(1), available=i(1), page_tokens=16, tokens=3, max_new=3, parents=i(-1, 0, 0))),
        axes=(ops.qk_norm_rope, dict(q=q, k=q, q_weight=None, k_weight=None, cos=cos, sin=cos, positions=i(0, 1, 2).expand(2, 3).contiguous(), axes=[0, 1] * 16)),
        attend=(ops.tree_attention, dict(q=q, cache=cache, page_table=i(0, 1).view(1, 2), context=i(15), q_start=i(0, 3), max_new=3, max_context=15, cap=5.0, **shaping)),
        verify=(ops.verify_drafts, dict(target=target, tokens=i(1, 2, 3), q_start=i(0, 3), uniforms=torch.full((3,), 0.5, device=device), max_new=3, draft=target.clone())),
        keep=(ops.kv_keep, dict(caches=[cache], page_table=i(0, 1).view(1, 2), context=i(15), path=i(0, 2, -1).view(1, 3), count=i(2))))
    return {name: (lambda f=f, a=a, **c: f(**{**a, **c}), a) for name, (f, a) in calls.items()}


def flat(x):
    return [] if x is None else [t for t in x if t is not None] if isinstance(x, tuple) else [x]


def test_nothing_to_do(ops, device):
    """No tokens, no requests, no new ones, no entries: results of these sizes, and nothing else changes."""
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)      # noqa: E731
    cache = ops.KvCache.allocate(2, 2, 16, 64, device=device)
    for t in cache._tensors:
        t.view(torch.uint8).fill_(5)
    q, cos = torch.ones((0, 2, 64), dtype=BF16, device=device), torch.ones((4, 32), device=device)
    assert [x.shape[0] for x in ops.qk_norm_rope(q, q, None, None, cos, cos, i(2, 0), axes=[0, 1] * 16)] == [0, 0]
    assert ops.qkv_to_cache(cache, q, q, q, i(0), None, None, cos, cos, i(2, 0), axes=[0, 1] * 16).shape == q.shape
    shaping = dict(cap=2.0, slopes=torch.ones(2, device=device), first=i(0), positions=i(0))
    assert ops.tree_attention(q, cache, i(1, 2), i(1), i(2), max_new=1, max_context=3, **shaping).shape == q.shape
    assert ops.tree_attention(q, cache, i(0, 2), i(0), i(1), max_new=1, max_context=3, prefix=i(0), **shaping).shape == q.shape
    some = torch.ones((3, 2, 64), dtype=BF16, device=device)
    for batch, max_new, width in ((0, 2, 2), (1, 0, 2), (1, 2, 0)):
        out = ops.tree_attention(some, cache, i(batch, width), i(batch), i(batch + 1), max_new=max_new, max_context=3, cap=2.0, prefix=i(batch))
        assert (out == 0).all()
        t = ops.step_tables(i(batch, width), i(batch), i(batch), i(batch) + 2, i(0), i(1), page_tokens=16, tokens=3, max_new=max_new, parents=i(3))
        assert t.q_start.tolist() == [0] * batch + [2 if batch and max_new else 0] and t.slots.tolist() == [-1] * 3 and t.held.tolist() == [0] * batch and t.available.tolist() == [0]
        ops.kv_keep(cache, i(batch, width), i(batch), i(batch, max_new), i(batch) + 2)
    for tokens, batch, max_new in ((0, 2, 3), (3, 0, 3), (3, 2, 0), (0, 0, 0)):
        v = ops.verify_drafts(torch.ones((tokens, 7), device=device), i(tokens), i(batch + 1), torch.ones(tokens, device=device), max_new=max_new)
        assert (v.count == 0).all() and v.path.shape == v.out.shape == (batch, max_new) and (v.path == -1).all() and (v.out == -1).all()
    ops.kv_keep([], i(1, 2), i(1), i(1, 3), i(1) + 3)
    assert all((t.view(torch.uint8) == 5).all() for t in cache._tensors)


def test_gradients_and_tangents_are_refused(ops, device):
    calls = a_step(ops, device)
    for name, argument in (("axes", "q"), ("axes", "cos"), ("attend", "q"), ("attend", "slopes"), ("verify", "target"), ("verify", "draft"), ("verify", "uniforms")):
        call, given = calls[name][0], calls[name][1][argument]
        call()
        with pytest.raises(ValueError, match=f"{argument} asks for a gradient"):
            call(**{argument: torch.nn.Parameter(given)})
        with torch.no_grad():
            call(**{argument: torch.nn.Parameter(given)})
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(ValueError, match=f"{argument} carries a forward-mode tangent"):
                call(**{argument: torch.autograd.forward_ad.make_dual(given, torch.ones_like(given))})


def test_tracers_are_refused(ops, device):
    from torch.fx.experimental.proxy_tensor import make_fx
    calls = a_step(ops, device)
    for name, argument in (("tables", "context"), ("axes", "q"), ("attend", "q"), ("verify", "target"), ("keep", "count")):
        call, given = calls[name][0], calls[name][1][argument]
        traced = lambda x: (flat(call(**{argument: x})) or [x])[0] + 1      # noqa: E731
        with pytest.raises(ValueError, match="tracer"):
            torch.jit.trace(traced, (given,))
        with pytest.raises(ValueError, match="tracer"):
            make_fx(traced)(given)


def test_inference_mode_and_other_streams_give_the_same(ops, device):
    calls = a_step(ops, device)
    want = {name: flat(call()) for name, (call, _) in calls.items()}
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.inference_mode():
        for name, (call, _) in a_step(ops, device).items():
            assert all(torch.equal(x, y) and x.is_inference() for x, y in zip(flat(call()), want[name]))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for name, (call, _) in a_step(ops, device).items():
            assert all(torch.equal(x, y) for x, y in zip(flat(call()), want[name]))


def test_results_of_one_allocation_are_tensors_of_their_own(ops, device):
    """Changed, viewed, saved and taken on by themselves; the memory stays as long as one of them does."""
    calls = a_step(ops, device)
    for name in ("tables", "verify"):
        call = calls[name][0]
        want = [x.clone() for x in flat(call())]
        got = flat(call())
        assert all(x.is_contiguous() and not x.requires_grad and x.data_ptr() % 16 == 0 and x._version == 0 for x in got)
        for k, x in enumerate(got):
            x.fill_(7)
            assert x._version == 1 and all(torch.equal(y, w) for y, w in zip(got[k + 1:], want[k + 1:])) and all((y == 7).all() for y in got[:k])
        last = flat(call())[-1]
        others = [torch.full((64,), 3, dtype=torch.int32, device=device) for _ in range(50)]
        assert torch.equal(last, want[-1]) and torch.equal(last.view(-1)[:1].clone(), want[-1].view(-1)[:1]) and all((t == 3).all() for t in others)
        weight = torch.ones(1, device=device, requires_grad=True)
        (weight * got[0].float()).sum().backward()
        assert float(weight.grad) == 7 * got[0].numel()
