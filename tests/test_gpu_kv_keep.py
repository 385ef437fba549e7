"""kv_keep: the cache afterwards is the cache before with the rows of the accepted tokens moved, byte for byte."""
import random

import pytest
import torch

from attention_reference import Slots
from fusedkernellibrary_amd import attention as ops

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def a_cache(pages, heads, page, dim, codes, seed):
    g = torch.Generator().manual_seed(seed)
    slots = Slots(pages * page, heads, dim, codes, g)
    return ops.KvCache(*slots.tensors(page, "cuda")), slots


def moved(slots, page, table, context, path, count):
    """The moves of one sequence after the other, each from what the cache was before its own path."""
    width, pages, most = len(table[0]) if table else 0, slots.k.shape[0] // page, len(path[0]) if path else 0
    def slot(b, j):
        return table[b][j // page] * page + j % page if j // page < width and 0 <= table[b][j // page] < pages else None
    for b in range(len(table)):
        c = min(max(context[b], 0), 1 << 30)
        moves = [(slot(b, c + path[b][i]), slot(b, c + i)) for i in range(1, min(count[b], most)) if i < path[b][i] < most]
        moves = [m for m in moves if None not in m]
        for x in (slots.k, slots.v, slots.ks, slots.vs):
            rows = [x[a].clone() for a, _ in moves]
            for r, (_, to) in zip(rows, moves):
                x[to] = r


def check(heads, page, dim, codes, context, path, count, layers=1, seed=0, table=None, extra=2):
    rng = random.Random(seed)
    batch, most = len(context), len(path[0])
    if table is None:
        width = max((max(c, 0) + most - 1) // page + 1 for c in context)
        order = rng.sample(range(batch * width + extra), batch * width)
        table = [order[b * width:(b + 1) * width] for b in range(batch)]
    pages = batch * len(table[0]) + extra
    both = [a_cache(pages, heads, page, dim, codes, seed + i) for i in range(layers)]
    ops.kv_keep([c for c, _ in both] if layers > 1 else both[0][0], ints(table).view(batch, -1), ints(context), ints(path).view(batch, -1), ints(count))
    for cache, slots in both:
        moved(slots, page, table, context, path, count)
        now = Slots.of(cache)
        for name in ("k", "v", "ks", "vs"):
            assert torch.equal(getattr(now, name), getattr(slots, name)), name


def a_path(n, most, rng):
    kept = rng.randint(1, n)
    row = [0] + sorted(rng.sample(range(1, n), kept - 1))
    return row + [-1] * (most - len(row)), len(row)


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("heads,page,dim", [(1, 16, 64), (2, 32, 128), (8, 64, 128), (5, 128, 96), (3, 256, 256), (20, 16, 8), (4, 16, 192), (7, 64, 40)])
def test_paths_through_trees(device, codes, heads, page, dim):
    rng = random.Random(dim + heads)
    for most in (2, 13, 64):
        rows = [a_path(rng.randint(1, most), most, rng) for _ in range(6)]
        check(heads, page, dim, codes, [rng.randint(0, 3 * page) for _ in rows], [r for r, _ in rows], [n for _, n in rows], seed=dim + most)


@pytest.mark.parametrize("most", [2, 8, 9, 17, 40, 300])
def test_everything_moves_by_one(device, most):
    """The second token refused, all behind it accepted: each row's place is where the one before it was."""
    path = [0] + list(range(2, most)) + [-1]
    for context in (0, 5, 63):
        check(2, 16, 64, torch.int8, [context, context + 1], [path, path], [most - 1, most - 1], seed=most)


def test_nothing_moves(device):
    check(2, 16, 64, torch.int8, [7, 0], [[0, 1, 2, 3], [0, -1, -1, -1]], [4, 1])
    check(2, 16, 64, torch.int8, [7, 0], [[0, 1, 2, 3], [0, 3, -1, -1]], [0, -4])


def test_many_layers(device):
    rng = random.Random(3)
    rows = [a_path(9, 9, rng) for _ in range(3)]
    check(2, 16, 16, torch.int8, [20, 3, 15], [r for r, _ in rows], [n for _, n in rows], layers=131)


def test_more_sequences_and_heads_than_fit_at_once(device):
    rng = random.Random(4)
    rows = [a_path(6, 6, rng) for _ in range(700)]
    check(9, 16, 16, torch.float8_e4m3fn, [rng.randint(0, 20) for _ in rows], [r for r, _ in rows], [n for _, n in rows])


def test_places_outside(device):
    """Paths that do not fit, counts above the path's room, pages and places outside of the cache: nothing moves there."""
    check(2, 16, 64, torch.int8, [3, 3, 3], [[0, 5, 6, 7], [0, 2, 4, -1], [9, -9, 2 ** 31 - 1, 3]], [9, 2 ** 31 - 1, 4])
    check(1, 16, 64, torch.int8, [10, 10, 10], [[0, 2, 3, 7, 9, 11, 12, 13, 14, 15, -1, -1, -1, -1, -1, 0]] * 3, [10] * 3, table=[[0, 2], [3, -1], [4, 99]])
    check(1, 16, 64, torch.int8, [30, -8, 2 ** 31 - 1], [[0, 2, 3, 5, 9, 10]] * 3, [4] * 3, table=[[0, 2], [3, 1], [4, 5]])


def test_no_sequences(device):
    cache, slots = a_cache(3, 2, 16, 64, torch.int8, 1)
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    ops.kv_keep(cache, empty.view(0, 2), empty, empty.view(0, 4), empty)
    ops.kv_keep([], ints([[0, 1]]), ints([3]), ints([[0, 2]]), ints([2]))
    ops.kv_keep(cache, ints([[]]).view(1, 0), ints([3]), ints([[0, 2]]), ints([2]))
    ops.kv_keep(cache, ints([[1]]), ints([3]), ints([[]]).view(1, 0), ints([2]))
    assert torch.equal(Slots.of(cache).k, slots.k)


def test_the_same_cache_twice_is_refused(device):
    cache, _ = a_cache(3, 2, 16, 64, torch.int8, 1)
    other, _ = a_cache(4, 2, 16, 64, torch.int8, 1)
    with pytest.raises(ValueError, match="twice"):
        ops.kv_keep([cache, cache], ints([[0, 1]]), ints([3]), ints([[0, 2]]), ints([2]))
    with pytest.raises(ValueError, match="different sizes"):
        ops.kv_keep([cache, other], ints([[0, 1]]), ints([3]), ints([[0, 2]]), ints([2]))


def test_a_moved_cache_counts_as_changed(device):
    cache, _ = a_cache(3, 2, 16, 64, torch.int8, 1)
    before = cache.k._version
    ops.kv_keep(cache, ints([[0, 1]]), ints([3]), ints([[0, 2]]), ints([2]))
    assert cache.k._version > before


def test_a_captured_call(device):
    rng = random.Random(6)
    cache, slots = a_cache(12, 2, 16, 64, torch.int8, 2)
    table, context = ints([[0, 1, 2], [5, 4, 3], [8, 9, 10]]), ints([1, 2, 3])
    path, count = ints([[0] * 12] * 3), ints([0, 0, 0])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.kv_keep(cache, table, context, path, count)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ops.kv_keep(cache, table, context, path, count)
    for _ in range(4):
        rows = [a_path(12, 12, rng) for _ in range(3)]
        c = [rng.randint(0, 30) for _ in rows]
        path.copy_(ints([r for r, _ in rows])), count.copy_(ints([n for _, n in rows])), context.copy_(ints(c))
        graph.replay()
        torch.cuda.synchronize()
        moved(slots, 16, table.tolist(), c, [r for r, _ in rows], [n for _, n in rows])
        assert torch.equal(Slots.of(cache).k, slots.k) and torch.equal(Slots.of(cache).v, slots.v)
