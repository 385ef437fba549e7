"""step_tables against its definition (tests/step_reference.py), number for number."""
import random

import pytest
import torch

import step_reference as ref
from fusedkernellibrary_amd import attention as ops

pytestmark = pytest.mark.gpu


def ints(x, device="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def requests(batch, most, rng, page=16, width=None, spare=5, context=(0, 300), held_more=0.3, none=0.1):
    new = [0 if rng.random() < none else rng.randint(1, max(1, most)) for _ in range(batch)]
    context = [rng.randint(*context) for _ in range(batch)]
    have = [-(-c // page) for c in context]
    held = [h + (rng.random() < held_more) for h in have]
    needs = [max(0, -(-(c + n) // page) - h) if n else 0 for c, n, h in zip(context, new, held)]
    width = width or max([h + n for h, n in zip(held, needs)], default=1) + 1
    pages = iter(rng.sample(range(100000), sum(held) + sum(needs) + 200))
    table = [[next(pages) if i < h else -7 for i in range(width)] for h in held]
    free = [next(pages) for _ in range(sum(needs) + spare + 3)]
    return dict(table=table, held=held, context=context, new=new, free=free, available=sum(needs) + spare, page=page, max_new=most)


def tree(new, rng, far=6):
    return [p for n in new for p in [-1] * (n > 0) + [rng.randint(max(0, t - far), t - 1) for t in range(1, n)]]


def check(r, tokens, parents=None):
    batch = len(r["table"])
    width = len(r["table"][0]) if batch else 3
    table = ints(r["table"]).view(batch, width)
    args = [ints(r[n]).view(-1) for n in ("held", "context", "new", "free")] + [ints([r["available"]])]
    got = ops.step_tables(table, *args, page_tokens=r["page"], tokens=tokens, max_new=r["max_new"], parents=None if parents is None else ints(parents).view(-1))
    want = ref.step_tables(r["table"], r["held"], r["context"], r["new"], r["free"], r["available"], r["page"], tokens, r["max_new"], parents)
    for name, x, y in zip(("page_table", "q_start", "slots", "positions", "held", "available"), (table, *got[:5]), want):
        assert x.cpu().flatten().tolist() == torch.tensor(y).flatten().tolist(), name
    if parents is None:
        assert got.mask is None
    else:
        assert got.mask.cpu().tolist() == want[6]
    return got


@pytest.mark.parametrize("batch,most", [(1, 1), (3, 1), (4, 7), (5, 64), (64, 3), (257, 2), (1030, 1), (2, 1025), (7, 2500)])
@pytest.mark.parametrize("padding", [0, 37])
def test_requests_of_all_sizes(device, batch, most, padding):
    r = requests(batch, most, random.Random(batch * 1000 + most), page=32 if most > 64 else 16)
    check(r, sum(r["new"]) + padding)


@pytest.mark.parametrize("batch,most", [(1, 1), (4, 2), (5, 29), (9, 63), (8, 64), (3, 65), (6, 128), (2, 200), (1, 700)])
@pytest.mark.parametrize("far", [1, 6, 1000])
def test_trees_see_their_ancestors(device, batch, most, far):
    """Chains (far 1), ordinary trees, and trees whose branches begin anywhere; more than 64 tokens in words behind each other."""
    rng = random.Random(batch * 1000 + most + far)
    r = requests(batch, most, rng, page=64)
    check(r, sum(r["new"]) + 5, tree(r["new"], rng, far) + [-1] * 5)


def test_no_requests(device):
    r = dict(table=[], held=[], context=[], new=[], free=[3, 4], available=2, page=16, max_new=4)
    check(r, 0)
    check(r, 300)
    check(r, 3, [-1] * 3)


def test_requests_without_new_tokens_take_no_page(device):
    r = requests(6, 4, random.Random(1))
    r["new"], r["held"] = [0] * 6, [0] * 6
    check(r, 10)


@pytest.mark.parametrize("available", [0, 1, 3, 6, -4, 1000])
def test_too_few_pages(device, available):
    """Pages go to the requests in their order; tokens without one have slot -1, and what is missing is counted."""
    r = requests(9, 70, random.Random(available), none=0.0)
    r["available"] = available
    got = check(r, sum(r["new"]))
    assert available > 50 or (got.slots == -1).any()


def test_a_narrow_table_cuts_off(device):
    r = requests(5, 60, random.Random(8), width=4, context=(0, 100))
    r["held"] = [min(4, h) for h in r["held"]]
    check(r, sum(r["new"]))
    r = requests(5, 60, random.Random(9), width=4)
    r["held"] = [9, -3, 4, 2 ** 31 - 1, -2 ** 31]
    check(r, sum(r["new"]))


def test_lengths_outside_of_what_was_said(device):
    r = requests(8, 5, random.Random(4), none=0.0)
    r["new"] = [3, -1, 9, 2 ** 31 - 1, -2 ** 31, 1, 0, 5]
    r["context"] = [0, 20, -5, 16, 7, 2 ** 31 - 1, 3, 1 << 30]
    check(r, 40)
    check(r, 11)                                               # (rows above the step's are cut off)
    check(r, 0)


def test_pages_that_are_no_pages(device):
    r = requests(4, 6, random.Random(2), none=0.0)
    r["table"][1] = [-1] * len(r["table"][1])
    r["table"][2] = [2 ** 31 - 1] * len(r["table"][2])
    check(r, sum(r["new"]))


def test_parents_that_are_none(device):
    """A parent that is not in front of its token counts as none."""
    r = requests(3, 70, random.Random(6), none=0.0)
    r["new"] = [70, 3, 66]
    check(r, 139, [random.Random(7).choice([-1, -9, t, t + 1, 2 ** 31 - 1, 0, t // 2]) for n in r["new"] for t in range(n)])


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_all_page_sizes(device, page):
    r = requests(6, 300, random.Random(page), page=page, context=(0, 2000))
    check(r, sum(r["new"]))


def test_a_captured_step_follows_its_lengths(device):
    """Captured once, replayed with other lengths, tables and parents in the same tensors; results equal the definition's each time."""
    rng = random.Random(3)
    sets = [requests(10, 20, rng, width=30) for _ in range(4)]
    trees = [tree(r["new"], rng) for r in sets]
    tokens, count = 200, max(len(r["free"]) for r in sets)
    table = ints(sets[0]["table"])
    args = [ints(sets[0][n]) for n in ("held", "context", "new")] + [ints([0] * count), ints([0])]
    parents = ints([-1] * tokens)
    run = lambda: ops.step_tables(table, *args, page_tokens=16, tokens=tokens, max_new=20, parents=parents)      # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = run()
    for r, p in zip(sets, trees):
        free = r["free"] + [0] * (count - len(r["free"]))
        for x, y in zip((table, *args), (r["table"], r["held"], r["context"], r["new"], free, [r["available"]])):
            x.copy_(ints(y))
        parents.copy_(ints(p + [-1] * (tokens - len(p))))
        graph.replay()
        torch.cuda.synchronize()
        want = ref.step_tables(r["table"], r["held"], r["context"], r["new"], free, r["available"], 16, tokens, 20, p + [-1] * (tokens - len(p)))
        for x, y in zip((table, *got), want):
            assert x.cpu().flatten().tolist() == torch.tensor(y).flatten().tolist()


def test_on_another_stream(device):
    rng = random.Random(5)
    r = requests(50, 8, rng)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        check(r, sum(r["new"]) + 3)
