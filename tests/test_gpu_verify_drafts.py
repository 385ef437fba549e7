"""verify_drafts against its definition (tests/step_reference.py), number for number."""
import math
import random

import pytest
import torch

import step_reference as ref
from fusedkernellibrary_amd import attention as ops

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def drafts(new, vocab, dtype, seed, kind, sharp=3.0):
    """Rows, tokens and uniforms of sequences of `new` rows: a chain with its draft's probabilities, without, or trees."""
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    tokens = sum(new)
    logits = torch.randn((tokens, vocab), generator=g) * sharp
    target = torch.softmax(logits, -1).to(dtype)
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    parents = [p for n in new for p in [-1] * (n > 0) + [rng.randint(max(0, t - 4), t - 1) if kind == "tree" else t - 1 for t in range(1, n)]]
    before = torch.tensor([starts[b] + max(0, parents[starts[b] + t]) for b, n in enumerate(new) for t in range(n)], dtype=torch.long)
    q = torch.softmax(logits[before] + 0.5 * torch.randn((tokens, vocab), generator=g), -1) if tokens else logits
    ids = torch.multinomial(q.double(), 1, generator=g)[:, 0].to(torch.int32) if tokens else torch.zeros(0, dtype=torch.int32)
    return dict(target=target, ids=ids, q_start=torch.tensor(starts, dtype=torch.int32), uniforms=torch.rand(tokens, generator=g), max_new=max(new, default=0),
                draft=q.to(dtype) if kind == "drafted" else None, parents=torch.tensor(parents, dtype=torch.int32) if kind == "tree" else None)


def want_of(d):
    rows = lambda t: None if t is None else t.double().tolist()      # noqa: E731
    return ref.verify(rows(d["target"]), d["ids"].tolist(), d["q_start"].tolist(), d["uniforms"].double().tolist(), d["max_new"], rows(d["draft"]),
                      None if d["parents"] is None else d["parents"].tolist())


def run(d):
    on = {n: t.cuda() if isinstance(t, torch.Tensor) and not t.is_cuda else t for n, t in d.items()}
    return ops.verify_drafts(on["target"], on["ids"], on["q_start"], on["uniforms"], max_new=on["max_new"], draft=on["draft"], parents=on["parents"])


def check(d, got=None):
    *want, margin = want_of(d)
    # Sums of v weights in 64 bits, in whatever order, are off by at most v 2^-53 of their total, on both sides.
    assert margin > 2 * d["target"].shape[1] * 2.0 ** -53, "a border too near to a running sum to say which token is right"
    got = got or run(d)
    for name, x, y in zip(ops.Verified._fields, got, want):
        assert x.dtype == torch.int32 and x.cpu().tolist() == y, name
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["drafted", "chain", "tree"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 100, 4095, 4096, 4097, 8200, 40001])
def test_vocabularies(device, dtype, kind, vocab):
    check(drafts([1, 4, 7, 2, 5], vocab, dtype, vocab, kind))


@pytest.mark.parametrize("new", [[1], [0], [0, 3, 0, 0, 2, 0], [9] * 40, [64, 1, 33], [65, 128, 70], [200]])
@pytest.mark.parametrize("kind", ["drafted", "chain", "tree"])
def test_lengths(device, new, kind):
    check(drafts(new, 50, torch.float32, sum(new), kind, sharp=0.3))


@pytest.mark.parametrize("new", [1023, 1024])
def test_long_chains_that_are_accepted(device, new):
    d = drafts([new, 3], 17, torch.float32, new, "chain")
    d["uniforms"][:] = 0.0
    got = check(d)
    assert int(got.count[0]) == new
    wide = drafts([new], 17, torch.float32, new, "tree", sharp=0.1)                 # children far behind their parents
    wide["parents"] = torch.tensor([-1] + [0 if t < 900 else 700 for t in range(1, new)], dtype=torch.int32)
    check(wide)


@pytest.mark.parametrize("vocab,batch", [(1 << 20, 2), ((1 << 20) + 3, 1), (131072, 5)])
def test_large_vocabularies(device, vocab, batch):
    for dtype in (torch.float32, torch.bfloat16):
        check(drafts([2] * batch, vocab, dtype, vocab + batch, "drafted", sharp=1.0))


def test_more_sequences_than_compute_units(device):
    check(drafts([2, 1, 3] * 200, 33, torch.float16, 5, "drafted"))


def test_rows_of_other_strides(device):
    """Rows with others in between, at odd elements, and one row for all."""
    for dtype in TYPES:
        d = drafts([3, 5, 1], 77, dtype, 4, "drafted")
        wide = [torch.zeros((9, 191), dtype=dtype, device="cuda") for _ in range(2)]
        on = dict(d)
        for w, n, at in zip(wide, ("target", "draft"), (1, 37)):
            w[:, at:at + 77] = d[n].cuda()
            on[n] = w[:, at:at + 77]
        check(d, run(on))
        one = dict(d, target=d["target"][:1].expand(9, 77), draft=None)
        check(one, run(dict(one, target=d["target"][:1].cuda().expand(9, 77))))


def test_greedy_targets(device):
    """One token with all probability: drafts that have it are accepted, whatever the uniforms are."""
    d = drafts([4, 4, 4], 6, torch.float32, 1, "chain")
    best = torch.randint(0, 6, (12,), generator=torch.Generator().manual_seed(2))
    d["target"] = torch.nn.functional.one_hot(best, 6).float()
    d["ids"][1:4] = best[0:3]
    d["ids"][5:8] = torch.stack([best[4], best[5], (best[6] + 1) % 6])
    d["ids"][9] = (best[8] + 1) % 6
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        d["uniforms"][:] = u
        for kind in ("chain", "tree"):
            got = check(dict(d, parents=torch.tensor([-1, 0, 1, 2] * 3, dtype=torch.int32) if kind == "tree" else None))
            assert got.count.tolist() == [4, 3, 1] and got.out[0].tolist() == best[:4].tolist()


def test_a_token_that_was_refused_is_refused_again(device):
    d = drafts([5, 4], 4, torch.float32, 3, "tree")
    d["target"][:] = torch.tensor([0.5, 0.25, 0.125, 0.125])
    d["parents"] = torch.tensor([-1, 0, 0, 0, 0, -1, 0, 0, 0], dtype=torch.int32)
    d["ids"] = torch.tensor([0, 0, 0, 1, 0, 0, 2, 2, 2], dtype=torch.int32)
    d["uniforms"] = torch.tensor([0.7, 0.9, 0.0, 0.6, 0.0, 0.3, 0.5, 0.0, 0.0])
    got = check(d)
    assert got.count.tolist() == [1, 1] and got.out[:, 0].tolist() == [3, 0]        # 0 and 1 are out, of 2 and 3 it is 3; 2 is out


def test_refused_tokens_across_64_rows(device):
    d = drafts([130], 5, torch.float32, 3, "tree")
    d["target"][:] = torch.tensor([0.1, 0.2, 0.3, 0.15, 0.25])
    d["parents"] = torch.tensor([-1] + [0] * 129, dtype=torch.int32)
    d["ids"] = torch.tensor([0] + [0] * 70 + [1, 0, 1, 2] * 14 + [4, 3, 3], dtype=torch.int32)
    d["uniforms"] = torch.tensor([0.5] + [0.95] * 127 + [0.95, 0.99])
    check(d)


def test_no_weight_left(device):
    """A draft that has all that the target has, and a child for each token: the target's row whole; a row of nothing: -1."""
    d = drafts([2, 2], 5, torch.float32, 3, "drafted")
    d["target"][0] = torch.tensor([0.5, 0.5, 0.0, 0.0, 0.0])
    d["draft"][1] = torch.tensor([0.5, 0.5, 0.0, 0.0, 0.0])
    d["ids"][1] = 2
    d["uniforms"][0] = 0.75
    d["target"][2] = 0.0
    got = check(d)
    assert got.out[:, 0].tolist() == [1, -1]
    d = drafts([6], 5, torch.float32, 3, "tree")
    d["parents"] = torch.tensor([-1, 0, 0, 0, 0, 0], dtype=torch.int32)
    d["ids"] = torch.tensor([0, 0, 1, 2, 3, 4], dtype=torch.int32)
    d["target"][0] = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0])
    assert check(d).out[0, 0] == -1


def test_what_is_no_probability(device):
    for dtype in TYPES:
        d = drafts([3, 2, 4], 40, dtype, 9, "drafted")
        for n in ("target", "draft"):
            d[n][:, 3], d[n][:, 5], d[n][:, 7], d[n][:, 11] = math.nan, math.inf, -math.inf, -0.25
        d["ids"][1], d["ids"][4], d["ids"][6] = 3, 5, 7
        check(d)
        d["target"][:] = math.nan
        assert (check(d).out[:, 0] == -1).all()


def test_tokens_and_uniforms_outside(device):
    for kind in ("drafted", "chain", "tree"):
        d = drafts([4] * 6, 20, torch.float32, 12, kind)
        d["ids"][1::3] = torch.tensor([-1, 20, 2 ** 31 - 1, -2 ** 31, 19, 0, 21, 5], dtype=torch.int32)
        check(d)
        d["uniforms"][:12] = torch.tensor([0.0, 1.0, 2.0, -1.0, math.nan, math.inf, -math.inf, 1.0, 1 - 2.0 ** -24, 0.0, 2.0 ** -149, 1.0])
        *want, _ = want_of(d)                                                     # (a uniform of 0 is a border of 0: no sum is near it)
        got = run(d)
        for x, y in zip(got, want):
            assert x.cpu().tolist() == y


def test_parents_that_are_none(device):
    d = drafts([70, 6], 9, torch.float32, 2, "tree", sharp=0.2)
    rng = random.Random(1)
    d["parents"] = torch.tensor([rng.choice([-1, -7, t, t + 2, 2 ** 31 - 1, 0, t // 2, max(0, t - 1)]) for n in (70, 6) for t in range(n)], dtype=torch.int32)
    d["uniforms"] *= 0.1
    check(d)


def test_sequences_outside_of_the_rows(device):
    d = drafts([3, 4, 2], 30, torch.float32, 7, "drafted")
    for starts, most in (([0, 3, 7, 9], 2), ([0, 3, 7, 100], 50), ([-5, 3, 7, 9], 4), ([2, 3, 3, 8], 4), ([9, 9, 9, 9], 3), ([20, 30, 40, 50], 3), ([5, 3, 7, 6], 4), ([-5, -3, -1, 2], 4)):
        check(dict(d, q_start=torch.tensor(starts, dtype=torch.int32), max_new=most))
    none = run(dict(d, max_new=0))
    assert none.count.tolist() == [0, 0, 0] and none.path.shape == (3, 0)
    none = run(dict(d, q_start=torch.zeros(1, dtype=torch.int32)))
    assert none.count.numel() == 0


def test_the_next_token_is_distributed_as_the_target(device):
    """All drafted tokens, and a grid of uniforms for the question and the draw: what a sequence's first decided token is, weighted
    by the draft's probabilities. A grid of N counts an interval to within 1 / N, and a token's chance is an interval of the
    question for its own draft and one of the draw for each draft: within 2 / N."""
    n = 128
    p, q = torch.tensor([0.31, 0.02, 0.2, 0.07, 0.4]), torch.tensor([0.1, 0.3, 0.25, 0.3, 0.05])
    grid = (torch.arange(n) + 0.5) / n
    ids, ask, draw = (x.reshape(-1) for x in torch.meshgrid(torch.arange(5).float(), grid, grid, indexing="ij"))
    ids = ids.long()
    batch = len(ids)
    assert batch > 65535
    chances = []
    for some in (slice(0, batch // 2), slice(batch // 2, batch)):                   # (two calls of fewer than 65536)
        m = len(ids[some])
        two = lambda a, b: torch.stack([a, b], 1).reshape(-1)      # noqa: E731
        d = dict(target=p.expand(2 * m, 5).contiguous(), draft=q.expand(2 * m, 5).contiguous(), ids=two(ids[some], ids[some]).to(torch.int32), uniforms=two(draw[some], ask[some]),
                 q_start=torch.arange(0, 2 * m + 1, 2, dtype=torch.int32), max_new=2, parents=None)
        chances.append(run(d).out[:, 0].cpu())
    first = torch.cat(chances).view(5, -1)
    got = sum(q[i].item() * torch.bincount(first[i].long(), minlength=5).double() / (n * n) for i in range(5))
    assert (got - p.double()).abs().max() <= 2 / n
    # without draft's probabilities: whatever is drafted, the target's come out
    d = dict(d, draft=None)
    first = run(d).out[:, 0].cpu()
    for i in (3, 4):
        mine = first[ids[batch // 2:] == i]
        assert (torch.bincount(mine.long(), minlength=5).double() / len(mine) - p.double()).abs().max() <= 2 / n


def test_a_captured_call(device):
    sets = [drafts([3, 6, 1, 4], 9000, torch.float32, s, "tree") for s in range(4)]
    on = {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in sets[0].items()}
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        run(on)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = run(on)
    for d in sets:
        for n in ("target", "ids", "uniforms", "parents", "q_start"):
            on[n].copy_(d[n])
        graph.replay()
        torch.cuda.synchronize()
        check(d, got)


def test_streams_at_once(device):
    """Calls on two streams, each with a workspace of its own."""
    sets = [drafts([5] * 30, 20000, torch.float32, s, "drafted", sharp=1.0) for s in range(2)]
    on = [{n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in d.items()} for d in sets]
    streams, got = [torch.cuda.Stream() for _ in sets], []
    torch.cuda.synchronize()
    for _ in range(5):
        for s, d in zip(streams, on):
            with torch.cuda.stream(s):
                got.append(run(d))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        if i < 2 or i > 7:
            check(sets[i % 2], g)
