"""Steps of drafted tokens as a server runs them, tables, norm and rotation by several axes into the caches of some layers,
attention with shaped scores, verification and the kept rows: each part against its reference, then the same steps in other
ways (replayed from a graph, spelled with the C++ host API), bit for bit."""
import ctypes as C
import os
import random

import pytest
import torch

import shaped_reference
import step_reference
from attention_reference import Slots, check
from test_attention_refusals import Attention, Cache, Heads, Rows
from test_gpu_attention import tables
from test_gpu_kv_keep import moved
from test_step_refusals import Drafts, Scores, Tables

pytestmark = pytest.mark.gpu

BF16, F16, INT8, E4M3 = torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
BATCH, TOKENS, MAX_NEW, HQ, HKV, LAYERS, VOCAB, PAGES, ENTRIES, MAX_CONTEXT, CAP = 4, 24, 9, 6, 2, 2, 50, 40, 12, 150, 20.0
STATE = "table", "held", "context", "available"


@pytest.fixture(scope="module")
def ops():
    from fusedkernellibrary_amd import attention
    return attention


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


class Server:
    """Caches, pages and requests' lengths; `step` takes one step's inputs, dicts of tensors on the device, from where they are."""

    def __init__(self, ops, device, dim, page, kind, dtype, start=0):
        g = torch.Generator().manual_seed(dim + page)
        self.ops, self.device, self.dim, self.page, self.kind, self.dtype = ops, device, dim, page, kind, dtype
        self.caches = [ops.KvCache(*Slots(PAGES * page, HKV, dim, kind, g).tensors(page, device)) for _ in range(LAYERS)]
        order = torch.randperm(PAGES, generator=g).to(torch.int32)
        # a request has its first tokens in the cache already (what they hold is random), another begins
        context = ints([37, 0, 1, 100])
        held = (context + page - 1) // page
        table = torch.full((BATCH, ENTRIES), -1, dtype=torch.int32)
        used = 0
        for b in range(BATCH):
            n = int(held[b])
            table[b, :n] = order[used:used + n]
            used += n
        self.table, self.held, self.context, self.available = (t.to(device) for t in (table, held, context, ints([PAGES - used])))
        self.free = order[used:].contiguous().to(device)
        self.weights = [(1 + 0.3 * torch.randn((2, dim), generator=g)).to(dtype).to(device) for _ in range(LAYERS)]
        self.cos, self.sin = (t.to(device) for t in tables(300, dim))
        self.slopes = (2.0 ** -torch.arange(1, HQ + 1)).to(device)
        self.axes = [i % 3 for i in range(dim // 2)]

    def state(self):
        return [getattr(self, n) for n in STATE] + [t.view(torch.int8) if t.dtype == E4M3 else t for c in self.caches for t in c._tensors]

    def front(self, x):
        t = self.ops.step_tables(self.table, self.held, self.context, x["new"], self.free, self.available, page_tokens=self.page, tokens=TOKENS, max_new=MAX_NEW, parents=x["parents"])
        at, got = torch.stack([t.positions, *x["frames"]]), []
        for cache, w, packed in zip(self.caches, self.weights, x["packed"]):
            q, k, v = packed.split([HQ, HKV, HKV], 1)
            q = self.ops.qkv_to_cache(cache, q, k, v, t.slots, w[0], w[1], self.cos, self.sin, at, axes=self.axes)
            out = self.ops.tree_attention(q, cache, self.table, self.context, t.q_start, max_new=MAX_NEW, max_context=MAX_CONTEXT, mask=t.mask, cap=CAP, slopes=self.slopes, positions=t.positions,
                                          first=x["first"])
            got.append((q, out))
        return t, got

    def back(self, x, t):
        v = self.ops.verify_drafts(x["target"], x["ids"], t.q_start, x["uniforms"], max_new=MAX_NEW, parents=x["parents"])
        self.ops.kv_keep(self.caches, self.table, self.context, v.path, v.count)
        self.held.copy_(t.held)
        self.available.copy_(t.available)
        self.context.add_(v.count)
        return v

    def step(self, x):
        t, got = self.front(x)
        return t, got, self.back(x, t)


def some_inputs(server, seed, new):
    """A step's inputs on the device; drafted tokens drawn from the target, so that some are accepted."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    parents = []
    for n in new:
        parents += [-1] + [rng.randint(max(0, t - 3), t - 1) for t in range(1, n)] if n else []
    parents += [rng.randint(-5, 5) for _ in range(TOKENS - len(parents))]
    target = (3 * torch.randn((TOKENS, VOCAB), generator=g)).softmax(-1)
    ids, lo = torch.randint(0, VOCAB, (TOKENS,), generator=g).to(torch.int32), 0
    for n in new:
        for t in range(1, n):
            ids[lo + t] = torch.multinomial(target[lo + parents[lo + t]], 1, generator=g)[0]
        lo += n
    context = server.context.tolist()
    want = step_reference.step_tables(server.table.tolist(), server.held.tolist(), context, new, server.free.tolist(), int(server.available), server.page, TOKENS, MAX_NEW, parents)
    first = (ints(want[3]) - 45).clamp(min=0).to(torch.int32)
    x = dict(new=ints(new), parents=ints(parents), frames=torch.randint(0, 300, (2, TOKENS), generator=g, dtype=torch.int32), first=first,
             packed=torch.randn((LAYERS, TOKENS, HQ + 2 * HKV, server.dim), generator=g).to(server.dtype), target=target, ids=ids, uniforms=torch.rand(TOKENS, generator=g))
    return {k: v.to(server.device) for k, v in x.items()}, want


NEW = [[9, 1, 5, 0], [4, 9, 1, 6], [1, 1, 1, 1], [0, 7, 9, 8]]
FORMS = [(64, 16, INT8, BF16), (128, 32, E4M3, F16)]


def copies(t, got, v):
    return [x.clone() for x in (t.q_start, t.slots, t.positions, t.held, t.available, t.mask, *sum(got, ()), v.path, v.count, v.out)]


def same(a, b):
    bits = lambda t: t.view(torch.int16) if t.dtype in (BF16, F16) else t.view(torch.int32) if t.dtype == torch.float32 else t      # noqa: E731
    return len(a) == len(b) and all(torch.equal(bits(x), bits(y)) for x, y in zip(a, b))


@pytest.mark.parametrize("dim,page,kind,dtype", FORMS)
def test_each_part_of_the_steps(ops, device, dim, page, kind, dtype):
    s = Server(ops, device, dim, page, kind, dtype)
    accepted = 0
    for i, new in enumerate(NEW):
        x, want = some_inputs(s, 10 + i, new)
        t, got = s.front(x)
        table, start, slots, positions, held, left, masks = want
        assert s.table.tolist() == table and t.q_start.tolist() == start and t.slots.tolist() == slots and t.positions.tolist() == positions
        assert t.held.tolist() == held and t.available.tolist() == [left] and t.mask.tolist() == masks and left >= 0
        before = [Slots.of(c) for c in s.caches]
        host = {k: v.cpu() for k, v in x.items()}
        for layer, (q, out) in zip(before, got):
            # int8 caches hold queries to 2^-16, as tests/shaped_reference.py counts
            ref, bound, _, _ = shaped_reference.attention(q.cpu(), layer, page, s.table.cpu(), s.context.tolist(), ints(start), dim ** -0.5, dtype, mask=t.mask.cpu(), cap=CAP, slopes=s.slopes.cpu(),
                                                          positions=t.positions.cpu(), first=host["first"])
            check(out.cpu(), ref, bound)
        context = s.context.tolist()
        v = s.back(x, t)
        exact = lambda m: [[float(p) for p in row] for row in m.double()]      # noqa: E731
        path, count, out, margin = step_reference.verify(exact(host["target"]), host["ids"].tolist(), start, host["uniforms"].tolist(), MAX_NEW, parents=host["parents"].tolist())
        assert margin > 1e-9 and (v.path.tolist(), v.count.tolist(), v.out.tolist()) == (path, count, out)
        for layer, cache in zip(before, s.caches):
            moved(layer, page, table, context, path, count)
            now = Slots.of(cache)
            assert all(torch.equal(getattr(now, n), getattr(layer, n)) for n in ("k", "v", "ks", "vs"))
        assert s.context.tolist() == [c + n for c, n in zip(context, count)]
        accepted += sum(max(0, n - 1) for n in count)
    assert accepted > 0                                                            # (the steps do keep drafted tokens)


@pytest.mark.parametrize("dim,page,kind,dtype", FORMS)
def test_replayed_steps(ops, device, dim, page, kind, dtype):
    """One graph is every step: lengths, pages and what is accepted live on the device."""
    s = Server(ops, device, dim, page, kind, dtype)
    start = [t.clone() for t in s.state()]
    steps, want = [], []
    for i, new in enumerate(NEW):
        x, _ = some_inputs(s, 20 + i, new)
        steps.append(x)
        want.append(copies(*s.step(x)) + [t.clone() for t in s.state()])

    def reset():
        for t, value in zip(s.state(), start):
            t.copy_(value)
    static = {k: v.clone() for k, v in steps[0].items()}
    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = s.step(static)
    for again in range(3):
        reset()
        for i, x in enumerate(steps):
            for k, v in x.items():
                static[k].copy_(v)
            graph.replay()
            assert same(copies(*results) + s.state(), want[i]), (again, i)
            if again:
                # a step of another server in between
                other = Server(ops, device, dim, page, kind, dtype)
                y, _ = some_inputs(other, 20, NEW[0])
                other.step(y)
                torch.cuda.synchronize()


def rows(t):
    return Rows(t.data_ptr(), t.stride(0), t.stride(1))


class Spelled:
    """A server's step as the C++ host API takes it, with results of its own."""

    def __init__(self, s, x):
        import fusedkernellibrary_amd as fkl
        fkl.lib()
        self.lib = lib = C.CDLL(os.path.join(os.path.dirname(os.path.abspath(__file__)), "cases", "libdrafts_step.so"))
        lib.drafts_step_error.restype = C.c_char_p
        lib.drafts_step_open.restype = C.c_void_p
        lib.drafts_step_close.argtypes = [C.c_void_p]
        lib.drafts_step_reserve.argtypes = [C.c_void_p, C.POINTER(Attention), C.POINTER(Drafts), C.POINTER(Cache)]
        lib.drafts_step_run.argtypes = [C.c_void_p, C.POINTER(Tables), C.POINTER(Heads), C.c_char_p, C.c_int32, C.c_int32, C.c_int64, C.POINTER(Attention), C.POINTER(Scores), C.POINTER(Drafts),
                                        C.POINTER(Cache), C.c_int32, C.c_void_p]
        lib.drafts_step_turn.argtypes = [C.POINTER(Heads), C.c_char_p, C.c_int32, C.c_int32, C.c_int64, C.c_void_p]
        make = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype, device=s.device)      # noqa: E731
        self.s, self.x = s, x
        self.at = make(3, TOKENS)
        self.q_start, self.slots, self.held, self.left, self.mask = make(BATCH + 1), make(TOKENS), make(BATCH), make(1), make(TOKENS, 1, dtype=torch.int64)
        self.path, self.count, self.out = make(BATCH, MAX_NEW), make(BATCH), make(BATCH, MAX_NEW)
        self.got = [(make(TOKENS, HQ, s.dim, dtype=s.dtype), make(TOKENS, HQ, s.dim, dtype=s.dtype)) for _ in range(LAYERS)]
        p = lambda t: t.data_ptr()      # noqa: E731
        self.tables = Tables(page_table=p(s.table), held=p(s.held), context=p(s.context), fresh=p(x["new"]), free_pages=p(s.free), available=p(s.available), parents=p(x["parents"]),
                             q_start=p(self.q_start), slots=p(self.slots), positions=p(self.at), held_out=p(self.held), left=p(self.left), mask=p(self.mask), tokens=TOKENS,
                             page_table_stride=ENTRIES, free_count=len(s.free), batch=BATCH, page_tokens=s.page, max_new=MAX_NEW, mask_words=1)
        self.heads, self.calls, self.caches = (Heads * LAYERS)(), (Attention * LAYERS)(), (Cache * LAYERS)()
        kind = int(s.dtype == F16)
        for i in range(LAYERS):
            packed, (q, out), c = x["packed"][i], self.got[i], s.caches[i]
            self.heads[i] = Heads(q=rows(packed[:, :HQ]), k=rows(packed[:, HQ:HQ + HKV]), v=rows(packed[:, HQ + HKV:]), q_out=rows(q), q_weight=p(s.weights[i][0]), k_weight=p(s.weights[i][1]),
                                  cos=p(s.cos), sin=p(s.sin), positions=p(self.at), slots=p(self.slots), tokens=TOKENS, table_rows=300, q_heads=HQ, kv_heads=HKV, head_dim=s.dim, rot_dim=s.dim,
                                  type=kind, eps=1e-6)
            self.calls[i] = Attention(q=rows(q), out=rows(out), page_table=p(s.table), context=p(s.context), q_start=p(self.q_start), mask=p(self.mask), tokens=TOKENS, page_table_stride=ENTRIES,
                                      batch=BATCH, max_new=MAX_NEW, max_context=MAX_CONTEXT, mask_words=1, q_heads=HQ, type=kind, scale=s.dim ** -0.5)
            self.caches[i] = Cache(p(c.k), p(c.v), p(c.k_scale), p(c.v_scale), c.pages, HKV, s.page, s.dim, int(s.kind == E4M3))
        self.scores = Scores(slopes=p(s.slopes), positions=p(self.at), first=p(x["first"]), cap=CAP)
        self.drafts = Drafts(target=p(x["target"]), ids=p(x["ids"]), q_start=p(self.q_start), parents=p(x["parents"]), uniforms=p(x["uniforms"]), path=p(self.path), count=p(self.count),
                             out=p(self.out), tokens=TOKENS, target_stride=VOCAB, batch=BATCH, max_new=MAX_NEW, vocab=VOCAB, type=2)
        self.server = lib.drafts_step_open()

    def reserve(self):
        assert self.lib.drafts_step_reserve(self.server, C.byref(self.calls[0]), C.byref(self.drafts), C.byref(self.caches[0])) == 0, self.lib.drafts_step_error()

    def run(self):
        self.at[1:].copy_(self.x["frames"])
        return self.lib.drafts_step_run(self.server, C.byref(self.tables), self.heads, bytes(self.s.axes), len(self.s.axes), 3, TOKENS, self.calls, C.byref(self.scores), C.byref(self.drafts),
                                        self.caches, LAYERS, torch.cuda.current_stream().cuda_stream)

    def after(self):
        self.s.held.copy_(self.held)
        self.s.available.copy_(self.left)
        self.s.context.add_(self.count)

    def results(self):
        return [x.clone() for x in (self.q_start, self.slots, self.at[0], self.held, self.left, self.mask, *sum(self.got, ()), self.path, self.count, self.out)] + self.s.state()


@pytest.mark.parametrize("dim,page,kind,dtype", FORMS)
def test_steps_of_the_host_api(ops, device, dim, page, kind, dtype):
    """The same results from C++, eagerly and replayed; captured without its workspaces a step is refused."""
    s = Server(ops, device, dim, page, kind, dtype)
    start = [t.clone() for t in s.state()]
    steps, want = [], []
    for i, new in enumerate(NEW):
        x, _ = some_inputs(s, 30 + i, new)
        steps.append(x)
        want.append(copies(*s.step(x)) + [t.clone() for t in s.state()])
    static = {k: v.clone() for k, v in steps[0].items()}
    spelled = Spelled(s, static)

    def through(run):
        for t, value in zip(s.state(), start):
            t.copy_(value)
        for i, x in enumerate(steps):
            for k, v in x.items():
                static[k].copy_(v)
            run()
            assert same(spelled.results(), want[i]), i

    def eager():
        assert spelled.run() == 0, spelled.lib.drafts_step_error()
        spelled.after()
    try:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            code = spelled.run()
        assert code == 3 and b"reserve" in spelled.lib.drafts_step_error()
        through(eager)
        spelled.reserve()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            code = spelled.run()
            spelled.after()
        assert code == 0, spelled.lib.drafts_step_error()
        for _ in range(3):
            through(graph.replay)
            through(eager)
        turned = torch.zeros_like(spelled.got[0][0])
        h = Heads.from_buffer_copy(spelled.heads[0])
        k = torch.zeros((TOKENS, HKV, dim), dtype=dtype, device=device)
        h.q_out, h.k_out = rows(turned), rows(k)
        assert spelled.lib.drafts_step_turn(C.byref(h), bytes(s.axes), dim // 2, 3, TOKENS, torch.cuda.current_stream().cuda_stream) == 0
        assert same([turned], [spelled.got[0][0]])
        assert spelled.lib.drafts_step_turn(C.byref(h), bytes(200), 200, 3, TOKENS, None) == 2 and b"128 pairs" in spelled.lib.drafts_step_error()
        assert spelled.lib.drafts_step_turn(C.byref(h), bytes(s.axes), dim // 2, 5, TOKENS, None) == 2
    finally:
        torch.cuda.synchronize()
        spelled.lib.drafts_step_close(spelled.server)


@pytest.mark.parametrize("drafts,codes", [(4, INT8), (1, E4M3)])
def test_the_example_goes_on_with_its_prompts(device, drafts, codes):
    import importlib.util
    spec = importlib.util.spec_from_file_location("verify_drafts", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "verify_drafts.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    written = example.generate(drafts=drafts, codes=codes)
    assert all(9 <= len(w) <= 1 + 8 * (drafts + 1) and all(0 <= x < 500 for x in w) for w in written)
    assert written == example.generate(drafts=drafts, codes=codes)
