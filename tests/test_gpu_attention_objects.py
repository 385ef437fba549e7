"""The objects of the C++ host API for attention: what a TreeAttention does with its workspace while graphs name it, and
a moved cache with its pages."""
import ctypes as C
import os

import pytest
import torch

import attention_reference as ref
from test_attention_refusals import Attention, Cache, Rows

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from fusedkernellibrary_amd import attention
    return attention


@pytest.fixture(scope="module")
def objects():
    import fusedkernellibrary_amd as fkl
    fkl.lib()
    lib = C.CDLL(os.path.join(os.path.dirname(os.path.abspath(__file__)), "cases", "libattention_objects.so"))
    lib.attention_objects_error.restype = C.c_char_p
    lib.attend_open.restype = C.c_void_p
    lib.attend_close.argtypes = [C.c_void_p]
    lib.attend_reserve.argtypes = [C.c_void_p, C.POINTER(Attention), C.POINTER(Cache)]
    lib.attend_run.argtypes = [C.c_void_p, C.POINTER(Attention), C.POINTER(Cache), C.c_void_p]
    return lib


def c_cache(cache):
    return Cache(cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), cache.pages, cache.kv_heads, cache.page_tokens, cache.head_dim, 0)


def rows(t):
    return Rows(t.data_ptr(), t.stride(0), t.stride(1))


class Call:
    """One token behind 3000 cached ones, of which there might be `said`: the more there might be, the larger the workspace."""

    def __init__(self, ops, device, said, tokens=1):
        g = torch.Generator().manual_seed(said)
        page, hkv, dim = 16, 2, 64
        self.cache = ops.KvCache(*ref.Slots(200 * page, hkv, dim, torch.int8, g).tensors(page, device))
        table = torch.randperm(200, generator=g).to(torch.int32)[:188 + tokens // 16]
        self.table = torch.nn.functional.pad(table, (0, max(0, said // page + 1 - len(table))), value=-1)[None].to(device)
        self.q = torch.randn((tokens, 4, dim), generator=g).to(BF16).to(device)
        self.out = torch.zeros_like(self.q)
        self.context, self.start = (torch.tensor(v, dtype=torch.int32, device=device) for v in ([2990], [0, tokens]))
        self.want = ops.tree_attention(self.q, self.cache, self.table, self.context, self.start, max_new=tokens, max_context=said)
        self.c = c_cache(self.cache)
        self.call = Attention(q=rows(self.q), out=rows(self.out), page_table=self.table.data_ptr(), context=self.context.data_ptr(), q_start=self.start.data_ptr(), tokens=tokens,
                              page_table_stride=self.table.shape[1], batch=1, max_new=tokens, max_context=said, q_heads=4, type=0, scale=0.125)

    def needs(self):
        import fusedkernellibrary_amd as fkl
        need = C.c_uint64()
        assert fkl.lib().fklhip_tree_attention_workspace(C.byref(self.call), C.byref(self.c), C.byref(need)) == 0
        return need.value

    def run(self, objects, attend):
        return objects.attend_run(attend, C.byref(self.call), C.byref(self.c), torch.cuda.current_stream().cuda_stream)

    def right(self):
        return torch.equal(self.out, self.want)


def test_graphs_keep_the_workspace_they_were_captured_with(ops, objects, device):
    """A larger eager call between capture and replay: the graph's workspace stays, and memory that is taken afterwards is not it."""
    small, large = Call(ops, device, 6000), Call(ops, device, 60000, tokens=9)
    assert 0 < small.needs() < large.needs()
    attend = objects.attend_open()
    try:
        assert objects.attend_reserve(attend, C.byref(small.call), C.byref(small.c)) == 0, objects.attention_objects_error()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            assert small.run(objects, attend) == 0, objects.attention_objects_error()
        for replay in range(4):
            assert large.run(objects, attend) == 0, objects.attention_objects_error()
            torch.cuda.synchronize()
            assert large.right()
            others = [torch.full((n,), 7, dtype=torch.uint8, device=device) for n in (1 << 16, 1 << 18, 1 << 20, 1 << 22)]
            small.out.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert small.right() and all((t == 7).all() for t in others), replay
            large.out.zero_()
    finally:
        torch.cuda.synchronize()
        objects.attend_close(attend)


def test_a_captured_call_that_needs_more_is_refused_and_the_capture_goes_on(ops, objects, device):
    small, large = Call(ops, device, 6000), Call(ops, device, 60000, tokens=9)
    assert 0 < small.needs() < large.needs()
    attend = objects.attend_open()
    try:
        assert small.run(objects, attend) == 0, objects.attention_objects_error()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            refused = large.run(objects, attend)
            taken = small.run(objects, attend)
        assert refused == 3 and b"reserve" in objects.attention_objects_error() and taken == 0
        small.out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert small.right() and (large.out == 0).all()
        assert objects.attend_reserve(attend, C.byref(large.call), C.byref(large.c)) == 0
        again = torch.cuda.CUDAGraph()
        with torch.cuda.graph(again):
            assert large.run(objects, attend) == 0, objects.attention_objects_error()
        for replay in range(3):
            large.out.zero_()
            torch.cuda.synchronize()
            again.replay()
            graph.replay()
            torch.cuda.synchronize()
            assert large.right() and small.right(), replay
            assert small.run(objects, attend) == 0
            torch.cuda.synchronize()
    finally:
        torch.cuda.synchronize()
        objects.attend_close(attend)


def test_a_cache_that_was_moved_from_has_no_pages_of_another(objects, device):
    """Its description goes along: what is left behind has none, or the pages it got in exchange, and no pointer that somebody else owns."""
    made, moves = (Cache * 2)(), (Cache * 4)()
    assert objects.cache_moves(made, moves) == 0, objects.attention_objects_error()
    fields = lambda c: tuple(getattr(c, name) for name, _ in Cache._fields_)      # noqa: E731
    first, other = map(fields, made)
    assert first[:4] != other[:4] and all(first[:4]) and all(other[:4])
    assert [fields(c) for c in moves] == [fields(Cache()), first, other, first]
