"""Which caches kv_keep takes together, without a GPU: the C ABI's checks (nothing is launched, pointers are not followed)."""
import ctypes as C

import pytest

import fusedkernellibrary_amd as fkl
from test_attention_refusals import AT, I32, I64, P, Cache, a_cache, refused

CODES, SCALES = 8 * 2 * 16 * 64, 8 * 2 * 16 * 4                  # bytes of a_cache's arrays


def keep(at, path=AT, batch=2):
    """Caches whose k, v, k_scale and v_scale are at `at`; a path that is not aligned is refused behind everything else but overlaps."""
    l = fkl.lib()
    l.fklhip_kv_keep.argtypes = [P, I32, P, I64, P, P, P, I32, I32, P]
    these = (Cache * len(at))(*[a_cache(**dict(zip(("k", "v", "k_scale", "v_scale"), x))) for x in at])
    return l.fklhip_kv_keep(these, len(at), AT, 3, AT, path, AT, batch, 3, None)


def apart(n, codes=CODES, scales=SCALES):
    """n caches, one array behind the other of its kind."""
    return [((1 << 32) + i * codes, (2 << 32) + i * codes, (3 << 32) + i * scales, (4 << 32) + i * scales) for i in range(n)]


@pytest.mark.parametrize("layers", [1, 2, 3, 64, 65, 1024])
def test_caches_side_by_side_are_taken(layers):
    """All that is wrong with these is the path, in whatever order they come."""
    at = apart(layers)
    for order in (at, at[::-1], at[1::2] + at[::2]):
        refused(keep(order, path=AT + 2), "aligned")


@pytest.mark.parametrize("layers", [2, 5, 300])
@pytest.mark.parametrize("kind", range(4))
@pytest.mark.parametrize("by", [16, -16, 1 << 11])
def test_caches_that_overlap(layers, kind, by):
    """One's array ends in another's, which need not be its neighbour in the call."""
    at = apart(layers, 2 * CODES, 2 * SCALES)
    size = CODES if kind < 2 else SCALES
    if abs(by) >= size:
        by = size // 2
    at[-1] = tuple(x + (at[0][kind] + by - x) * (i == kind) for i, x in enumerate(at[-1]))
    refused(keep(at), "overlap")
    refused(keep(at[::-1]), "overlap")
    assert keep(at, batch=0) == 0                                # (nothing moves)


@pytest.mark.parametrize("kind", range(4))
def test_the_same_cache_far_apart_in_a_call(kind):
    at = apart(1024)
    at[1023] = tuple(at[3][i] if i == kind else x for i, x in enumerate(at[1023]))
    refused(keep(at), "twice")
