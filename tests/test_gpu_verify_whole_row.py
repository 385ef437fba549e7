"""verify_drafts where the refused tokens had all that their row has: the next token is drawn from that row whole, theirs among it."""
import pytest
import torch

from test_gpu_verify_drafts import TYPES, check

pytestmark = pytest.mark.gpu


def rows_of(at, vocab, dtype):
    """A row of each {token: probability}."""
    t = torch.zeros((len(at), vocab), dtype=torch.float64)
    for row, some in zip(t, at):
        for token, p in some.items():
            row[token] = p
    return t.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,first,second", [(5, 0, 1), (9000, 3, 8999), (131072, 4096, 70001)])
@pytest.mark.parametrize("u,nth", [(0.25, 0), (0.75, 1)])
def test_children_for_all_that_a_row_has(device, dtype, vocab, first, second, u, nth):
    """0.25 is not above 0.9 of 1, nor above 0.9 of the 0.75 that are left: both are refused, and each is half of the row."""
    d = dict(target=rows_of([{first: 0.25, second: 0.25}, {0: 1.0}, {0: 1.0}], vocab, dtype), ids=torch.tensor([0, second, first], dtype=torch.int32), draft=None, max_new=3,
             q_start=torch.tensor([0, 3], dtype=torch.int32), uniforms=torch.tensor([u, 0.9, 0.9]), parents=torch.tensor([-1, 0, 0], dtype=torch.int32))
    got = check(d)
    assert got.count.tolist() == [1] and got.out.tolist() == [[(first, second)[nth], -1, -1]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,token", [(5, 4), (9000, 4095)])
def test_a_chain_whose_token_is_all_that_its_row_has(device, dtype, vocab, token):
    """In the first row, and behind an accepted one; next to a sequence that has something left."""
    half, one = {token: 0.5}, {1: 1.0}
    d = dict(target=rows_of([half, one, one, half, one, {token: 0.5, 2: 0.25}, one], vocab, dtype), ids=torch.tensor([0, token, 0, 1, token, 0, token], dtype=torch.int32), draft=None, max_new=3,
             q_start=torch.tensor([0, 2, 5, 7], dtype=torch.int32), uniforms=torch.tensor([0.5, 0.9, 0.25, 0.5, 0.75, 0.5, 0.9]), parents=None)
    got = check(d)
    assert got.count.tolist() == [1, 2, 1] and got.out[:, :2].tolist() == [[token, -1], [1, token], [2, -1]]
