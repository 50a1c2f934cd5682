"""ops.embed at the ends of its 32-bit sizes."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def ops():
    from ferrisboost_b200 import ops as o
    return o


@pytest.mark.parametrize("dim", [(1 << 29) + 5, (1 << 32) - 8])
def test_lookup_of_the_widest_rows(dim):
    """One row of up to almost 2^32 columns (8.6 GB; about 12 s, a warp takes a row): every element as it was,
    nothing after them.  A lane's 32-bit counter would pass 2^32 if it counted over the whole of the wider row;
    the other one ends just after a part of 2^29 columns, off the 16-byte boundaries."""
    table = torch.empty((1, dim), dtype=torch.bfloat16, device="cuda").uniform_(-1, 1)
    flat = torch.full((dim + 64,), 9.0, dtype=torch.bfloat16, device="cuda")
    tok = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops().embed(table, tok, out=flat[:dim].view(1, dim))
    part = 1 << 30
    for c in range(0, dim, part):
        assert torch.equal(flat[c:min(c + part, dim)], table[0, c:c + part]), c
    assert (flat[dim:] == 9.0).all()


def test_the_longest_list_of_tokens():
    """One row of 2^32 - 1 tokens (17 GB), summed in 256 parts of 2^24: the last part ends one token short of that,
    and the token behind the row is not one of its own."""
    buffer = torch.full((1 << 32,), -1, dtype=torch.int32, device="cuda")
    buffer[0] = buffer[(1 << 32) - 2] = 0
    buffer[(1 << 32) - 1] = 1
    table = torch.tensor([[1.0], [100.0]], device="cuda")
    assert ops().embed(table, buffer[:-1].view(1, -1)).item() == 2.0
