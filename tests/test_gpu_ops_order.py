"""The order of the sums of ops.embed and ops.embed_grad depends on the tokens,
the sizes and the element type: the same values in another layout (addresses
off 16-byte boundaries, padded rows) give the same bits."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

LAYOUTS = [(1, 0, 0, 0), (0, 0, 1, 0), (2, 0, 0, 0), (0, 2, 0, 0), (4, 0, 0, 4), (1, 1, 3, 5), (0, 8, 0, 2)]


def ops():
    from ferrisboost_b200 import ops as o
    return o


def laid_out(values, shift, pad):
    """The values in rows `pad` elements apart, `shift` elements behind an aligned address."""
    n, dim = values.shape
    flat = torch.full((shift + n * (dim + pad),), 5.0, dtype=values.dtype, device="cuda")
    out = flat[shift:].view(n, dim + pad)[:, :dim]
    out.copy_(values)
    return out


def random(shape, seed, dtype):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda").to(getattr(torch, dtype))


def tokens(n, k, vocab, seed, hot=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(0, vocab, (n, k), generator=gen, device="cuda")
    t[torch.rand((n, k), generator=gen, device="cuda") < hot] = vocab // 2
    return t


def same_bits(a, b):
    kind = torch.int32 if a.dtype == torch.float32 else torch.int16
    return torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,k,vocab,dim", [(1, 100, 900, 64), (1, 3000, 500, 8), (3, 500, 2000, 32), (40, 133, 700, 16),
                                           (2, 400, 300, 200), (1, 1000, 90, 2), (5, 700, 80, 1028), (300, 64, 90, 4)])
def test_embed(n, k, vocab, dim, dtype):
    table, tok = random((vocab, dim), 1, dtype), tokens(n, k, vocab, 2)
    want = ops().embed(table, tok, scale=0.37)
    for ts, tp, os, op in LAYOUTS:
        out = laid_out(torch.zeros((n, dim), dtype=table.dtype, device="cuda"), os, op)
        assert same_bits(ops().embed(laid_out(table, ts, tp), tok, scale=0.37, out=out), want), (ts, tp, os, op)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,k,vocab,dim,hot", [(3000, 4, 7, 64, 0.0), (40000, 3, 900, 32, 0.3), (5000, 1, 3, 8, 0.5),
                                               (2000, 40, 700, 24, 0.1), (9000, 2, 50, 130, 0.6), (700, 30, 5, 1024, 0.2),
                                               (30000, 4, 2, 4, 0.0), (100000, 5, 40, 2, 0.2)])
def test_embed_grad(n, k, vocab, dim, hot, dtype):
    grad, tok = random((n, dim), 1, dtype), tokens(n, k, vocab, 2, hot)
    want = ops().embed_grad(grad, tok, vocab, scale=0.37)
    for gs, gp, os, op in LAYOUTS:
        out = laid_out(torch.zeros((vocab, dim), dtype=grad.dtype, device="cuda"), os, op)
        assert same_bits(ops().embed_grad(laid_out(grad, gs, gp), tok, vocab, scale=0.37, out=out), want), (gs, gp, os, op)
