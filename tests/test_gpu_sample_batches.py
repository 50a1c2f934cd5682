"""ops.sample of large batches: the forms for many long rows, and blocks that
draw several rows one after another.  The draws are compared bit for bit with
those of few rows, and these with f64."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_ops import check_draw  # noqa: E402

LIMITS = [dict(), dict(top_p=0.9), dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.02), dict(temperature=0.0),
          dict(top_k=700), dict(temperature=20.0, top_p=0.6), dict(top_k=1500, top_p=0.8)]


def draw(x, u, limits, rows=slice(None)):
    from ferrisboost_b200 import ops
    part = {k: v[rows].contiguous() if isinstance(v, torch.Tensor) else v for k, v in limits.items()}
    return ops.sample(x[rows], u[rows], **part)


def scores_of(n, classes, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = 2 * torch.randn((n, classes), generator=gen, device="cuda")
    x[3] = 1.25                                              # every score equal
    x[4] = torch.round(x[4])                                 # many ties
    x[5] = -math.inf
    x[6] = math.nan
    x[7, ::3] = -math.inf
    x[8, classes // 2] = math.inf
    x[9] = 0.05 * x[9]                                       # flat
    x[10] = torch.finfo(torch.float32).min
    x[11, 1:] = -200.0
    x[n - 1, : classes - 1] = -math.inf
    return x.to(getattr(torch, dtype)), torch.rand(n, generator=gen, device="cuda")


def by_row(n, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    at = torch.randint(0, 4, (n,), generator=gen, device="cuda")
    return dict(temperature=0.5 * at.float(), top_k=torch.tensor([0, 1, 50, 1500], device="cuda", dtype=torch.int32)[at.flip(0)],
                top_p=torch.tensor([0.4, 0.9, 0.95, 1.0], device="cuda")[at.roll(1)], min_p=0.05 * (at.roll(2) == 1).float())


@pytest.mark.parametrize("n", [149, 296, 297])
@pytest.mark.parametrize("classes,dtype", [(8193, "float32"), (8193, "bfloat16"), (20000, "float16"), (32768, "bfloat16"),
                                           (32769, "bfloat16"), (16384, "float32"), (16385, "float32"),
                                           (40000, "float32"), (40001, "bfloat16")])
def test_many_long_rows_draw_as_few(n, classes, dtype):
    x, u = scores_of(n, classes, dtype, n + classes)
    for limits in LIMITS + [by_row(n, classes)]:
        got = draw(x, u, limits)
        for a in range(0, n, 100):  # at most 148 rows are drawn by another form
            want = draw(x, u, limits, slice(a, a + 100))
            for g, w in zip(got, want):
                assert torch.equal(g[a:a + 100], w), (limits, a)
        few = draw(x, u, limits, slice(2, 10))  # and up to 8 rows by a third, where they are long
        for g, w in zip(got, few):
            assert torch.equal(g[2:10], w), limits
        if n == 149:
            check_draw(x[2:10], u[2:10], **{k: v[2:10].contiguous() if isinstance(v, torch.Tensor) else v
                                            for k, v in limits.items()})
        assert got[0][5] == -1 and got[0][6] == -1 and got[1][5] == 0 and got[0][n - 1] == classes - 1


@pytest.mark.parametrize("classes,dtype", [(5, "float32"), (100, "bfloat16"), (257, "float32"), (300, "bfloat16"),
                                           (700, "float16"), (3000, "float32"), (9001, "bfloat16"), (40000, "bfloat16")])
def test_blocks_that_draw_several_rows(classes, dtype):
    """More rows than the largest grid of blocks a row (2^18), as windows of one vector three elements apart."""
    n, part = (1 << 18) + 77, 1 << 17
    gen = torch.Generator(device="cuda").manual_seed(classes)
    flat = (2 * torch.randn(3 * n + classes, generator=gen, device="cuda"))
    flat[1000:1000 + 2 * classes] = 0.5
    flat[300_000:300_000 + 2 * classes] = -math.inf
    x = flat.to(getattr(torch, dtype)).as_strided((n, classes), (3, 1))
    u = torch.rand(n, generator=gen, device="cuda")
    for limits in LIMITS[1:3] + [by_row(n, classes)]:
        got = draw(x, u, limits)
        for a in range(0, n, part):
            for g, w in zip(got, draw(x, u, limits, slice(a, a + part))):
                assert torch.equal(g[a:a + part], w), (limits, a)
        for a in (0, 333, (1 << 18) - 3, n - 4):
            for g, w in zip(got, draw(x, u, limits, slice(a, a + 4))):
                assert torch.equal(g[a:a + 4], w), (limits, a)
