"""ops.embed, ops.embed_grad, ops.dropout and ops.sample against plain
implementations in f64 (or whole numbers), at the sizes, strides, types and
masks where they can go wrong.

Tolerances.  A sum of k f32 terms in any order is within (k + 2) 2^-24 of the
sum of their magnitudes (the terms are exact f32 values, one more rounding for
the scale, one for the scale itself), and then rounded to the result's type:
it lies between the roundings of the two ends of that range.
A draw's weights are f32 exponentials, within CUDA's documented 2 ulp (2^-22
relative) of the exact ones of the same f32 arguments, so a share of their sum
is within 2^-20 of the exact share; u has to lie in the drawn class's part of
the distribution with 2^-20 to spare at either end."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def ops():
    from ferrisboost_b200 import ops as o
    return o


def dt(name):
    return getattr(torch, name)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, seed, dtype="float32"):
    return torch.randn(shape, generator=gen(seed), device="cuda").to(dt(dtype))


def tokens_of(n, k, vocab, seed, token="int32", hot=0.0, missing=0.1):
    g = gen(seed)
    t = torch.randint(0, max(vocab, 1), (n, k), generator=g, device="cuda")
    if hot:
        t[torch.rand((n, k), generator=g, device="cuda") < hot] = vocab // 2
    far = torch.rand((n, k), generator=g, device="cuda") < missing
    t[far] = torch.where(torch.rand((n, k), generator=g, device="cuda") < 0.5, -1, vocab)[far]
    if vocab == 0:
        t.fill_(-1)
    return t.to(dt(token))


def np64(t):
    return t.double().cpu().numpy()


def embed_ref(table, tok, scale):
    table, tok = np64(table), tok.cpu().numpy().astype(np.int64)
    V = len(table)
    ext = np.concatenate([table, np.zeros((1, table.shape[1]))])
    at = np.where((tok >= 0) & (tok < V), tok, V)
    return ext[at].sum(1) * scale, np.abs(ext[at]).sum(1) * abs(scale)


def grad_ref(grad, tok, V, scale):
    grad, tok = np64(grad), tok.cpu().numpy().astype(np.int64)
    n, k = tok.shape
    at = np.where((tok >= 0) & (tok < V), tok, V).ravel()
    rows = np.repeat(np.arange(n), k)
    out, mag = np.zeros((V + 1, grad.shape[1])), np.zeros((V + 1, grad.shape[1]))
    np.add.at(out, at, grad[rows])
    np.add.at(mag, at, np.abs(grad[rows]))
    count = np.bincount(at, minlength=V + 1)[:V]
    return out[:V] * scale, mag[:V] * abs(scale), count


def near(got, ref, mag, terms, dtype):
    got = np64(got)
    tol = (terms + 2) * 2.0 ** -24 * mag
    low, high = (np64(torch.from_numpy(v).to(torch.float32).to(dt(dtype))) for v in (ref - tol, ref + tol))
    bad = ~((low <= got) & (got <= high))
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], ref[bad][:5])


# ------------------------------------------------------------------ embed
EMBED = [  # n, k, vocab, dim
    (1, 1, 1, 1), (1, 100, 12700, 64), (3, 1, 5, 7), (5, 3, 17, 33), (1000, 20, 1280, 16), (257, 1, 300, 1024),
    (64, 500, 2000, 32), (2, 1000, 50, 8), (33, 7, 100, 201), (4097, 1, 900, 12), (7, 2, 9, 2050), (300, 37, 4000, 128),
    (150, 1, 40, 65), (1, 3000, 700, 24), (20000, 9, 500, 4),
]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,k,vocab,dim", EMBED)
def test_embed_matches_f64(n, k, vocab, dim, dtype):
    table = randn((vocab, dim), n + dim, dtype)
    tok = tokens_of(n, k, vocab, n + k, "int64" if (n + k) % 2 else "int32")
    got = ops().embed(table, tok if k > 1 else tok[:, 0], scale=0.37)
    assert got.shape == (n, dim) and got.dtype == table.dtype
    near(got, *embed_ref(table, tok, np.float32(0.37)), k, dtype)


def test_embed_missing_rows_and_empty_sizes():
    table = randn((10, 6), 1)
    tok = torch.full((4, 3), -1, dtype=torch.int64, device="cuda")
    tok[1] = torch.tensor([1 << 40, -(1 << 40), 10], device="cuda")
    assert not ops().embed(table, tok).any()
    assert ops().embed(table, tok[:0]).shape == (0, 6)
    assert not ops().embed(table, tok[:, :0]).any()
    assert ops().embed(table[:, :0], tok).shape == (4, 0)
    assert not ops().embed(table[:0], torch.zeros((2, 3), dtype=torch.int32, device="cuda")).any()
    # a missing token's row is not read: NaN and infinity elsewhere stay where they are
    table[3] = math.nan
    tok[2, 0] = 3
    got = ops().embed(table, tok)
    assert got[2].isnan().all() and not got[[0, 1, 3]].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shift,pad", [(0, 0), (0, 8), (1, 0), (1, 7), (2, 3), (4, 4)])
def test_embed_strides_and_alignment(dtype, shift, pad):
    dim, vocab, n, k = 24, 90, 130, 5
    wide = randn((vocab * (dim + pad) + shift,), 3, dtype)
    table = wide[shift:].view(vocab, dim + pad)[:, :dim]
    tok = tokens_of(n, k, vocab, 4)
    turned = tok.t().contiguous().t()  # strides (1, n)
    base = torch.full((n, dim + pad + 3), 9.0, dtype=dt(dtype), device="cuda")
    out = base[:, :dim]
    got = ops().embed(table, turned, scale=2.0, out=out)
    assert got is out and (base[:, dim:] == 9.0).all()
    near(got, *embed_ref(table, tok, 2.0), k, dtype)
    one = ops().embed(table, tok[:1].expand(n, k), scale=2.0)  # token rows of stride 0
    assert torch.equal(one, one[:1].expand(n, dim))
    # the sum depends on the row's tokens and the call's sizes only
    assert torch.equal(ops().embed(table, tok, scale=2.0), ops().embed(table.contiguous(), turned, scale=2.0))


# ------------------------------------------------------------- embed_grad
GRAD = [  # n, k, vocab, dim, hot
    (1, 1, 1, 1, 0.0), (512, 20, 1280, 16, 0.0), (3, 1, 70000, 7, 0.0), (1000, 1, 300, 33, 0.9), (64, 500, 2000, 32, 0.0),
    (4097, 3, 17, 65, 0.5), (5, 2, 9, 2050, 0.0), (9000, 1, 65534, 200, 0.1), (2000, 40, 700, 24, 0.3),
    (30000, 1, 2, 4, 0.0), (20000, 8, 1, 8, 0.0), (100, 1, 1000, 1024, 0.6), (33000, 4, 513, 12, 0.0),
    (70001, 3, 5000, 16, 0.05),
]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,k,vocab,dim,hot", GRAD)
def test_embed_grad_matches_f64(n, k, vocab, dim, hot, dtype):
    grad = randn((n, dim), n + dim, dtype)
    tok = tokens_of(n, k, vocab, n + k, "int64" if (n + k) % 2 else "int32", hot=hot)
    got = ops().embed_grad(grad, tok if k > 1 else tok[:, 0], vocab, scale=0.37)
    assert got.shape == (vocab, dim) and got.dtype == grad.dtype
    ref, mag, count = grad_ref(grad, tok, vocab, np.float32(0.37))
    near(got, ref, mag, count[:, None], dtype)
    # sorted, not atomic: the same bits again, whatever the buffers held
    again = ops().embed_grad(grad, tok if k > 1 else tok[:, 0], vocab, scale=0.37)
    assert torch.equal(again.view(torch.uint8), ops().embed_grad(grad, tok, vocab, scale=0.37).view(torch.uint8))


def test_embed_grad_empty_and_all_missing():
    for n, k in ((0, 3), (4, 0), (4, 3)):
        tok = torch.full((n, k), -1, dtype=torch.int32, device="cuda")
        out = torch.full((50, 6), 5.0, device="cuda")
        assert not ops().embed_grad(torch.ones((n, 6), device="cuda"), tok, 50, out=out).any()
    assert ops().embed_grad(torch.ones((4, 6), device="cuda"), tok, 0).shape == (0, 6)
    assert ops().embed_grad(torch.ones((4, 0), device="cuda"), tok, 5).shape == (5, 0)


@pytest.mark.parametrize("n,k", [(200, 5), (60000, 2)])
def test_embed_grad_strides_and_broadcast(n, k):
    vocab, dim = 90, 24
    tok = tokens_of(n, k, vocab, 4, "int64")
    wide = randn((n, dim + 5), 5)
    for grad in (wide[:, :dim], wide[:1, :dim].expand(n, dim), wide[:, 1:dim + 1]):
        base = torch.full((vocab, dim + 4), 9.0, device="cuda")
        got = ops().embed_grad(grad, tok.t().contiguous().t(), vocab, scale=-1.5, out=base[:, :dim])
        assert (base[:, dim:] == 9.0).all()
        ref, mag, count = grad_ref(grad, tok, vocab, -1.5)
        near(got, ref, mag, count[:, None], "float32")


@pytest.mark.parametrize("n,k,vocab,dim", [(40, 6, 30, 5), (3000, 4, 50, 8)])
def test_embed_grad_is_the_difference_of_embed(n, k, vocab, dim):
    """embed is linear in the table, and on small whole numbers every sum is
    exact: the difference quotient of sum(embed * g) is the gradient, bit for bit."""
    g = torch.randint(-3, 4, (n, dim), generator=gen(1), device="cuda").float()
    table = torch.randint(-3, 4, (vocab, dim), generator=gen(2), device="cuda").float()
    tok = tokens_of(n, k, vocab, 3)
    got = ops().embed_grad(g, tok, vocab, scale=2.0)
    for v, c in ((0, 0), (vocab // 2, dim - 1), (vocab - 1, 1)):
        step = torch.zeros_like(table)
        step[v, c] = 1.0
        f = [(ops().embed(table + s * step, tok, scale=2.0).double() * g.double()).sum() for s in (1, -1)]
        assert float(got[v, c]) == float((f[0] - f[1]) / 2)


# --------------------------------------------------------------- dropout
def mask_ref(count, p, seed, offset):
    """Kept elements offset .. offset + count, from Python integers."""
    M = (1 << 64) - 1

    def mix(z):
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & M
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & M
        return z ^ (z >> 31)

    key, limit = mix(seed & M), math.ceil(p * 2 ** 32)
    out = np.zeros(count, bool)
    for i in range(count):
        e = (offset + i) & M
        w = mix((key + ((e >> 1) + 1) * 0x9E3779B97F4A7C15) & M)
        out[i] = (w >> (32 * (e & 1)) & 0xFFFFFFFF) >= limit
    return out


def drop_ref(x, p, seed, offset):
    keep = mask_ref(x.numel(), p, seed, offset).reshape(x.shape)
    v = x.float().cpu().numpy() * np.float32(1.0 / (1.0 - p) if p < 1 else 0.0)
    return torch.from_numpy(np.where(keep, v, np.float32(0))).to(x.dtype), keep


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,dim,pad", [(1, 1, 0), (128, 64, 0), (37, 19, 1), (5, 1001, 0), (3, 2048, 8), (70, 33, 0),
                                       (2, 4096, 5), (1, 65537, 0), (300, 3, 2), (16, 24, 8)])
@pytest.mark.parametrize("offset", [0, 1, 1000003, (1 << 64) - 3])
def test_dropout_bit_for_bit(n, dim, pad, dtype, offset):
    x = randn((n, dim + pad), n * dim, dtype)[:, :dim]
    seed = 12345 + dim
    ref, _ = drop_ref(x, 0.3, seed, offset)
    got = ops().dropout(x, 0.3, seed, offset)
    assert torch.equal(got.cpu(), ref)


def test_dropout_mask_does_not_depend_on_layout_and_masks_what_is_there():
    x = randn((50, 40), 1)
    x[3, :] = math.nan
    x[4, :] = math.inf
    wide = torch.zeros((50, 47), device="cuda")
    wide[:, 3:43] = x
    a = ops().dropout(x, 0.5, 7)
    b = torch.full((50, 44), 8.0, device="cuda")
    ops().dropout(wide[:, 3:43], 0.5, 7, out=b[:, 1:41])
    assert torch.equal(a.nan_to_num(), b[:, 1:41].nan_to_num()) and (b[:, 41:] == 8.0).all() and (b[:, 0] == 8.0).all()
    keep = torch.from_numpy(mask_ref(2000, 0.5, 7, 0).reshape(50, 40)).cuda()
    assert (a[~keep] == 0).all() and a[3][keep[3]].isnan().all() and (a[4][keep[4]] == math.inf).all()
    y = x.clone()
    assert ops().dropout(y, 0.5, 7, out=y) is y
    assert torch.equal(y.nan_to_num(), a.nan_to_num())
    # the backward pass is the same call: d sum(dropout(x) g) / dx = dropout(g)
    g = randn((50, 40), 2)
    assert torch.equal(ops().dropout(g, 0.5, 7), torch.where(keep, g * 2, 0.0))
    assert torch.equal(ops().dropout(x.view(-1)[5:], 0.5, 7, offset=5).nan_to_num(), a.view(-1)[5:].nan_to_num())


def test_dropout_edges_of_p_and_sizes():
    x = randn((33, 65), 1, "bfloat16")
    assert torch.equal(ops().dropout(x, 0.0, 3), x)
    assert not ops().dropout(x, 1.0, 3).any()
    assert ops().dropout(x[:0], 0.5, 3).shape == (0, 65)
    assert ops().dropout(x[:, :0], 0.5, 3).shape == (33, 0)
    assert ops().dropout(x.view(3, 11, 65), 0.5, -1).shape == (3, 11, 65)
    # the share kept of N elements: 0.9 N within 5 standard deviations
    big = ops().dropout(torch.ones(1 << 22, device="cuda"), 0.1, 99)
    kept = int((big != 0).sum())
    assert abs(kept - 0.9 * (1 << 22)) < 5 * math.sqrt((1 << 22) * 0.09)


# ---------------------------------------------------------------- sample
def sample_ref(x, T, top_k, top_p, min_p):
    """The kept shares of one row by class (None: nothing to draw), from f64
    exponentials of the kernel's f32 arguments."""
    x = x.astype(np.float32)
    x = np.where(np.isnan(x), np.float32(-np.inf), x)
    top = x.max()
    if top == -np.inf:
        return None
    if not T > 0:
        return (np.arange(len(x)) == np.argmax(x)).astype(np.float64)
    with np.errstate(all="ignore"):
        z = (x - top) * (np.float32(1) / np.float32(T))
        e = np.exp(z.astype(np.float64))
    e = np.where(x == top, 1.0, np.where((x == -np.inf) | (top == np.inf), 0.0, e))
    w = np.floor(e * 2.0 ** 40) * 2.0 ** -40
    order = np.lexsort((np.arange(len(x)), -x.astype(np.float64)))
    ws = w[order]
    if 0 < top_k < len(x):
        ws[top_k:] = 0
    if top_p < 1:
        before = np.cumsum(ws) - ws
        ws[(before >= np.float64(np.float32(top_p)) * ws.sum()) & (np.arange(len(x)) > 0)] = 0
    ws[e[order] < np.float32(min_p)] = 0
    w = np.zeros_like(w)
    w[order] = ws
    return w / w.sum()


def check_draw(scores, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    classes, probs = ops().sample(scores, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    x, un = scores.float().cpu().numpy(), u.double().cpu().numpy()
    c, p = classes.cpu().numpy(), probs.double().cpu().numpy()

    def of(v, r):
        return v[r].item() if isinstance(v, torch.Tensor) else v

    tol = 2.0 ** -20
    for r in range(len(x)):
        share = sample_ref(x[r], *(of(v, r) for v in (temperature, top_k, top_p, min_p)))
        if share is None:
            assert c[r] == -1 and p[r] == 0
            continue
        assert share[c[r]] > 0, (r, c[r])
        below = share[:c[r]].sum()
        assert below - tol <= un[r] <= below + share[c[r]] + tol, (r, c[r], below, share[c[r]], un[r])
        assert abs(p[r] - share[c[r]]) <= tol * share[c[r]], (r, p[r], share[c[r]])
    return classes, probs


SIZES = [2, 3, 7, 8, 9, 16, 17, 31, 32, 33, 64, 100, 255, 257, 1000, 1024, 1025, 4097, 20000, 131071]
LIMITS = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 50, 0.95, 0.02),
          (1.0, 1, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (2.0, 3, 0.5, 0.3), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0),
          (100.0, 40, 0.999, 0.0), (0.01, 0, 0.9, 0.0)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("K", SIZES)
def test_sample_matches_f64(K, dtype):
    n = 40 if K <= 1025 else 6
    scores = 2 * randn((n, K), K, dtype)
    u = torch.rand(n, generator=gen(K + 1), device="cuda")
    for limits in LIMITS:
        check_draw(scores, u, *limits)


@pytest.mark.parametrize("K", [2, 7, 16, 40, 1000, 5000, 60001])
def test_sample_masks_ties_and_extremes(K):
    lowest = torch.finfo(torch.float32).min
    x = randn((14, K), K)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, :-1] = -math.inf
    x[3] = 1.25                       # every score equal
    x[4] = lowest                     # a mask of the type's lowest value, everywhere
    x[5, : K // 2] = lowest
    x[6, K // 2] = math.inf           # one class that is certain
    x[7] = math.inf
    x[8] = torch.where(torch.arange(K, device="cuda") % 2 == 0, 0.0, -0.0)
    x[9, K // 3] = math.nan
    x[10] = torch.round(x[10])        # many ties
    x[11, 1:] = -200.0                # weights below 2^-40: never drawn
    x[12, :] = -math.inf
    x[12, 0] = lowest
    x[13] = 3e38 * torch.sign(x[13])
    u = torch.rand(14, generator=gen(K), device="cuda")
    for limits in LIMITS + [(1.0, K, 1.0, 0.0), (1.0, K - 1, 0.97, 0.0), (1.0, max(K // 2, 1), 0.4, 0.0)]:
        c, p = check_draw(x, u, *limits)
        assert c[0] == -1 and c[1] == -1 and p[0] == 0 and p[1] == 0
        assert c[2] == K - 1 and p[2] == 1 and c[6] == K // 2 and c[12] == 0
        assert c[11] == 0 or limits[0] > 2
    # ties go by class: of equal scores, top_k keeps the lowest classes
    c, p = ops().sample(x[[3] * 14], u, top_k=2)
    assert torch.equal(c, (u >= 0.5).int()) and (p == 0.5).all()


@pytest.mark.parametrize("K", [5, 30, 300, 9000])
def test_sample_ends_of_u(K):
    x = randn((6, K), K)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan], device="cuda")
    c, p = ops().sample(x, u)
    assert (c >= 0).all() and (c < K).all() and (p > 0).all()
    assert c[0] == 0 and c[4] == 0 and c[5] == 0  # the first class has a weight here
    assert (c[1:4] == K - 1).all()


@pytest.mark.parametrize("K", [6, 60, 700, 30011])
def test_sample_limits_by_row_equal_single_calls(K):
    """Each row with its own limits; one row alone, a strided batch and the
    batch give the same draw, bit for bit."""
    n = 37
    wide = randn((n, K + 3), K)
    x = wide[:, 1:K + 1]
    g = gen(3)
    u = torch.rand(n, generator=g, device="cuda")
    t = torch.randint(0, 4, (n,), generator=g, device="cuda").float() * 0.5
    k = torch.randint(0, 9, (n,), generator=g, device="cuda").int()
    tp = 0.4 + 0.2 * torch.randint(0, 4, (n,), generator=g, device="cuda").float()
    mp = 0.1 * torch.randint(0, 2, (n,), generator=g, device="cuda").float()
    c, p = check_draw(x, u, t, k, tp, mp)
    c2, p2 = ops().sample(x.contiguous(), u, temperature=t, top_k=k, top_p=tp, min_p=mp)
    assert torch.equal(c, c2) and torch.equal(p, p2)
    for r in (0, 17, n - 1):
        c1, p1 = ops().sample(x[r:r + 1], u[r:r + 1], temperature=float(t[r]), top_k=int(k[r]),
                              top_p=min(float(tp[r]), 1.0), min_p=float(mp[r]))
        assert c1[0] == c[r] and p1[0] == p[r]


def test_sample_limits_outside_their_range_in_arrays():
    n, K = 8, 50
    x = randn((n, K), 1)
    u = torch.rand(n, generator=gen(2), device="cuda")
    f = dict(dtype=torch.float32, device="cuda")
    for name, odd, like in (("temperature", [-1.0, math.nan], 0.0), ("top_p", [-2.0], 0.0), ("top_p", [1.5, math.nan], 1.0),
                            ("min_p", [7.0], 1.0), ("min_p", [-1.0, math.nan], 0.0)):
        for v in odd:
            a = ops().sample(x, u, **{name: torch.full((n,), v, **f)})
            b = ops().sample(x, u, **{name: like})
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), (name, v)
    a = ops().sample(x, u, top_k=torch.full((n,), -5, dtype=torch.int32, device="cuda"))
    b = ops().sample(x, u, temperature=torch.full((n,), 1.0, **f))
    assert torch.equal(a[0], b[0])
    c = ops().sample(x, u, temperature=torch.full((n,), math.inf, **f))
    assert torch.equal(c[0], (u.double() * K).floor().int())


def test_sample_many_rows_and_empty():
    for K in (3, 7, 20):
        x = randn((70001, K), K)
        u = torch.rand(70001, generator=gen(9), device="cuda")
        c, p = ops().sample(x, u, top_p=0.8)
        for r in (0, 31, 32, 70000):
            c1, p1 = ops().sample(x[r:r + 1], u[r:r + 1], top_p=0.8)
            assert c1[0] == c[r] and p1[0] == p[r]
    c, p = ops().sample(x[:0], u[:0])
    assert c.shape == (0,) and p.shape == (0,)


# ------------------------------------------------- streams and graphs
def test_ops_run_on_the_current_stream_and_in_a_graph():
    table, tok = randn((500, 16), 1), tokens_of(300, 8, 500, 2)
    scores, u = randn((300, 50), 3), torch.rand(300, generator=gen(4), device="cuda")

    def step():
        e = ops().embed(table, tok)
        d = ops().dropout(e, 0.25, 11)
        return e, d, ops().embed_grad(d, tok, 500), *ops().sample(scores, u, top_p=0.9)

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    table.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0] * 2) and torch.equal(out[3], want[3])


def test_large_forms_in_a_graph_follow_new_inputs():
    """The sort in several launches, a cluster per row and a block per row,
    captured once and replayed on other tokens and scores."""
    n, k, vocab = 30000, 4, 3000
    tok, grad = tokens_of(n, k, vocab, 1), randn((n, 20), 2)
    scores = [randn((2, 70000), 3), randn((80, 5000), 4), randn((70, 20001), 5, "bfloat16")]
    u = [torch.rand(len(x), generator=gen(6), device="cuda") for x in scores]

    def step():
        return [ops().embed_grad(grad, tok, vocab)] + [
            ops().sample(x, r, top_k=k_, top_p=0.9)[0] for x, r in zip(scores, u) for k_ in (0, 30)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (7, 8):
        tok.copy_(tokens_of(n, k, vocab, seed))
        for i, x in enumerate(scores):
            x.copy_(randn(x.shape, seed + i, str(x.dtype)[6:]))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_two_streams_at_once():
    """Calls on two streams do not share anything."""
    tok = [tokens_of(40000, 3, 900, s) for s in (1, 2)]
    grad = [randn((40000, 24), s) for s in (3, 4)]
    x = [randn((4, 40000), s) for s in (5, 6)]
    u = torch.rand(4, generator=gen(7), device="cuda")
    want = [(ops().embed_grad(g, t, 900), ops().sample(s, u, top_p=0.7)[0]) for g, t, s in zip(grad, tok, x)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append((ops().embed_grad(grad[i], tok[i], 900), ops().sample(x[i], u, top_p=0.7)[0]))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])


def test_launches_are_counted():
    from ferrisboost_b200 import _lib
    before = _lib.load().fbgpu_launch_count()
    ops().embed(randn((5, 4), 1), tokens_of(3, 2, 5, 1))
    assert _lib.load().fbgpu_launch_count() == before + 1


@pytest.mark.parametrize("K", [1024, 1025, 8192, 8193, 32768, 32769, 262144, 262145, 300001, 1 << 20])
def test_sample_at_the_edges_of_the_variants(K):
    """Sizes at which another kernel takes over, with many and few rows and a
    row that starts off a 16-byte boundary."""
    base = randn((2 * K + 3,), K, "bfloat16")
    x = base[3:3 + 2 * K].view(2, K)
    u = torch.rand(2, generator=gen(K), device="cuda")
    for limits in ((1.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.0, 0, 0.5, 0.01), (1.0, K // 2, 0.95, 0.0), (1.0, 1000, 1.0, 0.0)):
        c, p = check_draw(x, u, *limits)
        if K <= 32769:
            c64, p64 = ops().sample(x[[0, 1] * 40], u.repeat(40), temperature=limits[0], top_k=limits[1],
                                    top_p=limits[2], min_p=limits[3])
            assert torch.equal(c64, c.repeat(40)) and torch.equal(p64, p.repeat(40))


@pytest.mark.parametrize("K", [257, 300, 512, 513, 1000, 2048])
def test_sample_batches_equal_few_rows(K):
    """Large batches of short rows take smaller blocks: the same draws."""
    x = 2 * randn((40, K), K, "float16")
    x[3] = 1.0
    x[4] = torch.round(x[4])
    x[5] = -math.inf
    u = torch.rand(40, generator=gen(K), device="cuda")
    for limits in LIMITS + [(0.9, 200, 0.95, 0.0), (50.0, 0, 0.6, 0.0)]:
        c, p = check_draw(x, u, *limits)
        for times in (30, 60):
            cm, pm = ops().sample(x.repeat(times, 1), u.repeat(times), temperature=limits[0], top_k=limits[1],
                                  top_p=limits[2], min_p=limits[3])
            assert torch.equal(cm, c.repeat(times)) and torch.equal(pm, p.repeat(times))


@pytest.mark.parametrize("K", [700, 3000, 40000])
def test_sample_temperatures_at_the_ends_of_f32(K):
    x = randn((4, K), K)
    u = torch.rand(4, generator=gen(1), device="cuda")
    for t in (1e-45, 1e-38, 1e-20, 1e20, 3e38):
        c, p = ops().sample(x, u, temperature=t, top_k=500, top_p=0.9)
        if t < 1:
            assert torch.equal(c, x.argmax(1).int()) and (p == 1).all()
        else:  # every class weighs the same: 450 of the 500 largest are left, drawn by class
            kept = x.argsort(dim=1, descending=True, stable=True)[:, :450].sort(1).values
            want = kept.gather(1, (u.double() * 450).long()[:, None])[:, 0]
            assert torch.equal(c.long(), want) and torch.allclose(p, torch.full_like(p, 1 / 450), rtol=2.0 ** -23)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim", [16, 31, 32, 33, 63, 65, 201, 1023, 2051])
def test_lookup_of_rows_off_16_byte_boundaries(dim, dtype):
    """One token a row: the same bits as indexing, at every distance of table
    and output from a 16-byte boundary, and nothing outside the rows is written."""
    n, vocab = 67, 29
    for tshift, tpad, oshift, opad in ((0, 0, 0, 0), (1, 0, 0, 0), (0, 1, 3, 0), (5, 7, 2, 1), (0, 0, 1, 2), (3, 5, 3, 5)):
        table = randn((tshift + vocab * (dim + tpad),), dim, dtype)[tshift:].view(vocab, dim + tpad)[:, :dim]
        tok = tokens_of(n, 1, vocab, dim)[:, 0]
        flat = torch.full((oshift + n * (dim + opad) + 9,), 9.0, dtype=dt(dtype), device="cuda")
        out = flat[oshift:oshift + n * (dim + opad)].view(n, dim + opad)[:, :dim]
        ops().embed(table, tok, scale=2.0, out=out)
        found = (tok >= 0) & (tok < vocab)
        want = torch.where(found[:, None], table[tok.clamp(0, vocab - 1).long()].float() * 2, 0.0).to(dt(dtype))
        assert torch.equal(out, want)
        spare = flat.clone()
        spare[oshift:oshift + n * (dim + opad)].view(n, dim + opad)[:, :dim] = 9.0
        assert (spare == 9.0).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n,dim", [(20011, 201), (60001, 37), (150001, 64), (200003, 5)])
def test_lookup_of_many_rows(n, dim, dtype):
    """More rows than groups: each group takes several, bits as by indexing."""
    table = randn((4000, dim), 1, dtype)
    tok = tokens_of(n, 1, 4000, 2, "int64")[:, 0]
    found = (tok >= 0) & (tok < 4000)
    want = torch.where(found[:, None], table[tok.clamp(0, 3999)].float() * 0.5, 0.0).to(dt(dtype))
    assert torch.equal(ops().embed(table, tok, scale=0.5), want)
