"""What ops.embed, ops.embed_grad, ops.dropout and ops.sample refuse, at the C
entries and in Python: every refusal comes before anything is enqueued, so no
device is needed."""
import ctypes as C

import pytest

from ferrisboost_b200 import _lib

A, B, D, E = (0x10000000 * (i + 1) for i in range(4))  # addresses that are never read: each call is refused first
F32, F16, I32, I64 = 0, 1, 0, 1


def refused(name, *args, match):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    text = lib.fbgpu_last_error(None).decode()
    assert match in text, text


def embed(**kw):
    a = dict(table=A, type=F32, vocab=10, dim=4, ts=4, tokens=B, tt=I32, n=3, k=2, tr=2, tc=1, scale=1.0, out=D, os=4,
             stream=None) | kw
    return list(a.values())


def grad(**kw):
    a = dict(grad=A, type=F32, n=3, k=2, dim=4, gs=4, tokens=B, tt=I32, tr=2, tc=1, vocab=10, scale=1.0, out=D, os=4,
             space=E, size=1 << 20, stream=None) | kw
    return list(a.values())


def drop(**kw):
    a = dict(x=A, type=F32, n=3, dim=4, xs=4, p=0.5, seed=1, offset=0, out=D, os=4, stream=None) | kw
    return list(a.values())


def draw(limits=None, **kw):
    p = _lib.FbgpuSampleParams(**(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) | (limits or {})))
    a = dict(x=A, type=F32, n=3, k=5, stride=5, u=B, params=C.byref(p), classes=D, probs=E, stream=None) | kw
    return list(a.values())


@pytest.mark.parametrize("kw,match", [
    (dict(type=3), "element type"), (dict(tt=2), "token type"), (dict(table=None), "table must be"),
    (dict(tokens=None), "tokens must be"), (dict(out=None), "out must be"), (dict(table=A + 2), "aligned"),
    (dict(tt=I64, tokens=B + 4), "aligned"), (dict(os=3), "overlap"), (dict(out=A), "overlap"),
    (dict(out=B + 4), "overlap"), (dict(ts=1 << 62), "too large"), (dict(tr=1 << 62), "too large"),
])
def test_embed_refusals(kw, match):
    refused("fbgpu_embed", *embed(**kw), match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(type=-1), "element type"), (dict(tt=7), "token type"), (dict(grad=None), "grad must be"),
    (dict(tokens=None), "tokens must be"), (dict(out=None), "out must be"), (dict(os=1), "overlap"),
    (dict(out=A), "overlap"), (dict(space=A), "overlap"), (dict(space=E + 128), "256-byte"),
    (dict(size=16), "workspace"), (dict(space=None), "workspace"), (dict(n=1 << 31), "2147483646"),
    (dict(vocab=1 << 31), "2147483646"), (dict(dim=1 << 22, gs=1 << 22, os=1 << 22), "2097120"),
])
def test_embed_grad_refusals(kw, match):
    refused("fbgpu_embed_grad", *grad(**kw), match=match)


@pytest.mark.parametrize("kw,match", [
    (dict(type=9), "element type"), (dict(p=-0.1), "p must be"), (dict(p=1.1), "p must be"),
    (dict(p=float("nan")), "p must be"), (dict(x=None), "x must be"), (dict(out=None), "out must be"),
    (dict(out=A + 4), "overlap"), (dict(out=A, xs=5), "overlap"), (dict(os=3), "overlap"), (dict(x=A + 1), "aligned"),
    (dict(n=1 << 40, dim=1 << 40, xs=1 << 40, os=1 << 40), "too large"),
])
def test_dropout_refusals(kw, match):
    refused("fbgpu_dropout", *drop(**kw), match=match)


@pytest.mark.parametrize("limits,kw,match", [
    ({}, dict(type=4), "element type"), ({}, dict(k=1), "classes must be"), ({}, dict(k=(1 << 20) + 1), "classes must be"),
    ({}, dict(x=None), "scores must be"), ({}, dict(u=None), "u must be"), ({}, dict(classes=None), "out_classes"),
    ({}, dict(params=None), "params"), ({}, dict(probs=D + 4), "overlap"), ({}, dict(classes=A), "overlap"),
    ({}, dict(probs=B), "overlap"), ({}, dict(u=B + 2), "aligned"), (dict(temperature=-1.0), {}, "temperature"),
    (dict(temperature=float("inf")), {}, "temperature"), (dict(temperature=float("nan")), {}, "temperature"),
    (dict(top_k=-1), {}, "top_k"), (dict(top_p=1.5), {}, "top_p"), (dict(top_p=float("nan")), {}, "top_p"),
    (dict(min_p=-0.5), {}, "min_p"), (dict(temperatures=B + 1), {}, "aligned"), (dict(top_ps=D), {}, "overlap"),
])
def test_sample_refusals(limits, kw, match):
    refused("fbgpu_sample", *draw(limits, **kw), match=match)


def test_nothing_to_do_is_not_refused():
    lib = _lib.load()
    assert lib.fbgpu_embed(*embed(n=0, tokens=None, out=None)) == 0
    assert lib.fbgpu_embed(*embed(dim=0, table=None, out=None)) == 0
    assert lib.fbgpu_embed_grad(*grad(vocab=0, out=None)) == 0
    assert lib.fbgpu_dropout(*drop(n=0, x=None, out=None)) == 0
    assert lib.fbgpu_sample(*draw(n=0, x=None, u=None, classes=None)) == 0
    assert lib.fbgpu_embed_grad_workspace(1 << 40, 1, 5, 5) == 0


def test_python_refuses_what_is_not_on_a_device():
    torch = pytest.importorskip("torch")
    from ferrisboost_b200 import ops
    x, t = torch.zeros((4, 3)), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.embed(x, t), lambda: ops.embed_grad(x, t, 5), lambda: ops.dropout(x, 0.5, 1),
                 lambda: ops.sample(x, x[:, 0])):
        with pytest.raises(ValueError, match="CUDA device"):
            call()
    with pytest.raises(ValueError, match="torch tensor"):
        ops.dropout([1.0], 0.5, 1)


@pytest.mark.gpu
def test_python_refusals_on_a_device():
    import torch
    from ferrisboost_b200 import ops
    x = torch.zeros((4, 6), device="cuda")
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    u = torch.zeros(4, device="cuda")
    bad = [
        (lambda: ops.embed(x[0], t), "dimension"), (lambda: ops.embed(x.double(), t), "must be one of"),
        (lambda: ops.embed(x, t.short()), "must be one of"), (lambda: ops.embed(x.t(), t), "contiguous rows"),
        (lambda: ops.embed(x, t.view(1, 2, 2)), "dimensions"), (lambda: ops.embed(x, t, out=x[:, :3]), "out must be"),
        (lambda: ops.embed(x, t, out=x), "overlap"), (lambda: ops.embed_grad(x, t[:3], 5), "rows"),
        (lambda: ops.embed_grad(x, t, -1), "negative"), (lambda: ops.embed_grad(x, t, 1 << 31), "2147483646"),
        (lambda: ops.dropout(x, 2.0, 1), "p must be"), (lambda: ops.dropout(x.t()[None], 0.1, 1), "contiguous"),
        (lambda: ops.dropout(x, 0.1, 1, out=x.half()), "out must be"),
        (lambda: ops.sample(x, u[:3]), "u must be"), (lambda: ops.sample(x[:, :1], u), "classes must be"),
        (lambda: ops.sample(x, u, temperature=-1.0), "temperature"), (lambda: ops.sample(x, u, top_k=-1), "top_k"),
        (lambda: ops.sample(x, u, top_k=1.5), "top_k"), (lambda: ops.sample(x, u, top_p=2.0), "top_p"),
        (lambda: ops.sample(x, u, min_p=u[:2]), "min_p"), (lambda: ops.sample(x, u, top_k=u), "top_k"),
        (lambda: ops.sample(x, u, classes=t[:2]), "classes must be"), (lambda: ops.sample(x, u.cpu()), "CUDA device"),
        (lambda: ops.sample(x, u, probs=u), "overlap"),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()
