"""ops next to autograd: no gradient is lost without a word, and a write to a
tensor that autograd has saved is seen."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def ops():
    from ferrisboost_b200 import ops as o
    return o


def tensors():
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((6, 8), generator=gen, device="cuda")
    return x, torch.arange(6, dtype=torch.int32, device="cuda"), torch.rand(6, generator=gen, device="cuda")


def calls(x, tok, u):
    o = ops()
    return [lambda: o.embed(x, tok), lambda: o.embed_grad(x, tok, 6), lambda: o.dropout(x, 0.5, 1),
            lambda: o.dropout(x.detach(), 0.5, 1, out=x), lambda: o.embed(x.detach().clone(), tok, out=x),
            lambda: o.embed_grad(x.detach().clone(), tok, 6, out=x), lambda: o.sample(x, u)[1],
            lambda: o.sample(x.detach(), u, temperature=x[:, 0].contiguous())[1],
            lambda: o.sample(x.detach(), u, probs=x.view(-1)[:6])[1]]


def test_a_tensor_that_asks_for_a_gradient_is_refused():
    x, tok, u = tensors()
    for call in calls(x.clone().requires_grad_(), tok, u):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()


def test_and_taken_where_none_is_recorded():
    x, tok, u = tensors()
    want = [call() for call in calls(x.clone(), tok, u)[:3] + calls(x, tok, u)[6:7]]
    for mode in (torch.no_grad, torch.inference_mode):
        y = x.clone().requires_grad_()
        with mode():
            got = [call() for call in calls(y, tok, u)[:3] + calls(y, tok, u)[6:7]]
        assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))
        assert torch.equal(x, y)
    with torch.inference_mode():  # a tensor without a count of its changes
        z = torch.empty_like(x)
        assert torch.equal(ops().dropout(x, 0.5, 1, out=z), want[2])


def test_a_write_to_a_saved_tensor_is_seen():
    x, tok, u = tensors()
    f = dict(device="cuda")
    writes = [
        lambda h: ops().embed(x, tok, out=h), lambda h: ops().embed_grad(x, tok, 6, out=h),
        lambda h: ops().dropout(h, 0.5, 1, out=h), lambda h: ops().sample(x, u, probs=h.view(-1)[:6]),
    ]
    for write in writes:
        h = x.clone()
        w = torch.ones_like(h).requires_grad_()
        loss = (w * h).sum()  # saves h
        write(h)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    classes = torch.empty(6, dtype=torch.int32, **f)
    version = classes._version
    ops().sample(x, u, classes=classes)
    assert classes._version > version
    # without out nothing that was there is touched
    version = x._version
    ops().dropout(x, 0.5, 1), ops().embed(x, tok), ops().sample(x, u)
    assert x._version == version
