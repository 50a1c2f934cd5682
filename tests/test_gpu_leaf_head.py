"""The operators together: a head on a boosted model's leaves (examples/leaf_head.py)
and Model.sample."""
import importlib.util
import pathlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ROOT = pathlib.Path(__file__).resolve().parents[1]


def example():
    spec = importlib.util.spec_from_file_location("leaf_head", ROOT / "examples" / "leaf_head.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_leaf_tokens_are_predict_s_leaves():
    import ferrisboost_b200 as fb
    ex = example()
    x, y = ex.data(3000, 4, 5)
    model = fb.train({"objective": "multi:softprob", "num_class": 4, "max_depth": 4}, x, label=y, num_boost_round=3)
    tokens = ex.LeafTokens(model)
    got = tokens(torch.from_numpy(x).cuda()).cpu().numpy()
    want = model.predict(x, pred_leaf=True).astype(np.int64)
    sizes = np.array([len(model.tree(t)["left"]) for t in range(model.num_trees)])
    assert np.array_equal(got, want + np.concatenate([[0], np.cumsum(sizes)[:-1]]))
    assert tokens.vocab == sizes.sum()


@pytest.mark.parametrize("p", [0.0, 0.3])
def test_gradients_match_autograd_in_f64(p):
    """The head's gradients against torch's differentiation of the same
    function in f64, the mask taken from dropout of ones.  f32 sums of a few
    hundred terms and two 32-wide products: 1e-4 of each gradient's norm."""
    ex = example()
    head = ex.LeafHead(vocab=300, trees=12, classes=5, dim=32, dropout=p, seed=4)
    gen = torch.Generator(device="cuda").manual_seed(1)
    leaves = torch.randint(0, 300, (500, 12), generator=gen, device="cuda").int()
    leaves[::7, 3] = -1
    labels = torch.randint(0, 5, (500,), generator=gen, device="cuda")
    loss, grads = head.gradients(leaves, labels, 77)
    mask = ex.ops.dropout(torch.ones((500, 32), device="cuda"), p, 77).double()
    params = [v.double().requires_grad_() for v in (head.table, head.weight, head.bias)]
    found = (leaves >= 0)[:, :, None]
    h = (params[0][leaves.clamp(min=0).long()] * found).sum(1) * head.scale * mask
    want = torch.nn.functional.cross_entropy(h @ params[1].T + params[2], labels)
    want.backward()
    assert abs(float(loss) - want.item()) < 1e-5
    for g, v in zip(grads, params):
        assert float((g.double() - v.grad).norm()) <= 1e-4 * float(v.grad.norm())


def test_head_learns_and_answers():
    r = example().main(n=60_000, classes=5, rounds=10, epochs=4, batch=4096)
    assert r["last_loss"] < 0.7 * r["first_loss"]
    assert r["best"] > 0.9 * r["boosted"] and r["best"] > 0.6
    assert r["drawn"] > 0.4 and 0.3 < r["share"] <= 1.0


def test_model_sample_draws_from_the_margins():
    import ferrisboost_b200 as fb
    from ferrisboost_b200 import ops
    x, y = example().data(5000, 4, 6)
    model = fb.train({"objective": "multi:softprob", "num_class": 4, "max_depth": 4}, x, label=y, num_boost_round=4)
    u = np.random.default_rng(1).random(len(x), dtype=np.float32)
    classes, probs = model.sample(x, u, temperature=0.8, top_p=0.9)
    margins = torch.from_numpy(model.predict(x, output_margin=True)).cuda()
    want = ops.sample(margins, torch.from_numpy(u).cuda(), temperature=0.8, top_p=0.9)
    assert np.array_equal(classes, want[0].cpu().numpy()) and np.array_equal(probs, want[1].cpu().numpy())
    assert np.array_equal(model.sample(x, u, temperature=0.0)[0], model.predict(x, output_margin=True).argmax(1))
    # without limits the shares are predict's probabilities, and u spreads the classes as they say
    classes, probs = model.sample(x, u)
    p = model.predict(x)
    assert np.allclose(probs, p[np.arange(len(x)), classes], rtol=1e-5)
    below = np.where(np.arange(4) < classes[:, None], p, 0).sum(1)
    assert np.all(u >= below - 1e-5) and np.all(u <= below + probs + 1e-5)
    with pytest.raises(ValueError, match="u must"):
        model.sample(x, u[:7])
    two = fb.train({"objective": "binary:logistic", "max_depth": 3}, x, label=(y > 1).astype(np.float32),
                   num_boost_round=2)
    with pytest.raises(ValueError, match="multiclass"):
        two.sample(x, u)
