"""Arguments of the operators on the Python side: what a conversion would
change without a word is refused, what means the same is taken."""
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")


class Predicted(Exception):
    pass


def model():
    def predict(*args, **kw):
        raise Predicted
    return types.SimpleNamespace(num_outputs=3, predict=predict)


@pytest.mark.parametrize("top_k", [[1.5, 2.0], [2**32 + 1, 5], np.array([2**31]), [float("nan")], [-2**31 - 1],
                                   [float("inf"), 1.0]])
def test_model_sample_refuses_top_k_that_is_no_int32(top_k):
    from ferrisboost_b200 import Model
    with pytest.raises(ValueError, match="top_k"):
        Model.sample(model(), None, None, top_k=top_k)


@pytest.mark.parametrize("top_k", [5, 0, [1, 2], [2.0, 3.0], np.array([2**31 - 1, -2**31]), np.array([3], np.uint8)])
def test_model_sample_takes_whole_top_k(top_k):
    from ferrisboost_b200 import Model
    with pytest.raises(Predicted):  # the check is over
        Model.sample(model(), None, None, top_k=top_k)


@pytest.mark.gpu
def test_numbers_of_numpy_are_numbers():
    from ferrisboost_b200 import ops
    x = torch.randn((5, 9), device="cuda")
    want = ops.dropout(x, 0.5, -7, 11)
    for kind in (np.int64, np.int32, np.int8):
        assert torch.equal(ops.dropout(x, np.float32(0.5), kind(-7), kind(11)), want)
    top = np.uint64(2**64 - 7)  # the same 64 bits
    assert torch.equal(ops.dropout(x, 0.5, top, np.uint8(11)), want)
    with pytest.raises(TypeError):
        ops.dropout(x, 0.5, 1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("top_k", [float("inf"), float("nan"), -1, 2**31, 1.5])
def test_sample_refuses_top_k(top_k):
    from ferrisboost_b200 import ops
    x = torch.zeros((5, 9), device="cuda")
    with pytest.raises(ValueError, match="top_k"):
        ops.sample(x, x[:, 0].contiguous(), top_k=top_k)
