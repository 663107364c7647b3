"""One class far above all others: the loss is what the others leave, however little."""
import numpy as np
import pytest
import torch

from oracle import vocab_oracle as VO

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from niti_b200 import ops  # noqa: E402
from tests.test_gpu_vocab import check_train, cu, same_loss, word  # noqa: E402
from tests.test_vocab_tail import GAPS, UNITS, peaked, sum_error  # noqa: E402

DEV = "cuda:0"


@pytest.mark.parametrize("e", UNITS)
@pytest.mark.parametrize("T,V", [(1, 65), (1, 131072), (4, 5000), (5, 131072), (len(GAPS), 131072), (70, 4999), (300, 5000)])
def test_the_rest_of_a_row(T, V, e):
    x, ex, w, ew, y, far = peaked(T, V, e)
    want = np.log1p((V - 1) * np.exp(-far))
    got = ops.vocab_loss(cu(x), word(ex), cu(w), word(ew), cu(y)).cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - want) <= want * 2.0 ** -24 + sum_error(want))
    check_train(ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y)), VO.vocab(x, ex, w, ew, y))


@pytest.mark.parametrize("T", [3, 40])
def test_the_rest_of_a_row_with_a_teacher(T):
    V = 20000
    x, ex, w, ew, y, far = peaked(T, V)
    idx, top = y[:, None], np.zeros((T, 1), np.int8)
    for temperature in (0, 1):
        rest = np.log1p((V - 1) * np.exp(-far / 2.0 ** temperature))
        got = ops.vocab_distill_loss(cu(x), word(ex), cu(w), word(ew), cu(idx), cu(top), word(-4), temperature)
        want = VO.vocab(x, ex, w, ew, idx, top=top, exp_top=-4, temperature_log2=temperature, train=False)["loss"]
        same_loss(got, want)
        assert np.all(np.abs(want - 4.0 ** temperature * rest) <= 4.0 ** temperature * sum_error(rest))
        check_train(ops.vocab_distill_train(cu(x), word(ex), cu(w), word(ew), cu(idx), cu(top), word(-4), temperature),
                    VO.vocab(x, ex, w, ew, idx, top=top, exp_top=-4, temperature_log2=temperature))
