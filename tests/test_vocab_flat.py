"""What the vocabulary losses' roundings leave of a row whose classes are all equal, as behind a ReLU that let nothing through."""
import numpy as np
import pytest
import torch

from oracle import niti_oracle as O, vocab_oracle as VO

# the other classes' errors of a wanted one's -127 (of 128): all equal, so pseudo-stochastic rounding sends all of them the same way.
# For p = 2^30 / V it is up where the upper twelve of its 23 dropped bits exceed twice the lower eleven.
SIZES = [300, 2048, 2056, 4096, 10000, 32768, 50257]


def flat(V, T=1):
    return np.zeros((T, 16), np.int8), np.ones((V, 16), np.int8), np.arange(T) % V


def goes_up(V):
    lo = int(VO.probabilities(np.zeros((1, V), np.int64), *VO.row_statistics(np.zeros((1, V), np.int64), 0), 0)[0, 0]) & 0x7FFFFF
    return (lo >> 11) > 2 * (lo & 0x7FF)


@pytest.mark.parametrize("V", SIZES)
def test_equal_classes_are_rounded_alike(V):
    x, w, y = flat(V)
    r = VO.vocab(x, 0, w, 0, y, loss_mode=O.PSEUDO_STOCHASTIC)
    assert abs(r["loss"][0] - np.log(V)) < 1e-5
    others = np.delete(r["err8"][0], 0).astype(int)
    assert np.all(others == goes_up(V)) and r["err8"][0, 0] == -127 and r["e32"][0, 0] == (V - 1) * goes_up(V) - 127
    assert goes_up(V) == (V == 2056)


@pytest.mark.parametrize("V", [v for v in SIZES if v >= 2048])
def test_stochastic_errors_of_equal_classes(V):
    x, w, y = flat(V)
    others = np.delete(VO.vocab(x, 0, w, 0, y, loss_mode=O.STOCHASTIC, seed=V)["err8"][0], 0).astype(int)
    assert set(np.unique(others)) <= {0, 1}
    assert abs(others.sum() - 128 * (V - 1) / V) < 6 * np.sqrt(128)  # each 1 with probability 128 / V: six standard deviations


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 40])
@pytest.mark.parametrize("V", SIZES)
def test_on_the_gpu(V, T):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from niti_b200 import ops
    dev = "cuda:0"
    x, w, y = flat(V, T)
    layer = [torch.from_numpy(x).to(dev), torch.zeros((), dtype=torch.int32, device=dev), torch.from_numpy(w).to(dev),
             torch.zeros((), dtype=torch.int32, device=dev), torch.from_numpy(y).to(dev)]
    # with features of zeros the weight gradient says nothing of the errors: the error of the features does, a sum over a row's classes
    for how, mode in ((ops.ROUND_PSEUDO_STOCHASTIC, O.PSEUDO_STOCHASTIC), (ops.ROUND_STOCHASTIC, O.STOCHASTIC)):
        want = VO.vocab(x, 0, w, 0, y, loss_mode=mode, seed=4)
        loss, e8, exp_err, g32, gmax = ops.vocab_train(*layer, loss_mode=how, seed=ops.seed_tensor(4, dev))
        assert np.array_equal(e8.cpu().numpy(), want["e8"]) and int(exp_err) == want["exp_err"] and not g32.any() and int(gmax) == 0
        if mode == O.PSEUDO_STOCHASTIC:
            total = (V - 1) * goes_up(V) - 127
            assert np.all(want["e32"] == total)
