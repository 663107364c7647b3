"""The vocabulary losses where one class stands far above all others, by their integer definition (oracle/vocab_oracle.py): the loss
is what the others leave, however little."""
import numpy as np
import pytest

from oracle import vocab_oracle as VO

GAPS = [8, 14, 16, 18, 20, 20.5, 21.5, 22, 24, 28, 31]  # the wanted class above all others, in nats
UNITS = {-7: (1, 64, 2), -15: (256, 64, 2), -1: (1, 1, 2)}  # exponent of an accumulator: features, weight, feature of a nat


def peaked(T, V, e=-7):
    """Rows of one class above V - 1 equal ones: (x, exp_x, w, exp_w, classes, the distances in nats)."""
    n, weight, per_nat = UNITS[e]
    x, w = np.zeros((T, max(16, n)), np.int8), np.zeros((V, max(16, n)), np.int8)
    gaps = np.array([GAPS[t % len(GAPS)] for t in range(T)])
    x[:, :n] = (gaps * per_nat)[:, None]
    w[V // 2, :n] = weight
    assert n * weight * per_nat * 2.0 ** e == 1
    return x, e + 7, w, -7, np.full(T, V // 2), gaps


def sum_error(loss):
    """How far a loss may be off by its row's sum: the pieces' exponentials by 2.9e-6 (less than 1 part in 10^7 more for the roundings
    of their argument), the wanted class's piece by 63 exponentials cut to 2^-30 and by a sum cut to 2^-24."""
    return np.minimum(1.0, np.expm1(loss)) * 3e-6 + 63 * 2.0 ** -30 + 2.0 ** -24


@pytest.mark.parametrize("e", UNITS)
@pytest.mark.parametrize("V", [65, 5000, 131072])
def test_the_rest_of_a_row(V, e):
    x, ex, w, ew, y, gaps = peaked(len(GAPS), V, e)
    want = np.log1p((V - 1) * np.exp(-gaps))
    got = VO.vocab(x, ex, w, ew, y, train=False)["loss"]
    assert np.all(np.abs(got - want) <= sum_error(want) + 1e-15), (got, want)


@pytest.mark.parametrize("e", [-70, -40, -31, -28, -27, -26, -20, -7, 0, 3, 5, 6, 9])
def test_row_sums_at_every_unit(e):
    """Two classes of two pieces, the lower one `d` units down, up to the ends of int32."""
    rng = np.random.default_rng(2)
    top = min(2 ** 32 - 1, int(70 * 2.0 ** -e) + 3)
    d = np.unique(np.concatenate([[0, 1, 2, 3, top], rng.integers(0, top + 1, 200), (top * rng.random(200) ** 4).astype(np.int64)]))
    acc = np.full((len(d), 65), -2 ** 31, np.int64)  # 63 of the first piece: far below wherever the unit tells them apart
    acc[:, 0], acc[:, 64] = 2 ** 31 - 1, 2 ** 31 - 1 - d
    L = VO.row_loss_sums(acc, e)
    far = 63 * np.exp(-min(700.0, (2.0 ** 32 - 1) * 2.0 ** e))
    want = 1 + np.exp(-np.minimum(d * 2.0 ** e, 700.0)) + far
    # quartics 2.9e-6, their arguments' roundings (those of an unshifted one of units below 2^-27 are the ones of
    # test_exponentials), the first piece's cuts
    const = 2.0 ** (32 + e) * min(1.0, 2.0 ** (-30 + min(31, -26 - e))) if e < -27 else 0.0
    assert np.all(np.abs(L / 2.0 ** 44 - want) <= (want - 1) * (3e-6 + const) + 63 * 2.0 ** -30 + 2.0 ** -24)
