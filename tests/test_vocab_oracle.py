"""The vocabulary losses' integer definition (oracle/vocab_oracle.py) against real softmaxes, and what the C entry point refuses
before it touches a GPU."""
import ctypes

import numpy as np
import pytest

from oracle import niti_oracle as O, vocab_oracle as VO


@pytest.mark.parametrize("e", [-70, -58, -40, -31, -28, -27, -26, -20, -13, -5, -1, 0, 1, 2, 3, 4, 5, 9])
def test_exponentials(e):
    rng = np.random.default_rng(3)
    top = min(2 ** 32 - 1, int(40 * 2.0 ** -e) + 3)
    d = np.unique(np.concatenate([[0, 1, 2, 3, top], rng.integers(0, top + 1, 20000), (top * rng.random(20000) ** 4).astype(np.int64)]))
    got = VO.exp_weights(d, e) / 2.0 ** 30
    want = np.exp(-d * 2.0 ** e)
    # quartic 2.82e-6 and its four roundings of at most one unit of 2^-30 each, 4e-9; u cut to 2^-25 of a power of two, 2.1e-8; the
    # constant's 2^-32 (or, shifted down, 2^-(31-s) of exponents that are below 2^(32+e) by then) times 31 powers of two, 5.1e-9;
    # the shift's truncation, one unit of 2^-30; from the cut on 0 for at most 2^-31
    const = 31 * np.log(2) * 2.0 ** -31 if e >= -27 else 2.0 ** (32 + e) * min(1.0, 2.0 ** (-30 + min(31, -26 - e)))
    assert np.all(np.abs(got - want) <= want * (2.82e-6 + 4e-9 + 2.1e-8 + const) + 2.0 ** -30)
    assert VO.exp_weights(np.array([0]), e)[0] == 1 << 30
    assert np.all(VO.exp_weights(np.array([1, 2, 2 ** 32 - 1]), 6) == 0)


def softmax_case(seed, T, F, V, spread=2.5):
    rng = np.random.default_rng(seed)
    w = np.clip(np.rint(rng.standard_normal((V, F)) * 30), -127, 127).astype(np.int8)
    x = np.clip(np.rint(rng.standard_normal((T, F)) * 24), -127, 127).astype(np.int8)
    e = int(round(np.log2(spread / (np.sqrt(F) * 720))))
    return rng, x, e + 9, w, -9


def log_softmax(z):
    z = z - z.max(1, keepdims=True)
    return z - np.log(np.exp(z).sum(1, keepdims=True))


@pytest.mark.parametrize("T,F,V", [(5, 16, 1), (4, 48, 63), (4, 48, 64), (3, 33, 65), (3, 64, 1000), (2, 100, 40001)])
def test_cross_entropy_is_a_softmax_cross_entropy(T, F, V):
    rng, x, ex, w, ew = softmax_case(V, T, F, V)
    y = rng.integers(0, V, T)
    r = VO.vocab(x, ex, w, ew, y, loss_mode=O.ROUND)
    z = (x.astype(np.float64) @ w.astype(np.float64).T) * 2.0 ** (ex + ew)
    want = -log_softmax(z)[np.arange(T), y]
    # the sum's relative error: exponentials 2.9e-6 twice (a class's, its piece's), 2^-24 of each piece (at least 1) and 2^-34 a piece
    rel = 2 * 2.9e-6 + 2.0 ** -24 + (V / 64 + 1) * 2.0 ** -34
    assert np.all(np.abs(r["loss"] - want) <= rel + 1e-12)
    p = np.exp(log_softmax(z))
    p[np.arange(T), y] -= 1
    # rounding 2^-8, or the cut to 127 of 128; p itself
    assert np.all(np.abs(r["err8"] / 128.0 - p) <= np.maximum(2.0 ** -8, (np.abs(p) > 127 / 128.0) * 2.0 ** -7) + 2 * rel + 2.0 ** -29)


def test_error_is_the_derivative_of_the_loss():
    T, F, V = 3, 24, 300
    rng, x, ex, w, ew = softmax_case(8, T, F, V)
    y = rng.integers(0, V, T)
    r = VO.vocab(x, ex, w, ew, y, loss_mode=O.ROUND)
    unit = 2.0 ** (ex + ew)
    real = lambda xs: -log_softmax((xs @ w.astype(np.float64).T) * unit)[np.arange(T), y]  # noqa: E731
    h = 1e-3
    for f in range(F):
        up, dn = x.astype(np.float64), x.astype(np.float64)
        up[:, f] += h
        dn[:, f] -= h
        diff = (real(up) - real(dn)) / (2 * h) / 2.0 ** ex  # with respect to the dequantised feature
        got = r["e8"][:, f] * 2.0 ** r["exp_err"]
        # each of V errors is off by at most 2^-8 (2^-7 for the one that is cut) and weighs |w| 2^ew; e8 is rounded by half its unit;
        # differences: h^2/6 of a third derivative of at most (max |w| unit)^3
        bound = (np.abs(w[:, f].astype(np.float64)).sum() * 2.0 ** -8 + 127 * 2.0 ** -8) * 2.0 ** ew + 2.0 ** (r["exp_err"] - 1)
        assert np.all(np.abs(got - diff) <= bound + 1e-6)
    # and the weight gradient is the same error against the features
    assert np.array_equal(r["g32"], r["err8"].astype(np.int64).T @ x.astype(np.int64))


def test_distillation_against_softmaxes():
    T, F, V, K = 4, 32, 500, 6
    rng, x, ex, w, ew = softmax_case(21, T, F, V)
    idx = np.stack([rng.choice(V, K, replace=False) for _ in range(T)])
    idx[1, 3:] = -1
    idx[2, :] = -1
    top = rng.integers(-127, 128, (T, K)).astype(np.int8)
    for k in (0, 2):
        r = VO.vocab(x, ex, w, ew, idx, top=top, exp_top=-5, temperature_log2=k, loss_mode=O.ROUND)
        z = (x.astype(np.float64) @ w.astype(np.float64).T) * 2.0 ** (ex + ew - k)
        lp = log_softmax(z)
        for t in range(T):
            used = idx[t] >= 0
            if not used.any():
                assert r["loss"][t] == 0 and not r["err8"][t].any()
                continue
            b = top[t][used] * 2.0 ** (-5 - k)
            lq = b - b.max() - np.log(np.exp(b - b.max()).sum())
            want = 4.0 ** k * (np.exp(lq) * (lq - lp[t, idx[t][used]])).sum()
            assert abs(r["loss"][t] - want) <= 4.0 ** k * 4e-5  # four exponentials of 2.9e-6, q's times terms of up to 2 (ln of 500 over ...)
            g = np.exp(lp[t])
            g[idx[t][used]] -= np.exp(lq)
            assert np.all(np.abs(r["err8"][t] / 128.0 - g) <= 2.0 ** -8 + 4e-5)


def test_rows_without_a_class_have_neither_loss_nor_error():
    rng, x, ex, w, ew = softmax_case(2, 4, 16, 70)
    r = VO.vocab(x, ex, w, ew, np.array([3, -100, 70, -5]))
    assert r["loss"][1] == 0 and np.isnan(r["loss"][2:]).all() and np.isfinite(r["loss"][0])
    assert not r["err8"][1:].any() and r["err8"][0].any()


def test_flat_rows_have_an_error_where_eleven_bits_had_none():
    V = 4096
    x, w = np.zeros((1, 16), np.int8), np.ones((V, 16), np.int8)
    y = np.array([7])
    r = VO.vocab(x, 0, w, 0, y, loss_mode=O.STOCHASTIC, seed=5)
    assert abs(r["loss"][0] - np.log(V)) < 1e-5
    assert r["err8"][0, 7] == -127 and r["err8"][0].astype(int).sum() + 127 > 0  # about V / 32 of the others are 1
    old, _ = O.ti_loss(np.zeros((1, V), np.int8), 0, y, np.zeros((1, V), np.uint32))
    assert not np.delete(old[0], 7).any()


def test_entry_point_refuses_before_it_touches_a_gpu():
    from niti_b200._lib import lib, VocabArgs
    assert lib.niti_vocab_supported(1, 1, 1, 1) == 1 and lib.niti_vocab_supported(131071, 131071, 262144, 128) == 1
    for bad in ((0, 16, 16, 1), (16, 0, 16, 1), (16, 16, 0, 1), (16, 16, 16, 0), (131072, 16, 16, 1), (16, 131072, 16, 1), (16, 16, 262145, 1), (16, 16, 16, 129)):
        assert lib.niti_vocab_supported(*bad) == 0 and lib.niti_vocab_scratch_bytes(*bad, 1) == 0
    assert lib.niti_vocab_scratch_bytes(128, 512, 10000, 1, 1) > lib.niti_vocab_scratch_bytes(128, 512, 10000, 1, 0) > 0
    assert lib.niti_vocab_loss_i8(None, None) == -1
    p = 1 << 20  # looks like an aligned pointer; no call below gets as far as following it

    def args(**kw):
        a = VocabArgs(x=p, exp_x=p, w=p, exp_w=p, index=p, ignore_index=-100, loss=p, scratch=p, scratch_bytes=1 << 40, T=8, F=16, V=100, entries=1, bits=7)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.niti_vocab_loss_i8(ctypes.byref(a), None)
    for name in ("x", "exp_x", "w", "exp_w", "index", "loss", "scratch"):
        assert args(**{name: None}) == -1, name
    assert args(entries=2) == -1 and args(top=p) == -1 and args(exp_top=p) == -1  # several entries need a teacher, a teacher its exponent
    assert args(x=p + 8) == -1 and args(w=p + 8) == -1
    train = dict(g32=p, e8=p, exp_err=p, grad_maxabs=p)
    for name in ("e8", "exp_err", "grad_maxabs"):
        assert args(**{**train, name: None}) == -1, name
    assert args(**train, loss_round=3) == -1 and args(**train, err_round=-1) == -1 and args(**train, loss_round=1) == -1  # no seed
    assert args(**{**train, "g32": p + 4}) == -1
    assert args(T=1 << 17) == -2 and args(V=(1 << 18) + 1) == -2 and args(temperature_log2=31) == -2
    assert args(scratch_bytes=64) == -4 and args(scratch=p + 8) == -4
