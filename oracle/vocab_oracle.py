"""The vocabulary losses in exact integers on NumPy arrays (TEST INFRASTRUCTURE, not product code): what
niti_vocab_loss_i8 computes, written from its definition.

The reference's counterparts are TiLinear.forward, TiLoss.forward and TiLinear.backward (ti_torch.py:241-266, ti_loss.py:6-36);
the softmax here is another one (30 bits on the int32 accumulators), see include/niti_b200.h.
"""
import math

import numpy as np

from . import niti_oracle as O, philox

PIECE = 64
LOG2E_31 = 0xB8AA3B29  # round(log2(e) * 2**31)
COEFF = (1 << 30, -744236436, 257956795, -60029066, 10289510)  # 2**-phi * 2**30, phi in [-1/2, 1/2)


def _mantissas(d, e):
    """(q, I): E(d) is q >> I.  d 2**e below 64."""
    up, down = max(0, 26 + e), max(0, -26 - e)
    u = ((d << up).astype(np.uint64) * np.uint64(LOG2E_31 >> down) >> np.uint64(32)).astype(np.int64) + (1 << 24)
    phi = ((u & ((1 << 25) - 1)) - (1 << 24)) << 7
    q = np.full_like(phi, COEFF[4])
    for c in COEFF[3::-1]:
        q = (phi * q >> 32) + c
    return q, u >> 25


def exp_weights(d, e):
    """E(d) = 2**30 exp(-d 2**e) for an int64 array d >= 0 and a Python int e."""
    d = np.asarray(d, dtype=np.int64)
    e = min(int(e), 5)
    if e >= 0:
        cut = (21 + (1 << e)) >> e
    elif e <= -28:
        cut = (1 << 32) - 1
    else:
        cut = 43 << (-e - 1)
    q, I = _mantissas(np.minimum(d, cut), e)
    return np.where(I < 63, q >> np.minimum(I, 63), 0)


def row_statistics(acc, e):
    """(maximum, sum of exponentials relative to it with 2**34 as 1) of each row."""
    acc = acc.astype(np.int64)
    M = acc.max(1)
    S = np.zeros(len(acc), dtype=np.int64)
    for c in range(0, acc.shape[1], PIECE):
        a = acc[:, c:c + PIECE]
        m = a.max(1)
        part = exp_weights(m[:, None] - a, e).sum(1) >> 6
        S += part * exp_weights(M - m, e) >> 20
    return M, S


def row_loss_sums(acc, e):
    """Each row's sum of exponentials for its loss, with 2**44 as 1: the pieces' sums are scaled by exponentials that are not cut to
    units of 2**-30 first."""
    acc = acc.astype(np.int64)
    M, e = acc.max(1), int(e)
    L = np.zeros(len(acc), dtype=np.int64)
    for c in range(0, acc.shape[1], PIECE):
        a = acc[:, c:c + PIECE]
        m = a.max(1)
        part, d = exp_weights(m[:, None] - a, e).sum(1) >> 6, M - m
        there = d <= (0 if e > 5 else (1 << 32) - 1 >> max(0, 26 + e))  # 64 nats; units of more than 32 nats tell 0 from the rest
        q, I = _mantissas(np.where(there, d, 0), min(e, 5))
        L += np.where(there, part * q >> np.minimum(10 + I, 63), 0)
    return L


def probabilities(acc, M, S, e):
    """p with 2**30 as 1."""
    p = np.empty(acc.shape, dtype=np.int64)
    for t in range(len(acc)):
        n = int(S[t]).bit_length() - 32
        R = ((1 << 63) - 1) // (int(S[t]) >> n)
        p[t] = (exp_weights(int(M[t]) - acc[t].astype(np.int64), e) * R >> 32) >> (n - 3)
    return p


def vocab(x, exp_x, w, exp_w, index, ignore_index=-100, top=None, exp_top=0, temperature_log2=0, train=True, bits=7,
          loss_mode=O.PSEUDO_STOCHASTIC, err_mode=O.ROUND, seed=0, loss_stream=0xFFFF, err_stream=1, sample_offset=0):
    """dict of loss (float64), and for training err8, e32, e8, exp_err, g32."""
    T, V = len(x), len(w)
    acc = x.astype(np.int64) @ w.astype(np.int64).T
    e = exp_x + exp_w - temperature_log2
    M, S = row_statistics(acc, e)
    L = row_loss_sums(acc, e)
    index = index.reshape(T, -1)
    loss = np.zeros(T)
    learns = np.zeros(T, dtype=bool)
    want = np.zeros((T, V), dtype=np.int64)
    for t in range(T):
        used = [k for k, j in enumerate(index[t]) if 0 <= j < V and (top is not None or j != ignore_index)]
        if any((j >= V or (top is None and j < 0)) and (top is not None or j != ignore_index) for j in index[t]):
            loss[t] = math.nan
            continue
        if not used:
            continue
        learns[t] = True
        if top is None:
            share, lnq = [1 << 30], [0.0]
        else:
            b = top[t].astype(np.int64)
            best = max(int(b[k]) for k in used)
            share = [int(exp_weights(best - int(b[k]), exp_top - temperature_log2)) for k in used]
            lnq = [-(best - int(b[k])) * 2.0 ** (exp_top - temperature_log2) - math.log(sum(share) / 2.0 ** 30) for k in used]
        total = sum(share)
        lnl = math.log(int(L[t]) / 2.0 ** 44)
        for k, s, l in zip(used, share, lnq):
            j = int(index[t, k])
            if s:
                loss[t] += s / total * ((int(M[t]) - int(acc[t, j])) * 2.0 ** e + lnl + l)
            want[t, j] += (s << 30) // total
        loss[t] *= 4.0 ** temperature_log2
    r = {"loss": loss}
    if not train:
        return r
    err = (probabilities(acc, M, S, e) - want) * learns[:, None]
    four = (V + 3) // 4 * 4
    rnd = philox.random_u32_tensor(seed, loss_stream, (T, four), sample_offset * four)[:, :V] if loss_mode == O.STOCHASTIC else None
    err8 = O.apply_shift(err, 23, loss_mode, rnd)
    e32 = err8.astype(np.int64) @ w.astype(np.int64)
    g32 = err8.astype(np.int64).T @ x.astype(np.int64)
    shift = max(0, O.range_estimate(e32) - bits)
    rnd = philox.random_u32_tensor(seed, err_stream, e32.shape, sample_offset * e32.shape[1]) if err_mode == O.STOCHASTIC else None
    e8 = O.apply_shift(e32, shift, err_mode, rnd) if shift > 0 else O.wrap_int8(e32)
    r.update(err8=err8, e32=e32, e8=e8, exp_err=shift + exp_w - 7 + temperature_log2, g32=g32)
    return r
