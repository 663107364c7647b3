"""Training calls whose errors do not fit into the workspace at once: the vocabulary's pieces together are one error, one maximum
and one gradient.  Whole numbers bit for bit against the same integers in plain 64-bit PyTorch (perf/operators.py), which is held
against the oracle first."""
import numpy as np
import pytest
import torch

from oracle import niti_oracle as O, vocab_oracle as VO

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from niti_b200 import ops  # noqa: E402
from niti_b200._lib import lib  # noqa: E402
from perf import operators as plain  # noqa: E402

DEV = "cuda:0"
ROUNDINGS = {plain.NEAREST: (ops.ROUND_NEAREST, ops.ROUND_NEAREST), plain.PSEUDO: (ops.ROUND_PSEUDO_STOCHASTIC, ops.ROUND_NEAREST),
             plain.STOCHASTIC: (ops.ROUND_STOCHASTIC, ops.ROUND_STOCHASTIC)}
ORACLE = {plain.NEAREST: O.ROUND, plain.PSEUDO: O.PSEUDO_STOCHASTIC, plain.STOCHASTIC: O.STOCHASTIC}


def word(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def case_of(T, F, V, rounding, **how):
    return plain._case(None, "distill_train" if how.get("top") else "train", T, F, V, rounding=rounding, **how)


def train(s):
    c = s["case"]
    loss_mode, err_mode = ROUNDINGS[c["rounding"]]
    how = dict(loss_mode=loss_mode, err_mode=err_mode, seed=s["seed"], loss_stream=0xFFFF, err_stream=1)
    layer = s["x"], s["exp_x"], s["w"], s["exp_w"]
    if c["top"]:
        return ops.vocab_distill_train(*layer, s["index"], s["top"], s["exp_top"], c["temperature"], **how)
    return ops.vocab_train(*layer, s["target"], **how)


def check(s):
    assert not plain.own
    want, got = plain.run(s), train(s)
    for name, a, b in zip(("e8", "exp_err", "g32", "max |g32|"), got[1:], want[1:]):
        assert a.shape == b.shape and a.dtype == b.dtype, name
        wrong = a != b
        assert not wrong.any(), f"{name}: {int(wrong.sum())} of {a.numel()} differ; exponents {int(got[2])} for {int(want[2])}"
    assert torch.isfinite(got[0]).all()
    ops.check_status(DEV)
    return got


@pytest.mark.parametrize("rounding", ROUNDINGS)
def test_the_plain_form_is_the_oracles(rounding):
    s = plain.prepare(case_of(70, 44, 900, rounding, ignored=0.2), 5)
    a = lambda t: t.cpu().numpy()  # noqa: E731
    want = VO.vocab(a(s["x"]), int(s["exp_x"]), a(s["w"]), int(s["exp_w"]), a(s["target"]), loss_mode=ORACLE[rounding],
                    err_mode=O.STOCHASTIC if rounding == plain.STOCHASTIC else O.ROUND, seed=int(s["seed"]))
    loss, e8, exp_err, g32, gmax = check(s)
    assert np.array_equal(a(e8), want["e8"]) and int(exp_err) == want["exp_err"] and np.array_equal(a(g32), want["g32"])


# first pieces whose product is one part (the first, second and fourth) or several; the later ones the other way round (the last two); rows
# of 16 bytes, of 4 and of 2
@pytest.mark.parametrize("rounding", ROUNDINGS)
@pytest.mark.parametrize("T,F,V", [(70000, 32, 3000), (6000, 700, 20000), (2500, 96, 50021), (9000, 130, 14000), (1500, 520, 70000), (5000, 250, 24000)])
def test_several_pieces(T, F, V, rounding):
    assert ops.vocab_pieces(T, V) > 1 and T * F > 131072
    check(plain.prepare(case_of(T, F, V, rounding, ignored=0.1), T + V))


@pytest.mark.parametrize("rounding", ROUNDINGS)
@pytest.mark.parametrize("T,F,V,K,kind,temperature", [(6000, 160, 20000, 9, "int8", 0), (2500, 96, 50021, 40, "int32", 1)])
def test_several_pieces_with_a_teacher(T, F, V, K, kind, temperature, rounding):
    assert ops.vocab_pieces(T, V) > 1 and T * F > 131072
    check(plain.prepare(case_of(T, F, V, rounding, top=K, top_type=kind, ragged=True, temperature=temperature), T + V))


@pytest.mark.parametrize("rounding", [plain.NEAREST, plain.PSEUDO])
@pytest.mark.parametrize("cooperative", [True, False])
@pytest.mark.parametrize("changed", [0, 1, 9])
@pytest.mark.parametrize("teacher", [False, True])
def test_a_later_piece_takes_back_the_first_ones_error(teacher, changed, cooperative, rounding):
    """Every wanted class lies in the first piece and has a copy behind it, each with half the probability: what the first piece
    adds to the error of the features, the last one takes away again, all of it or all but what `changed` of a copy's features differ
    by.  The error's unit is that of the sum."""
    T, F, V = 40000, 64, 3328
    first = lib.niti_vocab_piece(T, V)
    wanted = V - first
    assert ops.vocab_pieces(T, V) == 2 and wanted <= first and T * F > 131072
    g = torch.Generator(device=DEV).manual_seed(11)
    w = (torch.randint(0, 2, (V, F), device=DEV, generator=g) * 60 - 30).to(torch.int8)
    w[first:] = w[:wanted]
    w[first:, :changed] -= w[first:, :changed].sign()
    y = torch.arange(T, device=DEV) % wanted
    # a wanted class's logit: 900 F; any other's: 900 times a sum of F signs, far below by more than 31 powers of two
    ex, ew = -2, -7
    s = {"case": case_of(T, F, V, rounding, top=int(teacher)), "x": w[y].contiguous(), "w": w, "exp_x": word(ex), "exp_w": word(ew), "seed": None}
    if teacher:
        s.update(index=y.unsqueeze(1), top=torch.zeros((T, 1), dtype=torch.int8, device=DEV), exp_top=word(-4))
    else:
        s["target"] = y
    old = ops.set_cooperative_launch(cooperative)
    try:
        loss, e8, exp_err, g32, gmax = check(s)
    finally:
        ops.set_cooperative_launch(old)
    if not changed:
        assert not e8.any() and int(exp_err) == ew - 7
        assert int(gmax) > 0
