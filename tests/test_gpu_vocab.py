"""The vocabulary losses on the GPU against their integer definition (oracle/vocab_oracle.py): whole numbers bit for bit, losses to
float32's rounding."""
import numpy as np
import pytest
import torch

from oracle import niti_oracle as O, vocab_oracle as VO

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from niti_b200 import ops  # noqa: E402

DEV = "cuda:0"
MODES = {"nearest": O.ROUND, "stochastic": O.STOCHASTIC, "pseudo": O.PSEUDO_STOCHASTIC}


def cu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def word(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def layer(seed, T, F, V, spread=2.5, lift=True):
    """Features, weights and wanted classes of a last layer whose logits have the given spread."""
    rng = np.random.default_rng(seed)
    w = np.clip(np.rint(rng.standard_normal((V, F)) * 30), -127, 127).astype(np.int8)
    y = rng.integers(0, V, T)
    x = rng.standard_normal((T, F)) * 24
    if lift:
        x = x + rng.random((T, 1)) * (4.8 / np.sqrt(F)) * w[y]
    x = np.clip(np.rint(x), -127, 127).astype(np.int8)
    e = int(round(np.log2(spread / (np.sqrt(F) * 720))))
    return rng, x, e + 9, w, -9, y


def same(got, want, what):
    got = got.cpu().numpy()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = np.argwhere(got != want)
    assert not len(bad), f"{what}: {len(bad)} of {got.size} differ; first {bad[:5].tolist()}, {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"


def same_loss(got, want):
    got = got.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    # the same doubles up to the order of a row's entries and the libraries' logarithms, then one rounding to float32
    ok = np.abs(got - want) <= np.abs(want) * 2.0 ** -24 + 1e-11
    assert np.all(ok | np.isnan(want)), (got[~ok][:5], want[~ok][:5])


def check_train(r, want):
    loss, e8, exp_err, g32, gmax = r
    same_loss(loss, want["loss"])
    same(g32, want["g32"].astype(np.int32), "g32")
    assert int(gmax) == int(np.abs(want["g32"]).max())
    assert int(exp_err) == want["exp_err"]
    same(e8, want["e8"], "e8")
    ops.check_status(DEV)


SIZES = [  # tokens, features, classes
    (1, 16, 1), (1, 16, 2), (2, 32, 63), (3, 16, 64), (5, 48, 65), (1, 128, 255), (1, 128, 256), (1, 128, 257), (127, 128, 320),
    (128, 256, 512), (129, 144, 513), (130, 160, 1000), (257, 128, 777), (300, 272, 1536), (64, 512, 4099), (33, 1040, 300), (520, 64, 2500),
    # rows that are no multiples of 16 bytes, results that are none of four words
    (3, 1, 70), (7, 15, 129), (9, 17, 300), (140, 100, 700), (200, 130, 513), (65, 250, 1027),
]


@pytest.mark.parametrize("T,F,V", SIZES)
def test_loss(T, F, V):
    rng, x, ex, w, ew, y = layer(T + F + V, T, F, V)
    want = VO.vocab(x, ex, w, ew, y, train=False)
    same_loss(ops.vocab_loss(cu(x), word(ex), cu(w), word(ew), cu(y)), want["loss"])
    ops.check_status(DEV)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("T,F,V", SIZES)
def test_train(T, F, V, mode):
    rng, x, ex, w, ew, y = layer(T + F + V + 1, T, F, V)
    y[rng.random(T) < 0.2] = -100
    err_mode = O.STOCHASTIC if mode == "stochastic" else O.ROUND
    want = VO.vocab(x, ex, w, ew, y, loss_mode=MODES[mode], err_mode=err_mode, seed=2 ** 40 + 5, sample_offset=3, err_stream=17)
    r = ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y), loss_mode=MODES[mode], err_mode=err_mode, seed=ops.seed_tensor(2 ** 40 + 5, DEV),
                        sample_offset=3, err_stream=17)
    check_train(r, want)


@pytest.mark.parametrize("F,V", [(80, 5003), (80, 45001), (2064, 1500)])
@pytest.mark.parametrize("T", [5, 8, 31, 32, 33, 56, 63, 64, 65])
def test_few_tokens_in_a_row_tile(T, F, V):
    """Up to 64 tokens lie several times in a row tile: each row's every column is seen to once, in tiles of either width."""
    rng, x, ex, w, ew, y = layer(T + F + V + 2, T, F, V)
    y[T // 3] = -100
    mode = [O.PSEUDO_STOCHASTIC, O.STOCHASTIC, O.ROUND][T % 3]
    want = VO.vocab(x, ex, w, ew, y, loss_mode=mode, seed=77, sample_offset=1)
    same_loss(ops.vocab_loss(cu(x), word(ex), cu(w), word(ew), cu(y)), want["loss"])
    check_train(ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y), loss_mode=mode, seed=ops.seed_tensor(77, DEV), sample_offset=1), want)


@pytest.mark.parametrize("kind", ["int8", "int32"])
@pytest.mark.parametrize("T,F,V,K,temperature", [(1, 16, 1, 1, 0), (4, 32, 100, 3, 1), (40, 64, 300, 32, 0), (37, 96, 1000, 33, -1), (130, 128, 513, 64, 2),
                                                 (9, 20, 70, 128, 0), (300, 48, 90, 5, 3)])
def test_distill(T, F, V, K, temperature, kind):
    rng, x, ex, w, ew, y = layer(T + F + V + K, T, F, V)
    idx = rng.integers(0, V, (T, K))  # classes come twice
    idx[:, 0] = y
    idx = np.where(rng.random((T, K)) < 0.3, -1 - rng.integers(0, 3, (T, K)), idx)
    idx[T // 2] = -1  # a row without an entry
    top = rng.integers(-127, 128, (T, K)).astype(np.int8) if kind == "int8" else rng.integers(-2 ** 31, 2 ** 31, (T, K)).astype(np.int32)
    et = -4 if kind == "int8" else -28
    for mode in (O.PSEUDO_STOCHASTIC, O.STOCHASTIC):
        want = VO.vocab(x, ex, w, ew, idx, top=top, exp_top=et, temperature_log2=temperature, loss_mode=mode, seed=9)
        r = ops.vocab_distill_train(cu(x), word(ex), cu(w), word(ew), cu(idx), cu(top), word(et), temperature, loss_mode=mode, seed=ops.seed_tensor(9, DEV))
        check_train(r, want)
    same_loss(ops.vocab_distill_loss(cu(x), word(ex), cu(w), word(ew), cu(idx), cu(top), word(et), temperature), want["loss"])


@pytest.mark.parametrize("e", [-60, -35, -28, -27, -26, -14, -6, -1, 0, 1, 2, 3, 4, 5, 8])
def test_exponents_from_flat_to_one_hot(e):
    """Accumulator units from nothing to more than the softmax can tell apart, with accumulators at both ends of their range."""
    T, F, V = 6, 64, 700
    rng, x, _, w, _, y = layer(e + 100, T, F, V)
    x[0], w[3], w[5] = 127, 127, -128
    x[1] = -128
    want = VO.vocab(x, e + 4, w, -4, y)
    check_train(ops.vocab_train(cu(x), word(e + 4), cu(w), word(-4), cu(y)), want)


def test_rows_without_a_class():
    T, F, V = 200, 64, 600
    rng, x, ex, w, ew, y = layer(4, T, F, V)
    for fill in (-100, -1, V, 2 ** 40, -2 ** 40):
        y[:130] = fill  # a whole row tile without a loss
        y[150] = fill
        want = VO.vocab(x, ex, w, ew, y)
        check_train(ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y)), want)
    y[:] = -1
    want = VO.vocab(x, ex, w, ew, y, ignore_index=-1)
    loss, e8, exp_err, g32, gmax = ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y), ignore_index=-1)
    assert not loss.any() and not e8.any() and not g32.any() and int(gmax) == 0 and int(exp_err) == ew - 7
    check_train((loss, e8, exp_err, g32, gmax), want)


@pytest.mark.parametrize("ignore", [0, 5, 599, 600, 2 ** 33, -7])
def test_any_class_can_be_the_one_to_ignore(ignore):
    T, F, V = 150, 48, 600
    rng, x, ex, w, ew, y = layer(14, T, F, V)
    y[rng.random(T) < 0.3] = ignore
    want = VO.vocab(x, ex, w, ew, y, ignore_index=ignore)
    assert (want["loss"] == 0).any()
    check_train(ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y), ignore), want)
    same_loss(ops.vocab_loss(cu(x[:3]), word(ex), cu(w), word(ew), cu(y[:3]), ignore), want["loss"][:3])


def test_plain_launches_give_the_same():
    """Where cooperative launches are off, the error's maximum and its narrowing are two launches."""
    for T, F, V in ((300, 320, 3000), (40, 30, 2000)):
        rng, x, ex, w, ew, y = layer(16, T, F, V)
        a = ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y))
        old = ops.set_cooperative_launch(False)
        try:
            b = ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y))
        finally:
            ops.set_cooperative_launch(old)
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_no_tokens():
    w, ew = cu(np.ones((70, 16), np.int8)), word(-3)
    x = torch.empty((0, 16), dtype=torch.int8, device=DEV)
    y = torch.empty(0, dtype=torch.int64, device=DEV)
    assert ops.vocab_loss(x, word(0), w, ew, y).shape == (0,)
    g = torch.full((70, 16), 7, dtype=torch.int32, device=DEV)
    loss, e8, exp_err, g32, gmax = ops.vocab_train(x, word(0), w, ew, y, g32=g)
    assert loss.shape == (0,) and e8.shape == (0, 16) and int(exp_err) == -10 and g32 is g and not g.any() and int(gmax) == 0


@pytest.mark.parametrize("T,F,V", [(70000, 32, 3000), (131071, 16, 1100)])
def test_errors_that_take_several_pieces(T, F, V):
    """More tokens than a piece of the errors holds at once: adjointness and sums against the one-piece call on parts of the tokens."""
    rng, x, ex, w, ew, y = layer(T, T, F, V)
    assert ops.vocab_pieces(T, V) > 1
    args = (word(ex), cu(w), word(ew))
    loss, e8, exp_err, g32, gmax = ops.vocab_train(cu(x), *args, cu(y))
    total, parts, errs = torch.zeros_like(g32), [], []
    step = 16384
    for t in range(0, T, step):
        assert ops.vocab_pieces(min(step, T - t), V) == 1
        r = ops.vocab_train(cu(x[t:t + step]), *args, cu(y[t:t + step]))
        total += r[3]
        parts.append(r[0])
        errs.append((r[1], int(r[2])))
    assert torch.equal(loss, torch.cat(parts)) and torch.equal(g32, total) and int(gmax) == int(total.abs().max())
    for (part, e), t in zip(errs, range(0, T, step)):  # both round the same int32 sums, to units that may differ
        a, b = part.double() * 2.0 ** e, e8[t:t + step].double() * 2.0 ** int(exp_err)
        assert float((a - b).abs().max()) <= 2.0 ** (e - 1) + 2.0 ** (int(exp_err) - 1)
    ops.check_status(DEV)


@pytest.mark.parametrize("T", [2, 6, 40])
def test_the_largest_vocabulary(T):
    F, V = 48, 1 << 18
    rng, x, ex, w, ew, y = layer(T, T, F, V)
    y[0], y[1] = V - 1, 0
    idx = np.stack([y, np.full(T, V - 1), rng.integers(0, V, T)], axis=1)
    top = rng.integers(-9, 9, idx.shape).astype(np.int8)
    check_train(ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y)), VO.vocab(x, ex, w, ew, y))
    want = VO.vocab(x, ex, w, ew, idx, top=top, exp_top=-2, temperature_log2=1, loss_mode=O.STOCHASTIC, seed=3)
    check_train(ops.vocab_distill_train(cu(x), word(ex), cu(w), word(ew), cu(idx), cu(top), word(-2), 1, loss_mode=O.STOCHASTIC, seed=ops.seed_tensor(3, DEV)), want)


@pytest.mark.parametrize("T", [3, 5, 140])
def test_the_longest_rows(T):
    """Accumulators up to the ends of int32."""
    F, V = 131071, 70
    rng = np.random.default_rng(T)
    x = rng.choice(np.array([-128, 127], np.int8), (T, 1)).repeat(F, 1)
    w = rng.choice(np.array([-128, 127], np.int8), (V, 1)).repeat(F, 1)
    x[0], w[1] = -128, -128
    w[2, ::2] = 1
    y = rng.integers(0, V, T)
    for e in (-40, -31, -20):
        check_train(ops.vocab_train(cu(x), word(e + 9), cu(w), word(-9), cu(y)), VO.vocab(x, e + 9, w, -9, y))


def test_the_most_tokens_on_one_class():
    """Sums over tokens up to the ends of int32."""
    T, F, V = 131071, 16, 3
    x, w = np.full((T, F), -128, np.int8), np.zeros((V, F), np.int8)
    w[0] = 127
    y = np.zeros(T, np.int64)
    y[5] = 2
    r = ops.vocab_train(cu(x), word(-4), cu(w), word(-4), cu(y))
    check_train(r, VO.vocab(x, -4, w, -4, y))
    assert int(r[4]) > 2 ** 30


@pytest.mark.parametrize("cooperative", [True, False])
@pytest.mark.parametrize("T,F,V", [(128, 1024, 800), (129, 1024, 800), (700, 250, 513)])
def test_errors_about_the_size_that_one_cluster_narrows(T, F, V, cooperative):
    rng, x, ex, w, ew, y = layer(T + F + V + 3, T, F, V)
    want = VO.vocab(x, ex, w, ew, y, err_mode=O.STOCHASTIC, seed=8, sample_offset=5, err_stream=2)
    old = ops.set_cooperative_launch(cooperative)
    try:
        r = ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y), err_mode=O.STOCHASTIC, seed=ops.seed_tensor(8, DEV), sample_offset=5, err_stream=2)
    finally:
        ops.set_cooperative_launch(old)
    check_train(r, want)


def test_results_do_not_depend_on_pairs_of_thread_blocks():
    rng, x, ex, w, ew, y = layer(6, 300, 320, 3000)
    a = ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y))
    old = ops.set_cta_pairs(False)
    try:
        b = ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y))
    finally:
        ops.set_cta_pairs(old)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_given_gradient_buffer_unaligned_views_and_other_streams():
    T, F, V = 50, 64, 900
    rng, x, ex, w, ew, y = layer(7, T, F, V)
    want = VO.vocab(x, ex, w, ew, y)
    g = torch.full((V, F), 5, dtype=torch.int32, device=DEV)
    xo = torch.empty(T * F + 3, dtype=torch.int8, device=DEV)[3:].view(T, F).copy_(cu(x))  # starts off a 16-byte boundary
    wo = torch.empty(V * F + 1, dtype=torch.int8, device=DEV)[1:].view(V, F).copy_(cu(w))
    r = ops.vocab_train(xo, word(ex), wo, word(ew), cu(y), g32=g)
    assert r[3].data_ptr() == g.data_ptr()
    check_train(r, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = ops.vocab_train(cu(x), word(ex), cu(w), word(ew), cu(y))
    side.synchronize()
    check_train(r, want)


@pytest.mark.parametrize("T,F,V", [(3, 64, 500), (40, 64, 3000), (300, 100, 2000)])
def test_operands_written_right_before_a_call(T, F, V):
    """Launches set up under the one before: what that one writes, the operands among it, is seen all the same, call after call."""
    cases = []
    for seed in (1, 2):
        rng, x, ex, w, ew, y = layer(seed, T, F, V)
        idx = rng.integers(0, V, (T, 5))
        cases.append([cu(a) for a in (x, w, y, idx, rng.integers(-9, 9, (T, 5)).astype(np.int8))])
    wants = [(ops.vocab_loss(x, word(ex), w, word(ew), y), ops.vocab_distill_loss(x, word(ex), w, word(ew), idx, top, word(-2)),
              ops.vocab_train(x, word(ex), w, word(ew), y)) for x, w, y, idx, top in cases]
    x, w, y, idx, top = (torch.empty_like(t) for t in cases[0])
    exps = word(ex), word(ew), word(-2)
    got = []
    for i in range(40):
        for to, frm in zip((x, w, y, idx, top), cases[i % 2]):
            to.copy_(frm)
        a = ops.vocab_loss(x, exps[0], w, exps[1], y)
        b = ops.vocab_distill_loss(x, exps[0], w, exps[1], idx, top, exps[2])
        got.append((a, b, ops.vocab_train(x, exps[0], w, exps[1], y)))
    for i, (a, b, c) in enumerate(got):
        want = wants[i % 2]
        assert torch.equal(a, want[0]) and torch.equal(b, want[1]) and all(torch.equal(u, v) for u, v in zip(c, want[2])), i


def test_two_streams_at_once():
    cases = []
    for seed, (T, F, V) in enumerate([(500, 320, 6000), (30, 64, 9000)]):
        rng, x, ex, w, ew, y = layer(seed, T, F, V)
        cases.append((cu(x), word(ex), cu(w), word(ew), cu(y)))
    wants = [ops.vocab_train(*c) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], []
    for _ in range(20):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(ops.vocab_train(*c))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(u, v) for u, v in zip(r, wants[i % 2])), i
    ops.check_status(DEV)


def test_two_captured_steps_share_nothing():
    cases = [layer(s, 40 + s, 48, 600 + s) for s in (1, 2)]
    inputs = [(cu(x), word(ex), cu(w), word(ew), cu(y)) for _, x, ex, w, ew, y in cases]
    wants = [VO.vocab(x, ex, w, ew, y) for _, x, ex, w, ew, y in cases]
    for i in inputs:
        ops.vocab_train(*i)
    graphs, outs = [], []
    for i in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.vocab_train(*i))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, want in zip(outs, wants):
        check_train(o, want)


def test_refusals():
    rng, x, ex, w, ew, y = layer(9, 8, 32, 100)
    x, w, y, ex, ew = cu(x), cu(w), cu(y), word(ex), word(ew)
    top = torch.zeros((8, 4), dtype=torch.int8, device=DEV)
    idx = torch.zeros((8, 4), dtype=torch.int64, device=DEV)
    bad = [
        lambda: ops.vocab_loss(x.cpu(), ex, w, ew, y), lambda: ops.vocab_loss(x[:, ::2], ex, w[:, ::2], ew, y), lambda: ops.vocab_loss(x, ex, w.t(), ew, y),
        lambda: ops.vocab_loss(x.float(), ex, w, ew, y), lambda: ops.vocab_loss(x[:, :16].contiguous(), ex, w, ew, y),
        lambda: ops.vocab_loss(x, ex, w, ew, y[:7]), lambda: ops.vocab_loss(x, ex, w, ew, y.int()), lambda: ops.vocab_loss(x, ex, w, ew, idx),
        lambda: ops.vocab_loss(x, ex.float(), w, ew, y), lambda: ops.vocab_loss(x, torch.zeros(2, dtype=torch.int32, device=DEV), w, ew, y),
        lambda: ops.vocab_loss(x[None], ex, w, ew, y), lambda: ops.vocab_loss(x, ex, w[:0], ew, y),
        lambda: ops.vocab_distill_loss(x, ex, w, ew, idx, top[:, :3].contiguous(), ex), lambda: ops.vocab_distill_loss(x, ex, w, ew, idx, top.float(), ex),
        lambda: ops.vocab_distill_loss(x, ex, w, ew, idx, top, ex, 31), lambda: ops.vocab_distill_loss(x, ex, w, ew, y, top, ex),
        lambda: ops.vocab_distill_loss(x, ex, w, ew, idx.repeat(1, 33), top.repeat(1, 33), ex),
        lambda: ops.vocab_distill_loss(x, ex, w, ew, idx[:, :0], top[:, :0], ex),
        lambda: ops.vocab_train(x, ex, w, ew, y, loss_mode=1), lambda: ops.vocab_train(x, ex, w, ew, y, loss_mode=7), lambda: ops.vocab_train(x, ex, w, ew, y, err_mode=1),
        lambda: ops.vocab_train(x, ex, w, ew, y, bits=0), lambda: ops.vocab_train(x, ex, w, ew, y, bits=8),
        lambda: ops.vocab_train(x, ex, w, ew, y, g32=torch.zeros((100, 31), dtype=torch.int32, device=DEV)),
        lambda: ops.vocab_train(x, ex, w, ew, y, g32=torch.zeros((100, 32), dtype=torch.int64, device=DEV)),
        lambda: ops.vocab_train(x, ex, w, ew, y, g32=torch.zeros(100 * 32 + 1, dtype=torch.int32, device=DEV)[1:].view(100, 32)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError)):
            f()
            pytest.fail(f"call {i} was not refused")


# ----------------------------------------------------------------------------- the layer, the network, the trainer
def mlp(widths, vocab, seed):
    """A network of linear layers that ends in a vocabulary, and its weights on the host."""
    from torch.nn import Sequential
    from niti_b200 import ti_torch
    from niti_b200.ti_net import TiNet
    rng = np.random.default_rng(seed)
    net = TiNet()
    layers = []
    for a, b in zip(widths, widths[1:]):
        layers += [ti_torch.TiLinear(a, b), ti_torch.TiReLU()]
    layers += [ti_torch.TiVocabHead(widths[-1], vocab)]
    net.forward_layers = Sequential(*layers)
    net.assign_layer_ids()
    host = []
    for l in net.weighted_layers():
        w = np.clip(np.rint(rng.standard_normal(tuple(l.weight.shape)) * 30), -127, 127).astype(np.int8)
        e = -9 - int(np.log2(w.shape[1]) / 2)
        l.weight, l.weight_exp = cu(w), ti_torch.exp_tensor(e, DEV)
        host.append([w, e])
    return net, host


def oracle_step(host, x, target=None, teacher=None, temperature_log2=0, mu=5):
    """One step of that network; updates `host` in place and returns the losses."""
    a, e = O.float_to_int8(x)
    acts = []
    for w, we in host[:-1]:
        acts.append((a, e))
        a, e, _ = O.act_calc(O.int8_mm(a, w.T), e + we)
        acts.append((a, e))
        a = np.maximum(a, 0).astype(np.int8)
    w, we = host[-1]
    kw = dict(top=teacher[1], exp_top=teacher[2], temperature_log2=temperature_log2) if teacher else {}
    r = VO.vocab(a, e, w, we, teacher[0] if teacher else target, err_stream=16 * (len(host) - 1) + 1, **kw)
    err, err_e = r["e8"], r["exp_err"]
    grads = [r["g32"]]
    for i in range(len(host) - 2, -1, -1):
        pre, inp = acts[2 * i + 1][0], acts[2 * i][0]
        err = np.where(pre > 0, err, 0).astype(np.int8)
        grads.insert(0, O.int8_mm(err.T, inp))
        if i > 0:
            err, _ = O.err_calc(O.int8_mm(err, host[i][0]))
    for i, g in enumerate(grads):
        host[i][0] = O.weight_update(host[i][0], g, mu)[0]
    return r["loss"]


def test_a_network_learns_tokens_and_then_from_a_teacher():
    from niti_b200 import ti_torch
    ti_torch.GRAD_BITWIDTH, ti_torch.TRAINING = 5, True
    T, V, K = 130, 700, 7
    net, host = mlp([24, 48, 64], V, 3)
    rng = np.random.default_rng(4)
    x = rng.standard_normal((T, 24)).astype(np.float32)
    y = rng.integers(0, V, T)
    y[::9] = -100
    for _ in range(3):
        before = net.losses(cu(x), cu(y))
        loss = net.train_step(cu(x), cu(y))
        assert torch.equal(before, loss)
        same_loss(loss, oracle_step(host, x, y))
    teacher = (np.stack([rng.choice(V, K, replace=False) for _ in range(T)]), rng.integers(-100, 101, (T, K)).astype(np.int8), -4)
    teacher[0][5, 2:] = -1
    on_gpu = (cu(teacher[0]), cu(teacher[1]), teacher[2], 1)
    for _ in range(2):
        before = net.losses(cu(x), on_gpu)
        loss = net.train_step(cu(x), on_gpu)
        assert torch.equal(before, loss)
        same_loss(loss, oracle_step(host, x, teacher=teacher, temperature_log2=1))
    for l, (w, _) in zip(net.weighted_layers(), host):
        same(l.weight, w, "weights")
    ops.check_status(DEV)


def test_tokens_in_batches_of_positions():
    from niti_b200 import ti_torch
    net, _ = mlp([32], 300, 6)
    head = net.vocab_head()
    rng = np.random.default_rng(7)
    x = cu(rng.integers(-100, 101, (5, 9, 32)).astype(np.int8))
    y = cu(rng.integers(0, 300, (5, 9)))
    e = ti_torch.exp_tensor(-7, DEV)
    head.defer_update = True
    loss, (err, err_exp) = head.train_step((x, e), y)
    assert loss.shape == (5, 9) and err.shape == x.shape
    flat, (err1, err_exp1) = head.train_step((x.view(45, 32), e), y.view(45))
    assert torch.equal(loss.view(-1), flat) and torch.equal(err.view(45, 32), err1) and int(err_exp) == int(err_exp1)
    assert torch.equal(head.loss((x, e), y), loss)
    first = head.loss((x.transpose(0, 1), e), y.t())  # positions first, not contiguous
    assert torch.equal(first, loss.t())


def test_trainer_replays_steps_of_a_vocabulary():
    from niti_b200 import ti_torch
    from niti_b200.trainer import Trainer
    ti_torch.GRAD_BITWIDTH, ti_torch.TRAINING = 5, True
    T, V = 64, 500
    net, host = mlp([40, 32], V, 11)
    rng = np.random.default_rng(12)
    tr = Trainer(net, T, DEV, in_shape=(40,), warmup_steps=1, seed=1)
    for _ in range(4):  # one eager step, then replays
        x, y = rng.standard_normal((T, 40)).astype(np.float32), rng.integers(0, V, T)
        r = tr.step(torch.from_numpy(x).pin_memory(), torch.from_numpy(y).pin_memory())
        out, _ = r.wait()
        want = oracle_step(host, x, y)
        got = out.numpy().astype(np.float64)
        assert np.all(np.abs(got - want) <= np.abs(want) * 2.0 ** -24 + 1e-11)
    for l, (w, _) in zip(net.weighted_layers(), host):
        same(l.weight, w, "weights")
    ti_torch.SAMPLE_OFFSET = 0
