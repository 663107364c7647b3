"""Networks that end in a vocabulary of classes: blocks of layers, and what a classifier's network does beside them."""
import numpy as np
import pytest
import torch
from torch.nn import Sequential

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from niti_b200 import ops, ti_torch  # noqa: E402
from niti_b200.ti_net import TiNet  # noqa: E402
from tests.test_gpu_vocab import cu, mlp, oracle_step, same, same_loss  # noqa: E402

DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _training():
    old = ti_torch.GRAD_BITWIDTH, ti_torch.TRAINING
    ti_torch.GRAD_BITWIDTH, ti_torch.TRAINING = 5, True
    yield
    ti_torch.GRAD_BITWIDTH, ti_torch.TRAINING = old


def nested(layers, how):
    """The layers before the last in blocks: one of two layers; all of them in a block within a block."""
    body, last = layers[:-1], layers[-1]
    return Sequential(Sequential(*body[:2]), *body[2:], last) if how == "one block" else Sequential(Sequential(Sequential(*body[:2]), *body[2:]), last)


@pytest.mark.parametrize("how", ["one block", "blocks in a block"])
def test_a_vocabulary_behind_blocks_of_layers(how):
    T, V, K = 70, 300, 5
    rng = np.random.default_rng(8)
    x, y = rng.standard_normal((T, 24)).astype(np.float32), rng.integers(0, V, T)
    teacher = (rng.integers(0, V, (T, K)), rng.integers(-100, 101, (T, K)).astype(np.int8), -4)
    net, host = mlp([24, 48, 64], V, 3)
    weighted = net.weighted_layers()
    net.forward_layers = nested(list(net.forward_layers), how)
    assert net.vocab_head() is weighted[-1]
    for _ in range(2):
        before = net.losses(cu(x), cu(y))
        loss = net.train_step(cu(x), cu(y))
        assert torch.equal(before, loss)
        same_loss(loss, oracle_step(host, x, y))
        same_loss(net.train_step(cu(x), (cu(teacher[0]), cu(teacher[1]), teacher[2])), oracle_step(host, x, teacher=teacher))
    for l, (w, _) in zip(weighted, host):
        same(l.weight, w, "weights")
    ops.check_status(DEV)


@pytest.mark.parametrize("how", ["one block", "blocks in a block"])
@pytest.mark.parametrize("fused", [True, False])
def test_a_classifier_behind_blocks_of_layers(how, fused):
    """The same with ten classes, the classifier's one kernel and its several: as with the layers side by side."""
    T = 64
    rng = np.random.default_rng(9)
    x, y = cu(rng.standard_normal((T, 24)).astype(np.float32)), cu(rng.integers(0, 10, T))
    results = []
    old = ti_torch.FUSE_HEAD
    ti_torch.FUSE_HEAD = fused
    try:
        for blocks in (False, True):
            ti_torch.set_seed(5, torch.device(DEV))
            net = TiNet()
            w_rng = np.random.default_rng(10)
            layers = [ti_torch.TiLinear(24, 48), ti_torch.TiReLU(), ti_torch.TiLinear(48, 512), ti_torch.TiReLU(), ti_torch.TiLinear(512, 10, last_layer=True)]
            weighted = [l for l in layers if hasattr(l, "weight")]
            for l in weighted:
                l.weight = cu(w_rng.integers(-100, 101, tuple(l.weight.shape)).astype(np.int8))
            net.forward_layers = nested(layers, how) if blocks else Sequential(*layers)
            for i, l in enumerate(weighted):
                l.layer_id = i
            outs = [net.train_step(x, y)[0].clone() for _ in range(2)]
            results.append(outs + [l.weight for l in weighted])
    finally:
        ti_torch.FUSE_HEAD = old
    for a, b in zip(*results):
        assert torch.equal(a, b)
    ops.check_status(DEV)


def test_random_words_of_a_sample():
    """Stochastic errors are keyed by a row's number in the whole batch, whether the rows come together, as positions of samples or
    one at a time."""
    net, _ = mlp([32], 300, 6)
    head = net.vocab_head()
    head.defer_update = True
    rng = np.random.default_rng(7)
    x, y = cu(rng.integers(-100, 101, (12, 32)).astype(np.int8)), cu(rng.integers(0, 300, 12))
    e = ti_torch.exp_tensor(-7, DEV)
    old = ti_torch.VOCAB_ROUND_METHOD, ti_torch.SAMPLE_OFFSET
    ti_torch.VOCAB_ROUND_METHOD, ti_torch.SAMPLE_OFFSET = ti_torch.StoShift, 0
    try:
        ti_torch.set_seed(21, torch.device(DEV))

        def gradient(offset, x, y):
            ti_torch.SAMPLE_OFFSET = offset
            head.train_step((x, e), y)
            return head.grad_int32acc.clone()
        whole = gradient(0, x, y)
        assert torch.equal(whole, gradient(0, x.view(4, 3, 32), y.view(4, 3)))
        assert torch.equal(whole, gradient(0, x[:6].view(2, 3, 32), y[:6].view(2, 3)) + gradient(2, x[6:].view(2, 3, 32), y[6:].view(2, 3)))
        assert torch.equal(whole, sum(gradient(i, x[i], y[i]) for i in range(12)))
    finally:
        ti_torch.VOCAB_ROUND_METHOD, ti_torch.SAMPLE_OFFSET = old
