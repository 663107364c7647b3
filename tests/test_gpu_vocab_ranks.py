"""A convolutional network that ends in a vocabulary of classes, trained by Trainer: one process on the whole batch, and two with
unequal shares of it (gloo on the host; no kernel of one rank waits for one of the other), against oracle replicas whose int32 gradients
are summed before one update."""
import os
import socket

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

from oracle import niti_oracle as O, vocab_oracle as VO
from tests.golden.make_golden import synth_images, xavier_exp

pytestmark = pytest.mark.gpu

CFG = [128, "M", 128, "M", 512, "M"]
FEATURES, CLASSES = 8192, 333
GLOBAL_BATCH, STEPS, SEED = 25, 3, 37


def _data():
    rng = np.random.default_rng(SEED)
    shapes, cin = [], 3
    for c in CFG:
        if c != "M":
            shapes.append((c, 3, 3, cin))
            cin = c
    shapes.append((CLASSES, FEATURES))
    weights = [rng.integers(-127, 128, size=s).astype(np.int8) for s in shapes]
    batches = []
    for _ in range(STEPS):
        y = rng.integers(0, CLASSES, size=GLOBAL_BATCH)
        y[rng.integers(0, GLOBAL_BATCH, 3)] = -100
        batches.append((synth_images(rng, GLOBAL_BATCH), y))
    return shapes, weights, [xavier_exp(s) for s in shapes], batches


class VocabNet(O.Net):
    """oracle.Net with the losses over a vocabulary in place of its classifier."""

    def step(self, x, y, step, sample_offset):
        x8, xe = O.float_to_int8(x)
        self.forward(np.ascontiguousarray(x8.transpose(0, 2, 3, 1)), xe, step=step, sample_offset=sample_offset)
        _, li, a, e = self.trace["saved"].pop()
        r = VO.vocab(a, e, self.w[li], self.w_exp[li], y, err_stream=16 * li + 1, seed=self.seed + step, sample_offset=sample_offset)
        kept, O.ti_loss = O.ti_loss, lambda *_: (r["e8"], r["exp_err"])
        try:
            grads = self.backward(y, step=step, sample_offset=sample_offset, update=False)
        finally:
            O.ti_loss = kept
        grads[li] = r["g32"]
        return r["loss"], r["exp_err"], grads


def _expected(spans):
    shapes, weights, wexps, batches = _data()
    nets = [VocabNet(CFG, weights, wexps, dropout=True, mu=5, seed=SEED, classes=CLASSES) for _ in spans]
    want = {}
    for step, (x, y) in enumerate(batches):
        grads = []
        for net, (lo, hi) in zip(nets, spans):
            loss, exp_err, g = net.step(x[lo:hi], y[lo:hi], step, lo)
            want[(step, lo)] = loss, exp_err
            grads.append(g)
        summed = {i: sum(np.asarray(g[i], dtype=np.int64) for g in grads) for i in range(len(weights))}
        for net in nets:
            net.apply_grads(summed, step=step)
    return want, nets[0].w


def _train(rank, world):
    from niti_b200 import ti_torch, ti_vgg
    from niti_b200.dp import shard_range
    from niti_b200.trainer import Trainer
    shapes, weights, wexps, batches = _data()
    ti_torch.GRAD_BITWIDTH, ti_torch.TRAINING = 5, True
    model = ti_vgg.TiVGG_cifar(list(CFG), dropout=True, fuse_relu=True)
    model.forward_layers[-1] = ti_torch.TiVocabHead(FEATURES, CLASSES)
    model.assign_layer_ids()
    for l, w, e in zip(model.weighted_layers(), weights, wexps):
        l.weight = torch.from_numpy(w).to("cuda:0")
        l.weight_exp = ti_torch.exp_tensor(e, "cuda:0")
    lo, hi = shard_range(GLOBAL_BATCH, rank, world)
    tr = Trainer(model, hi - lo, "cuda:0", rank=rank, world=world, seed=SEED, warmup_steps=1, sample_offset=lo)
    losses = []
    for x, y in batches:
        out, exp = tr.step(torch.from_numpy(x[lo:hi].copy()).pin_memory(), torch.from_numpy(y[lo:hi].copy()).pin_memory())
        tr.sync()
        losses.append((out.numpy().copy(), int(exp)))
    ti_torch.SAMPLE_OFFSET = 0
    return rank, lo, hi, losses, [l.weight.cpu().numpy() for l in model.weighted_layers()]


def _worker(rank, world, port, q):
    import torch.distributed as dist
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        q.put(_train(rank, world))
    finally:
        dist.destroy_process_group()


def _check(results):
    want, weights = _expected([(lo, hi) for _, lo, hi, _, _ in sorted(results, key=lambda r: r[1])])
    for rank, lo, hi, losses, got in results:
        for step, (loss, exp) in enumerate(losses):
            l, e = want[(step, lo)]
            assert np.all(np.abs(loss.astype(np.float64) - l) <= np.abs(l) * 2.0 ** -24 + 1e-11) and exp == e, f"rank {rank} step {step}"
        for i, (a, b) in enumerate(zip(got, weights)):
            assert np.array_equal(a, b), f"rank {rank}: weights of layer {i}"


def test_one_process():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    _check([_train(0, 1)])


def test_two_ranks_with_unequal_shares():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    results = [q.get(timeout=240) for _ in procs]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    _check(results)
