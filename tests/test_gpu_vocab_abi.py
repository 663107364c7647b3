"""The vocabulary losses through the C entry point itself, as a host without torch's allocator calls it."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import vocab_oracle as VO

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from niti_b200 import ops  # noqa: E402
from niti_b200._lib import VocabArgs, lib  # noqa: E402
from tests.test_gpu_vocab import check_train, cu, layer, same_loss, word  # noqa: E402

DEV = "cuda:0"


@pytest.mark.parametrize("offset", [0, 16, 32, 48, 240])
@pytest.mark.parametrize("T,F,V", [(3, 48, 700), (5, 64, 300), (40, 100, 3000), (300, 128, 2000)])
def test_workspace_on_any_16_byte_boundary(T, F, V, offset):
    """A workspace of exactly the bytes that were asked for, at every place that the documentation allows."""
    rng, x, ex, w, ew, y = layer(T + F + V, T, F, V)
    want = VO.vocab(x, ex, w, ew, y)
    xd, exd, wd, ewd, yd = cu(x), word(ex), cu(w), word(ew), cu(y)
    loss = torch.empty(T, dtype=torch.float32, device=DEV)
    e8, exp_err = torch.empty((T, F), dtype=torch.int8, device=DEV), word(0)
    g32, gmax = torch.empty((V, F), dtype=torch.int32, device=DEV), word(0)
    status = ops.status_word(torch.device(DEV))
    for train in (0, 1):
        n = lib.niti_vocab_scratch_bytes(T, F, V, 1, train)
        room = torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=DEV)
        assert room.data_ptr() % 256 == 0
        a = VocabArgs(x=xd.data_ptr(), exp_x=exd.data_ptr(), w=wd.data_ptr(), exp_w=ewd.data_ptr(), index=yd.data_ptr(), ignore_index=-100,
                      loss=loss.data_ptr(), scratch=room.data_ptr() + offset, scratch_bytes=n, T=T, F=F, V=V, entries=1, status=status.data_ptr())
        if train:
            a.e8, a.exp_err, a.g32, a.grad_maxabs = e8.data_ptr(), exp_err.data_ptr(), g32.data_ptr(), gmax.data_ptr()
            a.bits, a.loss_round, a.err_round, a.loss_stream, a.err_stream = 7, ops.ROUND_PSEUDO_STOCHASTIC, ops.ROUND_NEAREST, 0xFFFF, 1
        assert lib.niti_vocab_loss_i8(ctypes.byref(a), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        torch.cuda.synchronize()
        same_loss(loss, want["loss"])
        if train:
            check_train((loss, e8, exp_err, g32, gmax), want)
        r = room.cpu().numpy()
        assert np.all(r[:offset] == 0xA5) and np.all(r[offset + n:] == 0xA5)
