"""What a network that ends in a vocabulary of classes, or does not, is refused before anything is set up."""
import pytest
import torch


def test_trainer_refuses_the_global_exact_mode():
    from niti_b200 import ti_torch
    from niti_b200.trainer import Trainer

    class Net:
        def vocab_head(self):
            return object()

        def weighted_layers(self):
            raise AssertionError("the trainer went on")
    before = ti_torch.GLOBAL_MAX_GROUP
    with pytest.raises(ValueError, match="global_exact"):
        Trainer(Net(), 4, "cpu", rank=0, world=2, global_exact=True)
    assert ti_torch.GLOBAL_MAX_GROUP is before


def test_losses_of_a_network_without_a_vocabulary():
    from niti_b200.ti_net import TiNet
    net = TiNet()
    net.forward_layers = torch.nn.Sequential(torch.nn.ReLU())
    with pytest.raises(RuntimeError, match="TiVocabHead"):
        net.losses(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
