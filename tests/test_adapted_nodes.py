"""Nodes whose model is adapted: which engine trains them, and what their checkpoints stand beside."""
import pytest
import torch

from p2pfl_amd.learning.exceptions import ModelNotMatchingError
from p2pfl_amd.learning.pytorch import layers as L
from p2pfl_amd.learning.pytorch.lightninglearner import LightningLearner
from p2pfl_amd.learning.pytorch.mnist.mnist import MNISTDataModule
from p2pfl_amd.learning.pytorch.mnist.models.mlp import MNISTModelMLP


def _learner(model):
    from p2pfl_amd.config.config import Config, default_participant
    p = default_participant()
    p["device_args"]["accelerator"] = "auto"
    return LightningLearner(model, MNISTDataModule(sub_id=0, number_sub=200), config=Config(participant=p))


def test_the_kernel_engine_takes_models_of_its_layout_alone():
    ln = _learner(MNISTModelMLP(seed=1))
    ln.device = torch.device("cuda", 0)
    assert ln._use_engine()
    ln.set_model(L.adapt(MNISTModelMLP(seed=1), rank=2))
    assert not ln._use_engine()                  # its state is adapters, not the layers that the engine's rows hold


@pytest.mark.gpu
def test_an_adapted_model_trains_on_the_gpu():
    ln = _learner(L.adapt(MNISTModelMLP(seed=1), rank=2, p=0.1))
    assert ln.device.type == "cuda"
    ln.set_epochs(1)
    ln.init()
    before = {k: v.detach().cpu().clone() for k, v in ln.get_parameters().items()}
    ln.fit()
    assert ln.evaluate() is not None
    after = ln.get_parameters()
    assert set(after) == set(before) and all(not torch.equal(before[k], after[k].cpu()) for k in before)
