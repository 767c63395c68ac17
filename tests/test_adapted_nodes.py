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


def _node(idx, model):
    from p2pfl_amd.config import Config
    from p2pfl_amd.node import Node
    c = Config(participant={"scenario_args": {"federation": "DFL", "n_nodes": 2, "name": "", "controller": ""},
                            "device_args": {"role": "aggregator", "idx": idx, "accelerator": "cpu"},
                            "tracking_args": {"local_tracking": "none", "log_dir": ""}})
    return Node(idx, "test", model, MNISTDataModule(sub_id=idx, number_sub=200), config=c)


def test_a_checkpoint_of_adapters_stands_beside_its_base(tmp_path):
    """Adapters of another base are a model that nobody trained: a checkpoint names its base and is refused beside another."""
    make = lambda seed: L.adapt(MNISTModelMLP(seed=seed), rank=2)
    nodes = [_node(i, m) for i, m in enumerate((make(1), make(1), make(2), MNISTModelMLP(seed=1)))]
    try:
        with torch.no_grad():
            nodes[0].learner.model.l1.b.normal_()
        path = str(tmp_path / "a.ckpt")
        nodes[0].save_checkpoint(path)
        assert nodes[1].load_checkpoint(path)["base"]
        assert torch.equal(nodes[1].learner.model.l1.b, nodes[0].learner.model.l1.b)
        before = nodes[2].learner.model.l1.b.clone()
        with pytest.raises(ModelNotMatchingError, match="base"):
            nodes[2].load_checkpoint(path)
        assert torch.equal(nodes[2].learner.model.l1.b, before)
        plain = str(tmp_path / "b.ckpt")
        nodes[3].save_checkpoint(plain)
        assert nodes[3].load_checkpoint(plain)["node"] and "base" not in nodes[3].load_checkpoint(plain)
    finally:
        for n in nodes:
            n.stop()


def test_the_kernel_engine_leaves_models_with_frozen_parameters_to_autograd():
    """It trains every row of its slab."""
    m = MNISTModelMLP(seed=1)
    m.l1.weight.requires_grad_(False)
    ln = _learner(m)
    ln.device = torch.device("cuda", 0)
    assert not ln._use_engine()
    m.l1.weight.requires_grad_(True)
    assert ln._use_engine()


@pytest.mark.gpu
def test_frozen_parameters_of_a_node_stay_on_the_gpu():
    m = MNISTModelMLP(seed=1)
    m.l1.weight.requires_grad_(False)
    start = {k: v.detach().clone() for k, v in m.state_dict().items()}
    ln = _learner(m)
    ln.set_epochs(1)
    ln.init()
    ln.fit()
    after = ln.get_parameters()
    assert {k for k in start if torch.equal(start[k], after[k].cpu())} == {"l1.weight"}
