"""Frozen weights, adapters and dropout masks of the nodes of a federation: in the engine that steps all nodes at once and one by
one, over shards, on both devices."""
import copy

import pytest
import torch
import torch.nn as nn

from p2pfl_amd.learning.pytorch import layers as L
from p2pfl_amd.models.torch_models import FederatedModule
from p2pfl_amd.runtime.module_engine import ModuleEngine, ModuleSpec

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


class Small(FederatedModule):
    """A convolution and two linear layers on 1 x 6 x 6 inputs."""

    def __init__(self, seed=None):
        super().__init__(1, 4, 1e-2, seed=seed)
        self.conv = nn.Conv2d(1, 3, 3)
        self.l1, self.l2 = nn.Linear(48, 16), nn.Linear(16, 4)

    def forward(self, x):
        x = torch.relu(self.conv(x.reshape(-1, 1, 6, 6))).flatten(1)
        return self.l2(torch.relu(self.l1(x)))


def engine(factory, device="cpu", batched=True, K=3, n=12, init=True, offset=0, epochs=1, active=None, total=None):
    """An engine that has trained ``epochs`` on data of its nodes among ``total``."""
    eng = ModuleEngine(ModuleSpec("small", factory, 4, (1, 6, 6)), K, device=device, batch_size=4, seed=5, batched=batched,
                       client_offset=offset)
    if init:
        eng.init_params()
    g = torch.Generator().manual_seed(11)
    x, y = torch.randn(total or K, n, 1, 6, 6, generator=g), torch.randint(0, 4, (total or K, n), generator=g)
    x, y = x[offset:offset + K], y[offset:offset + K]
    eng.set_data(x, y, x, y, x, y)
    if epochs:
        eng.fit(epochs, active=active)
    return eng


def close(a, b, steps):
    """Adam steps of 1e-2 from the same start, fp32 sums in another order: an entry whose gradient is all round-off may go either
    way (a step to each side), the others agree."""
    diff = (a.params - b.params).abs()
    assert diff.max() <= steps * 2.1e-2 and diff.mean() < 1e-3


@pytest.fixture(autouse=True)
def _strict(monkeypatch):
    monkeypatch.setenv("P2PFL_MODULE_VMAP_STRICT", "1")


def frozen_head(seed=7):
    m = Small(seed)
    for q in m.conv.parameters():
        q.requires_grad_(False)
    return m


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("batched", [True, False])
def test_frozen_parameters_stay_as_they_were(batched, device):
    eng = engine(frozen_head, device, batched, epochs=2)
    start = frozen_head().state_dict()
    for k in range(eng.K):
        now = eng.get_state_dict(k)
        for name in start:
            assert torch.equal(now[name].cpu(), start[name]) == name.startswith("conv"), name
    assert eng.batched == batched


def adapted(seed=7, p=0.0):
    return L.adapt(Small(seed), rank=2, p=p)


def test_only_adapters_are_state_of_an_adapted_model():
    base = Small(7)
    m = L.adapt(copy.deepcopy(base), rank=2)
    assert sorted(m.state_dict()) == ["l1.a", "l1.b", "l2.a", "l2.b"] == sorted(n for n, _ in m.named_parameters())
    x = torch.randn(3, 36)
    assert torch.equal(m(x), base(x))
    assert torch.equal(m.conv.weight, base.conv.weight) and not m.conv.weight.requires_grad
    again = copy.deepcopy(m)
    again.load_state_dict(m.state_dict())
    assert torch.equal(again(x), m(x))
    m.double()                                                # (buffers follow the module)
    assert m.conv.weight.dtype == torch.float64 == m.l1.weight.dtype


@pytest.mark.parametrize("device", DEVICES)
def test_an_adapted_convolution_network_trains_as_one_by_one(device):
    a, b = engine(adapted, device, True, epochs=2), engine(adapted, device, False, epochs=2)
    assert a.batched and not b.batched
    assert {s.name.split(".")[-1] for s in a.layout.slots} == {"a", "b"}
    start = Small(7)
    for eng in (a, b):
        for m in eng.modules:
            assert torch.equal(m.conv.weight.cpu(), start.conv.weight) and torch.equal(m.l1.weight.cpu(), start.l1.weight)
    close(a, b, 6)
    assert (a.params[0] != a.params[1]).any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("batched", [True, False])
def test_nodes_share_one_frozen_base(batched, device):
    """A factory that sets no seed makes another projection each time; adapters are averaged, so all nodes have the first one's."""
    eng = engine(lambda: adapted(None), device, batched, epochs=0)
    first = eng.modules[0]
    for m in eng.modules[1:]:
        for name, layer in m.named_modules():
            for b in getattr(layer, "frozen_buffers", ()):
                assert layer.get_buffer(b).data_ptr() == first.get_submodule(name).get_buffer(b).data_ptr()
        assert m.l1.weight is first.l1.weight and m.conv.bias is first.conv.bias
    x = torch.randn(2, 36, device=device)
    assert torch.equal(first(x), eng.modules[2](x))


def test_engines_of_two_shards_start_from_the_same_base():
    a, b = engine(lambda: adapted(None), epochs=0), engine(lambda: adapted(None), K=2, offset=3, total=5, epochs=0)
    assert torch.equal(a.modules[0].l1.weight, b.modules[0].l1.weight)
    assert torch.equal(a.modules[0].conv.weight, b.modules[0].conv.weight)


def test_unseeded_adapters_train_as_one_by_one():
    a, b = engine(lambda: adapted(None)), engine(lambda: adapted(None), batched=False)
    close(a, b, 3)


def test_replicas_of_another_base_are_refused():
    widths = iter((16, 16, 8))

    def odd():
        return L.adapt(nn.Sequential(nn.Linear(36, 4), nn.Linear(4, next(widths))), rank=2)
    with pytest.raises(ValueError, match="frozen"):
        engine(odd, epochs=0)


def test_adapters_of_a_model_in_evaluation_do_not_drop():
    m = L.adapt(Small(3).eval(), rank=2, p=0.9)
    with torch.no_grad():
        m.l1.b.normal_(), m.l2.b.normal_()
    x = torch.randn(5, 36)
    assert torch.equal(m(x), m(x)) and not m.l1.training
    m.train()
    assert not torch.equal(m(x), m(x))


def layers_with_dropout(device):
    return nn.Sequential(nn.Conv2d(1, 4, 3), L.GroupNormAct(2, 4, "relu", p=0.3, seed=1), nn.Flatten(), L.CounterDropout(0.3, seed=2),
                         L.AdapterLinear(nn.Linear(64, 5), rank=2, p=0.3, seed=3)).to(device)


@pytest.mark.parametrize("device", DEVICES)
def test_a_training_pass_between_an_evaluation_pass_and_its_gradients(device):
    net = layers_with_dropout(device)
    x = torch.randn(3, 1, 6, 6, device=device, requires_grad=True)
    (want,) = torch.autograd.grad(net.eval()(x).square().sum(), x)
    y = net(x)
    net.train()(x)                                            # moves the counters on
    (got,) = torch.autograd.grad(y.square().sum(), x)
    assert torch.equal(got, want)
    assert all(m.eval()._draw()[1] is not m.step for m in net.modules() if isinstance(m, L._Counted))


class Dropping(FederatedModule):
    """All three layers with dropout; what dropout leaves of ones is kept in ``seen``."""

    def __init__(self):
        super().__init__(1, 4, 1e-2)
        self.conv = nn.Conv2d(1, 4, 3)
        self.norm, self.drop = L.GroupNormAct(2, 4, "relu", p=0.3), L.CounterDropout(0.4)
        self.head = L.AdapterLinear(nn.Linear(64, 4), rank=2, p=0.3)

    def forward(self, x):
        return self.head(self.drop(self.norm(self.conv(x.reshape(-1, 1, 6, 6))).flatten(1)))


def masks_of(eng, steps=1):
    """[K, steps, 64]: what the engine's dropout layer would keep of each node in its next passes, without moving its counters."""
    out = []
    for m in eng.modules:
        d = copy.deepcopy(m.drop).train()
        out.append(torch.stack([d(torch.ones(1, 64, device=eng.device))[0] != 0 for _ in range(steps)]).cpu())
    return torch.stack(out)


@pytest.mark.parametrize("device", DEVICES)
def test_dropout_goes_by_the_node_however_nodes_are_run(device):
    a, b = engine(Dropping, device, True, init=False), engine(Dropping, device, False, init=False)
    assert a.batched and not b.batched
    close(a, b, 3)
    assert torch.equal(masks_of(a, 2), masks_of(b, 2))
    m = masks_of(a)[:, 0]
    assert all(not torch.equal(m[i], m[j]) for i in range(3) for j in range(i))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("batched", [True, False])
def test_dropout_goes_by_the_node_however_nodes_are_split(batched, device):
    """Nodes 0 .. 4 in one engine, and in engines of three and two."""
    whole = engine(Dropping, device, batched, K=5)
    parts = [engine(Dropping, device, batched, K=k, offset=o, total=5) for o, k in ((0, 3), (3, 2))]
    assert torch.equal(masks_of(whole), torch.cat([masks_of(e) for e in parts]))
    for o, e in ((0, parts[0]), (3, parts[1])):
        diff = (whole.params[o:o + e.K] - e.params).abs()      # (the same steps in other batched products: as in close())
        assert diff.max() <= 3 * 2.1e-2 and diff.mean() < 1e-3


@pytest.mark.parametrize("batched", [True, False])
def test_nodes_that_sit_a_fit_out_do_not_change_the_others_masks(batched):
    a, b = engine(Dropping, batched=batched, epochs=0), engine(Dropping, batched=batched, epochs=0)
    a.fit(1, active=torch.tensor([True, False, True]))
    b.fit(1)
    assert torch.equal(masks_of(a), masks_of(b))
    a.fit(1, active=torch.tensor([False, True, False]))
    b.fit(1, active=torch.tensor([True, False, False]))
    assert torch.equal(masks_of(a), masks_of(b))


def vmapped(device, net, x, **state):
    from torch.func import functional_call, vmap
    K = x.shape[0]
    state = {k: v.to(device) for k, v in state.items()}
    return vmap(lambda s, t: functional_call(net, s, (t,)), in_dims=(0, 0), randomness="different")(state, x) if state else \
        vmap(net, randomness="different")(x)


@pytest.mark.parametrize("device", DEVICES)
def test_vmapped_dropout_by_place_and_by_given_seeds(device):
    K, seeds = 4, torch.tensor([[5], [-9], [5], [10 ** 18]])
    x = torch.ones(K, 3, 21, device=device)
    d = L.CounterDropout(0.5, seed=1).to(device)
    by_place = vmapped(device, d, x) != 0
    want = L.keep_mask(1 + torch.arange(K) * L._GOLDEN, torch.zeros(1, dtype=torch.int64), d.site, 63, 0.5).view(x.shape)
    assert torch.equal(by_place.cpu(), want)
    assert torch.equal(by_place[0], L.CounterDropout.forward(_at(d, 0), x[0]) != 0)         # (the first is the layer alone)
    assert len({tuple(m.flatten().tolist()) for m in by_place}) == K
    given = vmapped(device, d, x, seed=seeds) != 0
    want = L.keep_mask(seeds[:, 0], torch.ones(1, dtype=torch.int64), d.site, 63, 0.5).view(x.shape)
    assert torch.equal(given.cpu(), want) and torch.equal(given[0], given[2])


def _at(d, step):
    """A copy of the layer at a step."""
    d = copy.deepcopy(d)
    d.step.fill_(step)
    return d


def test_vmapped_state_with_steps_of_its_own_on_the_cpu():
    d = L.CounterDropout(0.5, seed=1)
    x = torch.ones(3, 40)
    seeds, steps = torch.tensor([[5], [6], [5]]), torch.tensor([[0], [0], [4]])
    want = L.keep_mask(seeds[:, 0], steps[:, 0], d.site, 40, 0.5)
    got = vmapped("cpu", d, x, seed=seeds, step=steps) != 0
    assert torch.equal(got, want) and not torch.equal(got[0], got[2])
    assert steps[:, 0].tolist() == [1, 1, 5]                 # (the pass moves every client's counter on)


@pytest.mark.gpu
def test_vmapped_state_with_steps_of_its_own_is_refused_on_the_gpu():
    from p2pfl_amd.ops.hip import HipKernelError
    net = layers_with_dropout("cuda")
    x = torch.randn(2, 3, 1, 6, 6, device="cuda")
    for i in (1, 3, 4):
        with pytest.raises(HipKernelError, match="share one step"):
            vmapped("cuda", net, x, **{f"{i}.step": torch.zeros(2, 1, dtype=torch.int64)})


@pytest.mark.parametrize("device", DEVICES)
def test_vmapped_layers_of_nodes_are_the_nodes_one_by_one(device):
    """Results and gradients of all layers, with every node's own seed."""
    K = 3
    net = layers_with_dropout(device)
    with torch.no_grad():
        net[4].b.normal_()
    seeds = {f"{i}.seed": torch.tensor([[11], [12], [13]]) * (i + 1) for i in (1, 3, 4)}
    x = torch.randn(K, 5, 1, 6, 6, device=device, requires_grad=True)
    y = vmapped(device, net, x, **seeds)
    (dx,) = torch.autograd.grad(y.square().sum(), x)
    for k in range(K):
        one = copy.deepcopy(net)
        for i in (1, 3, 4):
            one[i].step.zero_()
            one[i].seed.copy_(seeds[f"{i}.seed"][k])
        xk = x[k].detach().clone().requires_grad_()
        yk = one(xk)
        (dk,) = torch.autograd.grad(yk.square().sum(), xk)
        # (fp32 sums of at most 64 terms around one another's order, through three layers)
        assert torch.allclose(yk, y[k], atol=1e-4) and (dk - dx[k]).abs().max() <= 1e-3 * dk.abs().max()


@pytest.mark.gpu
def test_transformed_gradients_are_refused():
    from torch.func import grad, vmap
    x = torch.randn(3, 2, 1, 6, 6, device="cuda")
    layers = [nn.Sequential(L.GroupNormAct(1, 1, "silu")).cuda(), L.CounterDropout(0.3, seed=2).cuda(),
              nn.Sequential(nn.Flatten(), L.AdapterLinear(nn.Linear(36, 5), rank=2)).cuda()]
    for net in layers:
        one = lambda t: net(t).square().sum()
        for call in (lambda: grad(one)(x[0]), lambda: vmap(grad(one), randomness="different")(x),
                     lambda: grad(lambda t: vmap(net, randomness="different")(t).square().sum())(x)):
            # (a dropout's counter is no argument of the transformed function: torch refuses to move it on)
            with pytest.raises(RuntimeError, match="captured Tensor" if isinstance(net, L.CounterDropout) else "autograd's"):
                call()
        t = x.clone().requires_grad_()
        (dx,) = torch.autograd.grad(vmap(net, randomness="different")(t).square().sum(), t)
        assert dx.isfinite().all() and dx.any()


class Normed(FederatedModule):
    def __init__(self):
        super().__init__(1, 4, 1e-2, seed=3)
        self.conv, self.bn, self.norm = nn.Conv2d(1, 4, 3), nn.BatchNorm2d(4), L.GroupNormAct(2, 4, "silu", p=0.2)
        self.head = nn.Linear(64, 4)

    def forward(self, x):
        return self.head(self.norm(self.bn(self.conv(x.reshape(-1, 1, 6, 6)))).flatten(1))


@pytest.mark.parametrize("device", DEVICES)
def test_an_adapted_model_with_norms_trains_as_one_by_one(device):
    make = lambda: L.adapt(Normed(), rank=2, p=0.1)
    a, b = engine(make, device, True), engine(make, device, False)
    assert {s.name for s in a.layout.slots} == {"bn.running_mean", "bn.running_var", "head.a", "head.b"}
    close(a, b, 3)
    assert torch.equal(a.modules[1].norm.weight.cpu(), torch.ones(4)) and a.modules[1].norm.weight is a.modules[0].norm.weight


def test_group_norm_layer_of_16_bit_maps_on_the_cpu():
    m = L.GroupNormAct(2, 4, "gelu")
    x, r = torch.randn(2, 4, 5, 5).bfloat16(), torch.randn(2, 4, 5, 5).bfloat16()
    y = m(x, r)
    want = m(x.float(), r.float())
    assert y.dtype == torch.bfloat16 and torch.allclose(y.float(), want, atol=0.05)
