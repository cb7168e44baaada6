"""ExpertMLP.decode describes its weights once for all calls: what it keeps between them,
and what makes it describe them anew. No device work."""

from __future__ import annotations

import copy
import pickle
import weakref

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import linear
from mlx_gptq.experts import ExpertMLP

BF, I32 = torch.bfloat16, torch.int32
CPU = torch.device("cpu")


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    """The launches' arguments; host tensors pass as the device's."""
    made = []
    monkeypatch.setattr(linear, "_device", lambda *tensors: CPU)
    monkeypatch.setattr(nat, "launch", lambda dev, name, *args: made.append((name, *args)))
    return made


def weight(n, k, mode, E=4, bits=4):
    if mode == "dense":
        return torch.zeros(E, n, k, dtype=BF)
    packed = torch.zeros(E, n, k * bits // 32, dtype=I32)
    if mode == "affine":
        return [packed, *(torch.zeros(E, n, k // 32, dtype=BF) for _ in range(2))]
    return [packed, torch.zeros(E, n, k // 32, dtype=torch.uint8)]


def layer_of(mode, H=64, I=32):
    return ExpertMLP(weight(2 * I, H, mode), weight(H, I, mode), mode)


def decode(layer, T=3, H=64):
    return layer.decode(torch.zeros(T, H, dtype=BF), torch.zeros(T, 2, dtype=torch.int64),
                        torch.zeros(T, 2))


@pytest.mark.parametrize("mode,place", [("mxfp4", 0), ("mxfp4", 1), ("affine", 0), ("affine", 1),
                                        ("affine", 2)])
@pytest.mark.parametrize("which", ["gate_up", "down"])
def test_a_tensor_replaced_in_a_list_is_seen(mode, place, which):
    layer = layer_of(mode)
    first = layer._decode_weights(64, BF, CPU)
    assert layer._decode_weights(64, BF, CPU) is first
    weights = getattr(layer, which)
    weights[place] = weights[place].clone()
    again = layer._decode_weights(64, BF, CPU)
    assert again is not first
    described = again.up if which == "gate_up" else again.down
    assert (described.data, described.scales, described.biases)[place] == weights[place].data_ptr()
    assert layer._decode_weights(64, BF, CPU) is again


def test_calls_at_once_take_their_own_description(monkeypatch):
    """Two threads: while one stores its description, the other stores one of other rows."""

    class Shared(ExpertMLP):
        other = None

        def __setattr__(self, name, value):
            super().__setattr__(name, value)
            if name == "_described" and value is not None and self.other is not None:
                super().__setattr__(name, self.other)

    layer = Shared(weight(64, 64, "dense"), weight(64, 32, "dense"))
    other = layer._decode_weights(64, BF, CPU)
    layer.gate_up, layer.down = weight(64, 64, "dense"), weight(64, 32, "dense")
    layer.other = other
    passed = []
    monkeypatch.setattr(nat, "launch", lambda dev, name, *args: passed.append(
        (nat.Weight.from_address(args[11]).data, nat.Weight.from_address(args[12]).data)))
    decode(layer)
    assert passed == [(layer.gate_up.data_ptr(), layer.down.data_ptr())]


@pytest.mark.parametrize("mode", ["dense", "mxfp4", "affine"])
def test_copies_go_with_their_call(mode, launches, monkeypatch):
    """Weights that had to be copied: no copy outlives its call."""
    layer = layer_of(mode)
    turned = layer.gate_up if mode == "dense" else layer.gate_up[0]
    turned = turned.transpose(1, 2).contiguous().transpose(1, 2)
    layer.gate_up = turned if mode == "dense" else [turned, *layer.gate_up[1:]]
    copies = []
    contiguous = torch.Tensor.contiguous

    def contiguous_seen(t):
        out = contiguous(t)
        if out is not t:
            copies.append(weakref.ref(out))
        return out

    monkeypatch.setattr(torch.Tensor, "contiguous", contiguous_seen)
    for calls in (1, 2):
        decode(layer)
        assert len(launches) == len(copies) == calls
        assert all(c() is None for c in copies)


@pytest.mark.parametrize("mode", ["dense", "mxfp4", "affine"])
def test_a_replaced_weight_is_let_go(mode):
    layer = layer_of(mode)
    decode(layer)
    old = weakref.ref(layer.gate_up if mode == "dense" else layer.gate_up[0])
    layer.gate_up = weight(64, 64, mode)
    assert old() is None
    decode(layer)


@pytest.mark.parametrize("mode", ["dense", "mxfp4", "affine"])
@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda layer: pickle.loads(pickle.dumps(layer))],
                         ids=["copy", "deepcopy", "pickle"])
def test_a_layer_that_has_decoded_can_be_copied(mode, how, launches):
    layer = layer_of(mode)
    decode(layer)
    twin = how(layer)
    assert (twin.mode, twin.num_experts) == (mode, 4)
    decode(twin)
    own = twin.gate_up if mode == "dense" else twin.gate_up[0]
    assert nat.Weight.from_address(launches[1][12]).data == own.data_ptr()
    decode(layer)
    assert launches[2][12] == launches[0][12]


@pytest.mark.parametrize("mode", ["dense", "mxfp4", "affine"])
def test_a_call_holds_its_weights_until_they_are_launched(mode, monkeypatch):
    """Another thread replaces the layer's weights once they are described."""

    class Replaced(ExpertMLP):
        def __setattr__(self, name, value):
            super().__setattr__(name, value)
            if name == "_described" and value is not None:
                self.gate_up, self.down = weight(64, 64, self.mode), weight(64, 32, self.mode)

    layer = Replaced(weight(64, 64, mode), weight(64, 32, mode), mode)
    given = [t for w in (layer.gate_up, layer.down) for t in ([w] if mode == "dense" else w)]
    pointers, alive = [t.data_ptr() for t in given], [weakref.ref(t) for t in given]
    del given
    seen = []

    def launch(dev, name, *args):
        parts = [nat.Weight.from_address(a) for a in args[11:13]]
        seen.extend(p for w in parts for p in (w.data, w.scales, w.biases) if p)
        seen.append(all(ref() is not None for ref in alive))

    monkeypatch.setattr(nat, "launch", launch)
    decode(layer)
    assert seen == [*pointers, True]
    assert all(ref() is None for ref in alive)
