"""What the optimizers queue and launch, on a library that only takes notes (no GPU)."""
from types import SimpleNamespace

import numpy as np
import pytest

import aether
from aether import layers as L


class Tensor:
    """Stands for a DeviceTensor: a shape and an address of its own."""
    made = 0

    def __init__(self, shape, dtype=np.float32):
        Tensor.made += 1
        self.ptr = Tensor.made << 20
        self.shape = tuple(np.atleast_1d(shape))
        self.size = int(np.prod(self.shape))

    def touched(self):
        pass

    def set(self, values):
        self.values = values

    @staticmethod
    def zeros(shape):
        return Tensor(shape)


class Library:
    """Every call's tensors: [(function, [addresses of the updated tensors])].  `refuse`: the call that fails next."""

    def __init__(self):
        self.calls, self.refuse = [], None

    def __getattr__(self, name):
        def call(n, theta, *rest):
            if self.refuse == name:
                self.refuse = None
                return -1
            self.calls.append((name, [int(theta[i]) for i in range(n)]))
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(L, "_L", lambda: lib)
    monkeypatch.setattr(L, "DeviceTensor", Tensor)

    def check(rc):
        if rc:
            raise ValueError("refused")
    monkeypatch.setattr(L, "_ck", check)
    return lib


def _layer(rows=6, cols=5):
    return SimpleNamespace(weights=Tensor((rows, cols)), biases=Tensor((1, cols)), dweights=Tensor((rows, cols)), dbiases=Tensor((1, cols)))


def _step(opt, layers):
    opt.pre_update_parameters()
    for layer in layers:
        opt.update_parameters(layer)
    opt.post_update_parameters()


def _all(layers):
    return sorted(t.ptr for layer in layers for t in (layer.weights, layer.biases))


def _updated(lib):
    return sorted(p for _, tensors in lib.calls for p in tensors)


@pytest.mark.parametrize("make,fails", [(aether.Optimizer_Adam, "aeth_adam_multi_f32"), (aether.Optimizer_Muon, "aeth_adam_multi_f32"),
                                        (aether.Optimizer_Muon, "aeth_muon_multi_f32")])
@pytest.mark.parametrize("count", [3, 20, 40])
def test_a_refused_step_leaves_nothing_queued(library, make, fails, count):
    """The step after it updates every tensor once."""
    opt, layers = make(), [_layer() for _ in range(count)]
    library.refuse = fails
    with pytest.raises(ValueError, match="refused"):
        _step(opt, layers)
    assert opt.iterations == 0
    del library.calls[:]
    _step(opt, layers)
    assert _updated(library) == _all(layers) and opt.iterations == 1


@pytest.mark.parametrize("make", [aether.Optimizer_Adam, aether.Optimizer_Muon])
@pytest.mark.parametrize("what", ["dweights", "dbiases"])
def test_a_wrong_or_missing_gradient_leaves_nothing_queued(library, make, what):
    opt, layers = make(), [_layer() for _ in range(3)]
    good = getattr(layers[2], what)
    setattr(layers[2], what, Tensor((2, 2)))
    with pytest.raises(ValueError, match="gradient shape"):
        _step(opt, layers)
    delattr(layers[2], what)
    with pytest.raises(AttributeError):
        _step(opt, layers)
    setattr(layers[2], what, good)
    del library.calls[:]
    _step(opt, layers)
    assert _updated(library) == _all(layers)


@pytest.mark.parametrize("make", [aether.Optimizer_Adam, aether.Optimizer_Muon])
def test_a_step_broken_off_is_not_mixed_into_the_next(library, make):
    """Updates that were queued (the reference applies them at once) go out before the next step's, in launches of their own."""
    opt, layers = make(), [_layer() for _ in range(3)]
    opt.pre_update_parameters()
    opt.update_parameters(layers[0])
    _step(opt, layers)
    assert _updated(library) == sorted(_all(layers) + _all(layers[:1]))
    assert all(len(set(tensors)) == len(tensors) for _, tensors in library.calls)


def test_a_layer_taken_out_of_muon_keeps_its_bias_moments(library):
    opt, layers = aether.Optimizer_Muon(), [_layer() for _ in range(2)]
    for _ in range(2):
        _step(opt, layers)
    held = layers[0].bias_momentums, layers[0].bias_cache
    layers[0].muon = False
    assert not opt.has_state(layers[0])
    _step(opt, layers)
    assert (layers[0].bias_momentums, layers[0].bias_cache) == held and opt.has_state(layers[0])
    assert layers[0].weight_momentums.shape == layers[0].weight_cache.shape == layers[0].weights.shape
    matrix = layers[0].muon_momentums
    layers[0].muon = True
    _step(opt, layers)
    assert (layers[0].muon_momentums, layers[0].bias_momentums, layers[0].bias_cache) == (matrix,) + held


def test_decay_and_step_number_of_muon_are_adams_too(library):
    """A resumed run sets them on the optimizer; both learning rates follow, in eager steps and in what a recording is checked by."""
    opt, layers = aether.Optimizer_Muon(learning_rate=.1, adam_learning_rate=.01), [_layer()]
    _step(opt, layers)
    assert opt.iterations == opt.adam.iterations == 1 and opt.decay == 0
    before = opt.recorded_settings(layers)
    opt.decay, opt.iterations = .5, 4
    opt.pre_update_parameters()
    assert opt.current_learning_rate == .1 * (1 / 3) and opt.adam.current_learning_rate == .01 * (1 / 3)    # (the formula's roundings)
    after = opt.recorded_settings(layers)
    assert after != before and after[6] != before[6]
    opt.update_parameters(layers[0])
    opt.post_update_parameters()
    assert opt.iterations == opt.adam.iterations == 5
    opt.replayed()
    assert opt.iterations == opt.adam.iterations == 6 and np.isclose(opt.current_learning_rate, .1 / 3.5)
    assert np.isclose(opt.adam.current_learning_rate, .01 / 3.5)
    assert aether.Optimizer_Muon(decay=.25).decay == .25


@pytest.mark.parametrize("make", [aether.Optimizer_Adam, aether.Optimizer_Muon])
def test_a_step_broken_off_goes_out_before_a_replayed_one(library, make):
    """Not with the next eager step, which may come much later."""
    opt, layers = make(), [_layer() for _ in range(3)]
    opt.pre_update_parameters()
    opt.update_parameters(layers[0])
    assert not library.calls
    opt.device_state()                                   # (what a recorded step asks for before its launch)
    assert _updated(library) == _all(layers[:1])
    opt.replayed()
    del library.calls[:]
    _step(opt, layers)
    assert _updated(library) == _all(layers)
