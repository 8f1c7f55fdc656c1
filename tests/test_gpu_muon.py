"""The orthogonalisation, the Muon update and Optimizer_Muon against the formulas in 64 bits (tests/muon_reference.py says
where the tolerances come from)."""
import ctypes as C

import numpy as np
import pytest

from tests import muon_reference as R

pytestmark = pytest.mark.gpu


def _lib():
    from aether import _lib
    return _lib.lib(), _lib.check


def _dev(a):
    from aether import DeviceTensor
    return DeviceTensor.from_numpy(a, np.float32)


def _ortho(g, steps=5):
    from aether import DeviceTensor
    lib, check = _lib()
    gd, o = _dev(g), DeviceTensor.full(g.shape, np.nan)
    check(lib.aeth_newton_schulz_f32(gd.ptr, o.ptr, g.shape[0], g.shape[1], steps))
    return o.get()


def _gradient(r, c, seed=0, strong=8):
    rng = np.random.RandomState(seed + 31 * r + c)
    k = max(1, min(r, c, strong))
    low = (rng.randn(r, k) * 2.0 ** (-np.arange(k) / 2.0)) @ rng.randn(k, c)
    return ((low + rng.randn(r, c)) * 1e-3).astype(np.float32)


def _check(g, steps=5, o=None):
    tol, exact = R.tolerance(g, steps)
    o = _ortho(g, steps) if o is None else o
    assert np.all(np.isfinite(o)), "non-finite values (unwritten output?)"
    off = np.linalg.norm(o - exact)
    assert off <= tol, "off by %.3g, allowed %.3g (norm %.3g)" % (off, tol, np.linalg.norm(exact))


# single rows and columns, both orientations, one less and one more than the tiles and slabs, long thin matrices
SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (2, 3), (5, 4), (15, 17), (16, 16), (27, 32), (31, 33), (32, 32), (33, 31), (48, 20),
          (63, 65), (64, 64), (64, 576), (576, 64), (65, 64), (10, 300), (300, 10), (96, 96), (100, 1000), (127, 129),
          (128, 128), (128, 576), (129, 128), (130, 1030), (160, 161), (191, 193), (192, 192), (255, 257), (256, 256),
          (256, 2048), (2048, 256), (257, 400), (320, 500), (1, 5000), (3, 4097), (4500, 33), (384, 384), (500, 640), (513, 700),
          (640, 512), (1000, 150), (1024, 512), (1025, 1030), (1300, 1100),
          # on both sides of what one workgroup takes, by column blocks a wave
          (32, 256), (20, 257), (20, 520), (1030, 20), (32, 1536), (1537, 32), (31, 1100), (64, 256), (33, 257), (520, 50), (64, 768),
          (768, 33), (64, 769), (769, 64), (61, 700)]


@pytest.mark.parametrize("r,c", SHAPES)
def test_orthogonalisation(r, c):
    g = _gradient(r, c)
    o = _ortho(g)
    _check(g, o=o)
    assert np.array_equal(_ortho(g), o)                    # the same bits again


# every tile of the larger products, ragged: their choice goes by the sizes
@pytest.mark.parametrize("r,c", [(810, 750), (1000, 4100), (1500, 1600), (2112, 2050), (2500, 6001), (3000, 3001), (4100, 3990),
                                 (4095, 4096)])
def test_large_matrices(r, c):
    _check(_gradient(r, c))


@pytest.mark.parametrize("r,tall", [(3, False), (3, True), (260, False), (260, True)])
def test_the_longest_matrices(r, tall):
    """2^21 columns (or rows), the buffers past 2^31 bytes at 260 rows.  n copies of a matrix H beside each other have H's
    left singular vectors and n of the right ones' copies: their result is H's, over sqrt(n), n times.  Sums of K products
    in float32, a rounding for 16 of them: at most 3 K / 16 2^-24 = 2.4 % of a sum for the three parts of a product; a
    singular value's change is the same part of itself or less; an offset that wraps changes all of a result."""
    from aether import DeviceTensor
    lib, check = _lib()
    h = _gradient(r, 4096, seed=9)
    tol, exact = R.tolerance(h)
    n = (1 << 21) // 4096
    g = np.tile(h, (1, n))
    gd = _dev(np.ascontiguousarray(g.T) if tall else g)
    o = DeviceTensor.full(gd.shape, np.nan)
    check(lib.aeth_newton_schulz_f32(gd.ptr, o.ptr, gd.shape[0], gd.shape[1], 5))
    del g
    o = o.get().T if tall else o.get()
    want = (exact / np.sqrt(n)).astype(np.float32)
    off = [np.linalg.norm(o[:, 4096 * k:4096 * (k + 1)] - want) for k in range(n)]
    bound = (tol + 3 * (1 << 21) / 16 * 2.0 ** -24 * np.linalg.norm(exact)) / np.sqrt(n)
    assert max(off) <= bound, (np.argmax(off), max(off), bound)


@pytest.mark.parametrize("steps", [1, 2, 3, 7, 12])
def test_steps(steps):
    for r, c in ((40, 70), (150, 90), (300, 260)):
        _check(_gradient(r, c, seed=1), steps)


@pytest.mark.parametrize("r,c", [(24, 40), (130, 70), (200, 300)])
def test_transposes_and_multiples(r, c):
    """The transposed matrix gives the transposed result; a power of two in front changes no bit, other multiples, up to the
    ends of float32, only the roundings."""
    g = _gradient(r, c, seed=2)
    o = _ortho(g)
    tol, _ = R.tolerance(g)
    assert np.linalg.norm(_ortho(np.ascontiguousarray(g.T)).T - o) <= 2 * tol
    for k in (-60, -3, 5, 90):
        assert np.array_equal(_ortho(g * np.float32(2.0) ** k), o)
    for f in (3e30, 1e-30):
        assert np.linalg.norm(_ortho(g * np.float32(f)) - o) <= 2 * tol
    tiny = (g * np.float32(1e-38)).astype(np.float32)      # denormal numbers: few bits, but a direction
    _check(tiny)


@pytest.mark.parametrize("r,c", [(1, 4), (30, 50), (150, 90), (300, 300)])
def test_zero_and_deficient_matrices(r, c):
    assert np.all(_ortho(np.zeros((r, c), np.float32)) == 0)
    rng = np.random.RandomState(r)
    one = (rng.randn(r, 1) @ rng.randn(1, c)).astype(np.float32)       # rank 1 up to float32
    tol, exact = R.tolerance(one)
    assert np.linalg.norm(_ortho(one) - exact) <= tol
    g = _gradient(r, c, seed=3)
    g[r // 2] = 0
    g[:, c // 3] = 0
    o = _ortho(g)
    _check(g, o=o)
    assert np.all(o[r // 2] == 0) and np.all(o[:, c // 3] == 0)         # products with zeros only
    single = np.zeros((r, c), np.float32)
    single[r - 1, c - 1] = -7.5
    _check(single)
    q = np.linalg.qr(rng.randn(max(r, c), min(r, c)))[0].astype(np.float32)
    _check(q if r >= c else np.ascontiguousarray(q.T))


@pytest.mark.parametrize("r,c", [(4, 6), (150, 90), (300, 300)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_bad_values(r, c, bad):
    g = _gradient(r, c, seed=4)
    g[r - 1, 1] = bad
    assert np.all(np.isnan(_ortho(g)))


def test_views_that_are_only_four_byte_aligned():
    from aether import DeviceTensor
    lib, check = _lib()
    for r, c in ((33, 47), (64, 64), (300, 130)):
        g = _gradient(r, c, seed=5)
        whole, out = np.full(r * c + 8, 5.0, np.float32), DeviceTensor.full(r * c + 8, 5.0)
        whole[3:3 + r * c] = g.reshape(-1)
        gd = _dev(whole)
        check(lib.aeth_newton_schulz_f32(gd.ptr + 12, out.ptr + 12, r, c, 5))
        o = out.get()
        assert np.all(o[:3] == 5) and np.all(o[3 + r * c:] == 5)
        _check(g, o=o[3:3 + r * c].reshape(r, c))


def _multi(tensors, lr=0.02, momentum=0.95, nesterov=1, wd=0.01, steps=5, state=None):
    """One call on [(theta, grad, mom)]; host copies of (theta, mom) afterwards."""
    lib, check = _lib()
    n = len(tensors)
    dev = [[_dev(a) for a in t] for t in tensors]
    table = [(C.c_void_p * n)(*[d[k].ptr for d in dev]) for k in range(3)]
    sizes = [(C.c_int * n)(*[t[0].shape[k] for t in tensors]) for k in range(2)]
    if state is None:
        check(lib.aeth_muon_multi_f32(n, *table, *sizes, lr, momentum, nesterov, wd, steps))
    else:
        check(lib.aeth_muon_multi_dev_f32(n, *table, *sizes, momentum, nesterov, wd, steps, state.ptr))
    for t, d in zip(tensors, dev):
        assert np.array_equal(d[1].get(), t[1])            # the gradients stay
    return [(d[0].get(), d[2].get()) for d in dev]


def _triple(r, c, seed=0):
    rng = np.random.RandomState(seed + r + 7 * c)
    return (0.01 * rng.randn(r, c)).astype(np.float32), _gradient(r, c, seed + 1), 3 * _gradient(r, c, seed + 2)


CNN3 = [(27, 32), (288, 64), (576, 128), (2048, 256)]


@pytest.mark.parametrize("shapes", [[(1, 1)], [(64, 64)], [(256, 10)], [(10, 256)], [(300, 500)], [(1100, 600)], CNN3,
                                    [(64, 64), (64, 64), (64, 64)], [(5, 9), (700, 700), (1, 3), (130, 64), (64, 130)],
                                    [(20 + 3 * i, 90 - 2 * i) for i in range(32)], [(64, 7), (3, 60), (300, 20), (40, 41)],
                                    [(33 + i, 30 + 8 * i) for i in range(32)]])
@pytest.mark.parametrize("nesterov", [0, 1])
def test_update(shapes, nesterov):
    tensors = [_triple(r, c, seed=10 * i) for i, (r, c) in enumerate(shapes)]
    got = _multi(tensors, nesterov=nesterov)
    alone = [_multi([t], nesterov=nesterov)[0] for t in tensors]
    for t, g, a in zip(tensors, got, alone):
        want, m, bound = R.update(*t, 0.02, 0.95, nesterov, 0.01)
        assert np.all(np.abs(g[1] - m) <= R.momentum_bound(t[1], t[2], 0.95))
        assert np.linalg.norm(g[0] - want) <= bound
        # a matrix does not depend on what else is in the call beyond the tolerance of its sums
        assert np.linalg.norm(a[0] - g[0]) <= 2 * bound and np.array_equal(a[1], g[1])
    again = _multi(tensors, nesterov=nesterov)
    assert all(np.array_equal(p[0], q[0]) and np.array_equal(p[1], q[1]) for p, q in zip(got, again))


def test_update_of_large_and_small_matrices_together():
    """Tiles of very different lengths in one launch, both orientations, more than the CUs at once."""
    tensors = [_triple(r, c, seed=r + c + i) for i, (r, c) in enumerate(
        [(500, 1200), (2000, 260), (1024, 3000), (64, 64), (3000, 1024), (700, 700), (1024, 3000), (3, 1), (1500, 1600)])]
    for t, g in zip(tensors, _multi(tensors)):
        want, m, bound = R.update(*t, 0.02, 0.95, 1, 0.01)
        assert np.all(np.abs(g[1] - m) <= R.momentum_bound(t[1], t[2], 0.95))
        assert np.linalg.norm(g[0] - want) <= bound


def test_update_without_momentum_decay_or_gradient():
    theta, grad, mom = _triple(40, 60)
    zero = np.zeros_like(grad)
    (t, m), = _multi([(theta, zero, zero)], wd=0.5, lr=0.1)
    keep = np.float32(1) - np.float32(0.1) * np.float32(0.5)
    assert np.allclose(t, theta * keep, rtol=2.0 ** -22, atol=0) and np.all(m == 0)
    (t, m), = _multi([(theta, grad, mom)], momentum=0.0, wd=0.0)
    want, _, bound = R.update(theta, grad, mom, 0.02, 0.0, 1, 0.0)
    assert np.array_equal(m, grad) and np.linalg.norm(t - want) <= bound
    (t, m), = _multi([(theta, grad, mom)], lr=0.0)
    assert np.array_equal(t, theta)


def test_learning_rate_on_the_device():
    from aether import DeviceTensor
    tensors = [_triple(48, 30), _triple(300, 200)]
    state = DeviceTensor.from_numpy(np.array([3.0, 1.0, 1.0, 0.0137]), np.float64)
    a, b = _multi(tensors, lr=0.0137), _multi(tensors, state=state)
    assert all(np.array_equal(p[0], q[0]) and np.array_equal(p[1], q[1]) for p, q in zip(a, b))


def test_matrices_whose_buffers_go_out_in_groups():
    """Buffers of more than 4 GiB together: one matrix after the other, with the bits of a call for each."""
    cols = 1 << 20
    tensors = []
    for seed in (1, 2):
        theta, grad, mom = _triple(260, 2048, seed)
        tensors.append((np.tile(theta, (1, cols // 2048)), np.tile(grad, (1, cols // 2048)), np.tile(mom, (1, cols // 2048))))
    both = _multi(tensors)
    for t, got in zip(tensors, both):
        want = _multi([t])[0]
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_empty_matrices_are_skipped():
    tensors = [_triple(20, 30)]
    lib, check = _lib()
    dev = [_dev(a) for a in tensors[0]]
    table = [(C.c_void_p * 2)(None, d.ptr) for d in dev]
    check(lib.aeth_muon_multi_f32(2, *table, (C.c_int * 2)(0, 20), (C.c_int * 2)(5, 30), 0.02, 0.95, 1, 0.01, 5))
    want = _multi(tensors)[0]
    assert np.array_equal(dev[0].get(), want[0]) and np.array_equal(dev[2].get(), want[1])
    check(lib.aeth_newton_schulz_f32(None, None, 0, 12, 5))
    check(lib.aeth_newton_schulz_f32(None, None, 12, 0, 5))


def test_recorded_and_replayed():
    """An update in a recording, replayed with eager updates of larger matrices (which replace the workspace) between: every
    replay equals the eager step from the same state bit for bit."""
    lib, check = _lib()
    tensors = [_triple(96, 130), _triple(40, 20)]
    _multi(tensors)
    dev = [[_dev(a) for a in t] for t in tensors]
    table = [(C.c_void_p * 2)(*[d[k].ptr for d in dev]) for k in range(3)]
    sizes = [(C.c_int * 2)(*[t[0].shape[k] for t in tensors]) for k in range(2)]
    check(lib.aeth_graph_begin())
    check(lib.aeth_muon_multi_f32(2, *table, *sizes, 0.02, 0.95, 1, 0.01, 5))
    graph = C.c_void_p()
    check(lib.aeth_graph_end(C.byref(graph)))
    state = tensors
    for k in range(4):
        check(lib.aeth_graph_launch(graph))
        after = [(d[0].get(), d[2].get()) for d in dev]
        want = _multi(state)
        assert all(np.array_equal(a[0], w[0]) and np.array_equal(a[1], w[1]) for a, w in zip(after, want))
        grads = [_gradient(*t[0].shape, seed=50 + k) for t in tensors]
        for d, g in zip(dev, grads):
            d[1].set(g)
        state = [(a[0], g, a[1]) for a, g in zip(after, grads)]
        _multi([_triple(300 * (k + 1), 250)])
    check(lib.aeth_graph_destroy(graph))


# ---- the optimizer ---------------------------------------------------------------------------------------------------
def _network(optimizer, seed=0, norm=True):
    import aether
    np.random.seed(seed)
    model = aether.Model()
    model.add(aether.Conv_Layer((8, 8, 3), num_filters=16))
    if norm:
        model.add(aether.Layer_Norm())
    model.add(aether.ReLU())
    model.add(aether.Pooling())
    model.add(aether.Flatten())
    model.add(aether.Layer_Dense(256, 48, weight_regularizer_l2=1e-4))
    if norm:
        model.add(aether.Layer_Norm())
    model.add(aether.Leaky_ReLU())
    model.add(aether.Layer_Dense(48, 10))
    model.add(aether.SoftMax())
    model.set(loss=aether.Loss_CategoricalCrossEntropy(label_smoothing=0.01), optimizer=optimizer,
              accuracy=aether.Accuracy_Categorical())
    model.finalize()
    model.loss.new_pass()
    model.accuracy.new_pass()
    return model


def _batches(n, rows=16, seed=1):
    r = np.random.RandomState(seed)
    return [(r.randn(rows, 8, 8, 3).astype(np.float32), r.randint(0, 10, rows)) for _ in range(n)]


def _host(model):
    return [np.asarray(a) for layer in model.trainable_layers for a in layer.get_parameters()]


def test_optimizer_steps_follow_the_formulas():
    """Layer norms, a convolution and dense layers under Muon: after every step matrices are where the formula puts them from
    the state and gradients before it; biases, gains and the classifier head where Adam's does."""
    import aether
    from tests import step_checks
    opt = aether.Optimizer_Muon(learning_rate=0.05, decay=0.1, weight_decay=0.02, adam_learning_rate=2e-3)
    model = _network(opt)
    conv, norm1, dense, norm2, head = model.trainable_layers
    for it, (x, y) in enumerate(_batches(4)):
        before = {}
        for l in model.trainable_layers:
            if l.weights is not None:
                before[id(l)] = (l.weights.get(), l.muon_momentums.get() if hasattr(l, "muon_momentums") else None)
        model.train_step(x, y)
        lr, lr_adam = 0.05 / (1 + 0.1 * it), 2e-3 / (1 + 0.1 * it)
        assert opt.iterations == opt.adam.iterations == it + 1 and np.isclose(opt.current_learning_rate, lr)
        assert [opt.takes(l) for l in model.trainable_layers] == [True, False, True, False, False]
        for l in (conv, dense):
            w0, m0 = before[id(l)]
            shape = (-1, w0.shape[-1])
            w0, g = w0.reshape(shape), l.dweights.get().reshape(shape)
            m0 = np.zeros_like(w0) if m0 is None else m0.reshape(shape)
            want, m, bound = R.update(w0, g, m0, lr, 0.95, True, 0.02)
            assert np.all(np.abs(l.muon_momentums.get().reshape(shape) - m) <= R.momentum_bound(g, m0, 0.95))
            assert np.linalg.norm(l.weights.get().reshape(shape) - want) <= bound
            assert not hasattr(l, "weight_cache")
        if it == 0:
            head0 = before[id(head)][0]
            e = step_checks.update_errors(head0, head.dweights.get(), 0 * head0, 0 * head0, head.weights.get(),
                                          head.weight_momentums.get(), head.weight_cache.get(), lr_adam, 0)
            assert max(e) <= 1
            for l in (conv, norm1, dense, norm2, head):
                z = np.zeros(l.biases.shape)
                e = step_checks.update_errors(z, l.dbiases.get(), z, z, l.biases.get(), l.bias_momentums.get(),
                                              l.bias_cache.get(), lr_adam, 0)
                assert max(e) <= 1


@pytest.mark.parametrize("decay", [0.0, 0.05])
def test_recorded_steps_equal_eager_steps(decay):
    """The whole network, norms and optimizer, replayed from a recording: the same bits as eager steps, with evaluations in
    between and batches of another size."""
    import aether
    steps = _batches(6)
    runs = []
    for record in (False, True):
        model = _network(aether.Optimizer_Muon(decay=decay))
        if record:
            model.record_steps(True)
            assert model.recording_active
        seen = []
        for k, (x, y) in enumerate(steps):
            seen.append(model.train_step(x, y)[:3])
            if k == 3:
                model.train_step(x[:5], y[:5])
                model.predict(x[:3])
        runs.append((seen, _host(model), model.optimizer.iterations, model.optimizer.current_learning_rate))
        if record:
            assert any(rec["graph"] for rec in model._recordings.values())
            model.record_steps(False)
    assert runs[0][0] == runs[1][0] and runs[0][2:] == runs[1][2:]
    assert all(np.array_equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))


def test_another_optimizer_makes_a_recording_stale():
    import aether
    steps = _batches(8)
    runs = []
    for record in (False, True):
        model = _network(aether.Optimizer_Adam(), norm=False)
        model.record_steps(record)
        for k, (x, y) in enumerate(steps):
            if k == 3:
                model.set(optimizer=aether.Optimizer_Muon())
            if k == 6:
                model.set(optimizer=aether.Optimizer_Adam(learning_rate=1e-2))
            model.train_step(x, y)
        runs.append(_host(model))
        model.record_steps(False)
    assert all(np.array_equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("change", ["momentum", "nesterov", "ns_steps", "weight_decay", "current_learning_rate", "adam", "muon"])
def test_other_settings_make_a_recording_stale(change):
    import aether
    steps = _batches(6)
    runs = []
    for record in (False, True):
        model = _network(aether.Optimizer_Muon(), norm=False)
        model.record_steps(record)
        for k, (x, y) in enumerate(steps):
            if k == 4:
                if change == "adam":
                    model.optimizer.adam.current_learning_rate = 3e-3
                elif change == "muon":
                    model.trainable_layers[0].muon = False
                else:
                    value = dict(momentum=.5, nesterov=False, ns_steps=3, weight_decay=.1, current_learning_rate=.1)[change]
                    setattr(model.optimizer, change, value)
            model.train_step(x, y)
        runs.append(_host(model))
        model.record_steps(False)
    assert all(np.array_equal(a, b) for a, b in zip(*runs))


def test_which_layers_are_matrices():
    import aether
    model = _network(aether.Optimizer_Muon())
    conv, norm1, dense, norm2, head = model.trainable_layers
    model.forward(_batches(1)[0][0], training=True)
    takes = aether.Optimizer_Muon.takes
    assert takes(conv) and takes(dense) and not takes(head) and not takes(norm1)
    head.muon, dense.muon = True, False
    assert takes(head) and not takes(dense)
    assert not takes(aether.Layer_Dense(1, 9)) and not takes(aether.Layer_Dense(9, 1)) and takes(aether.Layer_Dense(2, 2))


def test_a_shared_layer_is_refused_and_a_wrong_gradient_too():
    import aether
    opt = aether.Optimizer_Muon()
    layer = aether.Layer_Dense(6, 5)
    layer.forward(np.ones((2, 6), np.float32), True)
    layer.backward(np.ones((2, 5), np.float32))
    opt.update_parameters(layer)
    opt.update_parameters(layer)
    with pytest.raises(ValueError, match="overlap"):
        opt.post_update_parameters()
    opt = aether.Optimizer_Muon()
    layer.dweights = aether.DeviceTensor.zeros((6, 4))
    opt.update_parameters(layer)
    with pytest.raises(ValueError, match="gradient shape"):
        opt.post_update_parameters()


def test_training_prints_the_reference_lines_with_muon(capsys):
    import aether
    model = _network(aether.Optimizer_Muon(learning_rate=0.01))
    r = np.random.RandomState(3)
    X, y = r.randn(40, 8, 8, 3).astype(np.float32), r.randint(0, 10, 40)
    model.train(X, y, epochs=2, batch_size=16, print_every=1, validation_data=(X[:8], y[:8]))
    out = capsys.readouterr().out
    assert out.count("epoch: 2, acc:") == 3 and "lr:: 0.01" in out and "Valdiation" in out


def test_parameter_files_with_a_layer_norm(tmp_path):
    import aether
    model, other = _network(aether.Optimizer_Muon()), _network(aether.Optimizer_Muon(), seed=5)
    x, y = _batches(1)[0]
    model.train_step(x, y)
    path = str(tmp_path / "p")
    model.save_parameters(path)
    other.load_parameters(path)
    assert all(np.array_equal(a, b) for a, b in zip(_host(model), _host(other)))
    assert np.array_equal(model.predict(x), other.predict(x))


# ---- many steps ------------------------------------------------------------------------------------------------------
def _weak(r, c, scale, kind, seed=0):
    """A matrix of which a part is `scale` below the rest."""
    g = np.random.RandomState(seed + r + 3 * c).randn(r, c)
    if kind == "block":
        g[:r // 2, c // 2:] = 0
        g[r // 2:, :c // 2] = 0
        g[r // 2:] *= scale
    elif kind == "rows":
        g[r // 2:] *= scale
    elif kind == "columns":
        g[:, c // 2:] *= scale
    else:
        g *= np.logspace(0, np.log10(scale), r)[:, None]
    return g.astype(np.float32)


# on both sides of the steps that the halves carry (9 up to 236 columns, 8 up to 2800, 7 beyond), with one workgroup and with many
@pytest.mark.parametrize("r,c,steps", [(64, 96, 5), (64, 96, 9), (64, 96, 10), (64, 96, 12), (96, 64, 16), (64, 96, 25), (64, 96, 100),
                                       (150, 90, 9), (150, 90, 14), (90, 150, 20), (64, 700, 8), (700, 64, 9), (40, 2900, 7),
                                       (40, 2900, 8), (2900, 40, 14), (300, 260, 8), (300, 260, 20), (2, 3, 30)])
def test_steps_on_matrices_with_weak_parts(r, c, steps):
    """Every step brings a weak part nearer to full size: what was lost of it shows in the end."""
    for kind in ("block", "rows", "columns", "graded"):
        for scale in (1e-4, 1e-8, 1e-9, 1e-10, 1e-12, 1e-20, 1e-30):
            g = _weak(r, c, scale, kind)
            tol, exact = R.tolerance(g, steps)
            off = np.linalg.norm(_ortho(g, steps) - exact)
            assert off <= tol, (kind, scale, off / np.linalg.norm(exact), tol / np.linalg.norm(exact))


@pytest.mark.parametrize("r,c,steps", [(64, 96, 12), (96, 64, 20), (300, 260, 30), (40, 2900, 14), (64, 128, 100)])
def test_weak_rows_alone_after_many_steps(r, c, steps):
    """Row by row (of the shorter side): a float32 sum of products with a weak row is as exact for the row as for a strong one, so
    the worst row is off by what the worst row of a float32 evaluation is, and a factor of 8 for the other order of the sums."""
    for kind in ("block", "rows", "graded"):
        for scale in (1e-6, 1e-9, 1e-12):
            g = _weak(min(r, c), max(r, c), scale, kind, seed=1)
            exact, simple = R.newton_schulz(g, steps), R.newton_schulz(g, steps, np.float32)
            size = np.linalg.norm(exact, axis=1)
            worst = np.max(np.linalg.norm(simple - exact, axis=1) / size)
            o = _ortho(g, steps) if r <= c else _ortho(np.ascontiguousarray(g.T), steps).T
            off = np.max(np.linalg.norm(o - exact, axis=1) / size)
            assert off <= 8 * worst + 2.0 ** -17, (kind, scale, off, worst)


@pytest.mark.parametrize("steps", [9, 30])
def test_update_of_matrices_on_both_kinds_of_products(steps):
    """One call whose matrices need float32 products, or not, by their sizes."""
    shapes = [(20, 30), (5, 3000), (300, 500), (2000, 33), (64, 64), (1, 1), (129, 70), (230, 236), (230, 237)]
    tensors = [_triple(r, c, seed=10 * i) for i, (r, c) in enumerate(shapes)]
    got = _multi(tensors, steps=steps)
    for t, g in zip(tensors, got):
        want, m, bound = R.update(*t, 0.02, 0.95, 1, 0.01, steps)
        assert np.all(np.abs(g[1] - m) <= R.momentum_bound(t[1], t[2], 0.95))
        assert np.linalg.norm(g[0] - want) <= bound
    assert all(np.array_equal(p[0], q[0]) and np.array_equal(p[1], q[1]) for p, q in zip(got, _multi(tensors, steps=steps)))


@pytest.mark.parametrize("r,c", [(4, 6), (150, 90), (1, 500)])
def test_values_at_the_edge_with_many_steps(r, c):
    assert np.all(_ortho(np.zeros((r, c), np.float32), 20) == 0)
    for bad in (np.nan, np.inf):
        g = _gradient(r, c, seed=4)
        g[r - 1, 1] = bad
        assert np.all(np.isnan(_ortho(g, 20)))
    g = _gradient(r, c, seed=2)
    o = _ortho(g, 20)
    for k in (-60, 90):
        assert np.array_equal(_ortho(g * np.float32(2.0) ** k, 20), o)
    if min(r, c) > 1:
        g[r // 2] = 0
        o = _ortho(g, 20)
        _check(g, 20, o)
        assert np.all(o[r // 2] == 0)


def test_many_steps_of_a_long_row():
    """2^21 columns: the norm of a single row goes to p(p(...p(1))), every element its part of it."""
    g = np.tile(_gradient(1, 4096, seed=7), (1, 512))
    exact = R.newton_schulz(g, 6)
    # a sum of squares in float32, 2^9 pairs in line and 2^11 totals: off by at most e = (2^9 + 2^11) 2^-24 of itself.  A step's result
    # moves by |b A + 2 c A^2| s e, at most 1.1 e on [0.68, 1.2], and the slope of p along this orbit (1, 0.70, 1.11, 0.70, ...) is at
    # most 1.5 over two steps, 3.4 over six: at most 6 * 1.1 * 3.4 = 22 e
    assert np.linalg.norm(_ortho(g, 6) - exact) <= 22 * (2 ** 9 + 2 ** 11) * 2.0 ** -24 * np.linalg.norm(exact)


def test_more_steps_in_the_middle_of_recorded_training():
    """The float32 products need a workspace of their own, which has to be there before a step is recorded with them."""
    import aether
    steps = _batches(9)
    runs = []
    for record in (False, True):
        model = _network(aether.Optimizer_Muon(), norm=False)
        model.record_steps(record)
        for k, (x, y) in enumerate(steps):
            if k == 3:
                model.train_step(x[:6], y[:6])               # (a second shape, recorded only after the change)
                model.optimizer.ns_steps = 30
            model.train_step(x, y)
            if k == 5:
                model.train_step(x[:6], y[:6])
        runs.append(_host(model))
        model.record_steps(False)
    assert all(np.array_equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("muon", [False, True])
@pytest.mark.parametrize("change", [dict(beta_1=.5), dict(beta_2=.9), dict(epsilon=1e-3), dict(beta_1=.7, beta_2=.99)])
def test_other_betas_make_a_recording_stale(muon, change):
    """The betas are in a recording twice: in its kernels and, to the power of the step number, in the state on the device."""
    import aether
    steps = _batches(7)
    runs = []
    for record in (False, True):
        model = _network(aether.Optimizer_Muon() if muon else aether.Optimizer_Adam(), norm=False)
        model.record_steps(record)
        for k, (x, y) in enumerate(steps):
            if k == 4:
                for name, value in change.items():
                    setattr(model.optimizer.adam if muon else model.optimizer, name, value)
            model.train_step(x, y)
        if record:
            assert any(rec["graph"] for rec in model._recordings.values())
        runs.append(_host(model))
        model.record_steps(False)
    assert all(np.array_equal(a, b) for a, b in zip(*runs))


def test_the_state_on_the_device_follows_the_betas():
    """Between two replays, without a step that would move the step number."""
    import aether
    opt = aether.Optimizer_Adam()
    opt.iterations = 3
    for b1, b2 in ((.9, .999), (.5, .999), (.5, .75)):
        opt.beta_1, opt.beta_2 = b1, b2
        want = [3, float(np.float32(b1)) ** 3, float(np.float32(b2)) ** 3, opt.current_learning_rate]
        assert np.array_equal(opt.device_state().get(), np.array(want))


@pytest.mark.parametrize("muon", [False, True])
def test_moments_made_anew_make_every_recording_stale(muon):
    """Two batch shapes are recorded, then training starts over with fresh moments: the step that makes them runs normally, and the
    other shape's recording, which knows the old ones, may not be replayed."""
    import aether
    steps = _batches(8)
    runs = []
    for record in (False, True):
        model = _network(aether.Optimizer_Muon() if muon else aether.Optimizer_Adam(), norm=False)
        model.record_steps(record)
        for k, (x, y) in enumerate(steps):
            if k == 4:
                if record:
                    assert len([rec for rec in model._recordings.values() if rec["graph"]]) == 2
                for layer in model.trainable_layers:
                    for name in ("weight_momentums", "weight_cache", "bias_momentums", "bias_cache", "muon_momentums"):
                        if hasattr(layer, name):
                            delattr(layer, name)
            model.train_step(x, y)
            model.train_step(x[:7], y[:7])
            if k == 5:                                   # other moments in place of those that are there
                for layer in model.trainable_layers:
                    layer.bias_cache = aether.DeviceTensor.full(layer.biases.shape, 1e-3)
        runs.append((_host(model), [layer.bias_momentums.get() for layer in model.trainable_layers]))
        model.record_steps(False)
    for a, b in zip(*runs):
        assert all(np.array_equal(p, q) for p, q in zip(a, b))


def test_a_layer_taken_out_of_muon_goes_on_with_its_bias():
    """The step after it moves the bias by Adam's formula from the moments that it had."""
    import aether
    from tests import step_checks
    opt = aether.Optimizer_Muon(adam_learning_rate=2e-3)
    model = _network(opt, norm=False)
    steps = _batches(4)
    for x, y in steps[:3]:
        model.train_step(x, y)
    layer = model.trainable_layers[1]
    layer.muon = False
    before = [t.get() for t in (layer.biases, layer.bias_momentums, layer.bias_cache)]
    assert np.any(before[2] != 0)
    model.train_step(*steps[3])
    e = step_checks.update_errors(before[0], layer.dbiases.get(), before[1], before[2], layer.biases.get(),
                                  layer.bias_momentums.get(), layer.bias_cache.get(), 2e-3, 3)
    assert max(e) <= 1


def test_a_resumed_run_in_recorded_training():
    """The step number and the decay set in the middle: replays and eager steps go on alike, both learning rates lowered."""
    import aether
    steps = _batches(8)
    runs = []
    for record in (False, True):
        model = _network(aether.Optimizer_Muon(), norm=False)
        model.record_steps(record)
        for k, (x, y) in enumerate(steps):
            if k == 3:
                model.optimizer.iterations = 50
            if k == 5:
                model.optimizer.decay = .1
            model.train_step(x, y)
        assert model.optimizer.iterations == model.optimizer.adam.iterations == 55
        assert np.isclose(model.optimizer.adam.current_learning_rate, 1e-3 / (1 + .1 * 54))
        runs.append(_host(model))
        model.record_steps(False)
    assert all(np.array_equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("steps", [5, 9])
def test_a_call_that_cannot_have_its_scratch_changes_nothing(steps):
    """Two matrices that go out one after the other, with a workspace for the first: a recording refuses one that grows, and what it
    recorded of the call must be nothing.  (9 steps: both on float32 products.)  In a process of its own, whose workspace is small."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import ctypes as C, sys
sys.path[:0] = [%r, %r]
import numpy as np
from aether import DeviceTensor, _lib
lib, check = _lib.lib(), _lib.check
steps = %d
shapes = [(64, 1 << 20), (16000, 16000)]
t = [[DeviceTensor.full(s, 0.5 + k) for k in range(3)] for s in shapes]

def call(n):
    table = [(C.c_void_p * n)(*[m[k].ptr for m in t[:n]]) for k in range(3)]
    return lib.aeth_muon_multi_f32(n, *table, (C.c_int * n)(*[s[0] for s in shapes[:n]]), (C.c_int * n)(*[s[1] for s in shapes[:n]]),
                                   0.02, 0.95, 1, 0.01, steps)

check(call(1))
before = [m[k][:4].get() for m in t for k in range(3)]
check(lib.aeth_graph_begin())
rc = call(2)
graph = C.c_void_p()
check(lib.aeth_graph_end(C.byref(graph)))
assert rc == -4 and "grow" in lib.aeth_last_error().decode(), rc
check(lib.aeth_graph_launch(graph))
assert all(np.array_equal(a, b) for a, b in zip(before, [m[k][:4].get() for m in t for k in range(3)]))
check(lib.aeth_graph_destroy(graph))
check(call(2))
assert not np.array_equal(before[0], t[0][0][:4].get())
print("done")
""" % (root, os.path.join(root, "aether-ml_amd"), steps)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stderr[-2000:]
