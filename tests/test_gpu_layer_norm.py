"""Layer_Norm and the aeth_ln_* entry points against the formulas in 64 bits (tests/norm_reference.py derives the
tolerances), against differences, at the sizes, alignments and values where they can go wrong."""
import ctypes as C

import numpy as np
import pytest

from oracle import oracle as O
from tests import norm_reference as R

pytestmark = pytest.mark.gpu


def _dev(a):
    from aether import DeviceTensor
    return DeviceTensor.from_numpy(a, np.float32)


def _nan(shape, dtype=np.float32):
    from aether import DeviceTensor
    t = DeviceTensor(shape, dtype)
    return t.set(np.full(shape, np.nan if dtype == np.float32 else 0x7fff, dtype))


def _lib():
    from aether import _lib
    return _lib.lib(), _lib.check


def _forward(x, gamma, beta, eps=1e-5, saves=True, twin=False):
    lib, check = _lib()
    rows, c = x.shape
    y, m, s = _nan((rows, c)), _nan(rows), _nan(rows)
    xd, gd, bd = _dev(x), _dev(gamma), _dev(beta)
    head = (xd.ptr, gd.ptr, bd.ptr, m.ptr if saves else None, s.ptr if saves else None, y.ptr)
    y16 = _nan((rows, c), np.uint16) if twin else None
    if twin:
        check(lib.aeth_ln_fwd_twin_f32(*head, y16.ptr, rows, c, eps))
    else:
        check(lib.aeth_ln_fwd_f32(*head, rows, c, eps))
    return y.get(), m.get(), s.get(), y16.get() if twin else None


def _backward(x, dy, gamma, mean, invstd, twin=False):
    lib, check = _lib()
    rows, c = x.shape
    dx, dg, db = _nan((rows, c)), _nan(c), _nan(c)
    t = [_dev(a) for a in (x, dy, gamma, mean, invstd)]
    head = tuple(a.ptr for a in t) + (dx.ptr,)
    dx16 = _nan((rows, c), np.uint16) if twin else None
    if twin:
        check(lib.aeth_ln_bwd_twin_f32(*head, dx16.ptr, dg.ptr, db.ptr, rows, c))
    else:
        check(lib.aeth_ln_bwd_f32(*head, dg.ptr, db.ptr, rows, c))
    return dx.get(), dg.get(), db.get(), dx16.get() if twin else None


def _inputs(rows, c, seed=0):
    r = np.random.RandomState(seed + 7 * rows + c)
    x = (r.randn(rows, c) * (0.5 + r.rand(c)) + r.randn(c)).astype(np.float32)
    return x, (1 + 0.2 * r.randn(c)).astype(np.float32), r.randn(c).astype(np.float32), r.randn(rows, c).astype(np.float32)


# rows x features: one of each, row lengths on both sides of every power of two that a kernel could switch at, rows that
# no vector divides, rows longer than a workgroup's registers, many short rows
SIZES = [(1, 1), (1, 4), (5, 1), (3, 2), (7, 3), (1, 256), (128, 256), (2, 15), (2, 16), (9, 17), (33, 31), (64, 32), (65, 33),
         (31, 60), (130, 63), (257, 64), (17, 65), (19, 100), (5, 127), (66, 128), (5, 129), (12, 252), (3, 255), (3, 257),
         (7, 260), (4, 511), (6, 512), (3, 513), (5, 1000), (2, 1023), (9, 1024), (3, 1025), (2, 1537), (6, 2048), (3, 2049),
         (2, 4095), (5, 4096), (2, 4100), (2, 5001), (3, 8192), (2, 8193), (2, 8196), (2, 16384), (1, 16385), (3, 20000),
         (1, 32768), (2, 32769), (1, 40004), (1, 70001), (3, 100000), (1000, 8), (2000, 5), (1500, 64), (1030, 100), (700, 1024),
         # on both sides of the rows that the backward pass takes in one launch, every width above it
         (512, 256), (513, 256), (513, 1), (600, 3), (530, 15), (777, 33), (640, 60), (520, 129), (530, 513), (521, 1023), (514, 1025),
         # every width of a row, one launch and two
         (2, 30), (2, 40), (600, 40), (3, 90), (600, 90), (4, 190), (600, 190), (3, 380), (520, 380), (520, 700), (520, 1250), (2, 1500),
         (2, 1700), (2, 1900), (520, 1900), (2, 2300), (260, 2300), (2, 2500), (260, 2500), (2, 5000), (260, 6100), (2, 9000), (260, 9000),
         (2, 12000), (260, 12000), (2, 15000), (260, 15000), (2, 17000), (260, 18000), (2, 19000), (2, 21504), (260, 21500), (2, 25000),
         (2, 30000), (2, 23040), (600, 500), (600, 30), (600, 1500),
         (600, 1537), (513, 2048), (256, 2052), (257, 2052), (300, 4100), (258, 8193), (270, 16385), (257, 20000)]


@pytest.mark.parametrize("rows,c", SIZES)
def test_forward_and_backward(rows, c):
    x, gamma, beta, dy = _inputs(rows, c)
    (y, mean, inv), (e_y, e_mean, e_inv) = R.forward(x, gamma, beta, 1e-5)
    got = _forward(x, gamma, beta)
    assert R.worst(got[0], y, e_y) <= 1 and R.worst(got[1], mean, e_mean) <= 1 and R.worst(got[2], inv, e_inv) <= 1
    # without statistics the output has the same bits
    assert np.array_equal(_forward(x, gamma, beta, saves=False)[0], got[0])
    want, bounds = R.backward(x, dy, gamma, got[1], got[2])
    back = _backward(x, dy, gamma, got[1], got[2])
    for g, w, b, name in zip(back, want, bounds, ("dx", "dgamma", "dbeta")):
        assert R.worst(g, w, b) <= 1, name
    # the same call again gives the same bits
    again = _backward(x, dy, gamma, got[1], got[2])
    assert all(np.array_equal(a, b) for a, b in zip(again[:3], back[:3]))


@pytest.mark.parametrize("rows,c", [(1, 1), (5, 3), (129, 64), (7, 100), (3, 1025), (40, 1024), (2, 20000), (1, 40001), (600, 100), (600, 3),
                                    (300, 2500)])
def test_twins_are_the_rounded_outputs(rows, c):
    x, gamma, beta, dy = _inputs(rows, c, seed=1)
    plain, twin = _forward(x, gamma, beta), _forward(x, gamma, beta, twin=True)
    assert np.array_equal(plain[0], twin[0]) and np.array_equal(twin[3], O.bf16_bits(twin[0]))
    a, b = _backward(x, dy, gamma, plain[1], plain[2]), _backward(x, dy, gamma, plain[1], plain[2], twin=True)
    assert all(np.array_equal(p, q) for p, q in zip(a[:3], b[:3])) and np.array_equal(b[3], O.bf16_bits(b[0]))


@pytest.mark.parametrize("rows,c,skip", [(6, 64, 1), (6, 100, 2), (5, 1024, 3), (3, 4096, 1), (2, 20000, 3), (520, 100, 2), (520, 1023, 3),
                                         (260, 4099, 1)])
def test_pointers_that_are_only_four_byte_aligned(rows, c, skip):
    """Views that start `skip` floats into a block: no 16-byte load is aligned, the results are those of aligned ones within
    the tolerance, and the floats in front of and behind the outputs stay."""
    lib, check = _lib()
    x, gamma, beta, dy = _inputs(rows, c, seed=2)

    def shifted(a):
        whole = np.full(a.size + 8, 123.0, np.float32)
        whole[skip:skip + a.size] = a.reshape(-1)
        return _dev(whole)

    t = {k: shifted(v) for k, v in (("x", x), ("gamma", gamma), ("beta", beta), ("dy", dy))}
    out = {k: shifted(np.zeros(n, np.float32)) for k, n in (("y", rows * c), ("dx", rows * c), ("m", rows), ("s", rows),
                                                             ("dg", c), ("db", c))}
    at = lambda d, *names: [d[k].ptr + 4 * skip for k in names]  # noqa: E731
    check(lib.aeth_ln_fwd_f32(*at(t, "x", "gamma", "beta"), *at(out, "m", "s", "y"), rows, c, 1e-5))
    check(lib.aeth_ln_bwd_f32(*at(t, "x", "dy", "gamma"), *at(out, "m", "s", "dx", "dg", "db"), rows, c))
    got = {k: v.get() for k, v in out.items()}
    for k, v in got.items():
        n = v.size - 8
        assert np.all(v[:skip] == 123.0) and np.all(v[skip + n:] == 123.0), k
        got[k] = v[skip:skip + n]
    (y, mean, inv), (e_y, e_mean, e_inv) = R.forward(x, gamma, beta, 1e-5)
    assert R.worst(got["y"], y, e_y) <= 1 and R.worst(got["m"], mean, e_mean) <= 1 and R.worst(got["s"], inv, e_inv) <= 1
    want, bounds = R.backward(x, dy, gamma, got["m"], got["s"])
    for k, w, b in zip(("dx", "dg", "db"), want, bounds):
        assert R.worst(got[k], w, b) <= 1, k


@pytest.mark.parametrize("c", [48, 1000, 40000])
def test_rows_far_from_zero_and_constant_rows(c):
    """A mean a thousand times the spread costs what the inputs' own rounding costs and no more; a constant row has
    variance 0 and gives beta."""
    r = np.random.RandomState(c)
    x = (1000 + r.randn(4, c)).astype(np.float32)
    x[2] = 0.1
    x[3] = 0.0
    gamma, beta = np.ones(c, np.float32), r.randn(c).astype(np.float32)
    (y, _, _), (e_y, _, _) = R.forward(x, gamma, beta, 1e-5)
    got = _forward(x, gamma, beta)[0]
    assert R.worst(got[:2], y[:2], e_y[:2]) <= 1 and R.worst(got[2], y[2], e_y[2]) <= 1
    assert np.array_equal(got[3], beta)


@pytest.mark.parametrize("rows,c", [(6, 3), (6, 64), (6, 1024), (6, 33000), (530, 3), (530, 64), (530, 1024), (270, 4000)])
def test_bad_values_stay_in_their_row(rows, c):
    x, gamma, beta, dy = _inputs(rows, c, seed=3)
    clean = _forward(x, gamma, beta)
    x[1, c // 2], x[4, 0] = np.nan, np.inf
    got = _forward(x, gamma, beta)
    keep = [r for r in range(rows) if r not in (1, 4)]
    assert np.array_equal(got[0][keep], clean[0][keep])
    assert np.all(np.isnan(got[0][[1, 4]]))
    dx, dg, db, _ = _backward(x, dy, gamma, got[1], got[2])
    x0, _, _, _ = _inputs(rows, c, seed=3)
    want = _backward(x0, dy, gamma, clean[1], clean[2])
    assert np.array_equal(dx[keep], want[0][keep]) and np.all(np.isnan(dx[[1, 4]]))
    assert np.all(np.isnan(dg)) and np.array_equal(db, want[2])


def test_a_row_of_more_columns_than_a_launch_has_threads_for():
    c = (1 << 26) + 77
    x, dy = (np.resize(a, (1, c)) for a in _inputs(1, 1 << 18)[::3])
    gamma, beta = (np.resize(a, c) for a in _inputs(1, 100003)[1:3])
    (y, mean, inv), (e_y, e_mean, e_inv) = R.forward(x, gamma, beta, 1e-5)
    got = _forward(x, gamma, beta)
    assert R.worst(got[0], y, e_y) <= 1 and R.worst(got[1], mean, e_mean) <= 1 and R.worst(got[2], inv, e_inv) <= 1
    want, bounds = R.backward(x, dy, gamma, got[1], got[2])
    back = _backward(x, dy, gamma, got[1], got[2])
    for g, w, b, name in zip(back, want, bounds, ("dx", "dgamma", "dbeta")):
        assert R.worst(g, w, b) <= 1, name


@pytest.mark.parametrize("c", [64, 8192, 100000])
def test_tensors_past_two_to_the_thirty_second_bytes(c):
    """As many rows as the element limit allows, copies of a tile beside each other: every tile's output is the first one's,
    also where the offset passes 2^31 and 2^32 bytes; dbeta is a sum of small integers, so exact."""
    from aether import DeviceTensor
    lib, check = _lib()
    tile = (1 << 22) // c
    rows = ((1 << 31) - 1) // c
    x, gamma, beta, _ = _inputs(tile, c)
    dy = np.random.RandomState(c).randint(-2, 3, (tile, c)).astype(np.float32)

    def repeated(a):
        t, one = DeviceTensor((rows, c)), _dev(a)
        for r in range(0, rows, tile):
            part = t[r:min(r + tile, rows)]
            check(lib.aeth_memcpy_d2d(part.ptr, one.ptr, part.nbytes))
        return t

    xd, gd, bd = repeated(x), _dev(gamma), _dev(beta)
    out, m, s = DeviceTensor((rows, c)), _nan(rows), _nan(rows)
    check(lib.aeth_ln_fwd_f32(xd.ptr, gd.ptr, bd.ptr, m.ptr, s.ptr, out.ptr, rows, c, 1e-5))
    want = _forward(x, gamma, beta)
    places = [k * tile for k in (0, 1, (rows // tile) // 4, (rows // tile) // 2, rows // tile - 1, rows // tile)]
    for r in places:
        n = min(tile, rows - r)
        assert np.array_equal(out[r:r + n].get(), want[0][:n]) and np.array_equal(m[r:r + n].get(), want[1][:n])
    dyd, dg, db = repeated(dy), _nan(c), _nan(c)
    check(lib.aeth_ln_bwd_f32(xd.ptr, dyd.ptr, gd.ptr, m.ptr, s.ptr, out.ptr, dg.ptr, db.ptr, rows, c))
    back = _backward(x, dy, gamma, want[1], want[2])
    for r in places:
        n = min(tile, rows - r)
        assert np.array_equal(out[r:r + n].get(), back[0][:n])
    sums = dy.astype(np.int64).sum(0) * (rows // tile) + dy[:rows % tile].astype(np.int64).sum(0)
    assert np.abs(sums).max() < 1 << 24
    assert np.array_equal(db.get(), sums.astype(np.float32)) and np.all(np.isfinite(dg.get()))


def test_no_rows():
    x, gamma, beta, _ = _inputs(1, 12)
    empty = np.zeros((0, 12), np.float32)
    assert _forward(empty, gamma, beta)[0].shape == (0, 12)
    _, dg, db, _ = _backward(empty, empty, gamma, np.zeros(0, np.float32), np.zeros(0, np.float32))
    assert np.all(dg == 0) and np.all(db == 0)


@pytest.mark.parametrize("rows,c", [(3, 5), (2, 70)])
def test_gradients_against_differences(rows, c):
    """Central differences of sum(dy * y) in 64 bits of the float64 formula, at the point the kernel was given."""
    x, gamma, beta, dy = _inputs(rows, c, seed=4)
    fwd = _forward(x, gamma, beta)
    dx, dg, db, _ = _backward(x, dy, gamma, fwd[1], fwd[2])
    f = lambda a, g, b: float((R.forward_value(a, g, b, 1e-5) * dy).sum())  # noqa: E731
    h = 1e-5

    def slope(which):
        base = [np.asarray(a, np.float64) for a in (x, gamma, beta)]
        out = np.zeros(base[which].shape)
        for i in np.ndindex(out.shape):
            lo, hi = [a.copy() for a in base], [a.copy() for a in base]
            lo[which][i] -= h
            hi[which][i] += h
            out[i] = (f(*hi) - f(*lo)) / (2 * h)
        return out

    # differences: h^2 / 6 times the third derivative (of order 10 here: invstd up to 2) and rounding 1e-16 / h: below 1e-8;
    # the kernel: a few hundred roundings of 2^-24 of terms of order 10
    for got, which in ((dx, 0), (dg, 1), (db, 2)):
        assert np.allclose(got, slope(which), rtol=1e-4, atol=1e-4)


def test_layer_class():
    import aether
    r = np.random.RandomState(5)
    layer = aether.Layer_Norm()
    assert layer.weights is None and layer.epsilon == 1e-5
    x = r.randn(2, 3, 4, 20).astype(np.float32)
    dy = r.randn(2, 3, 4, 20).astype(np.float32)
    out = layer.forward(x, training=True)
    assert out is layer.output and out.shape == x.shape
    assert layer.weights is layer.gamma and layer.biases is layer.beta and layer.gamma.shape == (20,)
    gamma, beta = r.randn(20).astype(np.float32), r.randn(20).astype(np.float32)
    layer.set_parameters(gamma, beta.reshape(1, 20))
    assert layer.weights is layer.gamma and np.array_equal(layer.get_parameters()[1].get(), beta)
    y = layer.forward(x, training=True).get()
    (want, mean, inv), (e_y, _, _) = R.forward(x, gamma, beta, 1e-5)
    assert R.worst(y, want, e_y) <= 1
    assert layer.backward(dy) is layer.dinputs and layer.dinputs.shape == x.shape
    want, bounds = R.backward(x, dy, gamma, layer.row_mean.get(), layer.row_invstd.get())
    for got, w, b in zip((layer.dinputs, layer.dweights, layer.dbiases), want, bounds):
        assert R.worst(got.get(), w, b) <= 1
    assert np.array_equal(layer.forward(x, training=False).get(), y)
    with pytest.raises(ValueError, match="training=True"):
        layer.backward(dy)
    layer.forward(x, training=True)
    with pytest.raises(ValueError, match="gradient shape"):
        layer.backward(dy[:1])
    with pytest.raises(ValueError, match="features"):
        layer.forward(x[..., :19], training=True)
    with pytest.raises(ValueError, match="rows"):
        layer.forward(x[0, 0, 0], training=True)
    assert aether.Layer_Norm(n_features=7).gamma.shape == (7,)


def test_twin_for_a_bf16_convolution_and_behind_one():
    """Between two bf16 convolutions the norm leaves the bfloat16 copies they take (output forward, input gradient
    backward)."""
    import aether
    r = np.random.RandomState(6)
    first, last = aether.Conv_Layer((6, 6, 8), num_filters=8), aether.Conv_Layer((6, 6, 8), num_filters=8)
    norm = aether.Layer_Norm()
    norm.prev, norm.next = first, last
    x, dy = r.randn(2, 6, 6, 8).astype(np.float32), r.randn(2, 6, 6, 8).astype(np.float32)
    norm.forward(x, True)
    norm.backward(dy)
    assert norm.output._bf16 is None and norm.dinputs._bf16 is None
    first.precision = last.precision = "bf16"
    out = norm.forward(x, True)
    norm.backward(dy)
    assert np.array_equal(out._bf16.get(), O.bf16_bits(out.get()))
    assert np.array_equal(norm.dinputs._bf16.get(), O.bf16_bits(norm.dinputs.get()))


@pytest.mark.parametrize("rows", [300, 600])
def test_recorded_and_replayed(rows):
    """Forward and backward pass in a recording: every replay, with eager work of the same layer kind (and a larger
    workspace) between, equals the eager result bit for bit."""
    import aether
    lib, check = _lib()
    r = np.random.RandomState(7)
    c = 130
    gamma, beta = r.randn(c).astype(np.float32), r.randn(c).astype(np.float32)
    layer, other = aether.Layer_Norm(), aether.Layer_Norm()
    layer.set_parameters(gamma, beta)
    batches = [(r.randn(rows, c).astype(np.float32), r.randn(rows, c).astype(np.float32)) for _ in range(4)]
    want = []
    for x, dy in batches:
        layer.forward(x, True)
        layer.backward(dy)
        want.append([t.get() for t in (layer.output, layer.dinputs, layer.dweights, layer.dbiases)])
    xin, dyin = _dev(batches[0][0]), _dev(batches[0][1])
    check(lib.aeth_graph_begin())
    layer.forward(xin, True)
    layer.backward(dyin)
    graph = C.c_void_p()
    check(lib.aeth_graph_end(C.byref(graph)))
    outs = (layer.output, layer.dinputs, layer.dweights, layer.dbiases)
    for k, (x, dy) in enumerate(batches):
        xin.set(x)
        dyin.set(dy)
        check(lib.aeth_graph_launch(graph))
        for t, w in zip(outs, want[k]):
            assert np.array_equal(t.get(), w)
        other.forward(r.randn(900 * (k + 1), 700).astype(np.float32), True)
        other.backward(r.randn(900 * (k + 1), 700).astype(np.float32))
    check(lib.aeth_graph_destroy(graph))


# ---- long sums -------------------------------------------------------------------------------------------------------
U = R.U


@pytest.mark.parametrize("c", [32769, 200704, (1 << 20) + 37, 1 << 22])
def test_long_constant_rows_give_beta(c):
    """A sum of equal numbers in 64 bits is exact (24 bits times fewer than 2^29 of them), and so is its mean: what is left is 0."""
    beta = np.random.RandomState(c).randn(c).astype(np.float32)
    x = np.empty((3, c), np.float32)
    x[0], x[1], x[2] = 1000.3, -0.1, 3e7
    y, mean, inv, _ = _forward(x, np.ones(c, np.float32), beta)
    assert np.array_equal(mean, x[:, 0])
    assert all(np.array_equal(row, beta) for row in y)


def _long_forward(x, gamma, beta, eps):
    """R.forward with the bounds of sums in 64 bits: four terms by pairs in float32 (two roundings), the result (one); a square has
    one more."""
    (y, mean, inv), _ = R.forward(x, gamma, beta, eps)
    d = x.astype(np.float64) - mean[:, None]
    var = (d * d).mean(-1)
    e_mean = 3 * U * np.abs(x.astype(np.float64)).mean(-1)
    e_d = e_mean[:, None] + U * np.abs(d)
    e_var = 6 * U * var + e_mean ** 2 + 2 * U * float(np.float32(eps))
    e_inv = inv * (0.5 * e_var * inv ** 2 + 3 * U)
    xhat = d * inv[:, None]
    e_y = np.abs(gamma) * (e_d * inv[:, None] + np.abs(d) * e_inv[:, None] + 2 * U * np.abs(xhat)) + U * (np.abs(y) + np.abs(xhat * gamma))
    return (y, mean, inv), (e_y, e_mean, e_inv)


def _long_backward(x, dy, gamma, mean, invstd):
    """The same of R.backward."""
    want, (_, e_dgamma, e_dbeta) = R.backward(x, dy, gamma, mean, invstd)
    x, dy, gamma = (np.asarray(a, np.float64) for a in (x, dy, gamma))
    invstd = invstd.astype(np.float64)[:, None]
    xhat = (x - mean.astype(np.float64)[:, None]) * invstd
    g = dy * gamma
    mean_of = lambda a: a.mean(-1, keepdims=True)  # noqa: E731
    c1, c2 = mean_of(g), mean_of(g * xhat)
    e_c1 = 4 * U * mean_of(np.abs(g))                                    # the product, two sums, the result
    e_c2 = 7 * U * mean_of(np.abs(g * xhat))                             # xhat 2, g 1, the product 1, two sums, the result
    size = np.abs(g) + np.abs(c1) + np.abs(xhat * c2)
    e_dx = invstd * (e_c1 + np.abs(xhat) * e_c2 + 2 * U * np.abs(c2 * xhat) + 5 * U * size)
    return want, (e_dx, e_dgamma, e_dbeta)


@pytest.mark.parametrize("rows,c", [(3, 32769), (30, 23000), (3, 200704), (2, (1 << 20) + 37), (1, 1 << 24)])
def test_long_rows_of_like_numbers(rows, c):
    """Numbers far from zero and of one sign, whose sums grow with every term: the bounds are those of 64-bit sums."""
    r = np.random.RandomState(rows + c)
    x = (300 + 200 * r.rand(rows, c)).astype(np.float32)
    dy = (1 + 0.1 * r.randn(rows, c)).astype(np.float32)
    gamma, beta = (1 + 0.1 * r.randn(c)).astype(np.float32), r.randn(c).astype(np.float32)
    got = _forward(x, gamma, beta)
    if c > 32768:
        for g, w, b in zip(got, *_long_forward(x, gamma, beta, 1e-5)):
            assert R.worst(g, w, b) <= 1
    back = _backward(x, dy, gamma, got[1], got[2])
    for g, w, b, name in zip(back, *_long_backward(x, dy, gamma, got[1], got[2]), ("dx", "dgamma", "dbeta")):
        assert R.worst(g, w, b) <= 1, name


# blocks: partial rows, of 256 workgroups and for every 256 rows that a lane has
@pytest.mark.parametrize("rows,c,blocks", [(1 << 27, 8, 4096), (1 << 25, 3, 1024), (3000000, 250, 1536), (400000, 2500, 1792)])
def test_column_sums_of_like_rows(rows, c, blocks):
    """Copies of a tile of rows whose terms are all of one sign in a column, up to 2^30 elements: the sums are the tile's, in 64 bits,
    times the copies.  At most 256 terms are added in line by a lane, then by 6 + 7 levels of lanes and waves; of the partial rows that
    leaves, 128 lanes take their share each and 7 levels the rest."""
    from aether import DeviceTensor
    lib, check = _lib()
    tile = 4000
    rows = rows // tile * tile
    r = np.random.RandomState(c)
    x = (np.arange(c) - (c + 3) / 2 + 0.01 * r.randn(tile, c)).astype(np.float32)
    dy = np.full((tile, c), 0.1, np.float32)
    gamma = np.ones(c, np.float32)
    small = _forward(x, gamma, gamma)

    def repeated(a):
        t = DeviceTensor((rows,) + a.shape[1:])
        check(lib.aeth_memcpy_d2d(t.ptr, _dev(a).ptr, a.nbytes))
        done = tile
        while done < rows:
            n = min(done, rows - done)
            check(lib.aeth_memcpy_d2d(t[done:done + n].ptr, t.ptr, n * (a.nbytes // tile)))
            done += n
        return t

    xd, dyd, md, sd, gd = repeated(x), repeated(dy), repeated(small[1]), repeated(small[2]), _dev(gamma)
    dx, dg, db = DeviceTensor((rows, c)), _nan(c), _nan(c)
    check(lib.aeth_ln_bwd_f32(xd.ptr, dyd.ptr, gd.ptr, md.ptr, sd.ptr, dx.ptr, dg.ptr, db.ptr, rows, c))
    (_, dgamma, dbeta), _ = R.backward(x, dy, gamma, small[1], small[2])
    depth = 256 + 13 + blocks / 128 + 7
    n = rows // tile
    size = (np.abs(dy * (x - small[1][:, None]).astype(np.float64) * small[2][:, None])).sum(0)
    assert R.worst(db.get(), n * dbeta, depth * U * n * np.abs(dbeta)) <= 1
    assert R.worst(dg.get(), n * dgamma, (depth + 3) * U * n * size) <= 1


# one run of rows (16 and 17 of them, 64 with columns enough), several, the longest
@pytest.mark.parametrize("rows,c", [(1, 21505), (15, 21600), (16, 21505), (17, 21505), (64, 100000), (100, 40000), (513, 22001), (4100, 21507)])
def test_runs_of_long_rows(rows, c):
    x, gamma, beta, dy = _inputs(rows, c, seed=6)
    _, mean, inv, _ = _forward(x, gamma, beta)
    back = _backward(x, dy, gamma, mean, inv)
    for g, w, b, name in zip(back, *_long_backward(x, dy, gamma, mean, inv), ("dx", "dgamma", "dbeta")):
        assert R.worst(g, w, b) <= 1, name
    assert all(np.array_equal(a, b) for a, b in zip(back[:3], _backward(x, dy, gamma, mean, inv)[:3]))


def test_the_scratch_of_long_rows_stays_below_their_tensor():
    """64 rows of 2^23 (2 GiB): where they were given a run each, the partial rows took twice that.  A recording refuses a workspace
    that grows, so the calls go through one, after everything else that has grown it is gone (a process of its own)."""
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
rows, c = 64, 1 << 23
x, dy, dx = DeviceTensor.full((rows, c), 1.0), DeviceTensor.full((rows, c), 0.5), DeviceTensor((rows, c))
g, dg, db = DeviceTensor.full(c, 1.0), DeviceTensor(c), DeviceTensor(c)
m, s = DeviceTensor.zeros(rows), DeviceTensor.full(rows, 1.0)
check(lib.aeth_graph_begin())
rc = lib.aeth_ln_bwd_f32(x.ptr, dy.ptr, g.ptr, m.ptr, s.ptr, dx.ptr, dg.ptr, db.ptr, rows, c)
graph = C.c_void_p()
check(lib.aeth_graph_end(C.byref(graph)))
check(rc)
for _ in range(2):
    check(lib.aeth_graph_launch(graph))
    assert np.all(dg.get() == 32) and np.all(db.get() == 32)
check(lib.aeth_graph_destroy(graph))
print("done")
""" % (root, os.path.join(root, "aether-ml_amd"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), r.stderr[-2000:]


@pytest.mark.parametrize("rows,c", [(4, 1), (4, 3), (4, 5), (4, 6), (4, 7), (4, 64), (4, 101), (4, 255), (4, 1537), (4, 2050), (3, 4099),
                                    (3, 20001), (3, 30001), (600, 7), (600, 101), (300, 2050)])
def test_infinite_gradients(rows, c):
    """An infinity in dy, wherever it stands in its row, gives that row the formula's infinities and NaN, its column's dgamma and dbeta
    an infinity, and nothing else."""
    x, gamma, beta, dy = _inputs(rows, c, seed=8)
    fwd = _forward(x, gamma, beta)
    clean = _backward(x, dy, gamma, fwd[1], fwd[2])
    places = sorted({0, c // 2, c - 1, max(0, c - 2), max(0, c - 3), max(0, c - 4), max(0, c - 5)})
    for col in places:
        for value in (np.inf, -np.inf):
            bad = dy.copy()
            bad[1, col] = value
            got = _backward(x, bad, gamma, fwd[1], fwd[2])
            with np.errstate(invalid="ignore"):              # (a single column has xhat = 0: its dgamma is NaN)
                xhat = (x[1].astype(np.float64) - fwd[1][1]) * fwd[2][1]
                g = bad[1].astype(np.float64) * gamma
                dx = fwd[2][1] * (g - g.mean() - xhat * (g * xhat).mean())
                dgamma = value * np.sign(xhat[col])
            assert np.array_equal(got[0][1].astype(np.float64), dx, equal_nan=True), (col, value)
            others = [r for r in range(rows) if r != 1]
            assert np.array_equal(got[0][others], clean[0][others])
            rest = [k for k in range(c) if k != col]
            assert np.array_equal(got[1][rest], clean[1][rest]) and np.array_equal(got[2][rest], clean[2][rest])
            assert got[2][col] == value and np.array_equal(got[1][col], dgamma, equal_nan=True)
