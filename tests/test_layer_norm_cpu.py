"""Refusals of the layer norm's entry points (arguments are checked before the context, so a bad call is refused on any
machine) and checks of the 64-bit reference that its GPU tests compare with."""
import os

import numpy as np
import pytest

from tests import norm_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from aether import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _lib.load()


X, DY, G, B, M, S, Y, Y16, DG, DB = (0x10000000 + (i << 24) for i in range(10))      # addresses that are never read

GOOD = {
    "aeth_ln_fwd_f32": [X, G, B, M, S, Y, 4, 100, 1e-5],
    "aeth_ln_fwd_twin_f32": [X, G, B, M, S, Y, Y16, 4, 100, 1e-5],
    "aeth_ln_bwd_f32": [X, DY, G, M, S, Y, DG, DB, 4, 100],
    "aeth_ln_bwd_twin_f32": [X, DY, G, M, S, Y, Y16, DG, DB, 4, 100],
}


@pytest.mark.parametrize("name", sorted(GOOD))
def test_refusals(lib, name):
    call, good = getattr(lib, name), GOOD[name]
    pointers = [i for i, a in enumerate(good) if isinstance(a, int) and a > 1 << 20]
    at = {a: i for i, a in enumerate(good)}

    def refused(**changes):
        args = list(good)
        for i, v in changes.items():
            args[int(i[1:])] = v
        assert call(*args) == -1, changes
        assert name.replace("_twin", "").replace("aeth_", "").replace("_f32", "") in lib.aeth_last_error().decode()

    for i in pointers:                       # each tensor is needed (the statistics together, forward)
        refused(**{"_%d" % i: None})
    rows, c = at[4], at[100]
    refused(**{"_%d" % rows: -1})
    refused(**{"_%d" % c: 0})
    refused(**{"_%d" % c: -3})
    refused(**{"_%d" % rows: 1 << 16, "_%d" % c: 1 << 15})          # 2^31 elements
    refused(**{"_%d" % at[Y]: X})                                    # output over input
    refused(**{"_%d" % at[Y]: X + 4 * 399})
    refused(**{"_%d" % at[Y]: X - 4 * 399})
    if Y16 in at:
        refused(**{"_%d" % at[Y16]: Y + 64})
    if DY in at:
        refused(**{"_%d" % at[Y]: DY})
    outputs = [i for i, a in enumerate(good) if a in ((Y, Y16, M, S) if 1e-5 in at else (Y, Y16, DG, DB))]
    for i in outputs:                        # no output over any other tensor, whole or at one element
        for j in pointers:
            if i != j:
                refused(**{"_%d" % i: good[j]})
                refused(**{"_%d" % i: good[j] + 2})
    if 1e-5 in at:
        refused(**{"_%d" % at[1e-5]: -1e-3})
        refused(**{"_%d" % at[1e-5]: float("nan")})


def test_a_good_call_before_init_reports_the_state(lib):
    if os.path.exists("/dev/kfd"):
        pytest.skip("a GPU is present: the context may already be initialised by other tests")
    for name, args in GOOD.items():
        assert getattr(lib, name)(*args) == -4, name
    assert lib.aeth_ln_fwd_f32(X, G, B, None, None, Y, 4, 100, 1e-5) == -4
    assert lib.aeth_ln_fwd_f32(None, None, None, None, None, None, 0, 100, 1e-5) == -4


def test_the_class_refuses_a_bad_epsilon():
    import aether
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError, match="epsilon"):
            aether.Layer_Norm(epsilon=eps)


@pytest.mark.parametrize("rows,c", [(4, 3), (2, 40), (3, 700)])
def test_the_bounds_hold_float32_and_refuse_mistakes(rows, c):
    """NumPy's float32 evaluation is within the bounds; a variance over C - 1, a missing term of the gradient and a
    bfloat16-sized error are not (the mistakes are planted in the reference's own arithmetic)."""
    r = np.random.RandomState(c)
    f = np.float32
    x, dy = (r.randn(rows, c) + 0.5).astype(f), r.randn(rows, c).astype(f)
    gamma, beta = r.randn(c).astype(f), r.randn(c).astype(f)
    (y, mean, inv), (e_y, e_m, e_i) = R.forward(x, gamma, beta, 1e-5)
    d = x - x.mean(-1, keepdims=True, dtype=f)
    inv32 = f(1) / np.sqrt((d * d).mean(-1, keepdims=True, dtype=f) + f(1e-5))
    assert R.worst(d * inv32 * gamma + beta, y, e_y) <= 1
    unbiased = 1 / np.sqrt((d.astype(np.float64) ** 2).sum(-1, keepdims=True) / (c - 1) + 1e-5)
    assert R.worst(d * unbiased * gamma + beta, y, e_y) > 1
    assert R.worst(y * (1 + 2.0 ** -9), y, e_y) > 1
    m, s = mean.astype(f), inv.astype(f)
    want, bounds = R.backward(x, dy, gamma, m, s)
    xh = (x - m[:, None]) * s[:, None]
    g = dy * gamma
    c1, c2 = g.mean(-1, keepdims=True), (g * xh).mean(-1, keepdims=True)
    assert R.worst(s[:, None] * (g - c1 - xh * c2), want[0], bounds[0]) <= 1
    assert R.worst(s[:, None] * (g - xh * c2), want[0], bounds[0]) > 1
    assert R.worst(s[:, None] * (g - c1), want[0], bounds[0]) > 1
    assert R.worst((dy * xh).sum(0), want[1], bounds[1]) <= 1 and R.worst((dy * xh)[1:].sum(0), want[1], bounds[1]) > 1
