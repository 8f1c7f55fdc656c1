"""Refusals of the Muon entry points and of Optimizer_Muon (arguments are checked before the context: no GPU needed), and
checks of the reference that the GPU tests compare with."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from tests import muon_reference as R


@pytest.fixture(scope="module")
def lib():
    from aether import _lib
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _lib.load()


A, B, D, E = (0x10000000 + (i << 28) for i in range(4))         # addresses that are never read
GOOD = dict(count=2, theta=[A, A + (1 << 20)], grad=[B, B + (1 << 20)], mom=[D, D + (1 << 20)], rows=[8, 300], cols=[9, 200],
            lr=0.02, momentum=0.95, nesterov=1, wd=0.0, steps=5)


def _call(lib, dev=False, **changes):
    a = dict(GOOD, **changes)
    arr = lambda t, v: None if v is None else (t * len(v))(*v)  # noqa: E731
    table = [arr(C.c_void_p, a[k]) for k in ("theta", "grad", "mom")] + [arr(C.c_int, a[k]) for k in ("rows", "cols")]
    if dev:
        return lib.aeth_muon_multi_dev_f32(a["count"], *table, a["momentum"], a["nesterov"], a["wd"], a["steps"], a["state"])
    return lib.aeth_muon_multi_f32(a["count"], *table, a["lr"], a["momentum"], a["nesterov"], a["wd"], a["steps"])


@pytest.mark.parametrize("changes,word", [
    (dict(count=0), "count"), (dict(count=33), "count"), (dict(count=-1), "count"),
    (dict(theta=None), "NULL"), (dict(grad=None), "NULL"), (dict(mom=None), "NULL"), (dict(rows=None), "NULL"),
    (dict(cols=None), "NULL"), (dict(theta=[A, None]), "NULL"), (dict(grad=[None, B]), "NULL"), (dict(mom=[D, None]), "NULL"),
    (dict(rows=[-1, 3]), "-1"), (dict(cols=[9, -200]), "-200"), (dict(rows=[1 << 16, 3], cols=[1 << 15, 3]), "65536"),
    (dict(rows=[8, (1 << 21) + 1], cols=[9, 1]), "2097153"), (dict(rows=[8, 1], cols=[9, (1 << 21) + 1]), "2097153"),
    (dict(momentum=1.0), "momentum"), (dict(momentum=-0.1), "momentum"), (dict(momentum=float("nan")), "momentum"),
    (dict(lr=float("nan")), "learning rate"), (dict(lr=float("inf")), "learning rate"), (dict(wd=-1.0), "weight decay"),
    (dict(wd=float("nan")), "weight decay"), (dict(wd=float("inf")), "weight decay"),
    (dict(steps=0), "steps"), (dict(steps=101), "steps"),
    (dict(theta=[A, A]), "overlap"), (dict(theta=[A, A + 4]), "overlap"), (dict(mom=[D, D]), "overlap"),
    (dict(theta=[A, B + (1 << 20)]), "overlap"), (dict(mom=[B, D]), "overlap"), (dict(mom=[A, D]), "overlap"),
    (dict(theta=[A, D]), "overlap")])
def test_refusals(lib, changes, word):
    assert _call(lib, **changes) == -1
    assert word in lib.aeth_last_error().decode() and "aeth_muon_multi_f32" in lib.aeth_last_error().decode()
    if "lr" not in changes:
        assert _call(lib, dev=True, state=E, **changes) == -1
        assert "aeth_muon_multi_dev_f32" in lib.aeth_last_error().decode()


def test_refusals_of_the_orthogonalisation(lib):
    for args in ((None, B, 4, 5, 5), (A, None, 4, 5, 5), (A, A, 4, 5, 5), (A, A + 79 * 1, 4, 5, 5), (A + 4, A, 4, 5, 5),
                 (A, B, -1, 5, 5), (A, B, 4, -5, 5), (A, B, 1 << 16, 1 << 15, 5), (A, B, (1 << 21) + 1, 1, 5), (A, B, 1, (1 << 21) + 1, 5), (A, B, 4, 5, 0), (A, B, 4, 5, 101)):
        assert lib.aeth_newton_schulz_f32(*args) == -1, args
    assert _call(lib, dev=True, state=None) == -1


def test_good_calls_before_init_report_the_state(lib):
    if os.path.exists("/dev/kfd"):
        pytest.skip("a GPU is present: the context may already be initialised by other tests")
    assert _call(lib) == -4 and _call(lib, dev=True, state=E) == -4
    assert lib.aeth_newton_schulz_f32(A, B, 4, 5, 5) == -4
    assert _call(lib, grad=[B, B]) == -4                         # gradients are only read: they may be shared


def test_the_optimizer_refuses_bad_settings():
    import aether
    for kw in (dict(momentum=1.0), dict(momentum=-0.5), dict(momentum=float("nan")), dict(ns_steps=0), dict(ns_steps=101),
               dict(weight_decay=-0.1), dict(weight_decay=float("nan"))):
        with pytest.raises(ValueError):
            aether.Optimizer_Muon(**kw)
    opt = aether.Optimizer_Muon(learning_rate=0.1, decay=0.5)
    opt.pre_update_parameters()
    assert opt.current_learning_rate == 0.1 and opt.adam.current_learning_rate == 0.001
    opt.iterations = opt.adam.iterations = 2
    opt.pre_update_parameters()
    assert opt.current_learning_rate == 0.1 / 2 and opt.adam.current_learning_rate == 0.001 / 2


@pytest.mark.parametrize("r,c", [(6, 4), (40, 70), (90, 60)])
def test_the_tolerance_refuses_mistakes(r, c):
    """float32 and 22-bit factors are within the tolerance; 11-bit factors (one half of the pair alone), a wrong coefficient,
    a missing step, a forgotten transposition of the second factor are not (planted in the reference's own arithmetic)."""
    rng = np.random.RandomState(r)
    g = (rng.randn(r, c) + 2 * rng.randn(r, 1) @ rng.randn(1, c)).astype(np.float32)
    tol, exact = R.tolerance(g)
    off = lambda o: np.linalg.norm(o - exact)  # noqa: E731
    assert off(R.newton_schulz(g, 5, np.float32)) <= tol

    def rounded(x, bits):
        m, e = np.frexp(x)
        return np.ldexp(np.round(m * 2.0 ** bits), e - bits)

    def with_bits(bits, coef=R.COEF, steps=5):
        a, b, cc = coef
        x = np.asarray(g, np.float64)
        x = x.T if r > c else x
        x = x / np.linalg.norm(x)
        for _ in range(steps):
            x = rounded(x, bits)
            s = rounded(x @ x.T, bits)
            x = rounded(a * np.eye(len(s)) + b * s + cc * s @ s, bits) @ x
        return x.T if r > c else x

    assert off(with_bits(22)) <= tol
    assert off(with_bits(11)) > tol and off(with_bits(8)) > tol
    assert off(with_bits(30, (3.4445, -4.7750, 2.0300))) > tol
    assert off(with_bits(30, steps=4)) > tol
    assert off(-exact) > tol


def test_the_reference_sets_singular_values_near_one():
    rng = np.random.RandomState(0)
    g = rng.randn(30, 50)
    o = R.newton_schulz(g)
    s = np.linalg.svd(o, compute_uv=False)
    assert s.max() < 1.21 and s.min() > 0.6
    u, t, v = np.linalg.svd(g, full_matrices=False)
    p = t / np.linalg.norm(g)
    for _ in range(5):
        p = R.COEF[0] * p + R.COEF[1] * p ** 3 + R.COEF[2] * p ** 5
    assert np.allclose(o, (u * p) @ v, atol=1e-12)


def test_tiles_runs_and_buffers_cover_every_product(tmp_path):
    """aether-ml_amd/csrc/muon_plan.h: tile orders, the choice of tiles and runs, the workspace (tests/cpu/muon_plan_check.cpp
    walks them on the host)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "muon_plan_check")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(root, "aether-ml_amd", "csrc"),
                    os.path.join(root, "tests", "cpu", "muon_plan_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    assert [line.split()[1] for line in r.stdout.splitlines()] == ["triangles", "choices", "layouts"]


def test_the_limit_of_the_halves(tmp_path):
    """aether-ml_amd/csrc/muon_plan.h: which matrices go through the steps as two float16 halves."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "muon_halves_check")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", os.path.join(root, "aether-ml_amd", "csrc"),
                    os.path.join(root, "tests", "cpu", "muon_halves_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok halves\n", r.stdout + r.stderr


@pytest.mark.parametrize("steps,scale", [(16, 1e-9), (25, 1e-12)])
def test_the_tolerance_refuses_halves_beyond_their_limit(steps, scale):
    """Two float16 halves under one power of two, for more steps than they carry (planted in the reference's own arithmetic)."""
    rng = np.random.RandomState(steps)
    g = rng.randn(64, 96)
    g[:32, 48:] = 0
    g[32:, :48] = 0
    g[32:] *= scale
    tol, exact = R.tolerance(g.astype(np.float32), steps)

    def halves(x, s):
        y = (x * s).astype(np.float32)
        hi = y.astype(np.float16)
        return (hi.astype(np.float64) + (y - hi).astype(np.float16)) / s

    x = halves(g / np.linalg.norm(g), 32768.0)
    for _ in range(steps):
        a = halves(x @ x.T, 32768.0)
        x = halves(halves(R.COEF[0] * np.eye(64) + R.COEF[1] * a + R.COEF[2] * a @ a, 16384.0) @ x, 32768.0)
    assert np.linalg.norm(x - exact) > tol
