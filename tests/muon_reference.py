"""The Muon update in 64 bits, and how far the kernels may be from it.

A float32 evaluation of the same formula (NumPy, here on the CPU) is the measure: the kernels hold every factor of a product
in at least 22 bits where float32 has 24, so one rounding of a factor is at most 4 times float32's; leaving out the product
of two low halves is one more error of that size (together 8); sums are float32 in both.  Where the float32 evaluation happens
to be exact (tiny matrices), 32 roundings of 2^-22 remain, relative to the result's norm."""
import numpy as np

COEF = (3.4445, -4.7750, 2.0315)
U = 2.0 ** -24


def newton_schulz(g, steps=5, dtype=np.float64):
    a, b, c = (dtype(v) for v in COEF)
    g = np.asarray(g, dtype)
    tall = g.shape[0] > g.shape[1]
    x = g.T if tall else g
    norm = np.sqrt(np.sum(x.astype(np.float64) ** 2))
    x = (x.astype(np.float64) / norm).astype(dtype) if norm != 0 else x
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.T if tall else x


def tolerance(g, steps=5):
    """Bound of |o - exact| in the Frobenius norm, and the exact o."""
    exact = newton_schulz(g, steps)
    off = np.linalg.norm(newton_schulz(g, steps, np.float32) - exact)
    return 8 * off + 2.0 ** -17 * np.linalg.norm(exact), exact


def update(theta, grad, mom, lr, momentum, nesterov, weight_decay, steps=5):
    """(theta, momentum) after a step in 64 bits, and a bound of theta's error in the Frobenius norm."""
    theta, grad, mom = (np.asarray(t, np.float64) for t in (theta, grad, mom))
    lr, momentum, weight_decay = (float(np.float32(v)) for v in (lr, momentum, weight_decay))
    m = momentum * mom + grad
    u = grad + momentum * m if nesterov else m
    # the kernel's u carries three roundings of its terms; p amplifies a relative change of u like any other
    tol, o = tolerance(u, steps)
    step = lr * np.sqrt(max(1.0, theta.shape[1] / theta.shape[0]))
    want = theta * (1 - lr * weight_decay) - step * o
    bound = abs(step) * tol + 4 * U * (np.linalg.norm(theta) + abs(step) * np.linalg.norm(o)) + 1e-30
    return want, m, bound


def momentum_bound(grad, mom, momentum):
    """Two roundings: the product and the sum."""
    m = np.abs(momentum * np.asarray(mom, np.float64))
    return 2 * U * (m + np.abs(np.asarray(grad, np.float64))) + 1e-44
