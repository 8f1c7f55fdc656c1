"""Layer norm in 64 bits, and how far a float32 evaluation may be from it.

The bounds count roundings of u = 2^-24 (half a step of float32).  A float32 sum of n terms in any order is off by at most
(n - 1) u sum|terms| to first order; a tree over T lanes behind n / T terms each only makes that smaller, so `n` below is
the number of terms and no order is assumed, except where a row is long: there a lane adds at most n / 64 + 64 terms one
after the other (no kernel gives a row to fewer than 64 lanes unless the row has at most 512 elements)."""
import numpy as np

U = 2.0 ** -24


def _steps(n):
    return float(min(n, n / 64 + 64)) if n > 512 else float(n)


def forward(x, gamma, beta, eps):
    """(y, mean, invstd) in 64 bits of float32 inputs, and the bounds of the float32 results, element by element."""
    x, gamma, beta = (np.asarray(a, np.float64) for a in (x, gamma, beta))
    eps = float(np.float32(eps))
    C = x.shape[-1]
    n = _steps(C) + 2
    mean = x.mean(-1, keepdims=True)
    d = x - mean
    var = (d * d).mean(-1, keepdims=True)
    invstd = 1 / np.sqrt(var + eps)
    xhat = d * invstd
    y = xhat * gamma + beta
    e_mean = n * U * np.abs(x).mean(-1, keepdims=True)                  # the sum, the division
    e_d = e_mean + U * np.abs(d)                                         # the subtraction (of a mean that is off)
    # sum of squares: a common error e of d moves it by 2 e sum(d) + C e^2 = C e^2 (sum d = 0); each square and the sum: n + 2
    e_var = (n + 3) * U * var + e_mean ** 2 + 2 * U * eps
    e_inv = invstd * (0.5 * e_var * invstd ** 2 + 3 * U)                 # + square root, division, the sum with eps
    e_y = np.abs(gamma) * (e_d * invstd + np.abs(d) * e_inv + 2 * U * np.abs(xhat)) + U * (np.abs(y) + np.abs(xhat * gamma))
    return (y, mean[..., 0], invstd[..., 0]), (e_y, e_mean[..., 0], e_inv[..., 0])


def backward(x, dy, gamma, mean, invstd):
    """(dx, dgamma, dbeta) in 64 bits of float32 inputs (the saved statistics among them), and their bounds."""
    x, dy, gamma, mean, invstd = (np.asarray(a, np.float64) for a in (x, dy, gamma, mean, invstd))
    C = x.shape[-1]
    rows = x.size // C
    x, dy = x.reshape(rows, C), dy.reshape(rows, C)
    mean, invstd = mean.reshape(rows, 1), invstd.reshape(rows, 1)
    n, nr = _steps(C) + 2, rows + 2.0
    xhat = (x - mean) * invstd
    e_xhat = 2 * U * np.abs(xhat)                                        # one subtraction, one product
    g = dy * gamma
    c1, c2 = g.mean(-1, keepdims=True), (g * xhat).mean(-1, keepdims=True)
    e_c1 = (n + 1) * U * np.abs(g).mean(-1, keepdims=True)
    e_c2 = (n + 4) * U * np.abs(g * xhat).mean(-1, keepdims=True)
    dx = invstd * (g - c1 - xhat * c2)
    size = np.abs(g) + np.abs(c1) + np.abs(xhat * c2)
    e_dx = invstd * (e_c1 + np.abs(xhat) * e_c2 + np.abs(c2) * e_xhat + 5 * U * size)
    dgamma, dbeta = (dy * xhat).sum(0), dy.sum(0)
    e_dgamma = (nr + 3) * U * np.abs(dy * xhat).sum(0)
    e_dbeta = nr * U * np.abs(dy).sum(0)
    return (dx, dgamma, dbeta), (e_dx, e_dgamma, e_dbeta)


def worst(got, want, bound):
    """The largest error over its bound (a bound of zero allows none)."""
    got, want, bound = (np.asarray(a, np.float64).reshape(-1) for a in (got, want, bound))
    assert got.shape == want.shape
    if got.size == 0:
        return 0.0
    assert np.all(np.isfinite(got)), "non-finite values (unwritten output?)"
    err = np.abs(got - want)
    return float(np.max(np.where(err == 0, 0.0, err / np.maximum(bound, 1e-300))))


def forward_value(x, gamma, beta, eps):
    """y alone, for differences."""
    d = x - x.mean(-1, keepdims=True)
    return d / np.sqrt((d * d).mean(-1, keepdims=True) + float(np.float32(eps))) * gamma + beta
