"""Dense layers, the loss on top of one and clipped gradients in 64 bits, from their definitions (numpy), and how far the kernels may be off."""
import numpy as np

U = 2.0 ** -24          # half a step of float32, relative


def bits_of(words, frames):
    """[rows, words] int32 -> [rows, frames] of 0 and 1"""
    w = np.ascontiguousarray(words).view(np.uint32)
    f = np.arange(frames)
    return ((w[:, f // 32] >> (f % 32).astype(np.uint32)) & 1).astype(np.float64)


def activated(z, activation):
    if activation == "relu":
        return np.where(z <= 0, 0.0, z)
    if activation == "sigmoid":
        with np.errstate(over="ignore"):
            return 1.0 / (1.0 + np.exp(-z))
    if activation == "hard_tanh":
        return np.where(z <= -1, -1.0, np.where(z >= 1, 1.0, z))
    return z


def through(dy, y, activation):
    if activation == "relu":
        return np.where(y <= 0, 0.0, dy)
    if activation == "sigmoid":
        return dy * (y * (1.0 - y))
    if activation == "hard_tanh":
        return np.where((y <= -1) | (y >= 1), 0.0, dy)
    return dy


def product_bound(a, b):
    """How far a computed a @ b may be from the exact one, element by element.  Its sum of K products takes at most 3 K roundings to float32 (three products of halves for each k, in any
    order); a value is represented with 22 bits or better and the product of the two lower halves is left out: three times 2^-22 of a product at most, together 12 U; values far below the
    largest of their row are off by 2^-40 of that one."""
    a, b = np.abs(a), np.abs(b)
    k = a.shape[1]
    return (3 * k + 16) * U * (a @ b) + 2.0 ** -39 * k * a.max(1, initial=0)[:, None] * b.max(0, initial=0)[None]


def loss(x, W, b, label, weight, weight_sum):
    """x [inputs, frames], label and weight [frames] -> (loss, dz, dx, dW, db)"""
    C, F = W.shape[0], x.shape[1]
    counts = (label >= 0) & (label < C) & (weight != 0)
    x = np.where(counts[None], x, 0.0)
    z = W @ x + b[:, None]
    top = z.max(0)
    e = np.exp(z - top)
    s = e.sum(0)
    at = np.where(counts, label, 0)
    value = np.where(counts, weight * (np.log(s) - (z - top)[at, np.arange(F)]), 0.0)
    g = np.where(counts, weight / weight_sum, 0.0)
    dz = e / s * g
    dz[at, np.arange(F)] -= g
    return value, dz, W.T @ dz, dz @ x.T, dz.sum(1)
