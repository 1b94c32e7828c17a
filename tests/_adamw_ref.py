"""Plain AdamW for the tests, on the CPU.

``Plain64`` is the step in 64 bits, with bounds on what 32-bit arithmetic may be
off.  ``Plain32`` is the library's definition in numpy's fp32 (numpy rounds
every operation once), 8-bit codes included: the kernels have to give its bits.
"""

import math

import numpy as np

EPS32 = 2.0 ** -24  # half a step of fp32, relative
FLOOR = np.float32(2.0 ** -100)


def scalars(lr, betas, eps, wd, step):
    b1, b2 = betas
    return dict(b1=b1, o1=1 - b1, b2=b2, o2=1 - b2, decay=1 - lr * wd, size=lr / (1 - b1 ** step),
                rs=1 / math.sqrt(1 - b2 ** step), eps=eps)


class Plain64:
    """AdamW in 64 bits; ``round_to``: rounds the parameter (64-bit numpy in and
    out) as it is stored after each step, ``spacing`` its relative step and
    ``least`` the step below the type's smallest normal number."""

    def __init__(self, p, round_to=None, spacing=0.0, least=0.0):
        self.p = p.astype(np.float64)
        self.m = np.zeros_like(self.p)
        self.v = np.zeros_like(self.p)
        self.abs_m = np.zeros_like(self.p)  # the EMA of |g|: what rounding errors of m are relative to
        self.tol_p = np.zeros_like(self.p)
        self.round_to, self.spacing, self.least, self.t = round_to, spacing, least, 0

    def step(self, g, lr, betas, eps, wd, scale=1.0):
        self.t += 1
        s = scalars(lr, betas, eps, wd, self.t)
        g = g.astype(np.float64) * scale
        self.m = s["b1"] * self.m + s["o1"] * g
        self.abs_m = s["b1"] * self.abs_m + s["o1"] * np.abs(g)
        self.v = s["b2"] * self.v + s["o2"] * g * g
        den = np.sqrt(self.v) * s["rs"] + eps
        upd = s["size"] * self.m / den
        # a step rounds beta, 1 - beta, g * scale, the products (two for v) and the sum: at most 7 roundings each,
        # kept from step to step; v's error halves under the root; the update adds at most 8 more
        with np.errstate(invalid="ignore"):
            self.tol_m = 7 * self.t * EPS32 * self.abs_m
            self.tol_v = 7 * self.t * EPS32 * self.v
            self.tol_p = self.tol_p + 4 * EPS32 * np.abs(self.p) + s["size"] / den * self.tol_m \
                + (4 * self.t + 8) * EPS32 * np.abs(upd)
            self.p = self.p * s["decay"] - upd
            if self.round_to is not None:
                # a rounding that falls the other way is off by one step of the type
                self.p = self.round_to(self.p)
                self.tol_p = self.tol_p + np.maximum(self.spacing * np.abs(self.p), self.least)


def encode(x, top, block):
    """codes (nb, block) as integers and scales (nb, 1) of a flat fp32 array"""
    f = np.float32
    nb = -(-x.size // block)
    y = np.zeros(nb * block, f)
    y[:x.size] = x
    y = y.reshape(nb, block)
    with np.errstate(all="ignore"):
        s = np.maximum(np.abs(y).max(1, keepdims=True), FLOOR)
        r = np.abs(y) * (f(1) / s)
        r = np.where(np.isnan(r), f(0), r)
        c = np.rint(np.sqrt(np.maximum(r, FLOOR)) * f(top)).astype(np.int32)
    if top == 255:
        c = np.where((y > 0) & (c == 0), 1, c)
    return np.where(y < 0, -c, c), s


def decode(c, s, top):
    f = np.float32
    c = c.astype(f)
    with np.errstate(all="ignore"):
        return (c * np.abs(c)) * (s * f(1.0 / (top * top)))


class Plain32:
    """The definition in fp32; ``block``: 8-bit moments (None: fp32).

    ``tol_p`` bounds how far the parameter of the 8-bit step may be off, whose
    quotient is not rounded as defined: the reciprocal is within 2 half steps
    and its product rounds once more where the quotient rounds once; the
    denominator's and the parameter's multiply-adds round once instead of
    twice (1 for the denominator, 2 for the parameter).  With the difference
    of each pair counted for both: 8 half steps of the update, 4 of the
    parameter.  A stored type then rounds either way: one of its steps."""

    def __init__(self, p, block=None, round_to=None):
        self.p = p.astype(np.float32).reshape(-1)
        self.block, self.round_to, self.t = block, round_to, 0
        self.tol_p = np.zeros(self.p.size)
        self.m = np.zeros_like(self.p)
        self.v = np.zeros_like(self.p)
        if block:
            nb = -(-self.p.size // block)
            self.codes = [(np.zeros((nb, block), np.int32), np.zeros((nb, 1), np.float32)) for _ in range(2)]

    def step(self, g, lr, betas, eps, wd, scale=None):
        f = np.float32
        self.t += 1
        s = {k: f(x) for k, x in scalars(lr, betas, eps, wd, self.t).items()}
        g = g.astype(f).reshape(-1)
        n = self.p.size
        with np.errstate(all="ignore"):
            if scale is not None:
                g = g * f(scale)
            if self.block:
                self.m = decode(*self.codes[0], 127).reshape(-1)[:n]
                u = decode(*self.codes[1], 255).reshape(-1)[:n]
                self.v = u * u
            self.m = self.m * s["b1"] + g * s["o1"]
            self.v = self.v * s["b2"] + (g * s["o2"]) * g
            root = np.sqrt(self.v)
            upd = (self.m * s["size"]) / (root * s["rs"] + s["eps"])
            self.tol_p = self.tol_p + 8 * EPS32 * np.abs(upd.astype(np.float64)) + 4 * EPS32 * np.abs(self.p)
            self.p = self.p * s["decay"] - upd
            if self.round_to is not None:
                self.p = self.round_to(self.p)
                # the types' steps: from eps of the value, and not below their smallest number's
                eps = 2.0 ** -7 if self.round_to(np.float32([1 + 2.0 ** -9]))[0] == 1 else 2.0 ** -10
                least = eps * (2.0 ** -126 if eps == 2.0 ** -7 else 2.0 ** -14)
                self.tol_p = self.tol_p + np.maximum(eps * np.abs(self.p), least)
        if self.block:
            self.codes = [encode(self.m, 127, self.block), encode(root, 255, self.block)]
