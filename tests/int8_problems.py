"""Seeded int8 2:4 problems, the plain product in 64 bits, and its tolerance,
shared by the int8 tests."""
from __future__ import annotations

import numpy as np

import oracle as O


def bits_to_f64(bits, bf16):
    b = np.ascontiguousarray(bits).view(np.uint16)
    if bf16:
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.view(np.float16).astype(np.float64)


def round_bits(x, bf16):
    """fp32 values -> the nearest 16-bit patterns."""
    x = np.asarray(x, dtype=np.float32)
    if not bf16:
        return O.f32_to_f16_bits(x.reshape(-1)).reshape(x.shape)
    u = x.view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def act64(y, act):
    if act == 1:
        return np.maximum(y, 0)
    if act == 2:
        return y / (1 + np.exp(-y))
    if act == 3:
        return 0.5 * y * (1 + np.tanh(np.sqrt(2 / np.pi) * (y + 0.044715 * y ** 3)))
    return y


def prune_int8(a, M, K):
    """The two largest magnitudes of each group of four, ties to the lower index (numpy)."""
    g = a.reshape(-1, 4).astype(np.int32)
    order = np.argsort(-np.abs(g), axis=1, kind="stable")
    out = np.zeros_like(g)
    for i in range(2):
        np.put_along_axis(out, order[:, i:i + 1], np.take_along_axis(g, order[:, i:i + 1], 1), 1)
    return out.astype(np.int8).reshape(M, K)


def problem(M, N, K, seed, full_range=True):
    rng = np.random.default_rng(seed)
    lo = -128 if full_range else -4
    a = prune_int8(rng.integers(lo, -lo, (M, K)).astype(np.int8), M, K)
    b = rng.integers(lo, -lo, (N, K)).astype(np.int8)
    return a, b


def product(a, b):
    """The exact sums (fp64 holds every one: below 2^31)."""
    return a.astype(np.float64) @ b.astype(np.float64).T


def tolerance(ref, pre, extra, act, bf16):
    """|got - ref| for C = act(pre) + extra in fp32, rounded once.

    Half a step of C's type (2^-8 bf16, 2^-11 fp16; 2^-25 in fp16's subnormal
    range).  Before it, `pre` passes at most six fp32 roundings (the sum's
    conversion, two scales, alpha, the bias, the activation's own product), the
    addition of `extra` one; SiLU and GELU take a hardware tanh of relative
    error 2^-10.9, which moves 0.5 y tanh by 2^-11.9 |y|, and their slope is at
    most 1.13."""
    size = np.abs(pre)
    err = 1.13 * 6 * 2.0 ** -24 * size + 2.0 ** -24 * np.abs(ref)
    if act in (2, 3):
        err = err + 2.0 ** -11.9 * size
    half = 2.0 ** (-8 if bf16 else -11)
    # the last rounding sees ref + err
    return err * (1 + half) + half * np.abs(ref) + (0 if bf16 else 2.0 ** -25)
