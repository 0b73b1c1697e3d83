"""Fits the polynomial behind the capped scores of the masked attention (kTanhRatio in attention_masked.cuh).

tanh(y) = y p(y^2) on |y| <= 1 with p of degree 5, chosen to minimise the maximum RELATIVE error |y p(y^2) / tanh(y) - 1|
over a dense grid: a linear program in the coefficients and the error (minimax fit by linear programming). The
coefficients are rounded to f32 and the achieved error is re-measured in f32 arithmetic.

Run: python npu_ai_b200/csrc/fit_tanh_poly.py
"""
import numpy as np
from scipy.optimize import linprog

DEGREE, Y_MAX = 5, 1.0


def fit(n_grid: int = 4001):
    y = (1.0 - np.cos(np.pi * np.arange(1, n_grid) / (n_grid - 1))) / 2.0 * Y_MAX
    f = np.tanh(y) / y
    V = np.stack([(y * y) ** k for k in range(DEGREE + 1)], axis=1)
    # |V c - f| <= e f
    A = np.vstack([np.hstack([V, -f[:, None]]), np.hstack([-V, -f[:, None]])])
    res = linprog(c=[0] * (DEGREE + 1) + [1], A_ub=A, b_ub=np.concatenate([f, -f]),
                  bounds=[(None, None)] * (DEGREE + 1) + [(0, None)], method="highs")
    assert res.success, res.message
    return np.float32(res.x[:-1]), float(res.x[-1])


def poly_f32(y, c):
    """The kernel's evaluation order (Horner in y^2, then times y), in f32."""
    y = np.asarray(y, dtype=np.float32)
    z = (y * y).astype(np.float32)
    p = np.full_like(z, c[-1])
    for k in c[-2::-1]:
        p = (p.astype(np.float64) * z + np.float64(k)).astype(np.float32)  # a fused multiply-add rounds once
    return (p * y).astype(np.float32)


if __name__ == "__main__":
    c, e = fit()
    ys = np.linspace(1e-6, Y_MAX, 1_000_001).astype(np.float32)
    rel = np.abs(poly_f32(ys, c).astype(np.float64) / np.tanh(ys.astype(np.float64)) - 1.0).max()
    print("c =", ", ".join(f"{v:.9e}f" for v in c))
    print(f"LP minimax relative error {e:.3e}; measured in f32 on (0, {Y_MAX}]: {rel:.3e}")
