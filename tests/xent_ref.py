"""Softmax cross entropy of a classifier, its gradient, and the error bounds the GPU results are held to: plain numpy
in 64 bits.

Matrices are [rows, hidden]: W [vocab, hidden], X [tokens, hidden].  With u = 2^-24 the half step of fp32 and v that of
the operands' type (fp32 2^-24, bf16 2^-8), the bounds are sums of these parts:

* a logit is a sum of `hidden` products in fp32:  |dz| <= (hidden + 2) u |alpha| sum |x||w|   (+ 2: alpha, rounding);
* the sum of the exponentials is one of positive terms, at most 128 in a row inside a lane, 8 more joining the lanes
  and waves, one for every tile of 128 vocabulary rows; each exponential is off by at most 4 u of itself (2 u of the
  function, 2 u of its rounded argument near the maximum, where it counts);
* P = both * exp(z - lse) - gloss is off by (2 max|dz| + 2 u |lse| + 8 u) of both * exp, by 4 u of gloss, and by v of
  itself where it is rounded (not at the label, where what the rounding took is added in fp32);  z - lse is formed in fp32, hence the 2 u |z - lse| <= 2 u (|z| + |lse|) that is added;
* exp, P and the operands of the matrix cores may lose what lies below the smallest normal number, 2^-126 in both types:
  up to 2^-126 of each P, since a value under it may be rounded on coarser steps or to zero;
* the products sum tokens or vocabulary in fp32: (K + 8) u of the sum of absolute products, K their length;
* the result is rounded once more: v.
"""
import numpy as np

U = 2.0 ** -24


def half_step(prec):
    return {"s": 2.0 ** -24, "b": 2.0 ** -8}[prec]


def valid(label, vocab, ignore):
    return (label >= 0) & (label < vocab) & (label != ignore)


def forward(W, X, label, alpha, ignore, prec):
    """(loss, lse, bound of lse, bound of loss)"""
    V, H = W.shape
    has = valid(label, V, ignore)
    loss, lse = np.zeros(len(label)), np.zeros(len(label))
    blse, bloss = np.zeros(len(label)), np.zeros(len(label))
    t = np.flatnonzero(has)
    if t.size:
        z = alpha * (X[t] @ W.T)
        dz = (H + 2) * U * abs(alpha) * (np.abs(X[t]) @ np.abs(np.where(np.isfinite(W), W, 0.0)).T)
        top = z.max(axis=1)
        lse[t] = top + np.log(np.exp(z - top[:, None]).sum(axis=1))
        loss[t] = lse[t] - z[np.arange(t.size), label[t]]
        tiles = -(-V // 128)
        blse[t] = dz.max(axis=1) + (128 + 8 + tiles + 4) * U + 4 * U * np.abs(lse[t])
        bloss[t] = blse[t] + dz[np.arange(t.size), label[t]] + 2 * U * np.abs(loss[t])
    return loss, lse, blse, bloss


def backward(W, X, label, alpha, ignore, lse, gloss, glse, prec, beta=0.0, gW0=None):
    """(gW, gX, bound of gW, bound of gX) for the lse that is handed over"""
    V, H = W.shape
    T = len(label)
    v = half_step(prec)
    gW = np.zeros(W.shape) if gW0 is None else beta * gW0
    bW = 2 * U * np.abs(gW)
    gX, bX = np.zeros(X.shape), np.zeros(X.shape)
    t = np.flatnonzero(valid(label, V, ignore))
    if t.size:
        x, w = X[t], W
        z = alpha * (x @ w.T)
        dz = (H + 2) * U * abs(alpha) * (np.abs(x) @ np.abs(w).T)
        p = np.exp(z - lse[t][:, None])
        both = gloss[t] + (0.0 if glse is None else glse[t])
        hot = np.zeros(z.shape)
        hot[np.arange(t.size), label[t]] = 1.0
        P = alpha * (both[:, None] * p - gloss[t][:, None] * hot)
        # both is itself a rounded sum of two values
        size = (np.abs(gloss[t]) + (0.0 if glse is None else np.abs(glse[t])))[:, None]
        dP = abs(alpha) * (size * p * (2 * dz + 2 * U * (np.abs(z) + 2 * np.abs(lse[t][:, None])) + 12 * U)
                           + 4 * U * np.abs(gloss[t])[:, None] * hot)
        dP += np.where(hot == 1.0, 4 * U, v) * (np.abs(P) + dP) + 2.0 ** -126
        A = np.abs(P) + dP
        gX[t] = P @ w
        bX[t] = dP @ np.abs(w) + (V + 8) * U * (A @ np.abs(w))
        gW = gW + P.T @ x
        bW = bW + dP.T @ np.abs(x) + (t.size + 8) * U * (A.T @ np.abs(x))
    # the last rounding; a result below the normal range may be lost likewise
    tiny = 2.0 ** -126
    return gW, gX, bW + v * (np.abs(gW) + bW) + tiny, bX + v * (np.abs(gX) + bX) + tiny
