"""Mixture-of-experts layer in 64 bits, and bounds on the kernels' errors."""
import numpy as np

# code bytes of a block: zeroed, a block decodes to minus its minimums' part
CODES = {"Q2_K": [(20, 84)], "Q3_K": [(0, 96)], "Q4_K": [(16, 144)], "Q5_K": [(16, 176)], "Q6_K": [(0, 192)]}
BLOCK = {"Q8_0": (32, 34), "Q4_0": (32, 18), "Q2_K": (256, 84), "Q3_K": (256, 110), "Q4_K": (256, 144),
         "Q5_K": (256, 176), "Q6_K": (256, 210)}


class Weights:
    """Experts' packed rows, their values and the magnitudes that the kernel adds up: codes and minimums apart."""

    def __init__(self, orc, fmt, experts, rows, cols, rng, scale=1.0):
        self.fmt, self.shape = fmt, (experts, rows, cols)
        w = (rng.standard_normal((experts * rows, cols)) * scale).astype(np.float32)
        self.packed = orc.quantize(fmt, w)
        self.value = orc.dequantize(fmt, self.packed, experts * rows, cols).astype(np.float64).reshape(self.shape)
        self.size = np.abs(self.value)
        if fmt in CODES:
            be, bb = BLOCK[fmt]
            z = self.packed[: experts * rows * -(-cols // be) * bb].reshape(-1, bb).copy()
            for a, b in CODES[fmt]:
                z[:, a:b] = 0
            low = orc.dequantize(fmt, z.reshape(-1), experts * rows, cols).astype(np.float64).reshape(self.shape)
            self.size = np.abs(self.value - low) + np.abs(low)


def silu(v):
    with np.errstate(over="ignore"):
        return v / (1 + np.exp(-v))


def product_error(cols):
    """Relative to the sum of magnitudes: x in two fp16 terms (2^-22 of x, 2^-33 of the largest in its 256), codes
    exact; 256 terms and 16 minimums added in fp32 on the tensor core (each addition off by 2^-23 at most, as it may
    truncate), then one scale each and a sum over groups of 256 and eight warps."""
    return 2.0 ** -21 + (272 + -(-cols // 256) + 24) * 2.0 ** -23


def layer(x, ids, p, gate, up, down, eps):
    """(y, bound) for x [N x hidden] (float64 values of what the kernel gets)."""
    experts, ffn, hidden = gate.shape
    y, tol = np.zeros((x.shape[0], hidden)), np.zeros((x.shape[0], hidden))
    c1, c2 = product_error(hidden), product_error(ffn)
    big = np.abs(x).max(axis=1) if x.size else np.zeros(x.shape[0])
    for t in range(x.shape[0]):
        mag = np.zeros(hidden)
        for j in range(ids.shape[1]):
            e = ids[t, j]
            if not 0 <= e < experts:
                continue
            g, u = gate.value[e] @ x[t], up.value[e] @ x[t]
            low = 2.0 ** -33 * big[t]
            dg = c1 * (gate.size[e] @ np.abs(x[t])) + low * gate.size[e].sum(1)
            du = c1 * (up.size[e] @ np.abs(x[t])) + low * up.size[e].sum(1)
            h = silu(g) * u
            dh = 1.1 * dg * (np.abs(u) + du) + np.abs(silu(g)) * du + 8 * 2.0 ** -24 * np.abs(h)
            z = down.value[e] @ h
            dz = c2 * (down.size[e] @ (np.abs(h) + dh)) + np.abs(down.value[e]) @ dh
            if eps == 2.0 ** -7:  # a bf16 result: h enters the second product as one fp16 (half a step: 2^-11 of it)
                dz = dz + 2.0 ** -11 * (np.abs(down.value[e]) @ (np.abs(h) + dh))
            dz = dz + 2.0 ** -33 * (np.abs(h) + dh).max(initial=0) * down.size[e].sum(1)
            w = float(p[t, j])
            y[t] += w * z
            tol[t] += abs(w) * dz
            mag += abs(w) * np.abs(z)
        tol[t] += (ids.shape[1] + 2) * 2.0 ** -24 * mag + eps / 2 * (np.abs(y[t]) + tol[t]) + 1e-30
    return y, tol


def route(x, w, top_k):
    """(ids, logits, largest logit error) in 64 bits; the kernel adds hidden products in fp32."""
    logits = x @ w.T
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :top_k]
    err = (x.shape[1] / 32 + 8) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T)
    return ids, logits, err
