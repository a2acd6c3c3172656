"""AdamW with moments in 32 or 8 bits, restated in numpy: what rhp_adamw_step is tested against.

``update`` runs the step in one float type, operation by operation; with
float32 it is what the kernel does, with float64 the mathematics.  ``weight``
is its last line alone, from given moments.  The 8-bit
moments are integer arithmetic on the float32 moments' bits, so codes can be
compared exactly.
"""

from __future__ import annotations

import numpy as np

BLOCK = 128
M32 = 0xFFFFFFFF


def update(p, g, m, v, dtype, lr, betas, eps, weight_decay, step, scale=1.0, decay=True):
    """New (p, m, v) as arrays of ``dtype``; ``scale`` multiplies the gradient."""
    t = np.dtype(dtype).type
    b1, b2 = betas
    c1, c2 = t(1.0 - b1), t(1.0 - b2)
    g, m, v = (np.asarray(x).astype(dtype) for x in (g, m, v))
    with np.errstate(all="ignore"):
        g = g * t(scale)
        m = m * t(b1) + g * c1
        v = v * t(b2) + (g * c2) * g
    return weight(p, m, v, dtype, lr, betas, eps, weight_decay, step, decay), m, v


def weight(p, m, v, dtype, lr, betas, eps, weight_decay, step, decay=True):
    """The stepped weight from the stepped moments."""
    t = np.dtype(dtype).type
    b1, b2 = betas
    ibc2s = t(1.0 / np.sqrt(1.0 - b2 ** float(step)))
    a = t(lr / (1.0 - b1 ** float(step)))
    keep = t(1.0 - lr * weight_decay) if decay else t(1.0)
    p, m, v = (np.asarray(x).astype(dtype) for x in (p, m, v))
    with np.errstate(all="ignore"):
        return p * keep - a * (m / (np.sqrt(v) * ibc2s + t(eps)))


def mix(x):
    """A 32-bit hash: lowbias32 as C. Wellons published it (hash prospector)."""
    x = np.asarray(x, np.uint64) & np.uint64(M32)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D)) & np.uint64(M32)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x846CA68B)) & np.uint64(M32)
    return x ^ (x >> np.uint64(16))


def random_bits(n: int, seed: int, step: int, key: int, first: int = 0) -> np.ndarray:
    """32 random bits for each of n elements from index ``first`` on: a hash of (seed, step, key, index)."""
    salt = mix(int(mix(int(mix((step & M32) ^ (step >> 32))) ^ ((seed >> 32) & M32))) ^ (seed & M32))
    i = np.arange(first, first + n, dtype=np.uint64)
    x = mix((mix(np.uint64(key) ^ salt) + (i >> np.uint64(3))) & np.uint64(M32))
    x = (x + (i & np.uint64(7)) * np.uint64(0x9E3779B9)) & np.uint64(M32)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D)) & np.uint64(M32)
    return (x ^ (x >> np.uint64(15))).astype(np.int64)


def _blocks(bits: np.ndarray) -> np.ndarray:
    """[blocks, 128], the last block filled up with zeros."""
    out = np.zeros(-(-bits.size // BLOCK) * BLOCK, np.int64)
    out[: bits.size] = bits
    return out.reshape(-1, BLOCK)


def _exponent(mag: np.ndarray) -> np.ndarray:
    return np.minimum((mag.max(1) + 0xFFFFF) >> 23, 255)


def encode(m: np.ndarray, v: np.ndarray, r: np.ndarray):
    """(codes of m, codes of v, scales [blocks, 2]) of float32 moments under the random bits r."""
    n = m.size
    bm = m.astype(np.float32).view(np.uint32).astype(np.int64)
    bv = v.astype(np.float32).view(np.uint32).astype(np.int64)
    mag_m, mag_v = _blocks(bm & 0x7FFFFFFF), _blocks(bv & 0x7FFFFFFF)
    em, ev = _exponent(mag_m), _exponent(mag_v)
    rm, rv = _blocks(r & 0xFFFF), _blocks(r >> 16)
    cm = np.maximum(((mag_m + (rm << 4)) >> 20) - 8 * np.maximum(em - 15, 0)[:, None], 0)
    cm |= _blocks(bm >> 31) << 7
    with np.errstate(invalid="ignore"):
        pos = _blocks((v > 0).astype(np.int64)) > 0
    cv = np.maximum(((mag_v + (rv << 4)) >> 20) - 8 * np.maximum(ev - 31, 0)[:, None], 1)
    cv = np.where(pos, cv, 0)
    cm[em == 255] = 0
    cv[ev == 255] = 0
    return (cm.reshape(-1)[:n].astype(np.uint8), cv.reshape(-1)[:n].astype(np.uint8),
            np.stack([em, ev], 1).astype(np.uint8))


def decode(qm: np.ndarray, qv: np.ndarray, scales: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    n = qm.size
    em, ev = scales[:, 0].astype(np.int64), scales[:, 1].astype(np.int64)
    cm, cv = _blocks(qm.astype(np.int64)), _blocks(qv.astype(np.int64))
    c = cm & 127
    bits = np.where(c > 0, ((c + 8 * np.maximum(em - 15, 0)[:, None]) << 20) | ((cm & 128) << 24), 0)
    m = (bits & M32).astype(np.uint32).view(np.float32).copy()
    bits = np.where(cv > 0, (cv + 8 * np.maximum(ev - 31, 0)[:, None]) << 20, 0)
    v = (bits & M32).astype(np.uint32).view(np.float32).copy()
    m[em == 255] = np.nan
    v[ev == 255] = np.nan
    return m.reshape(-1)[:n], v.reshape(-1)[:n]


def nearest(n: int) -> np.ndarray:
    """The bits that round to the nearest code."""
    return np.full(n, 0x80008000, np.int64)
