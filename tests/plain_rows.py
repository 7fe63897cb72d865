"""Plain 64-bit forms of the operators over plain rows, and the helpers their
tests share.  Arrays are numpy; the GPU tests move them with torch."""
import numpy as np

import gotransformers_amd as gt

VALUES = {"f32": gt.VALUES_FLOAT32, "bf16": gt.VALUES_BFLOAT16, "f16": gt.VALUES_FLOAT16}
# half a step of each type relative to the value
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# and absolutely, where the value is below the type's normal numbers: fp16's
# steps stay 2^-24 from 2^-14 down, so a rounding there is off by up to 2^-25
HALF_LAST_STEP = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}


def philox4x32(counter, key, rounds=10):
    """Philox4x32 (Salmon et al., SC 2011): four uint32 arrays of counters and
    two key words to four uint32 arrays."""
    mask = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & mask,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [v.astype(np.uint32) for v in c]


def dropout_threshold(rate):
    return min(int(np.floor(rate * 65536 + 0.5)), 65535)


def dropout_factor(rows, columns, rate, seed, offset):
    """scale at the kept places of the mask, 0 at the dropped ones, and the mask."""
    blocks = (columns + 7) // 8
    b, r = np.meshgrid(np.arange(blocks), np.arange(rows))
    words = philox4x32([b, r, np.full_like(b, offset & 0xFFFFFFFF), np.full_like(b, offset >> 32)],
                       [seed & 0xFFFFFFFF, seed >> 32])
    halves = [h for w in words for h in (w & np.uint32(0xFFFF), w >> np.uint32(16))]
    bits = np.stack(halves, axis=2).reshape(rows, 8 * blocks)[:, :columns]
    t = dropout_threshold(rate)
    keep = bits >= t
    return np.where(keep, 65536.0 / (65536 - t), 0.0), keep


def grouped(offsets, x, w, dy):
    """(y, dx, dw) of every group in 64 bits; rows in no group stay zero."""
    y = np.zeros((x.shape[0], w.shape[1]))
    dx = np.zeros(x.shape)
    dw = np.zeros(w.shape)
    for g in range(len(offsets) - 1):
        at = slice(offsets[g], offsets[g + 1])
        y[at], dx[at], dw[g] = x[at] @ w[g].T, dy[at] @ w[g], dy[at].T @ x[at]
    return y, dx, dw


def adapted(x, w, b, adapter, down, up, scales, base=None):
    """y and the sum of its terms' magnitudes, in 64 bits."""
    y = x @ w.T if w is not None else base.copy()
    size = np.abs(x) @ np.abs(w).T if w is not None else np.abs(base)
    if b is not None:
        y, size = y + b, size + np.abs(b)
    adapter = np.asarray(adapter)
    for a in np.unique(adapter):
        if 0 <= a < len(scales):
            t = adapter == a
            y[t] += scales[a] * (x[t] @ down[a].T @ up[a].T)
            size[t] += abs(scales[a]) * (np.abs(x[t]) @ np.abs(down[a]).T @ np.abs(up[a]).T)
    return y, size


def offsets_of(sizes, first=0):
    return np.concatenate([[first], first + np.cumsum(sizes)]).astype(np.int32)
