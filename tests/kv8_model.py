"""The 8-bit cache, rotary positions and attention from their definitions, in float64 numpy."""
import numpy as np

HD, BLOCK, E_MIN, E_MAX = 256, 64, -60, 119


def code_values():
    """The 256 e4m3 values by their fields (code 0x7f / 0xff: NaN)."""
    c = np.arange(256)
    ex, man = (c >> 3) & 15, c & 7
    v = np.where(ex == 0, man * 2.0 ** -9, (1 + man / 8) * 2.0 ** (ex - 7.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


VALUES = code_values()


def to_code(x):
    """Nearest e4m3 code, ties to the even mantissa, largest magnitude 448."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    ex = np.maximum(np.frexp(np.where(a > 0, a, 1.0))[1] - 1, -6)
    n = np.rint(a * 2.0 ** (3.0 - ex)).astype(np.int64)       # 8 .. 16 steps (normal), 0 .. 8 (subnormal)
    up = n >= 16
    ex, n = np.where(up, ex + 1, ex), np.where(up, 8, n)
    code = np.where(n >= 8, ((ex + 7) << 3) | (n & 7), n)
    code = np.minimum(code, 0x7E)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def needed(amax):
    """Smallest e in range with amax <= 448 * 2^e."""
    if amax == 0:
        return E_MIN
    m, k = np.frexp(np.float64(amax))                        # 448 = 0.875 * 2^9
    return int(np.clip(k - 9 + (1 if m > 0.875 else 0), E_MIN, E_MAX))


class Cache:
    """One layer of K or V."""

    def __init__(self, kv_heads, ctx):
        self.codes = np.zeros((kv_heads, ctx, HD), np.uint8)
        self.exps = np.full((kv_heads, -(-ctx // BLOCK)), E_MIN, np.int64)

    def append(self, x, base):
        """x [rows, kv_heads, 256] at positions [base, base + rows)."""
        rows = x.shape[0]
        for h in range(x.shape[1]):
            for b in range(base // BLOCK, -(-(base + rows) // BLOCK)):
                t0 = b * BLOCK
                lo, hi = max(t0, base), min(t0 + BLOCK, base + rows)
                new = np.asarray(x[lo - base:hi - base, h], np.float64)
                new = np.where(np.isnan(new), 0.0, new)
                fin = np.abs(new[np.isfinite(new)])
                e = needed(fin.max() if fin.size else 0.0)
                if lo > t0:
                    was = int(self.exps[h, b])
                    e = max(e, was)
                    if e > was:
                        self.codes[h, t0:lo] = to_code(VALUES[self.codes[h, t0:lo]] * 2.0 ** (was - e))
                self.codes[h, lo:hi] = to_code(np.where(np.isinf(new), np.sign(new) * 1e300, new) * 2.0 ** -e)
                self.exps[h, b] = e

    def values(self, lo, hi):
        e = self.exps[:, np.arange(lo, hi) // BLOCK]
        return VALUES[self.codes[:, lo:hi]] * 2.0 ** e[..., None].astype(np.float64)

    def layer_bytes(self):
        """The plain buffer's bytes."""
        n = self.codes.size + self.exps.size
        out = np.zeros(-(-n // 256) * 256, np.uint8)
        out[:self.codes.size] = self.codes.ravel()
        out[self.codes.size:n] = (self.exps + 127).astype(np.uint8).ravel()
        return out


def attention(q, k, v, base, scale, gate=None):
    """q [rows, q_heads, 256], k and v [kv_heads, base + rows, 256] -> [rows, q_heads, 256]."""
    rows, qh, _ = q.shape
    grp = qh // k.shape[0]
    seen = np.arange(base + rows)[None] <= base + np.arange(rows)[:, None]
    out = np.empty(q.shape, np.float64)
    for h in range(qh):
        s = np.where(seen, q[:, h].astype(np.float64) @ k[h // grp].T * scale, -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        out[:, h] = (w @ np.where(np.isfinite(v[h // grp]), v[h // grp], 0.0)) / w.sum(1, keepdims=True)
    if gate is not None:
        out = out / (1 + np.exp(-gate.astype(np.float64)))
    return out


def rope(x, pos, freq, rotary, interleaved, amp=1.0):
    """x [rows, heads, head_dim]."""
    y = np.array(x, np.float64)
    a = pos.astype(np.float64)[:, None] * freq.astype(np.float64)
    co, si = np.cos(a)[:, None] * amp, np.sin(a)[:, None] * amp
    i0 = np.arange(0, rotary, 2) if interleaved else np.arange(rotary // 2)
    i1 = i0 + 1 if interleaved else i0 + rotary // 2
    x0, x1 = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = x0 * co - x1 * si, x1 * co + x0 * si
    return y
