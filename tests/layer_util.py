"""Plain forms of the layer loop's attention operators in 64 bits (numpy, CPU), for the tests."""
import numpy as np

NO_SLOT = 0xFFFFFFFF


def bf16(x):
    """x rounded to BF16 (nearest even), as float32."""
    u = np.asarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def bf16_bits(x):
    return (bf16(x).view(np.uint32) >> 16).astype(np.uint16)


def outward(x, up):
    """float32 x rounded to BF16 upwards or downwards, staying finite."""
    r = bf16(x)
    step = np.where(r.view(np.uint32) >> 31 == (0 if up else 1), 0x10000, -0x10000).astype(np.int64)
    wrong = (r < x) if up else (r > x)
    # one BF16 number further: up in magnitude away from zero, down towards it; past zero is the smallest of that sign
    bits = r.view(np.uint32).astype(np.int64) + np.where(wrong, step, 0)
    least = np.float32(np.array(0x10000, np.uint32).view(np.float32) * (1 if up else -1))
    return np.where(wrong & (r == 0), least, bits.astype(np.uint32).view(np.float32)).astype(np.float32)


def quantise(x, bits):
    """(codes, scale, bias) of the last axis's groups of 64, in the fp32 operations that define the format."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 64, 64)
    top = 2**bits - 1
    finite = (np.abs(g) < 2.0**103).all(axis=-1)
    safe = np.where(finite[..., None], g, np.float32(0))
    lo, hi = safe.min(axis=-1), safe.max(axis=-1)
    bias = outward(lo, False)
    scale = np.maximum(outward((hi - bias) / np.float32(top), True), np.float32(2.0**-126))
    codes = np.clip(np.rint((safe - bias[..., None]) / scale[..., None]), 0, top)
    nan = np.float32(np.nan)
    return codes, np.where(finite, scale, nan), np.where(finite, bias, nan)


def stored(x, bits):
    """What the cache holds of float32 x, as float64."""
    c, s, b = quantise(x, bits)
    return (c.astype(np.float64) * s[..., None] + b[..., None]).reshape(x.shape)


def norm(x, eps, w=None):
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps)
    return y if w is None else y * np.asarray(w, np.float64)


def rotate(x, positions, inv_freq, pairs):
    """x [tokens, heads, head_dim] turned; angles in 80-bit floats, so that far positions stay exact."""
    x = np.array(x, np.float64)
    r = 2 * len(inv_freq)
    if r == 0:
        return x
    two_pi = np.longdouble("6.283185307179586476925286766559")
    turns = np.asarray(positions, np.longdouble)[:, None] * (np.asarray(inv_freq, np.longdouble) / two_pi)[None]
    angle = ((turns - np.floor(turns)) * two_pi)[:, None]
    c, s = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    a, b = (x[..., 0:r:2].copy(), x[..., 1:r:2].copy()) if pairs else (x[..., :r // 2].copy(), x[..., r // 2:r].copy())
    u, v = a * c - b * s, b * c + a * s
    if pairs:
        x[..., 0:r:2], x[..., 1:r:2] = u, v
    else:
        x[..., :r // 2], x[..., r // 2:r] = u, v
    return x


def pair_size(x, r, pairs):
    """|(a, b)| of each element's pair (|x| for an element that has none): what a rotation's rounding scales with."""
    x = np.abs(np.asarray(x, np.float64))
    out = x.copy()
    if r == 0:
        return out
    if pairs:
        h = np.hypot(x[..., 0:r:2], x[..., 1:r:2])
        out[..., 0:r:2], out[..., 1:r:2] = h, h
    else:
        h = np.hypot(x[..., :r // 2], x[..., r // 2:r])
        out[..., :r // 2], out[..., r // 2:r] = h, h
    return out


def attention(q, k, v, own_first, window, scale):
    """q [rows, heads, d] at positions own_first ..., over k, v [keys, kv_heads, d]: zeros for a row that
    sees nothing."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    g = q.shape[1] // k.shape[1]
    out = np.zeros_like(q)
    for i in range(q.shape[0]):
        p = own_first + i
        lo, hi = (max(0, p - window + 1) if window else 0), p + 1
        if hi <= lo:
            continue
        for h in range(q.shape[1]):
            s = k[lo:hi, h // g] @ q[i, h] * scale
            w = np.exp(s - s.max())
            out[i, h] = w @ v[lo:hi, h // g] / w.sum()
    return out
