"""Plain 64-bit forms of the operators without a layer, on the host, and what the tests share."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# A rounding to the type is off by half a step at most.
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def route(logits, n_used, score="softmax", bias=None, n_groups=1, n_groups_used=1, renorm=True, scale=1.0):
    """ids, w, offsets, inv of logits [T][E] (64 bits), row by row from the definition."""
    T, E = logits.shape
    ids, w = np.full((T, n_used), -1, np.int32), np.zeros((T, n_used))
    for t in range(T):
        l = logits[t]
        b = np.zeros(E) if bias is None else bias.astype(np.float64)
        there = (l > -np.inf) & (b > -np.inf)  # false for NaN too
        if not there.any():
            continue
        e = np.where(there, l, -np.inf)
        with np.errstate(over="ignore", invalid="ignore"):
            if score == "softmax":
                top = e.max()
                p = np.where(e == top, 1.0, np.exp(e - top))
                p[~there] = 0
                s = p / p.sum()
            else:
                s = 1 / (1 + np.exp(-e))
        key = np.where(there, s + b, -np.inf)
        if n_groups > 1:
            rank = []
            for g in key.reshape(n_groups, -1):
                best = sorted((v for v in g if v > -np.inf), reverse=True)[:2]
                rank.append(sum(best) if best else -np.inf)
            stay = sorted((g for g in range(n_groups) if rank[g] > -np.inf), key=lambda g: (-rank[g], g))[:n_groups_used]
            key = np.where(np.isin(np.arange(E) // (E // n_groups), stay), key, -np.inf)
        order = key if bias is not None else np.where(key > -np.inf, l, -np.inf)
        chosen = sorted((i for i in range(E) if order[i] > -np.inf), key=lambda i: (-order[i], i))[:n_used]
        ids[t, :len(chosen)] = chosen
        if renorm:
            # In logarithms, so that scores too small for 64 bits keep their proportions.
            lc = l[chosen]
            with np.errstate(over="ignore"):
                ls = np.where(lc == np.inf, 0.0, lc) if score == "softmax" else -np.logaddexp(0, -lc)
            if score == "softmax" and (lc == np.inf).any():
                ls = np.where(lc == np.inf, 0.0, -np.inf)
            p = np.exp(ls - ls.max())
            w[t, :len(chosen)] = p / p.sum()
        else:
            w[t, :len(chosen)] = s[chosen]
    flat = ids.reshape(-1)
    inv = np.full(flat.size, -1, np.int32)
    offsets = np.zeros(E + 1, np.int32)
    row = 0
    for e in range(E):
        for a in np.flatnonzero(flat == e):
            inv[a] = row
            row += 1
        offsets[e + 1] = row
    return ids, w * scale, offsets, inv.reshape(T, n_used)


def scale_row_bytes(K):
    return (K // 32 + 3) // 4 * 4


def quantize(x):
    """Codes (one a byte, [R][K]) and scale bytes [R][K / 32] of rows x, in 64 bits."""
    b = np.asarray(x, np.float64).reshape(x.shape[0], -1, 32)
    top = np.abs(b).max(2)
    bad = ~np.isfinite(top)
    m, e = np.frexp(np.where(bad, 1.0, top))
    byte = np.where(top > 0, np.maximum(e - 1 - 2, -127) + 127, 0)
    v = np.where(bad[..., None], 0.0, b) * np.exp2(127.0 - byte)[..., None]
    a = np.abs(v)
    code = sum((a > t).astype(np.uint8) for t in (0.25, 1.25, 2.5, 5.0)) + sum((a >= t).astype(np.uint8) for t in (0.75, 1.75, 3.5))
    code = (code + 8 * (np.signbit(v) & ~bad[..., None])).astype(np.uint8)
    return code.reshape(x.shape[0], -1), np.where(bad, 255, byte).astype(np.uint8)


def values(code, byte):
    """What codes (one a byte) and scale bytes stand for."""
    v = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return v * np.repeat(s, 32, axis=-1)


def pack(code, byte):
    """As the device holds them: two codes a byte, scale rows filled up with zeros."""
    s = np.zeros(byte.shape[:-1] + (scale_row_bytes(code.shape[-1]),), np.uint8)
    s[..., :byte.shape[-1]] = byte
    return np.ascontiguousarray(code[..., 0::2] | code[..., 1::2] << 4), s


def unpack(codes, scales):
    c = np.empty(codes.shape[:-1] + (codes.shape[-1] * 2,), np.uint8)
    c[..., 0::2], c[..., 1::2] = codes & 15, codes >> 4
    return c, scales[..., :c.shape[-1] // 32]


def random_mx(rng, shape, lo=119, hi=124):
    """Random codes and scales: ((codes, scales) as the device holds them, values)."""
    code = rng.integers(0, 16, shape, dtype=np.uint8)
    byte = rng.integers(lo, hi, shape[:-1] + (shape[-1] // 32,), dtype=np.uint8)
    return pack(code, byte), values(code, byte)


def swiglu(g, u, limit):
    if limit > 0:
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u
