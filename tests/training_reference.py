"""Plain 64-bit forms of the training operators (word embedding, block norm, AdamW) and the bounds their results are held
to, for the tests.

Bounds are first-order rounding analysis.  u = 2^-24 is half a step of fp32 relative to the value.  A sum of n fp32 terms
taken in any order is off by at most n u (sum of the magnitudes); the kernels' row sums have at most 32 terms in a thread's
chain, six shuffle levels and 16 wavefronts, so a factor of C = 64 (sums, the products under them, the square root and the
division) covers a row's statistics.  For the rest every intermediate is carried along with its magnitude, the same formula
on absolute values: a result is off by at most C u times that magnitude, and by half a step of its storage type
(bf16: 2^-8 relative) once.
"""
import numpy as np

U = 2.0 ** -24
BF16 = 2.0 ** -8      # half a step of bf16, relative to the value (bf16 eps / 2)
C = 64.0
TINY = 1e-38


def bf16(x):
    """Round to bf16 (nearest even), as float64."""
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    r = ((b + (0x7FFF + ((b >> 16) & 1))) >> 16).astype(np.uint32) << 16
    return r.view(np.float32).astype(np.float64)


def storage(type_):
    return BF16 if type_ == "bfloat16" else U


# ---- embedding ------------------------------------------------------------------------------------------------
def valid_ids(ids, vocabulary):
    """Ids as the operator reads them: -1 where there is no token."""
    ids = np.asarray(ids)
    if ids.dtype.kind == "f":
        ok = np.isfinite(ids) & (ids > -1) & (ids < vocabulary)
        return np.where(ok, np.trunc(np.where(ok, ids, 0)), -1).astype(np.int64)
    return np.where((ids >= 0) & (ids < vocabulary), ids, -1).astype(np.int64)


def embedding_forward(ids, table, scale):
    t = valid_ids(ids, len(table)).reshape(-1)
    y = np.zeros((t.size, table.shape[1]))
    y[t >= 0] = float(np.float32(scale)) * table[t[t >= 0]].astype(np.float64)
    return y


def embedding_backward(ids, dy, vocabulary, scale, padding=-1):
    """(gradient, bound): a row of n tokens is a sum of n terms and one product."""
    t = valid_ids(ids, vocabulary).reshape(-1)
    keep = (t >= 0) & (t != padding)
    g, mag, n = np.zeros((vocabulary, dy.shape[1])), np.zeros((vocabulary, dy.shape[1])), np.zeros(vocabulary)
    np.add.at(g, t[keep], dy[keep].astype(np.float64))
    np.add.at(mag, t[keep], np.abs(dy[keep].astype(np.float64)))
    np.add.at(n, t[keep], 1)
    s = float(np.float32(scale))
    return s * g, (n[:, None] + 2) * U * abs(s) * mag + TINY


# ---- block norm -----------------------------------------------------------------------------------------------
def act(g, name):
    g = g.astype(np.float64)
    if name == "sigmoid":
        q = 1 / (1 + np.exp(-g))
        return q, q * (1 - q)
    if name == "tanh":
        q = np.tanh(g)
        return q, 1 - q * q
    return g, np.ones_like(g)


def statistics(z, kind, eps):
    z = z.astype(np.float64)
    mean = z.mean(1, keepdims=True) if kind == "layer" else np.zeros((len(z), 1))
    return mean, 1 / np.sqrt(((z - mean) ** 2).mean(1, keepdims=True) + eps)


def _one(v, dim):
    return np.ones(dim) if v is None else v.astype(np.float64)


def _zero(v, dim):
    return np.zeros(dim) if v is None else v.astype(np.float64)


def gate_per_row(gate, gate_rows, rows, dim):
    if gate is None:
        return None
    return np.broadcast_to(gate, (rows, dim)) if gate_rows == 0 else gate[np.arange(rows) // gate_rows]


def block_norm_forward(x, y, gate, gate_rows, pre, post, weights, scale, eps, activation, stream, block):
    """{name: (value, bound)} of u, h and the statistics; weights: dict of vectors by name (missing: ones / zeros)."""
    rows, dim = x.shape
    out = {}
    u, z = x.astype(np.float64), None
    if y is not None:
        z = y.astype(np.float64)
        n, mag = z, np.abs(z)
        if post:
            mean, rstd = statistics(z, post, eps)
            w, b = _one(weights.get("post_weight"), dim), _zero(weights.get("post_bias"), dim)
            n = (z - mean) * rstd * w + b
            mag = (np.abs(z) + np.abs(z).mean(1, keepdims=True)) * rstd * np.abs(w) + np.abs(b)
            out["post_statistics"] = _statistics_out(z, mean, rstd, post)
        g = gate_per_row(gate, gate_rows, rows, dim)
        if g is not None:
            q, _ = act(g, activation)
            n, mag = n * q, mag * np.abs(q)
        s = float(np.float32(scale))
        v = u + s * n
        err = C * U * (np.abs(u) + abs(s) * mag)
        out["u"] = v, err + storage(stream) * np.abs(v) + TINY
        u = v
        if stream == "bfloat16":  # the norm reads u as stored: a neighbour of the reference's u at most
            u, extra = bf16(v), err + 2 * BF16 * np.abs(v)
        else:
            extra = err + U * np.abs(v)
    else:
        extra = np.zeros_like(u)
    if pre:
        mean, rstd = statistics(u, pre, eps)
        w, b = _one(weights.get("pre_weight"), dim), _zero(weights.get("pre_bias"), dim)
        h = (u - mean) * rstd * w + b
        mag = (np.abs(u) + np.abs(u).mean(1, keepdims=True)) * rstd * np.abs(w) + np.abs(b)
        # an error of u moves h by rstd w (its own, the mean's, and through the deviation hat times the mean of |hat| err)
        hat = np.abs((u - mean) * rstd)
        moved = rstd * np.abs(w) * (extra + extra.mean(1, keepdims=True) + hat * (hat * extra).mean(1, keepdims=True))
        out["h"] = h, C * U * mag + moved + storage(block) * np.abs(h) + TINY
        mean_v, rstd_v = _statistics_out(u, mean, rstd, pre)
        rel = (hat * extra * rstd).mean(1, keepdims=True)
        out["pre_statistics"] = mean_v, rstd_v + np.concatenate((extra.mean(1, keepdims=True), rstd * rel), 1)
    return out


def _statistics_out(z, mean, rstd, kind):
    bound = np.concatenate((C * U * np.abs(z).mean(1, keepdims=True), C * U * rstd * (1 + np.abs(mean) * rstd)), 1)
    return np.concatenate((mean, rstd), 1), bound + TINY


def block_norm_backward(u, dh, du, y, gate, gate_rows, pre, post, weights, stats, scale, activation, stream, block):
    """{name: (value, bound)}; stats: {"pre": (rows, 2), "post": (rows, 2)} as the kernel is given them (fp32)."""
    rows, dim = (du if du is not None else dh).shape
    out = {}

    def back(z, dn, dn_mag, which, kind):
        mean, rstd = stats[which][:, :1].astype(np.float64), stats[which][:, 1:].astype(np.float64)
        w = _one(weights.get(which + "_weight"), dim)
        hat, hat_mag = (z - mean) * rstd, (np.abs(z) + np.abs(mean)) * rstd
        out["d_%s_weight" % which] = (dn * hat).sum(0), (rows + C) * U * (dn_mag * hat_mag).sum(0) + TINY
        out["d_%s_bias" % which] = dn.sum(0), (rows + C) * U * dn_mag.sum(0) + TINY
        a, a_mag = dn * w, dn_mag * np.abs(w)
        level = a.mean(1, keepdims=True) if kind == "layer" else 0.0
        level_mag = a_mag.mean(1, keepdims=True) if kind == "layer" else 0.0
        dz = rstd * (a - level - hat * (a * hat).mean(1, keepdims=True))
        return dz, rstd * (a_mag + level_mag + hat_mag * (a_mag * hat_mag).mean(1, keepdims=True))

    t = np.zeros((rows, dim)) if du is None else du.astype(np.float64)
    mag = np.abs(t)
    if dh is not None:
        d = dh.astype(np.float64)
        a, m = back(u.astype(np.float64), d, np.abs(d), "pre", pre)
        t, mag = t + a, mag + m
    out["dx"] = t, C * U * mag + storage(stream) * np.abs(t) + TINY
    if y is None:
        return out
    s = float(np.float32(scale))
    t, mag = s * t, abs(s) * mag
    z = y.astype(np.float64)
    g = gate_per_row(gate, gate_rows, rows, dim)
    if g is not None:
        q, slope = act(g, activation)
        n, n_mag = z, np.abs(z)
        if post:
            mean, rstd = stats["post"][:, :1].astype(np.float64), stats["post"][:, 1:].astype(np.float64)
            w, b = _one(weights.get("post_weight"), dim), _zero(weights.get("post_bias"), dim)
            n, n_mag = (z - mean) * rstd * w + b, (np.abs(z) + np.abs(mean)) * rstd * np.abs(w) + np.abs(b)
        dq, dq_mag = t * n * slope, mag * n_mag * (np.abs(slope) + (1.0 if activation in ("sigmoid", "tanh") else 0.0))
        if gate_rows == 0:
            out["d_gate"] = dq.sum(0), (rows + C) * U * dq_mag.sum(0) + TINY
        else:
            k = np.arange(rows) // gate_rows
            v, m = np.zeros((k[-1] + 1, dim)), np.zeros((k[-1] + 1, dim))
            np.add.at(v, k, dq)
            np.add.at(m, k, dq_mag)
            out["d_gate"] = v, (gate_rows + C) * U * m + storage(block) * np.abs(v) + TINY
        t, mag = t * q, mag * np.abs(q)
    if post:
        t, mag = back(z, t, mag, "post", post)
    out["dy"] = t, C * U * mag + storage(block) * np.abs(t) + TINY
    return out


# ---- AdamW ----------------------------------------------------------------------------------------------------
E4M3 = np.array([np.nan if (b & 0x7F) == 0x7F else (-1.0 if b & 0x80 else 1.0) *
                 ((b & 7) / 8 * 2.0 ** -6 if (b >> 3) & 15 == 0 else (1 + (b & 7) / 8) * 2.0 ** (((b >> 3) & 15) - 7))
                 for b in range(256)], dtype=np.float32)
E5M2 = np.array([np.nan if (b & 0x7F) > 0x7C else (-1.0 if b & 0x80 else 1.0) *
                 (np.inf if (b & 0x7F) == 0x7C else (b & 3) / 4 * 2.0 ** -14 if (b >> 2) & 31 == 0
                  else (1 + (b & 3) / 4) * 2.0 ** (((b >> 2) & 31) - 15)) for b in range(256)], dtype=np.float32)


def power(e):
    return ((np.asarray(e, dtype=np.int64) + 127) << 23).astype(np.uint32).view(np.float32)


def moments(m, v, g, beta1, beta2):
    """m' and v' in fp32, every product and sum rounded by itself: the kernels give these bits."""
    f = np.float32
    with np.errstate(over="ignore", invalid="ignore"):
        return m * f(beta1) + g * f(1 - beta1), v * f(beta2) + (g * g) * f(1 - beta2)


def new_parameters(p, m, v, rate, decay, beta1, beta2, eps, step):
    """(p', bound) from fp32 m' and v'."""
    p, m, v = (a.astype(np.float64) for a in (p, m, v))
    move = rate / (1 - beta1 ** step) * m / (np.sqrt(v) / np.sqrt(1 - beta2 ** step) + eps)
    new = p * (1 - rate * decay) - move
    # p: rate, decay, their product, 1 - it, the product with p, the difference; the move: step size, square root (and its
    # factor and product), epsilon, sum, division, product
    return new, U * (4 * np.abs(p) + 12 * np.abs(move) + np.abs(new)) + TINY


def philox(counter, key):
    """Philox4x32-10 on uint64 arrays holding 32-bit words."""
    c = [np.asarray(x, dtype=np.uint64) for x in counter]
    k0, k1 = key
    lo = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & lo, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & lo]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def random_words(count, tensor, step, seed):
    quad = np.arange((count + 3) // 4, dtype=np.uint64)
    z = np.zeros_like(quad)
    words = philox((quad & np.uint64(0xFFFFFFFF), quad >> np.uint64(32), z + np.uint64(tensor), z + np.uint64(step)),
                   (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    return np.stack(words, 1).reshape(-1)[:count].astype(np.int64)


def load8(codes, scales, table):
    unit = np.repeat(power(scales.astype(np.int64) - 127) * (scales > 0), 256)[:codes.size]
    with np.errstate(invalid="ignore"):
        return (table[codes] * unit).astype(np.float32)


def store8(x, room, mantissa, lowest, random, table, never_zero):
    """(codes, scales) of fp32 moments."""
    n = x.size
    pad = np.zeros(-n % 256, np.float32)
    finite = np.isfinite(x)
    blocks = np.concatenate((np.where(finite, np.abs(x), 0).astype(np.float32), pad)).reshape(-1, 256)
    scales = np.maximum((blocks.max(1).view(np.uint32) >> 23).astype(np.int64) - room, 1)
    a = np.where(finite, np.abs(x), 0).astype(np.float32) * np.repeat(power(127 - scales), 256)[:n]
    e = np.maximum((a.view(np.uint32) >> 23).astype(np.int64) - 127, lowest)
    k = ((a * power(23 - e)).astype(np.int64) + (random << (7 - mantissa))) >> (23 - mantissa)
    if never_zero:
        k = np.where((k == 0) & (a > 0), 1, k)
    value = np.copysign(k.astype(np.float32) * power(e - mantissa), x)
    positive = np.where(np.isnan(table[:128]), np.inf, table[:128])
    code = np.searchsorted(positive, np.abs(value)).astype(np.uint8)
    assert np.array_equal(table[code], np.abs(value))
    code = np.where(np.signbit(value), code | 0x80, code)
    return np.where(finite, code, 0x7F).astype(np.uint8), scales.astype(np.uint8)


def store_m(m, random):
    return store8(m, 7, 3, -6, random & 0xFFFF, E4M3, False)


def store_v(v, random):
    return store8(v, 14, 2, -14, random >> 16, E5M2, True)
