"""Plain implementations of the cache-eviction and logit operators (64-bit, or bit by bit where the operator
defines every rounding), and the bounds their tests use."""
import numpy as np

QK, BLOCK = 32, 36
U = 2.0 ** -24  # half a step of fp32, relative


def codes(planes):
    """int8 codes [..., nb, 32] of a uint8 plane."""
    return planes.reshape(*planes.shape[:-1], -1, BLOCK)[..., 4:].view(np.int8)


def scales(planes):
    """fp32 scales [..., nb] of a uint8 plane."""
    return planes.reshape(*planes.shape[:-1], -1, BLOCK)[..., :4].copy().view(np.float32)[..., 0]


def values(planes):
    """The float64 values [..., head_dim] a plane stands for."""
    c = codes(planes)
    return (c.astype(np.float64) * scales(planes).astype(np.float64)[..., None]).reshape(*c.shape[:-2], -1)


def attend64(q_planes, k_planes, v_planes, lens):
    """float64 attention of q [items, n_q, row] over caches [items, n_kv, tokens, row].  Returns the output
    [items, n_q, hd], the weights summed per kv head [items, n_kv, tokens] and the largest sum of absolute block
    products of any score (times 1/sqrt(hd)), which scales the scores' rounding errors."""
    q = values(q_planes)
    items, n_q, hd = q.shape
    n_kv, tokens = k_planes.shape[1:3]
    g = n_q // n_kv
    out, weight, big = np.zeros((items, n_q, hd)), np.zeros((items, n_kv, tokens)), 0.0
    for i, n in enumerate(lens):
        if n == 0:
            continue
        k, v = values(k_planes[i, :, :n]), values(v_planes[i, :, :n])
        for h in range(n_q):
            kv = h // g
            blocks = (k[kv] * q[i, h]).reshape(n, -1, QK).sum(-1) / np.sqrt(hd)
            big = max(big, float(np.abs(blocks).sum(-1).max()))
            s = blocks.sum(-1)
            p = np.exp(s - s.max())
            w = p / p.sum()
            out[i, h] = w @ v[kv]
            weight[i, kv, :n] += w
    return out, weight, big


def weight_bound(nb, big, n):
    """Relative bound on one q head's attention weight e^(s - m) / l in fp32.
    A score adds nb block products: two roundings each (scale product, times the exact integer dot), nb - 1
    sums, then the scale and the log2(e) factors, so it is off by at most (nb + 4) u times the sum of absolute block
    products; likewise the subtraction of the maximum, of at most twice that size: 2 u big.  The exponent's error is
    the weight's relative error (base 2 scores times ln 2), once for the numerator and once for l.  ex2.approx is off by
    2^-22, in both.  l adds positive terms in chains of at most n / 64 steps (four warps, 16 tokens a step) plus the
    sums within a step, over warps and over splits (under 64 in all), u each; the reciprocal, the product and the sum over
    heads round once each."""
    return 2 * ((nb + 4) * U * big + 2 * U * big) + 2 * 2.0 ** -22 + (n / 64 + 64) * U + 4 * U


def evict_ref(weight, position, n, budget, n_first, n_recent):
    """Kept slots of one head's n rows (boolean) and the moves (dst, src)."""
    if n <= budget:
        none = np.zeros(0, int)
        return np.ones(n, bool), none, none
    w = weight[:n].astype(np.float64) + 0.0
    w[np.isnan(weight[:n])] = -np.inf
    below = np.isnan(weight[:n]).astype(int)  # NaN ranks below -inf
    protected = np.zeros(n, bool)
    if position is not None:
        p = position[:n].astype(np.int64)
        protected = (p < n_first) | ((p > p.max() - n_recent) & (n_recent > 0))
    order = np.lexsort((np.arange(n), below, -w, ~protected))
    # among protected rows only the slot decides
    prot = np.flatnonzero(protected)
    rest = order[~protected[order]]
    keep = np.zeros(n, bool)
    keep[np.concatenate([prot, rest])[:budget]] = True
    return keep, np.flatnonzero(~keep[:budget]), budget + np.flatnonzero(keep[budget:])


def logits_ref(x, *, tokens=None, prompt=0, repetition=None, frequency=None, presence=None, bias=(), allowed=None):
    """One row, every step rounded to fp32 as the operator defines it.  Returns the row and the choice."""
    x = x.astype(np.float32).copy()
    f32 = np.float32
    with np.errstate(all="ignore"):
        if tokens is not None and (repetition is not None or frequency is not None or presence is not None):
            inside = (tokens >= 0) & (tokens < x.size)
            seen = np.unique(tokens[inside])
            if repetition is not None:
                x[seen] = np.where(x[seen] > 0, x[seen] / f32(repetition), x[seen] * f32(repetition))
            made = tokens[max(0, min(prompt, len(tokens))):]
            made, count = np.unique(made[(made >= 0) & (made < x.size)], return_counts=True)
            fr, pr = f32(frequency or 0), f32(presence or 0)
            x[made] = (x[made] - fr * count.astype(np.float32)) - pr
        total = {}
        for t, v in bias:
            if 0 <= t < x.size:
                total[t] = f32(total.get(t, f32(0)) + f32(v))
        for t, v in total.items():
            x[t] = x[t] + v
    if allowed is not None:
        x[~allowed] = -np.inf
    y = np.where(np.isnan(x), -np.inf, x)
    return x, int(np.argmax(y)) if y.max() > -np.inf else -1


def pack_bits(allowed):
    """Boolean [rows, vocab] as mask words [rows, ceil(vocab / 32)] (int32)."""
    rows, vocab = allowed.shape
    pad = np.zeros((rows, (vocab + 31) // 32 * 32), np.uint8)
    pad[:, :vocab] = allowed
    return np.packbits(pad, axis=1, bitorder="little").view(np.int32)
