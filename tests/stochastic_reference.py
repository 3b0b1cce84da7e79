"""Plain 64-bit numpy forms of litegs_amd/stochastic.py, written from the definitions in its docstrings."""
import numpy as np

M32 = np.uint64(0xFFFFFFFF)


def philox(counter, key, rounds=10):
    """Philox4x32: counter [..., 4], key (k0, k1) -> words [..., 4] (uint64 holding 32 bits)"""
    c = [np.asarray(counter[..., k], dtype=np.uint64) for k in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & M32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & M32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=-1)


def words(index, seed, offset):
    """word of every index (any shape, int64 / python ints below 2^63)"""
    index = np.asarray(index, dtype=np.uint64)
    block = index >> np.uint64(2)
    counter = np.stack([block & M32, block >> np.uint64(32), np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)], axis=-1)
    w = philox(counter, (seed & 0xFFFFFFFF, seed >> 32))
    return np.take_along_axis(w, (index & np.uint64(3)).astype(np.int64)[..., None], axis=-1)[..., 0]


def kept(index, p, seed, offset):
    return words(index, seed, offset) >= np.uint64(int(np.rint(p * 2.0 ** 32)))


def normals(n, seed, offset):
    """-> (N(0,1) draws in 64 bits, the radius of each one's pair)"""
    w = words(np.arange(n + n % 2), seed, offset).astype(np.float64)
    r = np.sqrt(-2.0 * np.log((w[0::2] + 0.5) / 2.0 ** 32))
    a = 2.0 * np.pi * w[1::2] / 2.0 ** 32
    return np.stack([r * np.cos(a), r * np.sin(a)], axis=-1).reshape(-1)[:n], np.repeat(r, 2)[:n]


def filtered(x, logits, temperature, top_k, top_p, min_p, big):
    """one row -> (indices kept, ascending; their log-masses; their masses)"""
    with np.errstate(all="ignore"):
        x = np.asarray(x, dtype=np.float64)
        x = np.minimum(np.where(np.isnan(x), -np.inf, x), big)
        who = np.flatnonzero(x > (-np.inf if logits else 0.0))
        who = who[np.argsort(-x[who], kind="stable")]
        v = x[who]
        l = (v if logits else np.log(v)) / temperature
        mass = v if (not logits and temperature == 1.0) else np.exp(l - l[:1])
        if top_k:
            who, l, mass = who[:top_k], l[:top_k], mass[:top_k]
        if top_p < 1.0 and len(who):
            run = np.cumsum(mass.astype(np.longdouble))
            before = np.concatenate([[0.0], run[:-1].astype(np.float64)])
            good = before < top_p * float(run[-1])
            who, l, mass = who[good], l[good], mass[good]
        if min_p > 0.0 and len(who):
            good = mass >= min_p * mass[0]
            who, l, mass = who[good], l[good], mass[good]
    order = np.argsort(who)
    return who[order], l[order], mass[order]


def sample_row(x, u, logits, temperature, top_k, top_p, min_p, big):
    who, _, mass = filtered(x, logits, temperature, top_k, top_p, min_p, big)
    who, mass = who[mass > 0], mass[mass > 0]
    if not len(who):
        return np.full(len(u), -1, dtype=np.int64)
    run = np.cumsum(mass.astype(np.longdouble))
    t = np.maximum(np.where(np.isnan(u), 0.0, u).astype(np.float64), 0.0) * float(run[-1])
    return who[np.minimum(np.searchsorted(run, t.astype(np.longdouble), side="right"), len(who) - 1)]


def distinct_row(x, u, n, logits, temperature, top_k, top_p, min_p, big):
    who, l, _ = filtered(x, logits, temperature, top_k, top_p, min_p, big)
    out = np.full(n, -1, dtype=np.int64)
    uu = np.where(np.isnan(u), 1.0, u).astype(np.float64)[who]
    key = l - np.log(-np.log1p(-np.clip(uu, 2.0 ** -33, 1.0 - 2.0 ** -24)))
    best = who[np.argsort(-key, kind="stable")[:n]]
    out[: len(best)] = np.sort(best)
    return out
