"""Plain 64-bit forms of the 8-bit cache operators, and how far the kernels may be from them."""

import math

import numpy as np
import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
FMTS = [torch.float8_e4m3fn, torch.int8]


def e4m3_table() -> np.ndarray:
    """The 256 values of e4m3 (bias 7, no infinities, NaN at 0x7f and 0xff)."""
    c = np.arange(128)
    e, m = c >> 3, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[127] = np.nan
    return np.concatenate([v, -v])


def decode_bytes(raw: np.ndarray, fmt) -> np.ndarray:
    """uint8 codes -> the values they stand for, without the scale."""
    if fmt == torch.int8:
        return raw.view(np.int8).astype(np.float64)
    return e4m3_table()[raw]


def encode(x: np.ndarray, fmt) -> np.ndarray:
    """Nearest code (ties to even) of values already divided by their scale, as uint8."""
    if fmt == torch.int8:
        y = np.clip(np.rint(np.where(np.isnan(x), 0.0, x)), -127, 127)
        return y.astype(np.int8).view(np.uint8)
    grid = e4m3_table()[:127]
    a = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), 448.0)
    i = np.clip(np.searchsorted(grid, a, side="right") - 1, 0, 126)
    j = np.minimum(i + 1, 126)
    below, above = a - grid[i], grid[j] - a
    code = np.where((above < below) | ((above == below) & (i % 2 == 1)), j, i).astype(np.uint8)
    code = np.where(np.signbit(x), code | 0x80, code)
    return np.where(np.isnan(x), code & 0x80 | 0x7F, code).astype(np.uint8)


def pow2_scale(a: float, fmt) -> float:
    s = 2.0 ** -126
    while a > QMAX[fmt] * s:
        s *= 2.0
    return s


def append_ref(raw, scale, fmt, x, tables, ctx, new):
    """The append by its definition, in place on raw uint8 [nb, H, bs, d] and f32 scale [nb, H];
    x f64 [T, H, d] packed new rows."""
    bs = raw.shape[2]
    t = 0
    for s in range(len(ctx)):
        p, L = int(ctx[s] - new[s]), int(ctx[s])
        while p < L:
            o = p % bs
            n = min(bs - o, L - p)
            blk = tables[s, p // bs]
            for h in range(raw.shape[1]):
                rows = x[t:t + n, h]
                fin = np.abs(rows[np.isfinite(rows)])
                to = pow2_scale(fin.max() if fin.size else 0.0, fmt)
                if o:
                    old = float(scale[blk, h])
                    to = max(old, to)
                    if to != old:
                        raw[blk, h, :o] = encode(decode_bytes(raw[blk, h, :o], fmt) * (old / to), fmt)
                raw[blk, h, o:o + n] = encode(rows / to, fmt)
                scale[blk, h] = to
            p += n
            t += n


def random_pool(nb, heads, bs, d, fmt, gen, device, spread=1.0):
    """Random codes (e4m3's NaN codes replaced by 0) and power-of-two scales of one device pool."""
    out = []
    for _ in range(2):
        raw = torch.randint(0, 256, (nb, heads, bs, d), generator=gen, device=device, dtype=torch.uint8)
        if fmt == torch.float8_e4m3fn:
            raw = torch.where((raw & 0x7F) >= 0x70, raw & 0x8F, raw)  # |value| < 256
        else:
            raw = torch.where(raw == 128, torch.zeros_like(raw), raw)
        e = torch.randint(-2, 3, (nb, heads), generator=gen, device=device).float() * spread
        base = 1 / 64.0 if fmt == torch.int8 else 1 / 32.0
        out.append((raw.view(fmt), torch.exp2(e) * base))
    (k, ks), (v, vs) = out
    return k, v, ks, vs


def dequant(cache, scale) -> np.ndarray:
    raw = cache.view(torch.uint8).cpu().numpy()
    return decode_bytes(raw, cache.dtype) * scale.cpu().numpy().astype(np.float64)[:, :, None, None]


def attention_ref(q, pool, tables, ctx, new, n_rep, scale, u_p):
    """f64 attention and, element by element, how far the kernel may be from it before its output
    is rounded. q f64 [T, Hq, d]; `new` query counts. The bound adds

      u_p * A           rounding of each probability (A = sum p |v|, p normalised),
      2 * ds * A        an error ds of a score, in nats: f32 accumulation of d products (2^-23 of
                        sum |q||k|, for each of 8 partial sums) and queries rounded 2^-24 below
                        their head's largest,
      2^-20 * A         2^x, the running sums and the division,
      2^-24 * sum |v|   probabilities under the smallest normal f16 (half a step of 2^-24; the
                        sum of probabilities is >= 1 before normalisation).
    """
    k, v = dequant(pool[0], pool[2]), dequant(pool[1], pool[3])
    tables = tables.cpu().numpy()
    bs = k.shape[2]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    t = 0
    for s in range(len(ctx)):
        L, n = int(ctx[s]), int(new[s])
        ids = tables[s, :(L + bs - 1) // bs]
        for h in range(q.shape[1]):
            kk = k[ids, h // n_rep].reshape(-1, k.shape[3])[:L]
            vv = v[ids, h // n_rep].reshape(-1, v.shape[3])[:L]
            qq = q[t:t + n, h]
            sc = qq @ kk.T * scale
            seen = np.arange(L)[None, :] <= (L - n + np.arange(n))[:, None]
            sc = np.where(seen, sc, -np.inf)
            p = np.exp(sc - sc.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[t:t + n, h] = p @ vv
            reach = (8 * 2.0 ** -23 * (np.abs(qq) @ np.abs(kk).T) +
                     2.0 ** -24 * np.abs(qq).max(1, keepdims=True) * np.abs(kk).sum(1)) * abs(scale)
            ds = np.where(seen, reach, 0).max(1, keepdims=True)
            A = p @ np.abs(vv)
            tol[t:t + n, h] = (u_p + 2 * ds + 2.0 ** -20) * A
            if u_p:
                tol[t:t + n, h] += 2.0 ** -24 * (seen @ np.abs(vv))
        t += n
    return out, tol


def assert_close(got: torch.Tensor, want: np.ndarray, tol: np.ndarray):
    g = got.double().cpu().numpy()
    u = torch.finfo(got.dtype).eps / 2
    bound = tol + u * (np.abs(want) + tol) + torch.finfo(got.dtype).tiny * u * 2
    worst = np.abs(g - want) - bound
    assert np.isfinite(g).all()
    assert (worst <= 0).all(), f"off by {np.abs(g - want).max()}, {worst.max()} past the bound"


def make_tables(ctx, bs, gen_seed, extra=3):
    """Disjoint, shuffled blocks for each sequence; returns int32 [S, max] and the pool size."""
    rng = np.random.default_rng(gen_seed)
    pages = [(int(c) + bs - 1) // bs for c in ctx]
    nb = sum(pages) + extra
    perm = rng.permutation(nb).astype(np.int32)
    bt = np.zeros((len(ctx), max(1, max(pages, default=1))), np.int32)
    o = 0
    for s, n in enumerate(pages):
        bt[s, :n] = perm[o:o + n]
        o += n
    return bt, nb


def inv_sqrt(d):
    return 1.0 / math.sqrt(d)
