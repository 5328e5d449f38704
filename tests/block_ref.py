"""Plain 64-bit forms of the block-sparse attention and of the low-rank
adapters, one row at a time, for the tests: written from the definitions in
include/granite4_layerops.h. Scores and ranges follow the definition's own f32
roundings (they are compared for equality), attention and adapters are float64.
"""
import numpy as np

D = 128
QMAX = {8: 127, 4: 7, 5: 15}


def bf16(x):
    """float32 -> bf16 bits, round to nearest even (no NaN)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def f32(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def codes(x, s):
    """clamp(round half away(x / s), +-127), 0 where s is 0 (float32 quotient)."""
    x, s = np.broadcast_arrays(np.asarray(x, np.float32), np.asarray(s, np.float32))
    r = np.divide(x, s, out=np.zeros_like(x), where=s != 0).astype(np.float64)
    return np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), -127, 127).astype(np.int64)


def pool(rng, bits, group, Hk, stride, kmean=1.0):
    """A filled pool: bytes K and V, scales, and the values float64 [Hk][stride][128]
    (code * scale as one float32 product)."""
    out = []
    for is_k in (True, False):
        x = rng.standard_normal((Hk, stride, D)).astype(np.float32)
        if is_k:
            x += (kmean * rng.standard_normal((Hk, 1, D))).astype(np.float32)
        if bits == 16:
            b = bf16(x)
            out.append((b.view(np.uint8), None, f32(b).astype(np.float64)))
            continue
        q = QMAX[bits] if is_k or bits == 8 else 7
        xg = x.reshape(Hk, stride, D // group, group)
        s = (np.abs(xg).max(-1) / np.float32(q)).astype(np.float32)
        c = np.clip(np.rint(xg / s[..., None]), -q, q).astype(np.int32).reshape(x.shape)
        v = (c.reshape(xg.shape).astype(np.float32) * s[..., None]).reshape(x.shape)
        if bits == 8:
            rows = c.astype(np.int8).view(np.uint8)
        else:
            u = c + q + 1
            rows = ((u[..., 0::2] & 15) | ((u[..., 1::2] & 15) << 4)).astype(np.uint8)
            if q == 15:
                p = (((u >> 4) & 1).reshape(Hk, stride, 16, 8) << np.arange(8)).sum(-1)
                rows = np.concatenate([rows, p.astype(np.uint8)], -1)
        out.append((np.ascontiguousarray(rows), s, v.astype(np.float64)))
    return out[0][0], out[1][0], out[0][1], out[1][1], out[0][2], out[1][2]


def table(rng, pages, page):
    """position -> arena row for a context of `pages` pages in random order."""
    order = rng.permutation(pages).astype(np.int32)
    return (order[:, None] * page + np.arange(page, dtype=np.int32)).reshape(-1)


def ranges(kval, block, pt, stride, done, codes_in, scale_in):
    """Updates (codes, scales) for the blocks numbered in `done` of the sequence pt."""
    c, s = codes_in.copy(), scale_in.copy()
    for b in done:
        rows = pt[b * block:(b + 1) * block]
        if not (0 <= rows[0] < stride) or rows[0] % block:
            continue
        rows = rows[(rows >= 0) & (rows < stride)]
        x = kval[:, rows].astype(np.float32)
        lo, hi = np.fmin.reduce(x, 1), np.fmax.reduce(x, 1)
        sc = (np.maximum(np.abs(lo), np.abs(hi)).max(-1) / np.float32(127)).astype(np.float32)
        at = pt[b * block] // block
        c[:, at, 0], c[:, at, 1], s[:, at] = codes(lo, sc[:, None]), codes(hi, sc[:, None]), sc
    return c, s


def select(q, rc, rs, block, pos, pt, stride, top_k, sink, recent):
    """One row: q [Hq][128] float32; the listed blocks [Hk][top_k]."""
    Hk = rc.shape[0]
    out = np.full((Hk, top_k), -1, np.int32)
    n = pos // block + 1 if pos >= 0 else 0
    if n == 0:
        return out
    first = np.array([pt[b * block] for b in range(n)])
    ok = (first >= 0) & (first < stride) & (first % block == 0)
    at = np.where(ok, first, 0) // block
    ids = np.arange(n)
    for h in range(Hk):
        best = np.full(n, -np.inf)
        for g in range(4):
            x = q[4 * h + g]
            sq = np.float32(np.abs(x).max()) / np.float32(127)
            qc = codes(x, sq)
            # the larger product where lo <= hi; by the sign of qc for any codes
            dot = np.where(qc < 0, qc * rc[h, at, 0].astype(np.int64), qc * rc[h, at, 1].astype(np.int64)).sum(-1)
            with np.errstate(invalid="ignore", over="ignore"):
                best = np.fmax(best, (dot.astype(np.float32) * rs[h, at]) * sq)
        best = best.astype(np.float64)
        kept = (ids < sink) | (ids >= n - recent)
        rank = np.where(kept, np.inf, best)
        order = sorted(ids[ok], key=lambda i: (not kept[i], -rank[i], i))[:top_k]
        out[h, :len(order)] = sorted(order)
    return out


def attend(q, kval, vval, block, pos, pt, stride, sel, scale):
    """One row: (out [Hq][128], bound on |kernel - out|) for lists sel [Hk][top_k].

    The kernel rounds p (times the V scale) to bf16: 2^-8 of sum p |v|; the result:
    2^-8 of it; and sums logits and values in f32 (128 products; at most a few
    thousand keys): 2^-15 of the absolute sums."""
    Hk = kval.shape[0]
    out, tol = np.zeros((4 * Hk, D)), np.zeros((4 * Hk, D))
    for h in range(Hk):
        p = (sel[h].astype(np.int64)[:, None] * block + np.arange(block)).reshape(-1)
        p = p[(np.repeat(sel[h], block) >= 0) & (p <= pos)]
        p = p[p < len(pt)]
        r = pt[p]
        r = r[(r >= 0) & (r < stride)]
        if not len(r):
            continue
        for g in range(4):
            x = q[4 * h + g].astype(np.float64)
            lg = scale * (kval[h, r] @ x)
            w = np.exp(lg - lg.max())
            w /= w.sum()
            out[4 * h + g] = w @ vval[h, r]
            mass = w @ np.abs(vval[h, r])
            lmax = abs(scale) * (np.abs(kval[h, r]) @ np.abs(x)).max()
            tol[4 * h + g] = 2.0 ** -8 * (mass + np.abs(out[4 * h + g])) + 2.0 ** -15 * (1 + lmax) * mass
            tol[4 * h + g] += 1e-30
    return out, tol


def lora(x, A, B, alpha, adapter, base, segs, mult):
    """y and a bound on the kernel's f32 result: x [M][K], A [n][parts][R][K],
    B [n][N][R], base [M][N] float64."""
    y, tol = base.copy(), np.abs(base) * 2.0 ** -23
    N, K, R = B.shape[1], x.shape[1], A.shape[2]
    cut = [0] + [s for s in segs if s < N] + [N]
    for m in range(x.shape[0]):
        a = adapter[m]
        if not 0 <= a < len(alpha):
            continue
        f = np.float64(mult) * alpha[a]
        for i in range(len(cut) - 1):
            t = A[a, i] @ x[m]
            # f32 sums of K products, t as two or three bf16 terms (2^-16 of it), f32 sums of 2 R
            # products, and the three roundings of base + (mult alpha) (.)
            dt = K * 2.0 ** -24 * (np.abs(A[a, i]) @ np.abs(x[m])) + 2.0 ** -16 * np.abs(t)
            b = B[a, cut[i]:cut[i + 1]]
            d = f * (b @ t)
            y[m, cut[i]:cut[i + 1]] += d
            tol[m, cut[i]:cut[i + 1]] += abs(f) * (np.abs(b) @ (dt + (2 * R + 4) * 2.0 ** -24 * np.abs(t)))
    return y, tol + np.abs(y) * 2.0 ** -24 + 1e-30
