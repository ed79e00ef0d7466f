"""Block-scaled e4m3 and the experts' routing in 64 bits (numpy): the definitions the fp8 kernels and the router
are held to. Test infrastructure only.

e4m3 here is the finite form: 1 sign, 4 exponent (bias 7), 3 mantissa bits, subnormals of 2^-9, largest value
448, NaN at 0x7f / 0xff, no infinity.
"""
from __future__ import annotations

import numpy as np

BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -100
MAGS = np.array([c * 2.0 ** -9 if c < 8 else (8 + c % 8) * 2.0 ** (c // 8 - 10) for c in range(127)])
MIDS = (MAGS[1:] + MAGS[:-1]) / 2


def codes_of(v):
    """Codes (u8) of the e4m3 values nearest to v (float64, |v| <= 464), ties to the even code."""
    a = np.abs(v)
    lo, hi = np.searchsorted(MIDS, a, side="left"), np.searchsorted(MIDS, a, side="right")
    c = np.minimum(np.where(lo % 2 == 0, lo, hi), 126)
    return (c | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def values_of(codes):
    """What codes (u8, none of them NaN) stand for, float64."""
    codes = np.asarray(codes)
    m = codes & 127
    assert (m < 127).all()
    return np.where(codes >= 128, -MAGS[np.minimum(m, 126)], MAGS[np.minimum(m, 126)])


def blocks(n):
    return -(-n // BLOCK)


def quantize(x, rows=1):
    """x [M, K] (values of an fp32 or narrower type) -> (codes u8 [M, K_pad], scale float32 [ceil(M / rows), K_pad / 128])."""
    x = np.asarray(x, dtype=np.float64)
    M, K = x.shape
    mb, nb = -(-M // rows), blocks(K)
    p = np.zeros((mb * rows, nb * BLOCK))
    p[:M, :K] = x
    p = p.reshape(mb, rows, nb, BLOCK)
    bad = ~np.isfinite(p).all(axis=(1, 3))
    amax = np.abs(np.where(np.isfinite(p), p, 0.0)).max(axis=(1, 3)).astype(np.float32)
    s = np.maximum(amax / np.float32(TOP), np.float32(LEAST))
    with np.errstate(invalid="ignore"):
        q = codes_of(np.where(bad[:, None, :, None], 0.0, p / s.astype(np.float64)[:, None, :, None]))
    s = np.where(bad, np.float32(np.nan), s)
    return q.reshape(mb * rows, nb * BLOCK)[:M], s


def dequantize(codes, scale, rows=1):
    """Codes [M, K_pad] and scales [ceil(M / rows), K_pad / 128] -> values, float64."""
    v = values_of(codes)
    s = np.repeat(np.asarray(scale, dtype=np.float64), rows, axis=0)[:v.shape[0]]
    return v * np.repeat(s, BLOCK, axis=1)


def sum_slack(K, rows=1):
    """Relative to the sum of the magnitudes: `rows` sums of K products each, taken as one. The products of a block of 128 columns
    are exact and summed first, in any order, each addition off by at most a whole step of 2^-23 (an instruction may cut);
    then every block is taken times one factor, which is rounded, and joined by an fma, the waves' sums and those of K
    ranges by additions, all off by half a step: at most three roundings a block, and four besides."""
    return (2 * min(K, BLOCK) + 3 * rows * blocks(K) + 4) * 2.0 ** -24


def cut_slack(xv, wv):
    """What the e4m3 matrix instruction may lose besides: before it adds the products of 8 neighbouring columns it cuts each
    off (toward zero) below u = 2^-13 of the binade of the largest of the eight, so at 2^-13 max|x| max|w| over them at
    most. For operands of random signs the losses, each in [0, u) with its product's sign, have mean 0 and variance
    u^2 / 3 at most, so their sum over the groups stays within six standard deviations but for one output in 10^9."""
    gx, gw = (np.abs(v).reshape(v.shape[0], -1, 8).max(axis=2) for v in (xv, wv))
    return 6 * 2.0 ** -13 * np.sqrt(8 / 3 * ((gx * gx) @ (gw * gw).T))


def linear(xv, wv):
    """(y, bound): the product of dequantized operands, and how far an fp32 sum rounded to bf16 may be off."""
    y = xv @ wv.T
    e = sum_slack(xv.shape[1]) * (np.abs(xv) @ np.abs(wv).T) + cut_slack(xv, wv)
    return y, 2.0 ** -8 * np.abs(y) + (1 + 2.0 ** -8) * e


def experts(xv, ids, w, gu, dn, H, I):
    """(out, bound) of a MoE layer's experts on quantized rows xv [T, H_pad]; gu / dn = (codes [E, .., K_pad], scales).
    Gate and up are sums of exact products. The bound follows the sums' errors through silu, through the second
    quantization (a value of h that close to a rounding border may take either code) and the down projection; the routed
    rows are summed in fp32 and the result is rounded."""
    (gq, gs), (dq, ds) = gu, dn
    T, k = ids.shape
    ib = blocks(I)
    out, tol = np.zeros((T, H)), np.zeros((T, H))
    for e in np.unique(ids):
        t, j = np.nonzero(ids == e)
        W = [dequantize(gq[e, p * I:(p + 1) * I], gs[e, p * ib:(p + 1) * ib], BLOCK) for p in range(2)]
        wd = dequantize(dq[e], ds[e], BLOCK)
        x = xv[t]
        (g, u), (eg, eu) = zip(*((x @ v.T, sum_slack(x.shape[1]) * (np.abs(x) @ np.abs(v).T)) for v in W))
        sig = 1.0 / (1.0 + np.exp(-g))
        h = g * sig * u
        # |d silu / dg| <= 1.1; the fp32 evaluation of exp, the division and two products: 8 steps
        eh = 1.1 * eg * (np.abs(u) + eu) + np.abs(g * sig) * eu + 8 * 2.0 ** -23 * np.abs(h)
        codes, s = quantize(h)
        hv = dequantize(codes, s)
        sv = np.repeat(s.astype(np.float64), BLOCK, axis=1)
        pad = np.zeros((h.shape[0], ib * BLOCK))
        hp, ep = pad.copy(), pad.copy()
        hp[:, :I], ep[:, :I] = h, eh
        es = ep.reshape(-1, ib, BLOCK).max(axis=2) / TOP + 2.0 ** -23 * s    # the scale's own error
        es = np.repeat(es, BLOCK, axis=1)
        move = (ep + np.abs(hp) * es / sv) / sv * (1 + 2.0 ** -20) + 2.0 ** -40
        a = np.abs(hp) / sv
        lo, hi = (values_of(codes_of(np.clip(a + d, 0.0, TOP))) for d in (-move, move))
        width = np.maximum(np.abs(hi * sv - np.abs(hv)), np.abs(lo * sv - np.abs(hv))) + np.maximum(hi, np.abs(hv) / sv) * es
        y = hv @ wd.T
        ey = width @ np.abs(wd).T + sum_slack(hv.shape[1], k) * ((np.abs(hv) + width) @ np.abs(wd).T) + cut_slack(np.abs(hv) + width, wd)
        c = w[t, j].astype(np.float64)[:, None]
        np.add.at(out, t, c * y)
        np.add.at(tol, t, np.abs(c) * ey + k * 2.0 ** -23 * np.abs(c * y))
    return out, tol + 2.0 ** -8 * (np.abs(out) + tol)


def route(logits, k, score="softmax", bias=None, n_group=1, topk_group=1, group_top=2, renorm=True, scale=1.0):
    """(weights float64 [T, k], ids [T, k]) of the router; logits / bias: values of fp32 or narrower types."""
    v = np.asarray(logits, dtype=np.float64)
    T, E = v.shape
    b = np.zeros(E) if bias is None else np.asarray(bias, dtype=np.float64)
    w, ids = np.zeros((T, k)), np.zeros((T, k), dtype=np.int64)
    for t in range(T):
        live = [e for e in range(E) if v[t, e] > -np.inf and b[e] > -np.inf]
        l = np.minimum(v[t], np.finfo(np.float32).max)
        s = np.zeros(E)
        if live:
            if score == "softmax":
                p = np.exp(l[live] - l[live].max())
                s[live] = p / p.sum()
            else:
                with np.errstate(over="ignore"):
                    s[live] = 1.0 / (1.0 + np.exp(-l[live]))
        c = s + b
        by = l if bias is None else c                      # without a bias the order of the logits
        if n_group > 1:
            size, gv = E // n_group, []
            for g in range(n_group):
                top = sorted((e for e in live if e // size == g), key=lambda e: -(c if group_top > 1 or bias is not None else l)[e])
                top = top[:group_top]
                gv.append(sum((c if group_top > 1 or bias is not None else l)[e] for e in top) if top else -np.inf)
            keep = sorted(range(n_group), key=lambda g: (-gv[g], g))[:topk_group]
            live = [e for e in live if e // size in keep]
        order = sorted(live, key=lambda e: (-by[e], e))
        order += [e for e in range(E) if e not in set(order)]
        ids[t] = order[:k]
        chosen = [e for e in order[:k] if e in set(live)]
        if score == "sigmoid" and renorm and chosen:
            m = min(0.0, max(l[e] for e in chosen))
            part = {e: np.exp(min(l[e], 0.0) - m) / (1.0 + np.exp(-abs(l[e]))) for e in chosen}
        elif score == "softmax" and renorm and chosen:
            m = max(l[e] for e in chosen)
            part = {e: np.exp(l[e] - m) for e in chosen}
        else:
            part = {e: s[e] for e in chosen}
        total = sum(part.values()) if renorm else 1.0
        for j, e in enumerate(order[:k]):
            w[t, j] = scale * part[e] / total if e in part and total > 0 else 0.0
    return w, ids


def route_slack(logits, E):
    """Relative error of a weight taken in fp32: the exponent's argument rounds by 2^-24 of itself, exp and the
    division by a few steps, the sum by one per expert."""
    v = np.asarray(logits, dtype=np.float64)
    v = np.clip(np.where(np.isfinite(v), v, 0.0), -1e4, 1e4)
    return (E + 16 + 2 * np.abs(v).max()) * 2.0 ** -23
