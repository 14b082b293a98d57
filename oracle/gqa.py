"""The GQA layer over the block-scaled 8-bit cache in numpy, 64 bits: what include/hk.h states for
hk_qk_norm_rope, hk_gqa_append_fp8, hk_gqa_decode_fp8, hk_gqa_select_blocks and hk_gqa_sparse_fp8."""
import numpy as np


def _e4m3_values():
    v = np.zeros(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        x = (1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6
        v[b] = -x if b & 128 else x
    v[0x7F] = v[0xFF] = np.nan
    return v


E4M3 = _e4m3_values()


def to_e4m3(x):
    """Codes of x rounded to e4m3, ties to even, saturating at 448 (NaN: 0x7f)."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.floor(np.log2(np.where(a >= 2.0 ** -6, a, 2.0 ** -6)))
    n = np.rint(a / np.exp2(e - 3))  # a = n * 2^(e-3); n may reach 16
    up = n >= 16
    e, n = np.where(up, e + 1, e), np.where(up, 8, n)
    code = np.where(n >= 8, (e + 7) * 8 + n - 8, n)
    code = np.where(np.isnan(x), 0x7F, np.nan_to_num(code)).astype(np.uint8)
    return code | np.where(np.signbit(x) & ~np.isnan(x), 0x80, 0).astype(np.uint8)


def norm_rope(x, gain, positions, table, interleaved, eps):
    """x [T, H, D]; gain [D] or None; rows with a negative position are returned as they are."""
    x = np.asarray(x, np.float64)
    rot = table.shape[1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if gain is not None:
        y = y * np.asarray(gain, np.float64)
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    line = table[np.maximum(positions, 0)].astype(np.float64)[:, None]
    c, s = line[..., :rot // 2], line[..., rot // 2:]
    out = y.copy()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    return np.where((positions < 0)[:, None, None], x, out)


def pow2_scale(top):
    top = max(float(top), 2.0 ** -32)
    m, e = np.frexp(top)
    return 2.0 ** (int(e) - 9 + (1 if m > 0.875 else 0))


def append(k_new, v_new, slots, cache):
    """Updates cache = dict(k, v uint8 [N, G, R, D], ks, vs fp32 [N, G], cen int8 or None, cs) in place."""
    N, G, R, D = cache["k"].shape
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= N * R:
            t += 1
            continue
        p, o = divmod(int(slots[t]), R)
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and o + n < R:
            n += 1
        skip = n
        while t + skip < len(slots) and slots[t + skip] >= 0 and slots[t + skip] // R == p:
            skip += 1  # rows of the page that do not continue the run
        for x, c, sc in ((k_new, "k", "ks"), (v_new, "v", "vs")):
            for g in range(G):
                r = np.asarray(x[t:t + n, g], np.float64)
                fin = np.abs(r[np.isfinite(r)])
                s = pow2_scale(fin.max() if fin.size else 0.0)
                old = float(cache[sc][p, g])
                if o > 0:
                    s = max(s, old)
                    if old < s:
                        ratio = np.float32(np.float32(old) * (np.float32(1) / np.float32(s)))
                        cache[c][p, g, :o] = to_e4m3((E4M3[cache[c][p, g, :o]].astype(np.float32) * ratio))
                inv = np.float32(1) / np.float32(s)
                with np.errstate(over="ignore", under="ignore"):
                    cache[c][p, g, o:o + n] = to_e4m3(np.where(np.isnan(r), 0, r).astype(np.float32) * inv)
                cache[sc][p, g] = s
        if cache.get("cen") is not None and o + n == R:
            centroid(cache, p)
        t += skip


def centroid(cache, p):
    R = cache["k"].shape[2]
    S = (np.nan_to_num(E4M3[cache["k"][p]]) * 512).sum(1)  # [G, D] whole numbers
    m = np.abs(S).max(-1).astype(np.float32)
    with np.errstate(divide="ignore"):
        r = np.where(m > 0, np.float32(127) / m, np.float32(0)).astype(np.float32)
    cache["cen"][p] = np.rint(S.astype(np.float32) * r[:, None]).astype(np.int8)
    cache["cs"][p] = cache["ks"][p] * (m / np.float32(127.0 * 512.0 * R))


def select(q, cache, block_table, cu, positions, top, sink, local):
    """int32 [T, G, top]; q [T, H, D] as float64 values."""
    N, G, R, D = cache["k"].shape
    T, H, _ = q.shape
    out = np.full((T, G, top), -1, np.int32)
    for b in range(len(cu) - 1):
        for t in range(cu[b], min(cu[b + 1], T)):
            n = 0 if positions[t] < 0 else int(positions[t]) // R + 1
            for g in range(G):
                if n <= top:
                    out[t, g, :n] = np.arange(n)
                    continue
                u = q[t].reshape(G, H // G, D)[g].astype(np.float64).sum(0).astype(np.float32)
                m = np.abs(u).max()
                c = np.zeros(D)
                if m < 2.0 ** -64:  # 127 / m could pass fp32: a power of two changes nothing else
                    u, m = u * np.float32(2.0 ** 64), m * np.float32(2.0 ** 64)
                if m > 0 and np.isfinite(m):
                    c = np.rint(u * (np.float32(127) / m)).astype(np.float64)
                pg = block_table[b, :n]
                dot = cache["cen"][pg, g].astype(np.float64) @ c
                score = (dot.astype(np.float32) * cache["cs"][pg, g]).astype(np.float64) + 0.0
                score[:sink] = np.inf
                score[n - local:] = np.inf
                out[t, g] = np.sort(np.argsort(-score, kind="stable")[:top])
    return out


def attend(q, cache, block_table, cu, positions, scale, blocks=None):
    """(out [T, H, D], lse [T, H], absolute weight sum [T, H, D], score size [T, H]) in 64 bits.  The
    last two size the error bounds: sum_j p_j |v_j|, and max_j scale * sum_d |q_d k_jd|."""
    N, G, R, D = cache["k"].shape
    T, H, _ = q.shape
    out, mag = np.zeros((T, H, D)), np.zeros((T, H, D))
    lse, size = np.full((T, H), -np.inf), np.zeros((T, H))
    grp = H // G
    for b in range(len(cu) - 1):
        for t in range(cu[b], min(cu[b + 1], T)):
            if positions[t] < 0:
                continue
            n = int(positions[t]) + 1
            for g in range(G):
                idx = np.arange(n)
                if blocks is not None:
                    keep = blocks[t, g][blocks[t, g] >= 0]
                    idx = idx[np.isin(idx // R, keep)]
                pg = block_table[b, idx // R]
                ok = (pg > 0) & (pg < N)
                idx, pg = idx[ok], pg[ok]
                if not len(idx):
                    continue
                k = E4M3[cache["k"][pg, g, idx % R]] * cache["ks"][pg, g].astype(np.float64)[:, None]
                v = E4M3[cache["v"][pg, g, idx % R]] * cache["vs"][pg, g].astype(np.float64)[:, None]
                qh = q[t, g * grp:(g + 1) * grp].astype(np.float64)
                s = qh @ k.T * scale
                m = s.max(1, keepdims=True)
                w = np.exp(s - m)
                z = w.sum(1, keepdims=True)
                hs = slice(g * grp, (g + 1) * grp)
                out[t, hs], mag[t, hs] = w @ v / z, w @ np.abs(v) / z
                lse[t, hs] = (m + np.log(z))[:, 0]
                size[t, hs] = (np.abs(qh) @ np.abs(k).T * scale).max(1)
    return out, lse, mag, size
