"""The operators of include/talos_b200_lm.h written out in 64 bits: what their tests compare the kernels with, each with a bound
on what fp32 arithmetic may lose, element by element.  U is half a step of fp32: one rounding is off by at most U relative.

The bounds count roundings in the first order: a sum of terms a_i over a chain of c additions is off by at most c U sum |a_i|."""
import numpy as np

U = 2.0 ** -24


def philox(block, offset, seed):
    """philox4x32-10 (Salmon, Moraes, Dror and Shaw, SC 2011): the four words of each counter (block, offset)."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    block = np.asarray(block, dtype=np.uint64)
    c = [block & low, block >> u(32), np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k0), b & low, (a >> u(32)) ^ c[3] ^ u(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, -1)


def keep(n, p, seed, offset):
    """Which of n elements dropout keeps."""
    words = philox(np.arange((n + 3) // 4), offset % 2 ** 64, seed % 2 ** 64).reshape(-1)[:n]
    return words >= int(np.floor(float(np.float32(p)) * 2.0 ** 32 + 0.5))


def dropout(x, p, seed, offset):
    return np.where(keep(x.size, p, seed, offset).reshape(x.shape), x, 0.0) / (1.0 - float(np.float32(p)))


def layernorm(x, gamma, beta, eps):
    mean = x.mean(1)
    inv = 1.0 / np.sqrt(((x - mean[:, None]) ** 2).mean(1) + eps)
    y = (x - mean[:, None]) * inv[:, None]
    if gamma is not None: y = y * gamma
    if beta is not None: y = y + beta
    return y, mean, inv


# A thread adds at most 16 values of a row, five shuffles and at most 32 warps follow: 53 additions.
ROW_ADDS = 53


def layernorm_bound(x, gamma, beta, eps):
    """Bounds of y, mean and inv_std."""
    y, mean, inv = layernorm(x, gamma, beta, eps)
    g = np.ones(x.shape[1]) if gamma is None else np.abs(gamma)
    d_mean = (ROW_ADDS + 2) * U * np.abs(x).mean(1)
    # sum of squares: each (x - mean)^2 is off by 3 U relative and by the shift of the mean, whose first order cancels over the row; root and
    # quotient add half of the sum's error and 3 roundings
    rel_inv = 0.5 * (ROW_ADDS + 6) * U + 4 * U + 0.5 * (d_mean * inv) ** 2
    xh = np.abs(x - mean[:, None]) * inv[:, None]
    d_y = (d_mean * inv)[:, None] * g + xh * g * (5 * U + rel_inv[:, None]) + 2 * U * np.abs(y)
    return d_y, d_mean + U * np.abs(mean), rel_inv * inv + U * inv


def layernorm_bwd(dy, x, gamma, mean, inv):
    g = dy if gamma is None else dy * gamma
    xh = (x - mean[:, None]) * inv[:, None]
    dx = inv[:, None] * (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


# A column: at most 64 rows a thread (tests of at most 8 192 rows), 32 groups of a CTA, up to 1 184 CTAs by 32 lanes, five shuffles.
COL_ADDS = 64 + 32 + 1184 // 32 + 5


def layernorm_bwd_bound(dy, x, gamma, mean, inv):
    """Bounds of dx, dgamma and dbeta where mean and inv_std come rounded to fp32."""
    g = np.abs(dy if gamma is None else dy * gamma)
    xh = np.abs(x - mean[:, None]) * inv[:, None]
    d_xh = U * (4 * xh + (np.abs(mean) * inv)[:, None])
    m1, m2 = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    c = ROW_ADDS + 6
    d_dx = inv[:, None] * (c * U * (g + m1 + xh * m2) + d_xh * m2 + xh * (g * d_xh).mean(1, keepdims=True)) + 4 * U * inv[:, None] * (g + m1 + xh * m2)
    return d_dx, COL_ADDS * U * (np.abs(dy) * xh).sum(0) + (np.abs(dy) * d_xh).sum(0), COL_ADDS * U * np.abs(dy).sum(0)


def policy_loss(z, tokens, old, ref, adv, w, low, high, c_kl, c_ent, denom):
    """(stats[5], logp, dlogits, and bounds of the three).  z [rows, vocab]; rows that do not count have token < 0 or weight 0."""
    rows, vocab = z.shape
    low, high = float(np.float32(1) - np.float32(low)), float(np.float32(1) + np.float32(high))
    c_kl, c_ent = float(np.float32(c_kl)), float(np.float32(c_ent))
    stats, logp, dz = np.zeros(5), np.zeros(rows), np.zeros((rows, vocab))
    sizes = np.zeros(5)
    e_stats, e_logp, e_dz = np.zeros(5), np.zeros(rows), np.zeros((rows, vocab))
    for r in range(rows):
        a, wt = int(tokens[r]), 1.0 if w is None else float(w[r])
        if a < 0 or wt == 0.0: continue
        m = z[r].max()
        if m == -np.inf:
            logp[r] = -np.inf
            continue
        lse = m + np.log(np.exp(z[r] - m).sum())
        logs = z[r] - lse
        p = np.exp(logs)
        plog = np.where(p > 0, p * np.where(p > 0, logs, 0.0), 0.0)
        H, lp = -plog.sum(), logs[a]
        size = np.abs(z[r][np.isfinite(z[r])]).max() + abs(lse)
        # an exponent's argument is off by the roundings of z - m and m - lse, a sum by at most 128 additions, exp and log by 2 U each
        e = U * (8 * (size + (abs(old[r]) if old is not None else 0) + (abs(ref[r]) if ref is not None else 0)) + 160)
        loss = kl = g = dg = clipped = mag = 0.0
        if adv is not None:
            ratio = np.exp(lp - old[r]); s1 = ratio * adv[r]; s2 = min(max(ratio, low), high) * adv[r]
            loss = -min(s1, s2)
            inside = low <= ratio <= high
            g = -s1 if (s1 < s2 or inside) else 0.0
            clipped = float(s2 < s1 and not inside)
            mag += abs(s1); dg += abs(s1) * e
        if ref is not None:
            d = ref[r] - lp
            kl = np.expm1(d) - d
            loss += c_kl * kl; g -= c_kl * np.expm1(d)
            mag += c_kl * (abs(np.expm1(d)) + abs(d)); dg += c_kl * (np.exp(d) + 1) * e
        loss -= c_ent * H
        k = wt / denom
        logp[r] = lp; e_logp[r] = e
        e_H = e * (1 + H + np.abs(logs[np.isfinite(logs)]).max() * 2)
        stats += wt * np.array([loss, kl, H, clipped, 1.0])
        sizes += abs(wt) * np.array([mag + c_ent * H, abs(kl), H, clipped, 1.0])
        e_kl = 0.0 if ref is None else (np.exp(ref[r] - lp) + 1) * e
        e_stats += abs(wt) * np.array([dg + mag * e + c_ent * e_H, e_kl + abs(kl) * e, e_H, 0.0, 0.0])
        onehot = np.arange(vocab) == a
        ent = np.where(p > 0, p * (np.where(p > 0, logs, 0.0) + H), 0.0)
        dz[r] = k * (g * (onehot - p) + c_ent * ent)
        e_dz[r] = abs(k) * ((dg + abs(g) * e * 2) * (onehot + p) + c_ent * p * (e_H + e * (np.where(p > 0, np.abs(np.where(p > 0, logs, 0.0)), 0.0) + H + 1)) + 4 * U * (abs(g) * (onehot + p) + c_ent * np.abs(ent)))
    # a CTA adds its rows in fp32 (at most 64 here, then five shuffles and eight warps), the CTAs' sums are added in 64 bits and rounded once
    return stats, logp, dz, e_stats + 80 * U * sizes, e_logp, e_dz


# One product of the tensor cores' operands: values are sums of bf16 terms, and a term leaves at most half a step, 2^-8, of what it is rounded from: x = x0 + x1
# + x2 + r with |x1| <= 2^-8 |x|, |x2| <= 2^-16 |x|, |r| <= 2^-24 |x|.  Three terms leave 2^-24 of either factor and drop x1 y2 and x2 y1, 2^-24 each, and x2 y2,
# 2^-32: below 4.02 2^-24.  Two terms (the fast mode) leave 2^-16 of either and drop x1 y1, 2^-16, less than 2^-16 of that again: 3.02 2^-16.
PRODUCT = {0: 4.02 * 2.0 ** -24, 1: 4.02 * 2.0 ** -24, 2: 3.02 * 2.0 ** -16}


def attention(q, k, v, key_len, scale, causal, dout=None, mode=1):
    """(out, lse[, dq, dk, dv]) and bounds of each.  q [B, H, Sq, D], k and v [B, Hkv, Sk, .]; a query that sees no key has out 0, lse -inf.

    Bounds: a score is a chain of d products and additions, a probability is off by the score's and the log-sum-exp's error plus 2^-21
    (the hardware's exp2 is within 2^-22, twice), an output by a chain of sk additions; 2 U for an addition, since tensor cores truncate."""
    B, H, Sq, D = q.shape
    Hk, Sk = k.shape[1:3]
    G = H // Hk
    kk, vv = np.repeat(k, G, 1), np.repeat(v, G, 1)
    see = np.ones((B, 1, Sq, Sk), dtype=bool)
    if causal: see &= np.arange(Sk)[None, :] <= np.arange(Sq)[:, None] + Sk - Sq
    if key_len is not None: see &= np.arange(Sk)[None, None, None, :] < np.clip(np.asarray(key_len), 0, Sk)[:, None, None, None]
    T = lambda a: a.swapaxes(-1, -2)  # noqa: E731
    t = np.where(see, q @ T(kk) * scale, -np.inf)
    top = np.maximum(t.max(-1, keepdims=True, initial=-np.inf), -1e300)
    p = np.exp(t - top)
    total = p.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"): lse = np.where(total > 0, top + np.log(total), -np.inf)[..., 0]
    p = np.where(total > 0, p / np.where(total > 0, total, 1), 0.0)
    out = p @ vv
    A = np.abs
    prod = PRODUCT[mode]
    e_t = np.where(see, ((2 * D + 8) * U + prod) * (A(q) @ T(A(kk))) * abs(scale) + 6 * U * A(np.where(see, t, 0)) , 0.0)
    e_row = e_t.max(-1, keepdims=True, initial=0.0) + 4 * U * A(np.where(np.isfinite(lse), lse, 0))[..., None]
    adds = 2 * (Sk + Sk // 16 + 16) * U
    rel = e_t + e_row + 2.0 ** -20
    # fp32 ends at 2^-126: what lies below, and what a split leaves below, counts as 0
    e_p = rel * p + see * 2.0 ** -125
    e_out = e_p @ A(vv) + (adds + 8 * U + prod) * (p @ A(vv))
    e_lse = e_row[..., 0] + adds + 2.0 ** -20
    if dout is None: return out, lse, e_out, e_lse
    dp = dout @ T(vv)
    delta = (dout * out).sum(-1, keepdims=True)
    ds = p * (dp - delta) * scale
    Dv = v.shape[-1]
    e_dp = ((2 * Dv + 8) * U + prod) * (A(dout) @ T(A(vv)))
    # delta is taken from the forward call's out: its sum's own roundings, and out's error carried through the same sum
    e_delta = ((Dv + 8) * U * A(dout) * A(out) + A(dout) * e_out).sum(-1, keepdims=True)
    e_ds = abs(scale) * (e_p * A(dp - delta) + p * (e_dp + e_delta + 4 * U * (A(dp) + A(delta)))) + see * 2.0 ** -125
    fold = lambda a: a.reshape(B, Hk, G, *a.shape[2:]).sum(2)  # noqa: E731
    adds_q = 2 * (G * (Sq + Sq // 16 + 16)) * U
    dq, dk, dv = ds @ kk, fold(T(ds) @ q), fold(T(p) @ dout)
    e_dq = e_ds @ A(kk) + (adds + 8 * U + prod) * (A(ds) @ A(kk))
    e_dk = fold(T(e_ds) @ A(q)) + (adds_q + 8 * U + prod) * fold(T(A(ds)) @ A(q))
    e_dv = fold(T(e_p) @ A(dout)) + (adds_q + 8 * U + prod) * fold(T(p) @ A(dout))
    return out, lse, dq, dk, dv, e_out, e_lse, e_dq, e_dk, e_dv
