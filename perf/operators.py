"""Performance cases of the operators for training language-model-shaped policies.

  layernorm   layer norm, forward and (training) backward with the gradients of weight and bias
  dropout     dropout from a counter-based generator, with or without a residual, and its backward pass
  fused       dropout + residual add + layer norm, forward and (training) backward
  policy      clipped policy loss with a KL term from a head's logits, with the gradient
  attention   attention over long sequences that saves one number a row: forward and (training) a backward pass that computes
              the probabilities again; heads may share keys, batches may be padded, a decode step has one query a sequence

Everything is fp32, as the framework's other operators.  The sizes are those of the repository's own configurations (batch
1 024 x 64 tokens of width 256, minibatches of 65 536 with 16 actions, blocks of 24 x 50 tokens) and generic ones of larger models.
"""
import importlib
import math

import numpy as np
import torch

own = False
_CTX = {}
DEV = "cuda:0"


def _own():
    """The framework and the one context a program creates at start-up, on torch's current stream."""
    if "ctx" not in _CTX:
        _CTX["talos"] = importlib.import_module("talos-xii_b200")
        _CTX["ctx"] = _CTX["talos"].torch_context(0)
    return _CTX["talos"].lib, _CTX["talos"].ptr, _CTX["ctx"].handle


def listed():
    return [
        # one new token in a decode step: latency is all there is
        dict(name="norm_token", kind="layernorm", rows=1, dim=64, affine=True, train=False),
        # a wide model's norm over a batch whose row count divides nothing
        dict(name="norm_wide", kind="layernorm", rows=8191, dim=4096, affine=True, train=True),
        # dropout in the residual branch of the benchmark's block
        dict(name="dropout_block", kind="dropout", n=65536 * 256, p=0.1, residual=True),
        # dropout of activations of a small odd-sized layer
        dict(name="dropout_odd", kind="dropout", n=123457, p=0.35, residual=False),
        # the junction between the halves of the benchmark's block, training
        dict(name="fused_block", kind="fused", rows=65536, dim=256, p=0.1, train=True),
        # the same junction for a batch of 24 x 50 tokens of a width that no vector divides
        dict(name="fused_odd", kind="fused", rows=1200, dim=771, p=0.2, train=True),
        # the benchmark's policy head: a minibatch of 65 536 transitions, 16 actions of which some are illegal
        dict(name="policy_actions", kind="policy", rows=65536, vocab=16, pad=0, masked=0.1, padded=0.0, kl=0.0, entropy=0.01),
        # a batch of generated text with its padding, vocabulary of 32 000
        dict(name="policy_vocab", kind="policy", rows=4096, vocab=32000, pad=0, masked=0.0, padded=0.1, kl=0.05, entropy=0.0),
        # an odd vocabulary, rows that are not aligned to anything
        dict(name="policy_odd", kind="policy", rows=777, vocab=50257, pad=0, masked=0.0, padded=0.0, kl=0.05, entropy=0.01),
        # a decode step: one new token of 16 sequences, four query heads to a key head, caches filled to different lengths
        dict(name="attn_token", kind="attention", batch=16, heads=16, kv_heads=4, sq=1, sk=4096, d=64, dv=64, causal=True, ragged=True, train=False, mode="tf32x3"),
        # training on sequences of 2 048 tokens, heads of 64
        dict(name="attn_train", kind="attention", batch=4, heads=8, kv_heads=8, sq=2048, sk=2048, d=64, dv=64, causal=True, ragged=False, train=True, mode="tf32x3"),
        # training on a padded batch whose length fits no tile, heads that share keys, no causal mask
        dict(name="attn_padded", kind="attention", batch=3, heads=12, kv_heads=4, sq=777, sk=777, d=64, dv=64, causal=False, ragged=True, train=True, mode="tf32x3"),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]; about half of them odd."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v))


def _width(rng, lo, hi):
    """A row width: half of them multiples of four, as models have them."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.5 else min(hi, (v + 3) // 4 * 4)


def draw(rng):
    kind = rng.choice(["layernorm", "dropout", "fused", "policy", "policy", "attention", "attention"])
    if kind in ("layernorm", "fused"):
        dim = _width(rng, 8, 16384)
        case = dict(kind=kind, rows=_log(rng, 1, (1 << 25) // dim), dim=dim, train=rng.random() < 0.7)
        case.update(dict(affine=rng.random() < 0.8) if kind == "layernorm" else dict(p=rng.choice([0.0, 0.05, 0.1, 0.3])))
        return case
    if kind == "dropout":
        return dict(kind=kind, n=_log(rng, 1, 1 << 25), p=rng.choice([0.05, 0.1, 0.25, 0.5]), residual=rng.random() < 0.5)
    if kind == "policy":
        vocab = _width(rng, 4, 160000)
        return dict(kind=kind, rows=_log(rng, 1, min(65536, (1 << 27) // vocab)), vocab=vocab, pad=rng.choice([0, 0, 0, 4, 7]), masked=rng.choice([0.0, 0.0, 0.1]),
                    padded=rng.choice([0.0, 0.2]), kl=rng.choice([0.0, 0.05, 0.2]), entropy=rng.choice([0.0, 0.01]))
    d, dv = rng.choice([(64, 64), (64, 64), (32, 32), (96, 64), (128, 128), (40, 40)])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4])
    case = dict(kind=kind, batch=0, heads=kv_heads * group, kv_heads=kv_heads, sq=0, sk=0, d=d, dv=dv, causal=rng.random() < 0.7, ragged=rng.random() < 0.5,
                mode=rng.choice(["tf32x3", "tf32x3", "fp32"]))
    if rng.random() < 0.4:      # serving: a few new tokens of each sequence over a cache
        case.update(sq=rng.choice([1, 1, 1, rng.randint(2, 8)]), sk=_log(rng, 16, 16384), train=False)
        case.update(batch=_log(rng, 1, max(1, min(64, (1 << 25) // (case["sk"] * kv_heads * (d + dv))))))
    else:
        s = _log(rng, 16, 2048)
        case.update(sq=s, sk=s, train=rng.random() < 0.8, batch=_log(rng, 1, max(1, min(64, (1 << 26) // (s * s * kv_heads * group)))))
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------

EPS, CLIP_LOW, CLIP_HIGH = 1e-5, 0.2, 0.28


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)


def _normal(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _empty(*shape):
    return torch.empty(*shape, device=DEV)


def _stream_values(gen, rows, dim):
    """A residual stream: an offset, and a few channels that are far larger than the others."""
    wide = torch.where(torch.rand(dim, device=DEV, generator=gen) < 0.01, 10.0, 1.0)
    return _normal(gen, rows, dim) * wide + 0.5


def _padded_rows(case):
    return int(case["padded"] * case["rows"])


def _head(gen, rows, vocab, pad, masked):
    """Logits of a head [rows, vocab] (rows `pad` values further apart), the rows' tokens, their log-probabilities in 64 bits."""
    logits = torch.empty(rows, vocab + pad, device=DEV).normal_(0.0, 2.0, generator=gen)
    tokens = torch.randint(0, vocab, (rows,), device=DEV, generator=gen, dtype=torch.int32)
    at = tokens.long().unsqueeze(1)
    if masked:
        logits.masked_fill_(torch.rand(rows, vocab + pad, device=DEV, generator=gen) < masked, -math.inf)
    logits.scatter_(1, at, 4.0 + _normal(gen, rows, 1))
    z = logits[:, :vocab]
    logp = (z.gather(1, at).squeeze(1).double() - torch.logsumexp(z.double(), 1))
    return logits, tokens, logp


def prepare(case, seed):
    gen, s = _gen(seed), {"case": case, "seed": seed}
    kind = case["kind"]
    if kind in ("layernorm", "fused"):
        rows, dim = case["rows"], case["dim"]
        affine = case.get("affine", True)
        s.update(x=_stream_values(gen, rows, dim), gamma=1.0 + 0.2 * _normal(gen, dim) if affine else None, beta=0.1 * _normal(gen, dim) if affine else None,
                 y=_empty(rows, dim), mean=_empty(rows), inv=_empty(rows))
        if kind == "fused":
            s.update(residual=_stream_values(gen, rows, dim), h=_empty(rows, dim))
        if case["train"]:
            s.update(dy=_normal(gen, rows, dim), dx=_empty(rows, dim), dgamma=_empty(dim), dbeta=_empty(dim))
            if kind == "fused":
                s.update(dh=_normal(gen, rows, dim), dresidual=_empty(rows, dim))
    elif kind == "dropout":
        n = case["n"]
        s.update(x=_normal(gen, n), residual=_normal(gen, n) if case["residual"] else None, dy=_normal(gen, n), y=_empty(n), dx=_empty(n))
    elif kind == "policy":
        rows, vocab = case["rows"], case["vocab"]
        logits, tokens, logp = _head(gen, rows, vocab, case["pad"], case["masked"])
        # the policy has moved a little since the rollout; ratios next to the clip's two borders are moved off them
        shift = 0.2 * _normal(gen, rows).double()
        for border in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
            shift = torch.where((shift - border).abs() < 1e-3, shift + 4e-3, shift)
        weights = torch.ones(rows, device=DEV)
        weights[torch.randperm(rows, device=DEV, generator=gen)[: _padded_rows(case)]] = 0.0
        s.update(logits=logits, tokens=tokens, old=(logp - shift).float(), ref=(logp + 0.3 * _normal(gen, rows).double()).float(), adv=_normal(gen, rows),
                 weights=weights if case["padded"] else None, denom=float(rows - _padded_rows(case)) or 1.0, logp=_empty(rows), dlogits=_empty(rows, vocab), stats=_empty(5))
    else:
        b, hq, hkv, sq, sk, d, dv = (case[k] for k in ("batch", "heads", "kv_heads", "sq", "sk", "d", "dv"))
        s.update(q=2.0 * _normal(gen, b, hq, sq, d), k=_normal(gen, b, hkv, sk, d), v=_normal(gen, b, hkv, sk, dv), key_len=None, out=_empty(b, hq, sq, dv), lse=_empty(b, hq, sq))
        if case["ragged"]:      # at least half of the longest sequence
            s["key_len"] = torch.tensor(_lengths(case, seed), dtype=torch.int32, device=DEV)
        if case["train"]:
            s.update(dout=_normal(gen, b, hq, sq, dv), dq=_empty(b, hq, sq, d), dk=_empty(b, hkv, sk, d), dv=_empty(b, hkv, sk, dv))
    return s


def _lengths(case, seed):
    """The sequences' key counts: the case's own, in another order for each seed."""
    counts = np.random.RandomState(case["sk"] + 7 * case["batch"]).randint((case["sk"] + 1) // 2, case["sk"] + 1, case["batch"])
    return [int(v) for v in np.random.RandomState(seed % (1 << 31)).permutation(counts)]


# ---- the operators ---------------------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"layernorm": _own_layernorm, "dropout": _own_dropout, "fused": _own_fused, "policy": _own_policy, "attention": _own_attention}[kind](state)
    return {"layernorm": _layernorm, "dropout": _dropout, "fused": _fused, "policy": _policy, "attention": _attention}[kind](state)


def _own_layernorm(s):
    L, P, c = _own()
    rows, dim, train = s["case"]["rows"], s["case"]["dim"], s["case"]["train"]
    L.talos_layernorm_fwd(c, P(s["x"]), P(s["gamma"]), P(s["beta"]), EPS, rows, dim, P(s["y"]), P(s["mean"]) if train else None, P(s["inv"]) if train else None)
    if not train:
        return {"y": s["y"]}
    affine = s["gamma"] is not None
    L.talos_layernorm_bwd(c, P(s["dy"]), P(s["x"]), P(s["gamma"]), P(s["mean"]), P(s["inv"]), rows, dim, P(s["dx"]), P(s["dgamma"]) if affine else None,
                          P(s["dbeta"]) if affine else None, 0)
    out = {"y": s["y"], "mean": s["mean"], "inv": s["inv"], "dx": s["dx"]}
    return {**out, "dgamma": s["dgamma"], "dbeta": s["dbeta"]} if affine else out


def _own_dropout(s):
    L, P, c = _own()
    n, p, seed = s["case"]["n"], s["case"]["p"], s["seed"]
    L.talos_dropout_fwd(c, P(s["x"]), P(s["residual"]), P(s["y"]), n, p, seed, 3, None)
    L.talos_dropout_bwd(c, P(s["dy"]), P(s["dx"]), n, p, seed, 3, None, 0)
    return {"y": s["y"], "dx": s["dx"]}


def _own_fused(s):
    L, P, c = _own()
    rows, dim, p, seed, train = s["case"]["rows"], s["case"]["dim"], s["case"]["p"], s["seed"], s["case"]["train"]
    L.talos_dropout_add_layernorm_fwd(c, P(s["x"]), P(s["residual"]), P(s["gamma"]), P(s["beta"]), EPS, p, seed, 5, None, rows, dim, P(s["h"]), P(s["y"]),
                                      P(s["mean"]) if train else None, P(s["inv"]) if train else None)
    if not train:
        return {"h": s["h"], "y": s["y"]}
    L.talos_dropout_add_layernorm_bwd(c, P(s["dy"]), P(s["dh"]), P(s["h"]), P(s["gamma"]), P(s["mean"]), P(s["inv"]), p, seed, 5, None, rows, dim, P(s["dx"]),
                                      P(s["dresidual"]), P(s["dgamma"]), P(s["dbeta"]), 0)
    return {k: s[k] for k in ("h", "y", "dx", "dresidual", "dgamma", "dbeta")}


def _own_policy(s):
    L, P, c = _own()
    k = s["case"]
    L.talos_policy_loss_fwd_bwd(c, P(s["logits"]), k["vocab"] + k["pad"], P(s["tokens"]), P(s["old"]), P(s["ref"]) if k["kl"] else None, P(s["adv"]), P(s["weights"]),
                                k["rows"], k["vocab"], CLIP_LOW, CLIP_HIGH, k["kl"], k["entropy"], s["denom"], P(s["logp"]), P(s["dlogits"]), k["vocab"], P(s["stats"]), 0)
    return {"stats": s["stats"], "logp": s["logp"], "dlogits": s["dlogits"]}


def _own_attention(s):
    L, P, c = _own()
    k = s["case"]
    mode = _CTX["talos"].MODES[k["mode"]]
    shape = (k["batch"], k["heads"], k["kv_heads"], k["sq"], k["sk"], k["d"], k["dv"], 1.0 / math.sqrt(k["d"]), 1 if k["causal"] else 0, 0, mode)
    L.talos_attention_lse_fwd(c, P(s["q"]), P(s["k"]), P(s["v"]), P(s["key_len"]), P(s["out"]), P(s["lse"]) if k["train"] else None, *shape)
    if not k["train"]:
        return {"out": s["out"]}
    L.talos_attention_lse_bwd(c, P(s["q"]), P(s["k"]), P(s["v"]), P(s["key_len"]), P(s["out"]), P(s["lse"]), P(s["dout"]), P(s["dq"]), P(s["dk"]), P(s["dv"]), *shape)
    return {k: s[k] for k in ("out", "lse", "dq", "dk", "dv")}


# plain forms

def _normed(x, gamma, beta):
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    inv = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    hat = centred * inv
    return mean, inv, hat, hat if gamma is None else hat * gamma + beta


def _normed_bwd(dy, hat, inv, gamma):
    g = dy if gamma is None else dy * gamma
    return inv * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True)), (dy * hat).sum(0), dy.sum(0)


def _layernorm(s):
    mean, inv, hat, y = _normed(s["x"], s["gamma"], s["beta"])
    if not s["case"]["train"]:
        return {"y": y}
    dx, dgamma, dbeta = _normed_bwd(s["dy"], hat, inv, s["gamma"])
    out = {"y": y, "mean": mean[:, 0], "inv": inv[:, 0], "dx": dx}
    return {**out, "dgamma": dgamma, "dbeta": dbeta} if s["gamma"] is not None else out


def _words(n, seed, offset):
    """The generator's first n 32-bit words, as int64: philox4x32-10 of key = seed, counter = (word / 4, offset)."""
    low = 0xFFFFFFFF
    i = torch.arange((n + 3) // 4, device=DEV, dtype=torch.int64)
    c0, c1, c2, c3 = i & low, i >> 32, torch.full_like(i, offset & low), torch.full_like(i, offset >> 32)
    k0, k1 = seed & low, (seed >> 32) & low

    def times(m, b):        # high and low word of the 64-bit product, from halves that fit int64
        top = m * (b >> 16) + ((m * (b & 0xFFFF)) >> 16)
        return top >> 16, (m * b) & low

    for _ in range(10):     # the generator's ten rounds
        h0, l0 = times(0xD2511F53, c0)
        h1, l1 = times(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n]


def _scale(shape, p, seed, offset):
    """0 where a value is dropped, 1 / (1 - p) where it is kept."""
    keep = _words(math.prod(shape), seed, offset) >= int(math.floor(float(np.float32(p)) * 2.0 ** 32 + 0.5))
    return torch.where(keep, 1.0 / (1.0 - float(np.float32(p))), 0.0).float().reshape(shape)


def _dropout(s):
    scale = _scale(s["x"].shape, s["case"]["p"], s["seed"], 3)
    y = s["x"] * scale
    return {"y": y if s["residual"] is None else s["residual"] + y, "dx": s["dy"] * scale}


def _fused(s):
    scale = _scale(s["x"].shape, s["case"]["p"], s["seed"], 5)
    h = s["residual"] + s["x"] * scale
    mean, inv, hat, y = _normed(h, s["gamma"], s["beta"])
    if not s["case"]["train"]:
        return {"h": h, "y": y}
    dh, dgamma, dbeta = _normed_bwd(s["dy"], hat, inv, s["gamma"])
    dh = dh + s["dh"]
    return {"h": h, "y": y, "dx": dh * scale, "dresidual": dh, "dgamma": dgamma, "dbeta": dbeta}


def _log_softmax(z):
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    return e, total, z - (top + torch.log(total))


def _policy(s):
    k, at = s["case"], s["tokens"].long().unsqueeze(1)
    e, total, logs = _log_softmax(s["logits"][:, : k["vocab"]])
    p = e / total
    logp = logs.gather(1, at)
    plogs = torch.where(p > 0, p * logs, 0.0)
    entropy = -plogs.sum(1, keepdim=True)
    w = (torch.ones_like(s["adv"]) if s["weights"] is None else s["weights"]).unsqueeze(1)
    adv = s["adv"].unsqueeze(1)
    ratio = torch.exp(logp - s["old"].unsqueeze(1))
    s1, s2 = ratio * adv, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv
    inside = (ratio >= 1 - CLIP_LOW) & (ratio <= 1 + CLIP_HIGH)
    delta = s["ref"].unsqueeze(1) - logp if k["kl"] else torch.zeros_like(logp)
    kl = torch.expm1(delta) - delta
    loss = -torch.minimum(s1, s2) + k["kl"] * kl - k["entropy"] * entropy
    clipped = ((s2 < s1) & ~inside).float()
    dlogp = w / s["denom"] * (-torch.where((s1 < s2) | inside, s1, 0.0) - k["kl"] * torch.expm1(delta))
    dlogits = -dlogp * p + w / s["denom"] * k["entropy"] * (plogs + p * entropy)
    dlogits.scatter_add_(1, at, dlogp)
    sums = torch.cat([w * loss, w * kl, w * entropy, w * clipped, w], 1).double().sum(0).float()
    return {"stats": sums, "logp": torch.where(w[:, 0] == 0, 0.0, logp[:, 0]), "dlogits": dlogits}


def _visible(case, key_len):
    """[batch or 1, 1, 1, sq, sk]: which keys a query sees."""
    i, j = torch.arange(case["sq"], device=DEV).unsqueeze(1), torch.arange(case["sk"], device=DEV)
    see = (j <= i + case["sk"] - case["sq"]) if case["causal"] else torch.ones(case["sq"], case["sk"], device=DEV, dtype=torch.bool)
    return see[None, None, None] if key_len is None else see & (j < key_len.view(-1, 1, 1, 1, 1))


def _attention(s):
    c = s["case"]
    scale = 1.0 / math.sqrt(c["d"])
    q = s["q"].unflatten(1, (c["kv_heads"], -1))                          # [batch, key heads, queries' group, sq, d]
    k, v = s["k"].unsqueeze(2), s["v"].unsqueeze(2)
    scores = (q @ k.transpose(-1, -2) * scale).masked_fill_(~_visible(c, s["key_len"]), -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)                  # a row that sees no key: exp(-inf - top) = 0
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    out = p @ v
    if not c["train"]:
        return {"out": out.flatten(1, 2)}
    dout = s["dout"].unflatten(1, (c["kv_heads"], -1))
    dp = dout @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    return {"out": out.flatten(1, 2), "lse": lse[..., 0].flatten(1, 2), "dq": (ds @ k).flatten(1, 2), "dk": (ds.transpose(-1, -2) @ q).sum(2),
            "dv": (p.transpose(-1, -2) @ dout).sum(2)}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def _kept(n, p, seed, offset):
    """1 / (1 - p) where a value is kept, 0 where not, in 64 bits: the generator in numpy's unsigned words."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    block = np.arange(-(-n // 4), dtype=np.uint64)
    ctr = [block & low, block >> u(32), np.full_like(block, offset % 2 ** 32), np.full_like(block, offset // 2 ** 32)]
    key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
    for r in range(10):
        a, b = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ctr = [(b >> u(32)) ^ ctr[1] ^ u((key[0] + r * 0x9E3779B9) % 2 ** 32), b & low, (a >> u(32)) ^ ctr[3] ^ u((key[1] + r * 0xBB67AE85) % 2 ** 32), a & low]
    words = np.stack(ctr, 1).reshape(-1)[:n]
    p = float(np.float32(p))
    return torch.from_numpy(np.where(words < round(p * 2 ** 32), 0.0, 1.0 / (1.0 - p))).to(DEV)


def _exact_norm(x, s, extra):
    """Layer norm and, where there is an upstream gradient, its gradients through torch's tape."""
    dim = x.shape[1]
    x = x.detach().requires_grad_(True)
    gamma = (torch.ones(dim, device=DEV) if s["gamma"] is None else s["gamma"]).double().requires_grad_(True)
    beta = (torch.zeros(dim, device=DEV) if s["beta"] is None else s["beta"]).double().requires_grad_(True)
    mean, var = x.mean(1, keepdim=True), x.var(1, keepdim=True, unbiased=False)
    inv = (var + EPS) ** -0.5
    y = (x - mean) * inv * gamma + beta
    if not extra:
        return y.detach(), None, None, (None, None, None)
    return y.detach(), mean.detach()[:, 0], inv.detach()[:, 0], torch.autograd.grad(y, (x, gamma, beta), s["dy"].double())


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "layernorm":
        y, mean, inv, (dx, dgamma, dbeta) = _exact_norm(s["x"].double(), s, case["train"])
        if not case["train"]:
            return {"y": y}
        out = {"y": y, "mean": mean, "inv": inv, "dx": dx}
        return {**out, "dgamma": dgamma, "dbeta": dbeta} if case["affine"] else out
    if kind == "dropout":
        k = _kept(case["n"], case["p"], seed, 3)
        y = s["x"].double() * k
        return {"y": y + s["residual"].double() if case["residual"] else y, "dx": s["dy"].double() * k}
    if kind == "fused":
        k = _kept(case["rows"] * case["dim"], case["p"], seed, 5).reshape(case["rows"], case["dim"])
        h = s["x"].double() * k + s["residual"].double()
        y, _, _, (dn, dgamma, dbeta) = _exact_norm(h, s, case["train"])
        if not case["train"]:
            return {"h": h, "y": y}
        dh = dn + s["dh"].double()
        return {"h": h, "y": y, "dx": dh * k, "dresidual": dh, "dgamma": dgamma, "dbeta": dbeta}
    if kind == "policy":
        at = s["tokens"].long().unsqueeze(1)
        z = s["logits"][:, : case["vocab"]].double()
        logs = torch.log_softmax(z, 1)
        del z
        lp = logs.gather(1, at)[:, 0]
        p = logs.exp()
        p_logs = torch.special.entr(p)                                   # -p log p, 0 where p is 0
        entropy = p_logs.sum(1)
        w = torch.ones_like(lp) if s["weights"] is None else s["weights"].double()
        adv, ratio = s["adv"].double(), (lp - s["old"].double()).exp()
        low, high = float(np.float32(1) - np.float32(CLIP_LOW)), float(np.float32(1) + np.float32(CLIP_HIGH))
        free, held = ratio * adv, ratio.clip(low, high) * adv
        active = torch.where(held < free, (ratio > low) & (ratio < high), torch.ones_like(ratio, dtype=torch.bool))
        d = s["ref"].double() - lp if case["kl"] else torch.zeros_like(lp)
        kl = d.exp() - d - 1
        loss = -torch.where(held < free, held, free) + case["kl"] * kl - case["entropy"] * entropy
        g = w / s["denom"] * (case["kl"] * (1 - d.exp()) - active * free)
        dz = p_logs.neg_().addcmul_(p, entropy.unsqueeze(1)).mul_((case["entropy"] * w / s["denom"]).unsqueeze(1))
        dz.addcmul_(p, g.unsqueeze(1), value=-1.0)
        dz[torch.arange(case["rows"], device=DEV), at[:, 0]] += g
        stats = torch.stack([(w * loss).sum(), (w * kl).sum(), (w * entropy).sum(), w[~active].sum(), w.sum()])
        return {"stats": stats, "logp": lp * (w != 0), "dlogits": dz}
    q, k, v = (s[n].double().requires_grad_(case["train"]) for n in ("q", "k", "v"))
    group = case["heads"] // case["kv_heads"]
    rows = torch.einsum("bhid,bhjd->bhij", q, k.repeat_interleave(group, 1)) / math.sqrt(case["d"])
    hidden = torch.zeros(case["batch"], 1, case["sq"], case["sk"], device=DEV, dtype=torch.bool)
    for b, n in enumerate(_lengths(case, seed) if case["ragged"] else []):
        hidden[b, :, :, n:] = True
    if case["causal"]:
        hidden = hidden | torch.ones(case["sq"], case["sk"], device=DEV, dtype=torch.bool).triu(case["sk"] - case["sq"] + 1)
    rows = rows.masked_fill(hidden, -math.inf)
    out = torch.einsum("bhij,bhjd->bhid", torch.softmax(rows, -1), v.repeat_interleave(group, 1))      # (every query of these cases sees a key)
    if not case["train"]:
        return {"out": out}
    lse = torch.logsumexp(rows, -1).detach()
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"].double())
    return {"out": out.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("layernorm", "fused"):
        rows, dim = case["rows"], case["dim"]
        e = rows * dim
        fused = kind == "fused"
        moved, ops = (16 if fused else 8) * e + 8 * dim, (10 + 8) * e if fused else 8 * e
        if case["train"]:
            moved += (20 if fused else 12) * e + 16 * rows + 16 * dim
            ops += (14 + 8) * e if fused else 14 * e
        return {"bytes": moved, "flops": ops}
    if kind == "dropout":
        return {"bytes": (20 if case["residual"] else 16) * case["n"], "flops": 4 * case["n"]}
    if kind == "policy":
        rows, read = case["rows"], case["rows"] - _padded_rows(case)      # padding is not read, its gradient is zero
        return {"bytes": 4 * case["vocab"] * (read + rows) + 28 * rows, "flops": 12 * case["vocab"] * read}
    b, hq, hkv, sq, sk, d, dv = (case[k] for k in ("batch", "heads", "kv_heads", "sq", "sk", "d", "dv"))
    keys = _lengths(case, 0) if case["ragged"] else [sk] * b
    first = sk - sq                                                       # a causal query i sees the keys up to i + first
    pairs = hq * sum(sum(min(n, i + first + 1) for i in range(sq)) if case["causal"] else sq * n for n in keys)
    moved, ops = 4 * (b * hq * sq * (d + dv) + hkv * sum(keys) * (d + dv)), 2 * (d + dv) * pairs
    if case["train"]:
        moved += 4 * (b * hq * sq * (2 * d + 2 * dv + 2) + hkv * (sum(keys) + b * sk) * (d + dv))
        ops += (6 * d + 4 * dv) * pairs
    return {"bytes": moved, "flops": ops}
