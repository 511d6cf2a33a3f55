"""The operators together, as they are used: a language-model-shaped policy (layer norm, attention over the whole padded sequence with shared key heads,
dropout + residual + layer norm, feed-forward with dropout, head, clipped policy loss with a KL term) through the C++ host layer, loss and every gradient
against the same network in 64 bits on torch's tape."""
import os
import subprocess

import numpy as np
import pytest
import torch

import lm_reference as ref

pytestmark = pytest.mark.gpu
BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin", "lm_driver")


def shapes(D, Hd, ff, V):
    return [("n1.w", (D,)), ("n1.b", (D,)), ("q", (D, D)), ("k", (D, Hd)), ("v", (D, Hd)), ("o", (D, D)), ("o.b", (D,)), ("n2.w", (D,)), ("n2.b", (D,)), ("f1", (D, ff)), ("f1.b", (ff,)),
            ("f2", (ff, D)), ("f2.b", (D,)), ("nf.w", (D,)), ("nf.b", (D,)), ("head", (D, V)), ("head.b", (V,))]


def norm(x, w, b):
    m = x.mean(-1, keepdim=True)
    return (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + float(np.float32(1e-5))) * w + b


# Relative 2-norm: the framework's tolerance of one fp32-faithful product is 1e-5 and of a fast one 2e-3; a gradient of this network passes through a
# dozen of them whose errors add like independent ones (sqrt(12) = 3.5), and the worst of seventeen is looked at.
@pytest.mark.parametrize("mode,tol", [(0, 4e-5), (1, 4e-5), (2, 8e-3)])
@pytest.mark.parametrize("B,S,D,H,Hk,ff,V,p", [(2, 90, 64, 4, 2, 96, 300, 0.1), (3, 33, 48, 3, 3, 64, 1001, 0.3), (1, 200, 128, 2, 1, 128, 512, 0.0)])
def test_policy_loss_and_gradients(tmp_path, mode, tol, B, S, D, H, Hk, ff, V, p):
    rng = np.random.RandomState(B + S)
    f32 = lambda a: np.asarray(a, dtype=np.float32).astype(np.float64)  # noqa: E731
    seed, step, dh = 1234567, 3, D // H
    x = f32(rng.randn(B, S, D))
    params = {}
    for name, s in shapes(D, dh * Hk, ff, V):
        params[name] = f32(rng.randn(*s) * (0.3 / np.sqrt(s[0]) * 2 if len(s) == 2 else 0.1) + (1.0 if name.endswith(".w") else 0.0))
    n, lens = B * S, rng.randint(S // 2, S + 1, B)
    tokens = rng.randint(0, V, n); tokens[::11] = -1
    adv, w = f32(rng.randn(n)), f32(0.5 + rng.rand(n))
    w[5::13] = 0.0

    tx = torch.tensor(x, requires_grad=True)
    tp = {k: torch.tensor(v, requires_grad=True) for k, v in params.items()}
    drop = lambda t, offset: t * torch.tensor(ref.keep(t.numel(), p, seed, offset).reshape(t.shape) / (1.0 - float(np.float32(p))))  # noqa: E731
    a = norm(tx, tp["n1.w"], tp["n1.b"])
    q, k, v = (a @ tp["q"]).view(B, S, H, dh), (a @ tp["k"]).view(B, S, Hk, dh), (a @ tp["v"]).view(B, S, Hk, dh)
    k, v = k.repeat_interleave(H // Hk, 2), v.repeat_interleave(H // Hk, 2)
    see = torch.tril(torch.ones(S, S, dtype=torch.bool))[None, None] & (torch.arange(S)[None, None, None] < torch.tensor(lens)[:, None, None, None])
    scores = torch.einsum("bihd,bjhd->bhij", q, k) / np.sqrt(dh)
    att = torch.einsum("bhij,bjhd->bihd", torch.softmax(scores.masked_fill(~see, -np.inf), -1), v).reshape(B, S, D)
    h = tx + drop(att @ tp["o"] + tp["o.b"], 2 * step)
    y = norm(h, tp["n2.w"], tp["n2.b"])
    u = y @ tp["f1"] + tp["f1.b"]
    out = h + drop((u * torch.sigmoid(u)) @ tp["f2"] + tp["f2.b"], 2 * step + 1)
    logits = norm(out, tp["nf.w"], tp["nf.b"]) @ tp["head"] + tp["head.b"]
    z = logits.detach().numpy().reshape(n, V)
    lp = np.where(tokens >= 0, z[np.arange(n), np.maximum(tokens, 0)] - np.logaddexp.reduce(z, 1), 0.0)
    shift = 0.2 * rng.randn(n)
    for border in (np.log(0.8), np.log(1.28)): shift = np.where(np.abs(shift - border) < 0.05, shift + 0.11, shift)      # no ratio where an error of the fast mode moves it over a border
    old, rf = f32(lp - shift), f32(lp + 0.2 * rng.randn(n))
    stats, logp, dz = ref.policy_loss(z, tokens, old, rf, adv, w, 0.2, 0.28, 0.05, 0.01, float(n))[:3]
    want = torch.autograd.grad(logits, [tx, *tp.values()], torch.tensor(dz.reshape(B, S, V)))

    (tmp_path / "in").write_bytes(np.concatenate([x.ravel(), *[v.ravel() for v in params.values()], tokens, old, rf, adv, w, lens]).astype(np.float64).tobytes())
    r = subprocess.run([BIN, str(mode), str(tmp_path / "in"), str(tmp_path / "out"), *[str(i) for i in (B, S, D, H, Hk, ff, V, p, seed, step)]], stdout=subprocess.PIPE,
                       stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    flat, at = np.fromfile(tmp_path / "out"), 0
    wanted = [("logits", z), ("loss", np.array([stats[0] / n])), ("logp", logp_all(z, tokens)), ("x", want[0].numpy()), *[(k, g.numpy()) for k, g in zip(params, want[1:])]]
    for name, ref_value in wanted:
        got = flat[at:at + ref_value.size].reshape(ref_value.shape); at += ref_value.size
        scale = np.abs(w).sum() / n if name == "loss" else np.linalg.norm(ref_value)      # (the loss is a sum of terms of either sign)
        assert np.linalg.norm(got - ref_value) <= tol * scale, (name, np.linalg.norm(got - ref_value) / scale)
    assert at == flat.size


def logp_all(z, tokens):
    return np.where(tokens >= 0, z[np.arange(len(tokens)), np.maximum(tokens, 0)] - np.logaddexp.reduce(z, 1), 0.0)


# x + dropout(x): both gradients go into one buffer; then h alone, over the same nodes.  Tolerance: a dozen fp32 roundings of the row's own sums (2^-24 each, the
# sums over the rows of a column included, at 70 rows) is below 1e-5 of the 2-norm.
@pytest.mark.parametrize("R,D,p", [(70, 96, 0.25), (1, 5, 0.5)])
def test_junction_of_a_tensor_with_itself(tmp_path, R, D, p):
    rng = np.random.RandomState(R)
    x, w, b, gh, gy = [rng.randn(*s).astype(np.float32).astype(np.float64) for s in ((R, D), (D,), (D,), (R, D), (R, D))]
    (tmp_path / "in").write_bytes(np.concatenate([t.ravel() for t in (x, w, b, gh, gy)]).tobytes())
    r = subprocess.run([BIN, "junction", str(tmp_path / "in"), str(tmp_path / "out"), str(R), str(D), str(p), "42"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    got = np.split(np.fromfile(tmp_path / "out"), np.cumsum([R * D, D, D, R * D, D]))
    t = [torch.tensor(a, requires_grad=True) for a in (x, w, b)]
    h = t[0] + t[0] * torch.tensor(ref.keep(R * D, p, 42, 5).reshape(R, D) / (1.0 - p))
    first = torch.autograd.grad((h * torch.tensor(gh)).sum() + (norm(h, t[1], t[2]) * torch.tensor(gy)).sum(), t, retain_graph=True)
    for name, value, g in zip("xwb", got, first):
        assert np.linalg.norm(value - g.numpy().ravel()) <= 1e-5 * np.linalg.norm(g.numpy()), name
    second = torch.autograd.grad((h * torch.tensor(gh)).sum(), t[0])[0].numpy().ravel()
    assert np.linalg.norm(got[3] - second) <= 1e-5 * np.linalg.norm(second)
    assert not got[4].any() and not got[5].any()
