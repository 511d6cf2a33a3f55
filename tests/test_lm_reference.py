"""CPU tests of the operators in include/talos_b200_lm.h: the 64-bit forms that the GPU tests compare with (published vectors,
finite differences) and the calls that the entry points refuse, which they do before they look at the context."""
import numpy as np
import pytest

import lm_reference as ref


def test_philox_published_vectors():
    # the known-answer vectors published with the generator: zeros, ones, digits of pi (counter words low first)
    assert [hex(w) for w in ref.philox([0], 0, 0)[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = 2 ** 64 - 1
    assert [hex(w) for w in ref.philox(np.array([ones], dtype=np.uint64), ones, ones)[0]] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]
    block = np.array([0x85a308d3243f6a88], dtype=np.uint64)
    assert [hex(w) for w in ref.philox(block, 0x0370734413198a2e, 0x299f31d0a4093822)[0]] == ["0xd16cfe09", "0x94fdcceb", "0x5001e420", "0x24126ea1"]


def test_dropout_keeps_its_share():
    n, p = 200000, 0.3
    kept = ref.keep(n, p, 99, 7).mean()
    assert abs(kept - 0.7) < 5 * np.sqrt(0.21 / n)                        # five standard deviations
    assert ref.keep(n, 0.0, 99, 7).all()


def differences(f, x, h=1e-6):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h; b[i] -= h
        g[i] = (f(a) - f(b)) / (2 * h)
    return g


def test_layernorm_gradients_are_differences():
    rng = np.random.RandomState(0)
    x, dy, gamma, beta = rng.randn(4, 7) * 2 + 1, rng.randn(4, 7), rng.randn(7), rng.randn(7)
    _, mean, inv = ref.layernorm(x, gamma, beta, 1e-5)
    dx, dgamma, dbeta = ref.layernorm_bwd(dy, x, gamma, mean, inv)
    assert np.abs(dx - differences(lambda v: (dy * ref.layernorm(v, gamma, beta, 1e-5)[0]).sum(), x)).max() < 1e-8
    assert np.abs(dgamma - differences(lambda v: (dy * ref.layernorm(x, v, beta, 1e-5)[0]).sum(), gamma)).max() < 1e-8
    assert np.abs(dbeta - differences(lambda v: (dy * ref.layernorm(x, gamma, v, 1e-5)[0]).sum(), beta)).max() < 1e-8


@pytest.mark.parametrize("c_kl,c_ent", [(0.0, 0.0), (0.1, 0.0), (0.0, 0.02), (0.1, 0.02)])
def test_policy_loss_gradients_are_differences(c_kl, c_ent):
    rng = np.random.RandomState(1)
    rows, vocab = 12, 5
    z, tokens = rng.randn(rows, vocab), rng.randint(0, vocab, rows)
    z[3, (tokens[3] + 1) % vocab] = -np.inf                               # a masked token
    tokens[5] = -1                                                        # padding
    lp = z[np.arange(rows), tokens] - np.log(np.exp(z).sum(1))
    old, rf, adv, w = lp + 0.4 * rng.randn(rows), lp + 0.3 * rng.randn(rows), rng.randn(rows), rng.rand(rows) + 0.5
    w[7] = 0.0
    f = lambda v: ref.policy_loss(v, tokens, old, rf, adv, w, 0.2, 0.3, c_kl, c_ent, 4.0)  # noqa: E731
    stats, logp, dz = f(z)[:3]
    assert stats[3] > 0 and abs(stats[4] - (w.sum() - w[5])) < 1e-12
    free = np.isfinite(z)
    num = differences(lambda v: f(v)[0][0] / 4.0, np.where(free, z, -800.0))
    assert np.abs(dz - num)[free].max() < 1e-8 and (dz[~free] == 0).all() and (dz[[5, 7]] == 0).all()


@pytest.mark.parametrize("causal,key_len", [(False, None), (True, None), (True, [3, 0]), (False, [5, 2])])
def test_attention_gradients_are_differences(causal, key_len):
    rng = np.random.RandomState(2)
    q, k, v, do = rng.randn(2, 4, 3, 6), rng.randn(2, 2, 5, 6), rng.randn(2, 2, 5, 4), rng.randn(2, 4, 3, 4)
    out, lse, dq, dk, dv = ref.attention(q, k, v, key_len, 0.4, causal, do)[:5]
    f = lambda a, b, c: (ref.attention(a, b, c, key_len, 0.4, causal)[0] * do).sum()  # noqa: E731
    assert np.abs(dq - differences(lambda a: f(a, k, v), q)).max() < 1e-8
    assert np.abs(dk - differences(lambda a: f(q, a, v), k)).max() < 1e-8
    assert np.abs(dv - differences(lambda a: f(q, k, a), v)).max() < 1e-8
    if key_len and key_len[1] == 0: assert (out[1] == 0).all() and (lse[1] == -np.inf).all()


P = 4096     # an address that is never read: the call is refused first, or fails for want of a context


@pytest.mark.parametrize("args,status,text", [
    ((P, P, P, -1.0, 4, 8, P, P, P), 1, "eps"), ((P, P, P, 1e-5, 4, 16385, P, P, P), 2, "16384"), ((P, P, P, 1e-5, 4, 0, P, P, P), 2, "16384"),
    ((P, P, P, 1e-5, -1, 8, P, P, P), 2, "rows"), ((None, P, P, 1e-5, 4, 8, P, P, P), 1, "null pointer"), ((P, P, P, 1e-5, 4, 8, None, P, P), 1, "null pointer"),
    ((P, None, None, 1e-5, 4, 8, P, None, None), 1, "null context")])
def test_layernorm_fwd_refuses(talos, args, status, text):
    with pytest.raises(talos.TalosError) as e: talos.lib.talos_layernorm_fwd(None, *args)
    assert e.value.status == status and text in str(e.value)


@pytest.mark.parametrize("args,status,text", [
    ((P, P, P, P, P, 4, 20000, P, P, P, 0), 2, "16384"), ((P, P, P, P, P, 4, 8, P, P, P, 8), 1, "accumulate"), ((P, P, P, None, P, 4, 8, P, P, P, 0), 1, "null pointer"),
    ((P, P, None, P, P, 4, 8, None, None, None, 0), 1, "null context")])
def test_layernorm_bwd_refuses(talos, args, status, text):
    with pytest.raises(talos.TalosError) as e: talos.lib.talos_layernorm_bwd(None, *args)
    assert e.value.status == status and text in str(e.value)


def test_dropout_refuses(talos):
    L = talos.lib
    for p in (1.0, -0.1, float("nan"), 2.0):
        for call in (lambda: L.talos_dropout_fwd(None, P, None, P, 8, p, 1, 0, None), lambda: L.talos_dropout_bwd(None, P, P, 8, p, 1, 0, None, 0),
                     lambda: L.talos_dropout_add_layernorm_fwd(None, P, P, P, P, 1e-5, p, 1, 0, None, 4, 8, P, 2 * P, P, P),
                     lambda: L.talos_dropout_add_layernorm_bwd(None, P, P, P, P, P, P, p, 1, 0, None, 4, 8, P, 2 * P, P, P, 0)):
            with pytest.raises(talos.TalosError) as e: call()
            assert e.value.status == 1 and "probability" in str(e.value)
    for call, text in ((lambda: L.talos_dropout_fwd(None, P, None, P, -1, 0.1, 1, 0, None), "negative"), (lambda: L.talos_dropout_fwd(None, None, None, P, 8, 0.1, 1, 0, None), "null pointer"),
                       (lambda: L.talos_dropout_bwd(None, P, P, 8, 0.1, 1, 0, None, 2), "accumulate"), (lambda: L.talos_dropout_bwd(None, P, None, 8, 0.1, 1, 0, None, 0), "null pointer"),
                       (lambda: L.talos_dropout_add_layernorm_fwd(None, P, P, P, P, 1e-5, 0.1, 1, 0, None, 4, 8, P, P, P, P), "two results"),
                       (lambda: L.talos_dropout_add_layernorm_bwd(None, P, P, P, P, P, P, 0.1, 1, 0, None, 4, 8, P, P, P, P, 0), "two results"),
                       (lambda: L.talos_dropout_add_layernorm_bwd(None, P, P, P, P, P, P, 0.1, 1, 0, None, 4, 8, P, 2 * P, P, P, 16), "accumulate"),
                       (lambda: L.talos_dropout_fwd(None, P, None, P, 8, 0.1, 2 ** 64 - 1, 2 ** 64 - 1, None), "null context")):
        with pytest.raises(talos.TalosError) as e: call()
        assert text in str(e.value)


POLICY = dict(logits=P, ld=8, tokens=P, old=P, ref=P, adv=P, w=P, rows=4, vocab=8, lo=0.2, hi=0.2, kl=0.1, ent=0.0, denom=4.0, logp=P, dlogits=2 * P, ld_out=8, stats=P, acc=0)


@pytest.mark.parametrize("change,status,text", [
    (dict(vocab=0), 2, "shape"), (dict(rows=-1), 2, "shape"), (dict(ld=7), 2, "stride"), (dict(ld_out=7), 2, "stride"), (dict(lo=1.5), 1, "clip"), (dict(lo=-0.1), 1, "clip"),
    (dict(hi=-0.1), 1, "clip"), (dict(denom=0.0), 1, "denominator"), (dict(denom=float("nan")), 1, "denominator"), (dict(acc=2), 1, "accumulate"), (dict(ref=None), 1, "ref_logp"),
    (dict(dlogits=P, ld_out=12), 1, "same row stride"), (dict(old=None), 1, "old_logp"), (dict(old=None, adv=None), 1, "old_logp"), (dict(logits=None), 1, "null pointer"),
    (dict(tokens=None), 1, "null pointer"), (dict(), 1, "null context"), (dict(old=None, adv=None, dlogits=None), 1, "null context"), (dict(ref=None, kl=0.0), 1, "null context")])
def test_policy_loss_refuses(talos, change, status, text):
    with pytest.raises(talos.TalosError) as e: talos.lib.talos_policy_loss_fwd_bwd(None, *{**POLICY, **change}.values())
    assert e.value.status == status and text in str(e.value)


ATTN = dict(q=P, k=P, v=P, key_len=P, out=P, lse=P, batch=2, heads=4, kv_heads=2, sq=16, sk=32, d=64, dv=64, scale=0.125, causal=0, layout=0, mode=1)


@pytest.mark.parametrize("change,status,text", [
    (dict(kv_heads=3), 2, "kv_heads"), (dict(kv_heads=0), 2, "kv_heads"), (dict(sq=-1), 2, "negative"), (dict(d=0), 2, "1 to 128"), (dict(d=129), 2, "1 to 128"), (dict(dv=160), 2, "1 to 128"),
    (dict(sq=2 ** 25), 2, "too large"), (dict(layout=2), 1, "layout"), (dict(mode=3), 1, "mode"), (dict(scale=float("nan")), 1, "scale"), (dict(causal=2), 1, "causal"),
    (dict(q=None), 1, "null pointer"), (dict(k=None), 1, "null pointer"), (dict(out=None), 1, "null pointer"), (dict(lse=None, key_len=None), 1, "null context")])
def test_attention_refuses(talos, change, status, text):
    args = {**ATTN, **change}
    with pytest.raises(talos.TalosError) as e: talos.lib.talos_attention_lse_fwd(None, *args.values())
    assert e.value.status == status and text in str(e.value)
    if change.get("lse", P) is None: args["lse"], text = None, "null pointer"     # the backward pass needs it
    head = {n: args.pop(n) for n in ("q", "k", "v", "key_len", "out", "lse")}
    with pytest.raises(talos.TalosError) as e: talos.lib.talos_attention_lse_bwd(None, *head.values(), P, P, P, P, *args.values())
    assert e.value.status == status and text in str(e.value)
