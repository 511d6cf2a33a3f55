"""The policy loss over a vocabulary on the GPU against its 64-bit form, with bounds counted from roundings."""
import numpy as np
import pytest

import lm_reference as ref
from test_gpu_norm_dropout import blank, get, put

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(talos):
    c = talos.torch_context(0)
    yield c
    c.synchronize()


def f32(a):
    return np.asarray(a, dtype=np.float32).astype(np.float64)


def ints(a):
    import torch
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda:0")


def make(rows, vocab, seed, masked=0.1):
    rng = np.random.RandomState(seed)
    z = f32(3 * rng.randn(rows, vocab))
    tokens = rng.randint(0, vocab, rows)
    z[rng.rand(rows, vocab) < masked] = -np.inf
    z[np.arange(rows), tokens] = f32(2 + rng.randn(rows))
    lp = z[np.arange(rows), tokens] - np.logaddexp.reduce(z, 1)
    # ratios at least 1e-3 away from the clip's borders, where a rounding would change the formula's branch
    shift = 0.25 * rng.randn(rows)
    for border in (np.log(0.8), np.log(1.3)): shift = np.where(np.abs(shift - border) < 1e-3, shift + 4e-3, shift)
    old, rf, adv, w = f32(lp - shift), f32(lp + 0.3 * rng.randn(rows)), f32(rng.randn(rows)), f32(0.5 + rng.rand(rows))
    return z, tokens, old, rf, adv, w


class Call:
    """One call's device buffers; rows are `pad` (logits) and `pad_out` (gradient) values further apart than the vocabulary."""
    def __init__(self, z, tokens, old, rf, adv, w, pad=0, pad_out=0, off=0):
        rows, vocab = z.shape
        wide = np.full((rows, vocab + pad), 1e30); wide[:, :vocab] = z
        self.shape, self.ld, self.ld_out = z.shape, vocab + pad, vocab + pad_out
        self.z, self.tokens = put(wide, off), ints(tokens)
        self.old, self.ref, self.adv, self.w = (None if a is None else put(a) for a in (old, rf, adv, w))
        self.logp, self.dz, self.stats = blank(rows), blank((rows, vocab + pad_out), off, -55.0), blank(5)

    def run(self, talos, ctx, c_kl, c_ent, denom, acc=0, dz=True, in_place=False):
        p = talos.ptr
        out = p(self.z) if in_place else p(self.dz) if dz else None
        talos.lib.talos_policy_loss_fwd_bwd(ctx.handle, p(self.z), self.ld, p(self.tokens), p(self.old), p(self.ref), p(self.adv), p(self.w), self.shape[0], self.shape[1], 0.2, 0.3,
                                            c_kl, c_ent, denom, p(self.logp), out, self.ld if in_place else self.ld_out, p(self.stats), acc)
        return get(self.stats), get(self.logp), get(self.z if in_place else self.dz)


def check(got, want, what):
    for g, w, b, name in zip(got, want[:3], want[3:], ("stats", "logp", "dlogits")):
        inf = np.isinf(w)
        assert (g[inf] == w[inf]).all() and np.isfinite(g[~inf]).all(), (what, name)
        err = np.abs(g - np.where(inf, 0, w))[~inf]
        assert (err <= b[~inf]).all(), "%s %s: off by %.3g, %.2f of the bound" % (what, name, err.max(), (err / np.maximum(b[~inf], 1e-300)).max())


@pytest.mark.parametrize("c_kl,c_ent", [(0.0, 0.0), (0.05, 0.0), (0.05, 0.01)])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (5, 2), (70, 5), (300, 16), (129, 17), (33, 64), (40, 65), (9, 256), (17, 257), (20, 1000), (7, 1024), (6, 1031), (5, 4096), (3, 4099),
                                        (4, 8192), (3, 8195), (3, 16000), (2, 16411), (3, 32000), (2, 32771), (2, 50257), (2, 65536), (2, 70001), (1, 131072), (2, 151000), (1, 160003),
                                        (2, 163844), (1, 200001), (1, 256000), (1, 425987), (1, 430000), (3, 6144), (3, 6145), (3, 12285), (2, 24576), (2, 49153), (1, 98301), (1, 98304)])
def test_policy_loss(talos, ctx, rows, vocab, c_kl, c_ent):
    z, tokens, old, rf, adv, w = make(rows, vocab, rows * 7 + vocab)
    if rows > 4:
        tokens[1] = -100                                                  # padding by token, by weight
        w[3] = 0.0; z[3] = np.nan; adv[3] = np.nan
    for pad, pad_out, off in ((0, 0, 0), (4, 8, 0), (3, 0, 0), (0, 0, 1)):
        c = Call(z, tokens, old, rf, adv, w, pad, pad_out, off)
        want = ref.policy_loss(z, tokens, old, rf, adv, w, 0.2, 0.3, c_kl, c_ent, 7.0)
        got = c.run(talos, ctx, c_kl, c_ent, 7.0)
        check((got[0], got[1], got[2][:, :vocab]), want, (pad, pad_out, off))
        assert (got[2][:, vocab:] == -55.0).all()
        again = Call(z, tokens, old, rf, adv, w, pad, pad_out, off).run(talos, ctx, c_kl, c_ent, 7.0)
        assert all((a == b).all() for a, b in zip(got, again))            # the same bits
        over = c.run(talos, ctx, c_kl, c_ent, 7.0, in_place=True)
        check((over[0], over[1], over[2][:, :vocab]), want, (pad, off, "in place"))
        ctx.synchronize()


def test_without_weights_reference_or_gradient(talos, ctx):
    z, tokens, old, rf, adv, _ = make(50, 100, 5)
    want = ref.policy_loss(z, tokens, old, None, adv, None, 0.2, 0.3, 0.0, 0.0, 50.0)
    check(Call(z, tokens, old, None, adv, None).run(talos, ctx, 0.0, 0.0, 50.0), want, "no reference")
    c = Call(z, tokens, None, None, None, None)                           # what a rollout asks for: log-probabilities alone
    c.run(talos, ctx, 0.0, 0.0, 1.0, dz=False)
    assert (np.abs(get(c.logp) - want[1]) <= want[4]).all() and (get(c.dz) == -55.0).all()
    c = Call(z, tokens, old, rf, adv, None)
    first = c.run(talos, ctx, 0.1, 0.0, 1.0)[0]
    twice = c.run(talos, ctx, 0.1, 0.0, 1.0, acc=1)[0]
    assert (np.abs(twice - 2 * first) <= 2 * ref.U * np.abs(2 * first)).all()


def test_rows_that_leave_nothing(talos, ctx):
    for vocab in (6, 700, 5000, 20000, 170000, 430001):
        z, tokens, old, rf, adv, w = make(6, vocab, vocab)
        z[0] = -np.inf                                                    # no action at all
        z[2, :] = -np.inf; z[2, tokens[2]] = -3.0                         # one action: probability 1
        z[4, (tokens[4] + 1) % vocab] = -3.4028234663852886e38            # the type's lowest value as a mask
        z, old = f32(z), old.copy()
        old[2] = 0.0
        for c_ent in (0.0, 0.01):
            want = ref.policy_loss(z, tokens, old, None, adv, w, 0.2, 0.3, 0.0, c_ent, 3.0)
            got = Call(z, tokens, old, None, adv, w).run(talos, ctx, 0.0, c_ent, 3.0)
            assert got[1][0] == -np.inf and (got[2][0] == 0).all() and got[1][2] == 0.0
            rest = [1, 3, 5]                                              # (a magnitude of 1e38 makes row 4's counted bound empty)
            assert (np.abs(got[1] - want[1])[rest] <= want[4][rest]).all() and (np.abs(got[2] - want[2])[rest] <= want[5][rest]).all()
            assert np.isfinite(got[2]).all() and np.isfinite(got[0]).all()
            assert abs(got[1][4] - want[1][4]) < 1e-4 and np.abs(got[2][4] - want[2][4]).max() < 1e-5
            assert got[0][4] == pytest.approx(w.sum() - w[0], rel=1e-6)
    z, tokens, old, rf, adv, w = make(6, 300, 2)
    z[1, 7] = np.nan                                                      # a NaN stays in its row and in the sums
    got = Call(z, tokens, old, rf, adv, w).run(talos, ctx, 0.1, 0.0, 3.0)
    assert np.isnan(got[2][1]).all() and np.isfinite(np.delete(got[2], 1, 0)).all() and np.isnan(got[0][0])
    z[1] = np.nan
    got = Call(z, tokens, old, rf, adv, w).run(talos, ctx, 0.1, 0.0, 3.0)
    assert np.isnan(got[2][1]).all() and np.isnan(got[1][1])


def test_token_outside_the_vocabulary(talos, ctx):
    for vocab in (10, 9000, 170000, 430001):
        z, tokens, old, rf, adv, w = make(5, vocab, 4)
        bad = tokens.copy(); bad[2] = vocab
        got = Call(z, bad, old, rf, adv, w).run(talos, ctx, 0.05, 0.0, 5.0)
        with pytest.raises(talos.TalosError) as e: ctx.synchronize()
        assert e.value.status == talos.ERR_ARG
        tokens[2] = -1
        check(got, ref.policy_loss(z, tokens, old, rf, adv, w, 0.2, 0.3, 0.05, 0.0, 5.0), "as padding")
        ctx.synchronize()


def test_no_rows(talos, ctx):
    stats = blank(5, 0, 9.0)
    args = (None, None, None, None, None)
    talos.lib.talos_policy_loss_fwd_bwd(ctx.handle, None, 8, None, None, None, None, None, 0, 8, 0.2, 0.2, 0.0, 0.0, 1.0, None, None, 8, talos.ptr(stats), 1)
    assert (get(stats) == 9).all() and args
    talos.lib.talos_policy_loss_fwd_bwd(ctx.handle, None, 8, None, None, None, None, None, 0, 8, 0.2, 0.2, 0.0, 0.0, 1.0, None, None, 8, talos.ptr(stats), 0)
    assert (get(stats) == 0).all()


def test_agrees_with_the_small_loss(talos, ctx):
    # the framework's per-transition loss (at most 64 actions, no reference policy) on the same rows: value terms switched off
    import torch
    z, tokens, old, _, adv, _ = make(500, 16, 77, masked=0.0)
    shift = 0.15 * np.random.RandomState(4).randn(500)                    # symmetric clip 0.2 there
    lp = z[np.arange(500), tokens] - np.logaddexp.reduce(z, 1)
    for border in (np.log(0.8), np.log(1.2)): shift = np.where(np.abs(shift - border) < 1e-3, shift + 4e-3, shift)
    old = f32(lp - shift)
    c = Call(z, tokens, old, None, adv, None)
    p = talos.ptr
    talos.lib.talos_policy_loss_fwd_bwd(ctx.handle, p(c.z), 16, p(c.tokens), p(c.old), None, p(c.adv), None, 500, 16, 0.2, 0.2, 0.0, 0.01, 500.0, p(c.logp), p(c.dz), 16, p(c.stats), 0)
    v, dv, dz, stats = torch.zeros(500, device="cuda:0"), blank(500), blank((500, 16)), torch.zeros(3, device="cuda:0")
    talos.lib.talos_ppo_loss_fwd_bwd(ctx.handle, p(c.z), 16, p(v), 1, p(c.tokens), p(c.old), p(c.adv), p(v), 500, 16, 0.2, 0.0, 0.01, 500.0, p(dz), 16, p(dv), 1, p(stats))
    ctx.synchronize()
    want = ref.policy_loss(z, tokens, old, None, adv, None, 0.2, 0.2, 0.0, 0.01, 500.0)
    assert (np.abs(get(c.dz) - get(dz)) <= 2 * want[5]).all() and abs(get(c.stats)[0] - get(stats)[0]) <= 2 * want[3][0] + 1e-6 * 500
