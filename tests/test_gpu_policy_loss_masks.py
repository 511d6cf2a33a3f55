"""The policy loss of rows of which a mask leaves a few tokens, over all routes of its kernels: most of a row's warps, and CTAs, then hold nothing but masked
logits, and what they contribute must be nothing, wherever the row's own logits lie (a softmax does not see an offset)."""
import numpy as np
import pytest

import lm_reference as ref
from test_gpu_policy_loss import Call, check, ctx, f32  # noqa: F401

pytestmark = pytest.mark.gpu

# one CTA, shifted rows, clusters of two, four and eight, a cluster's shared memory in units of four and of one, a row that is read twice
VOCABS = [1031, 5000, 20000, 50257, 100000, 170000, 170001, 430001]


def masked_rows(vocab, mask, seed):
    """Rows of five legal tokens at different offsets; the legal ones first, last, or anywhere.  `mask` stands in the others; the second result has -inf there
    (both have probability 0 to the last bit: a distance of at least 1e30 from the legal logits)."""
    rng = np.random.RandomState(seed)
    offsets = (0.0, -95.0, -200.0, -1000.0, 200.0, -88.0)
    z, want = np.full((len(offsets), vocab), mask), np.full((len(offsets), vocab), -np.inf)
    tokens = np.zeros(len(offsets), dtype=np.int64)
    for r, offset in enumerate(offsets):
        legal = [np.arange(5), np.arange(vocab - 5, vocab), rng.choice(vocab, 5, replace=False)][r % 3]
        z[r, legal] = want[r, legal] = f32(offset + rng.randn(5))
        tokens[r] = legal[rng.randint(5)]
    lp = want[np.arange(len(offsets)), tokens] - np.logaddexp.reduce(want, 1)
    old, rf, adv, w = f32(lp - 0.1 * rng.rand(len(offsets))), f32(lp + 0.3 * rng.randn(len(offsets))), f32(rng.randn(len(offsets))), f32(0.5 + rng.rand(len(offsets)))
    return z, want, tokens, old, rf, adv, w


def check_masked(talos, ctx, vocab, mask, c_ent):  # noqa: F811
    z, plain, tokens, old, rf, adv, w = masked_rows(vocab, mask, vocab)
    want = ref.policy_loss(plain, tokens, old, rf, adv, w, 0.2, 0.3, 0.05, c_ent, 3.0)
    for pad, off in ((0, 0), (3, 1)):
        got = Call(z, tokens, old, rf, adv, w, pad, pad, off).run(talos, ctx, 0.05, c_ent, 3.0)
        dz = got[2][:, :vocab]
        check((got[0], got[1], dz), want, (vocab, mask, pad, off))
        assert (dz[plain == -np.inf] == 0).all()
    ctx.synchronize()


@pytest.mark.parametrize("c_ent", [0.0, 0.01])
@pytest.mark.parametrize("vocab", VOCABS)
def test_few_legal_tokens_others_minus_infinity(talos, ctx, vocab, c_ent):  # noqa: F811
    check_masked(talos, ctx, vocab, -np.inf, c_ent)


@pytest.mark.parametrize("c_ent", [0.0, 0.01])
@pytest.mark.parametrize("mask", [np.finfo(np.float32).min, -1e36, -1e30])
@pytest.mark.parametrize("vocab", VOCABS)
def test_few_legal_tokens_others_a_low_value(talos, ctx, vocab, mask, c_ent):  # noqa: F811
    check_masked(talos, ctx, vocab, float(np.float32(mask)), c_ent)


@pytest.mark.parametrize("vocab", VOCABS)
def test_a_nan_among_masked_tokens_stays(talos, ctx, vocab):  # noqa: F811
    """A NaN whose warp holds nothing else but -inf reaches its row's results, and no other row's."""
    z, plain, tokens, old, rf, adv, w = masked_rows(vocab, -np.inf, vocab)
    z[1, vocab // 2] = np.nan
    got = Call(z, tokens, old, rf, adv, w).run(talos, ctx, 0.05, 0.0, 3.0)
    assert np.isnan(got[1][1]) and np.isnan(got[2][1]).all() and np.isnan(got[0][0])
    assert np.isfinite(np.delete(got[1], 1)).all() and np.isfinite(np.delete(got[2], 1, 0)).all()
