"""The policy loss of more rows than its kernels have places for: a CTA or a cluster takes several rows one after the other, copies the next one ahead, alternates
its sums' places and meets padding between them, in place, aligned and not; and the form without a gradient on every route."""
import numpy as np
import pytest

import lm_reference as ref
from test_gpu_norm_dropout import blank, put
from test_gpu_policy_loss import ctx, ints, make  # noqa: F401

pytestmark = pytest.mark.gpu

KINDS = 7
# (rows, vocabulary): at least two rows a CTA or cluster, up to eight
MANY = [(9000, 1000), (2000, 1031), (1500, 4100), (1500, 6144), (1500, 8191), (1000, 12000), (1000, 16411), (400, 24576), (400, 32771), (300, 50257), (300, 65536), (120, 98301), (120, 131072),
        (120, 131071), (120, 151000), (90, 160003), (90, 262144), (700, 430001)]


def repeated(rows, vocab, seed):
    """`rows` rows of KINDS different ones in no order, the first, the last and runs in between being padding, by token and by weight.  Returns which kind each is (-1: padding by
    token, -2: by weight) and the kinds."""
    rng = np.random.RandomState(seed)
    kind = rng.randint(0, KINDS, rows)
    pad = rng.rand(rows) < 0.15
    pad[[0, 1, rows - 1]] = True
    pad[rows // 2:rows // 2 + 3] = True
    kind[pad] = np.where(rng.rand(int(pad.sum())) < 0.5, -1, -2)
    return kind, make(KINDS, vocab, seed)


class Many:
    """The device buffers of one call; the rows are put together on the device.  Padded rows hold NaN."""
    def __init__(self, rows, vocab, seed, c_ent, pad, off):
        import torch
        kind, (z, tokens, old, rf, adv, w) = repeated(rows, vocab, seed)
        self.rows, self.vocab, self.c_ent, self.ld = rows, vocab, c_ent, vocab + pad
        self.of = torch.tensor(np.maximum(kind, 0), device="cuda:0")
        self.on = torch.tensor(kind >= 0, device="cuda:0")
        flat = torch.full((rows * self.ld + off,), float("nan"), device="cuda:0")[off:]
        self.z = flat.view(rows, self.ld)
        base = put(z)
        for r in range(0, rows, 64):
            part = self.z[r:r + 64, :vocab]
            part.copy_(torch.where(self.on[r:r + 64, None], base[self.of[r:r + 64]], float("nan")))
        one = lambda a, bad: torch.where(self.on, put(a)[self.of], bad)  # noqa: E731
        self.old, self.ref, self.adv = (one(a, float("nan")) for a in (old, rf, adv))
        weight = one(w, 1.0)
        weight[torch.tensor(kind == -2, device="cuda:0")] = 0.0
        self.w = weight
        token = np.where(kind >= 0, tokens[np.maximum(kind, 0)], np.where(kind == -1, -7, 0))
        self.tokens = ints(token)
        self.logp, self.stats = blank(rows), blank(5)
        each = [ref.policy_loss(z[k:k + 1], tokens[k:k + 1], old[k:k + 1], rf[k:k + 1], adv[k:k + 1], w[k:k + 1], 0.2, 0.3, 0.05, c_ent, 7.0) for k in range(KINDS)]
        count = np.bincount(kind[kind >= 0], minlength=KINDS)
        self.want_stats, self.e_stats = sum(n * e[0] for n, e in zip(count, each)), sum(n * e[3] for n, e in zip(count, each))
        dev = lambda i: torch.tensor(np.concatenate([e[i] for e in each]), device="cuda:0")  # noqa: E731
        self.want = {"logp": (dev(1), dev(4)), "dz": (dev(2), dev(5))}

    def run(self, talos, ctx, dz):  # noqa: F811
        p = talos.ptr
        talos.lib.talos_policy_loss_fwd_bwd(ctx.handle, p(self.z), self.ld, p(self.tokens), p(self.old), p(self.ref), p(self.adv), p(self.w), self.rows, self.vocab, 0.2, 0.3, 0.05, self.c_ent,
                                            7.0, p(self.logp), None if dz is None else p(dz), self.ld, p(self.stats), 0)

    def near(self, got, name, rows=slice(None)):
        import torch
        of, on, (want, bound) = self.of[rows], self.on[rows], self.want[name]
        if got.dim() == 2: on = on[:, None]
        w, b = torch.where(on, want[of], 0.0), torch.where(on, bound[of], 0.0)
        err = (got.double() - w).abs()
        assert bool((err <= b).all()), "%s: off by %.3g, %.2f of the bound" % (name, float(err.max()), float((err / b.clamp(min=1e-300)).max()))

    def check(self, dz):
        self.near(self.logp, "logp")
        got = self.stats.double().cpu().numpy()
        assert (np.abs(got - self.want_stats) <= self.e_stats).all(), (got, self.want_stats, self.e_stats)
        if dz is not None:
            for r in range(0, self.rows, 64): self.near(dz[r:r + 64, :self.vocab], "dz", slice(r, r + 64))


@pytest.mark.parametrize("c_ent", [0.0, 0.01])
@pytest.mark.parametrize("pad,off", [(0, 0), (3, 1)])
@pytest.mark.parametrize("rows,vocab", MANY)
def test_many_rows(talos, ctx, rows, vocab, pad, off, c_ent):  # noqa: F811
    import torch
    c = Many(rows, vocab, rows + vocab, c_ent, pad, off)
    dz = torch.full((rows * c.ld + off,), -55.0, device="cuda:0")[off:].view(rows, c.ld)
    c.run(talos, ctx, dz)
    ctx.synchronize()
    c.check(dz)
    if pad: assert bool((dz[:, vocab:] == -55.0).all())
    first, logp, stats = dz, c.logp.clone(), c.stats.clone()
    c.logp.fill_(float("nan")); c.stats.fill_(float("nan"))
    c.run(talos, ctx, None)                                               # without a gradient: the same numbers
    ctx.synchronize()
    assert torch.equal(c.logp, logp) and torch.equal(c.stats, stats)
    c.run(talos, ctx, c.z)                                                # over the logits: the same bits
    ctx.synchronize()
    assert torch.equal(c.z[:, :vocab], first[:, :vocab]) and torch.equal(c.logp, logp) and torch.equal(c.stats, stats)
    del c, dz, first
    torch.cuda.empty_cache()


@pytest.mark.parametrize("pad,off", [(0, 0), (3, 1)])
@pytest.mark.parametrize("rows,vocab", [(40, 16), (40, 1000), (700, 5000), (700, 16411), (300, 32000), (150, 50257), (60, 98301), (60, 170000), (30, 170001), (20, 430001)])
def test_log_probabilities_alone(talos, ctx, rows, vocab, pad, off):  # noqa: F811
    """What a rollout stores and a reference policy answers: neither old_logp nor adv, no sums, no gradient."""
    import torch
    c = Many(rows, vocab, 3 * rows + vocab, 0.0, pad, off)
    before = c.z.clone()
    p = talos.ptr
    talos.lib.talos_policy_loss_fwd_bwd(ctx.handle, p(c.z), c.ld, p(c.tokens), None, None, None, p(c.w), rows, vocab, 0.2, 0.2, 0.0, 0.0, 1.0, p(c.logp), None, c.ld, None, 0)
    ctx.synchronize()
    c.near(c.logp, "logp")
    assert torch.equal(torch.nan_to_num(c.z), torch.nan_to_num(before))
    del c, before
    torch.cuda.empty_cache()
