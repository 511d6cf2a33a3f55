"""How the operators of include/talos_b200_lm.h may be called: captured and replayed, from two graphs that share scratch, by two contexts at once, with offsets
beyond 32 bits, with more sequences than are split at a time.  Their arithmetic is tested elsewhere; where a call has been made before in another way the
same bits are asked for, since every sum has a fixed order."""
import numpy as np
import pytest

import lm_reference as ref
from test_gpu_attention_long import near
from test_gpu_norm_dropout import blank, get, put

pytestmark = pytest.mark.gpu

B, S, H, HK, D, V, ROWS = 2, 90, 4, 2, 64, 515, 180


class Step:
    """Layer norm, attention, junction and loss, each with its gradients, over buffers of its own; `results` are overwritten."""

    def __init__(self, talos, ctx, seed):
        self.lib, self.ctx, p = talos.lib, ctx, talos.ptr
        self.seed = seed
        rng = np.random.RandomState(seed)
        self.source = {"x": (ROWS, 256), "gamma": (256,), "beta": (256,), "dy": (ROWS, 256), "q": (B, S, H, D), "k": (B, S, HK, D), "v": (B, S, HK, D), "do": (B, S, H, D), "z": (ROWS, V),
                       "old": (ROWS,), "adv": (ROWS,), "q1": (B, 1, H, D), "kc": (B, 700, HK, D)}
        import torch
        self.t = {k: put(0.5 * rng.randn(*s)) for k, s in self.source.items()}
        self.tokens = torch.tensor(rng.randint(0, V, ROWS), dtype=torch.int32, device="cuda:0")
        self.lens = torch.tensor([S, 31], dtype=torch.int32, device="cuda:0")
        names = {"y": (ROWS, 256), "mean": (ROWS,), "inv": (ROWS,), "dx": (ROWS, 256), "dgamma": (256,), "dbeta": (256,), "h": (ROWS, 256), "hy": (ROWS, 256), "hmean": (ROWS,), "hinv": (ROWS,),
                 "hdx": (ROWS, 256), "hdr": (ROWS, 256), "hdg": (256,), "hdb": (256,), "out": (B, S, H, D), "lse": (B, H, S), "dq": (B, S, H, D), "dk": (B, S, HK, D), "dv": (B, S, HK, D),
                 "o1": (B, 1, H, D), "lse1": (B, H, 1), "logp": (ROWS,), "dz": (ROWS, V), "stats": (5,), "drop": (ROWS, 256)}
        self.results = {k: blank(s) for k, s in names.items()}
        self.p = {k: p(v) for k, v in {**self.t, **self.results, "tokens": self.tokens, "lens": self.lens}.items()}

    def refill(self, seed):
        rng = np.random.RandomState(seed)
        for k, s in self.source.items(): self.t[k].copy_(put(0.5 * rng.randn(*s)))

    def run(self):
        p, L, c, s = self.p, self.lib, self.ctx.handle, self.seed
        L.talos_layernorm_fwd(c, p["x"], p["gamma"], p["beta"], 1e-5, ROWS, 256, p["y"], p["mean"], p["inv"])
        L.talos_layernorm_bwd(c, p["dy"], p["x"], p["gamma"], p["mean"], p["inv"], ROWS, 256, p["dx"], p["dgamma"], p["dbeta"], 0)
        att = (B, H, HK, S, S, D, D, 0.125, 1, 1, 1)
        L.talos_attention_lse_fwd(c, p["q"], p["k"], p["v"], p["lens"], p["out"], p["lse"], *att)
        L.talos_attention_lse_bwd(c, p["q"], p["k"], p["v"], p["lens"], p["out"], p["lse"], p["do"], p["dq"], p["dk"], p["dv"], *att)
        L.talos_attention_lse_fwd(c, p["q1"], p["kc"], p["kc"], None, p["o1"], p["lse1"], B, H, HK, 1, 700, D, D, 0.125, 1, 1, 1)
        L.talos_dropout_fwd(c, p["x"], p["dy"], p["drop"], ROWS * 256, 0.1, s, 4, None)
        L.talos_dropout_add_layernorm_fwd(c, p["y"], p["x"], p["gamma"], p["beta"], 1e-5, 0.1, s, 1, None, ROWS, 256, p["h"], p["hy"], p["hmean"], p["hinv"])
        L.talos_dropout_add_layernorm_bwd(c, p["dy"], p["x"], p["h"], p["gamma"], p["hmean"], p["hinv"], 0.1, s, 1, None, ROWS, 256, p["hdx"], p["hdr"], p["hdg"], p["hdb"], 0)
        L.talos_policy_loss_fwd_bwd(c, p["z"], V, p["tokens"], p["old"], None, p["adv"], None, ROWS, V, 0.2, 0.2, 0.0, 0.01, 180.0, p["logp"], p["dz"], V, p["stats"], 0)

    def take(self):
        got = {k: get(v) for k, v in self.results.items()}
        assert all(np.isfinite(v).all() for v in got.values())
        for v in self.results.values(): v.fill_(float("nan"))
        return got


def same(a, b):
    for k in a: assert (a[k] == b[k]).all(), k


def test_two_graphs_of_one_context(talos):
    import torch
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        own = talos.torch_context(0)
        steps = [Step(talos, own, 5), Step(talos, own, 6)]
        for s in steps: s.run()
        eager = [s.take() for s in steps]
        stream.synchronize()
        graphs = []
        for s in steps:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream): s.run()
            graphs.append(g)
        for _ in range(2):                                    # in turn: both use the context's scratch
            for g in graphs: g.replay()
            for s, e in zip(steps, eager): same(s.take(), e)
        for i, s in enumerate(steps): s.refill(50 + i)
        for g in graphs: g.replay()
        fresh = [s.take() for s in steps]
        for s in steps: s.run()
        for s, f, e in zip(steps, fresh, eager):
            same(s.take(), f)
            assert (f["dz"] != e["dz"]).any()
        stream.synchronize()
    del g, graphs
    own.close()


def test_two_contexts_at_once(talos):
    import torch
    streams, steps, alone = [torch.cuda.Stream() for _ in range(2)], [], []
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            steps.append(Step(talos, talos.torch_context(0), 7 + i))
            steps[i].run()
            alone.append(steps[i].take())
            stream.synchronize()
    for _ in range(5):
        for s in steps: s.run()
    for stream, s, a in zip(streams, steps, alone):
        stream.synchronize()
        with torch.cuda.stream(stream): same(s.take(), a)
        s.ctx.close()


@pytest.fixture(scope="module")
def ctx(talos):
    c = talos.torch_context(0)
    yield c
    c.synchronize()


def test_more_sequences_than_are_split_at_a_time(talos, ctx):
    """2 000 sequences of 72 tokens: scratch for 1 820 of them forward, 1 365 backward; a slice must find its own key counts, rows and saved numbers."""
    import torch
    n, h, s, d = 2000, 4, 72, 8
    rng = np.random.RandomState(1)
    lens = rng.randint(1, s + 1, n)
    q, k, v, do = [rng.randn(n, h, s, d).astype(np.float32).astype(np.float64) for _ in range(4)]
    dev, out, lse, tl = [put(a) for a in (q, k, v, do)], blank((n, h, s, d)), blank((n, h, s)), torch.tensor(lens, dtype=torch.int32, device="cuda:0")
    grads, p, tail = [blank((n, h, s, d)) for _ in range(3)], talos.ptr, (n, h, h, s, s, d, d, 0.25, 1, 0, 1)
    talos.lib.talos_attention_lse_fwd(ctx.handle, *(p(t) for t in dev[:3]), p(tl), p(out), p(lse), *tail)
    talos.lib.talos_attention_lse_bwd(ctx.handle, *(p(t) for t in dev[:3]), p(tl), p(out), p(lse), p(dev[3]), *(p(t) for t in grads), *tail)
    got = [get(t) for t in (out, lse, *grads)]
    for part in (slice(0, 3), slice(1363, 1367), slice(1818, 1822), slice(1997, 2000)):
        w = ref.attention(q[part], k[part], v[part], list(lens[part]), 0.25, True, do[part], 1)
        for g, a, b, what in zip(got, w[:5], w[5:], ("out", "lse", "dq", "dk", "dv")): near(g[part], a, b, what)
    assert all(np.isfinite(g).all() for g in got)


@pytest.mark.parametrize("sq", [1, 70])
def test_a_cache_beyond_32_bits(talos, ctx, sq):
    """k and v share one tensor of 3 x 2 heads x 2^22 rows of 128: the last sequence starts at element 2^31.  Only the rows in front of the key counts are filled."""
    import torch
    rows, d, lens = 1 << 22, 128, [3, 70, 200]
    rng = np.random.RandomState(sq)
    cache = torch.empty((3, 2, rows, d), device="cuda:0")
    keys = np.zeros((3, 2, 256, d))
    for b, n in enumerate(lens):
        keys[b, :, :n] = rng.randn(2, n, d).astype(np.float32)
        cache[b, :, :256] = float("nan")
        cache[b, :, :n] = put(keys[b, :, :n])
    q = rng.randn(3, 4, sq, d).astype(np.float32).astype(np.float64)
    qd, out, lse, tl, p = put(q), blank(q.shape), blank((3, 4, sq)), torch.tensor(lens, dtype=torch.int32, device="cuda:0"), talos.ptr
    talos.lib.talos_attention_lse_fwd(ctx.handle, p(qd), p(cache), p(cache), p(tl), p(out), p(lse), 3, 4, 2, sq, rows, d, d, 0.0625, 0, 0, 1)
    got = [get(out), get(lse)]
    w = ref.attention(q, keys, keys, lens, 0.0625, False, None, 1)
    near(got[0], w[0], w[2], "out"); near(got[1], w[1], w[3], "lse")
    del cache
    torch.cuda.empty_cache()


def test_rows_beyond_32_bits(talos, ctx):
    import torch
    p, L, rng = talos.ptr, talos.lib, np.random.RandomState(3)
    rows, dim = (1 << 17) + 3, 16384                          # 2^31 elements lie before the last three rows
    x = torch.zeros((rows, dim), device="cuda:0")
    tail, dy = rng.randn(3, dim).astype(np.float32).astype(np.float64), rng.randn(3, dim).astype(np.float32).astype(np.float64)
    x[-3:] = put(tail)
    mean, inv = blank(rows), blank(rows)
    L.talos_layernorm_fwd(ctx.handle, p(x), None, None, 1e-5, rows, dim, p(x), p(mean), p(inv))
    want, bound = ref.layernorm(tail, None, None, float(np.float32(1e-5))), ref.layernorm_bound(tail, None, None, float(np.float32(1e-5)))
    assert (np.abs(get(x[-3:]) - want[0]) <= bound[0]).all() and (get(x[0]) == 0).all()
    # dropout of the same elements: their words are counted in 64 bits
    x[-3:] = 1.0
    L.talos_dropout_fwd(ctx.handle, p(x), None, p(x), rows * dim, 0.5, 99, 1 << 40, None)
    first = (rows - 3) * dim // 4
    kept = ref.philox(np.arange(first, first + 3 * dim // 4), 1 << 40, 99).reshape(3, dim) >= 1 << 31
    assert (get(x[-3:]) == 2.0 * kept).all()
    del x
    z = torch.empty((4, 1 << 30), device="cuda:0")            # rows of 100 logits, 2^30 apart
    values = rng.randn(4, 100).astype(np.float32).astype(np.float64)
    z[:, :100] = put(values)
    dz, tokens, zero, one = blank((4, 100)), torch.tensor([1, 99, 0, 42], dtype=torch.int32, device="cuda:0"), blank(4), blank(4, value=1.0)
    logp = values[np.arange(4), [1, 99, 0, 42]] - np.logaddexp.reduce(values, 1)
    zero.copy_(put(logp))
    L.talos_policy_loss_fwd_bwd(ctx.handle, p(z), 1 << 30, p(tokens), p(zero), None, p(one), None, 4, 100, 0.2, 0.2, 0.0, 0.0, 1.0, None, p(dz), 100, None, 0)
    soft = np.exp(values - np.logaddexp.reduce(values, 1)[:, None])
    soft[np.arange(4), [1, 99, 0, 42]] -= 1.0
    # (softmax of 100 logits of order 1: a hundred roundings at most)
    assert (np.abs(get(dz) - soft) <= 100 * ref.U).all()
    del z
    torch.cuda.empty_cache()
