"""Attention over long sequences on the GPU against its 64-bit form, with bounds counted from roundings."""
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


def lens(key_len):
    import torch
    return None if key_len is None else torch.tensor(key_len, dtype=torch.int32, device="cuda:0")


class Problem:
    def __init__(self, B, H, Hk, Sq, Sk, d, dv, causal=False, key_len=None, layout=0, mode=0, off=0, seed=0):
        rng = np.random.RandomState(seed + B + H + Sq + 3 * Sk + d)
        self.q, self.k, self.v, self.do = f32(2 * rng.randn(B, H, Sq, d)), f32(rng.randn(B, Hk, Sk, d)), f32(rng.randn(B, Hk, Sk, dv)), f32(rng.randn(B, H, Sq, dv))
        if key_len is not None:                                           # what lies behind a sequence's keys is not read
            for b, n in enumerate(key_len): self.k[b, :, max(n, 0):] = np.nan; self.v[b, :, max(n, 0):] = np.inf
        self.layout, self.scale, self.causal, self.key_len = layout, 1.0 / np.sqrt(d), causal, key_len
        self.tail = (B, H, Hk, Sq, Sk, d, dv, self.scale, int(causal), layout, mode)
        self.dev = [self.send(a, off) for a in (self.q, self.k, self.v, self.do)]
        self.lens = lens(key_len)
        self.out, self.lse = self.send(np.full(self.do.shape, np.nan), off), blank((B, H, Sq))
        self.grads = [self.send(np.full(a.shape, np.nan), off) for a in (self.q, self.k, self.v)]

    def send(self, a, off=0):
        return put(a.swapaxes(1, 2) if self.layout else a, off)

    def fetch(self, t):
        return get(t).swapaxes(1, 2) if self.layout else get(t)

    def forward(self, talos, ctx, lse=True):
        p = talos.ptr
        talos.lib.talos_attention_lse_fwd(ctx.handle, *(p(t) for t in self.dev[:3]), p(self.lens), p(self.out), p(self.lse) if lse else None, *self.tail)
        return self.fetch(self.out), get(self.lse)

    def backward(self, talos, ctx):
        p = talos.ptr
        talos.lib.talos_attention_lse_bwd(ctx.handle, *(p(t) for t in self.dev[:3]), p(self.lens), p(self.out), p(self.lse), p(self.dev[3]), *(p(t) for t in self.grads), *self.tail)
        return [self.fetch(t) for t in self.grads]

    def want(self, grads):
        k, v = np.where(np.isfinite(self.k), self.k, 0.0), np.where(np.isfinite(self.v), self.v, 0.0)
        scale = float(np.float32(self.scale))
        return ref.attention(self.q, k, v, self.key_len, scale, self.causal, self.do if grads else None, self.tail[-1])


def near(got, want, bound, what):
    same = np.isinf(want)
    assert (got[same] == want[same]).all() and np.isfinite(got[~same]).all(), what
    err = np.abs(got - np.where(same, 0.0, want))[~same]
    b = bound[~same]
    assert (err <= b).all(), "%s: off by %.3g, %.2f of the bound" % (what, err.max(), (err / np.maximum(b, 1e-300)).max())


def check(talos, ctx, pr, grads=True):
    w = pr.want(grads)
    out, lse = pr.forward(talos, ctx)
    n = len(w) // 2
    near(out, w[0], w[n], "out"); near(lse, w[1], w[n + 1], "lse")
    first = out.copy()
    assert (pr.forward(talos, ctx, lse=False)[0] == first).all()          # without lse; the same bits
    if not grads: return
    got = pr.backward(talos, ctx)
    for g, a, b, what in zip(got, w[2:5], w[n + 2:], ("dq", "dk", "dv")): near(g, a, b, what)
    assert all((a == b).all() for a, b in zip(got, pr.backward(talos, ctx)))


@pytest.fixture(params=["tensor", "cuda"])
def route(request, monkeypatch):
    """Products of more than 64 queries or keys run on the tensor cores; "cuda" takes them away, so that the other kernels see all sizes, too."""
    if request.param == "cuda": monkeypatch.setenv("TALOS_DISABLE_TENSOR_CORES", "1")
    return request.param


def kernels(ctx, call):
    call()
    ctx.timeline_begin()
    call()
    return {name for name, _ in ctx.timeline_end()}


def test_the_routes_are_taken(talos, ctx, route):
    for shape, tensor in (((1, 2, 1, 100, 130, 64, 64), True), ((1, 2, 1, 64, 64, 64, 64), False), ((1, 1, 1, 20, 90, 96, 128), True), ((2, 2, 2, 70, 70, 128, 40), True)):
        pr = Problem(*shape, mode=1)
        ran = kernels(ctx, lambda: (pr.forward(talos, ctx), pr.backward(talos, ctx)))
        assert ("attention_tc_fwd" in ran and "attention_tc_bwd_q" in ran) == (tensor and route == "tensor"), (shape, ran)
        assert ("attention_lse_fwd" in ran and "attention_lse_bwd_q" in ran) != (tensor and route == "tensor"), (shape, ran)


SHAPES = [(1, 1, 1, 1, 1, 4, 4), (2, 2, 1, 9, 9, 8, 8), (1, 3, 3, 17, 17, 32, 32), (2, 4, 2, 64, 64, 64, 64), (1, 2, 2, 65, 65, 64, 64), (1, 2, 1, 100, 130, 40, 24), (1, 1, 1, 129, 63, 64, 32),
          (2, 2, 2, 200, 200, 96, 64), (1, 2, 1, 77, 201, 128, 128), (1, 4, 1, 300, 300, 64, 64), (1, 1, 1, 33, 70, 5, 3), (1, 1, 1, 257, 513, 64, 64), (1, 2, 2, 90, 90, 7, 65),
          (1, 4, 2, 300, 300, 128, 128), (1, 2, 1, 129, 260, 65, 64), (2, 2, 2, 150, 150, 80, 128), (1, 2, 2, 200, 333, 128, 31), (2, 7, 1, 99, 93, 1, 1)]


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(talos, ctx, shape, causal, mode, route):
    check(talos, ctx, Problem(*shape, causal=causal, mode=mode))


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("layout,off", [(1, 0), (0, 1), (1, 3)])
@pytest.mark.parametrize("shape,key_len", [((3, 4, 2, 100, 100, 64, 64), [100, 1, 37]), ((3, 2, 2, 70, 150, 32, 32), [0, 64, 151]), ((2, 2, 1, 200, 200, 64, 64), [129, -5]),
                                           ((2, 2, 1, 50, 50, 96, 64), [50, 20]), ((3, 4, 2, 130, 130, 96, 64), [130, 0, 66]), ((2, 2, 1, 100, 200, 128, 128), [200, 65])])
def test_padded_batches_and_layouts(talos, ctx, shape, key_len, layout, off, causal, mode, route):
    check(talos, ctx, Problem(*shape, causal=causal, key_len=key_len, layout=layout, off=off, mode=mode))


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("shape,key_len", [((2, 4, 1, 1, 300, 64, 64), [300, 17]), ((1, 16, 2, 1, 1000, 64, 64), None), ((3, 2, 2, 1, 40, 96, 64), [0, 40, 1]), ((2, 8, 2, 5, 513, 32, 32), [513, 200]),
                                           ((1, 8, 1, 8, 257, 128, 128), None), ((2, 1, 1, 3, 4097, 40, 24), [4097, 2000]), ((1, 3, 1, 2, 7, 9, 5), None), ((64, 4, 4, 1, 17, 64, 64), None)])
@pytest.mark.parametrize("causal", [False, True])
def test_decode(talos, ctx, shape, key_len, causal, layout):
    check(talos, ctx, Problem(*shape, causal=causal, key_len=key_len, layout=layout, mode=1))


@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(16, 8, 8, 200, 200, 64, 64), (24, 8, 4, 140, 270, 32, 32), (16, 8, 8, 200, 200, 96, 128)])
def test_more_tiles_than_the_gpu_has_places(talos, ctx, shape, causal, mode):
    """(Of fewer tiles, as everywhere above, several CTAs share each in backward.)"""
    check(talos, ctx, Problem(*shape, causal=causal, mode=mode))


def test_causal_with_fewer_keys_than_queries(talos, ctx):
    check(talos, ctx, Problem(1, 2, 2, 150, 60, 64, 64, causal=True, mode=1))      # the first 90 queries see nothing


def test_far_scores(talos, ctx):
    for mode in (0, 1):
        pr = Problem(1, 1, 1, 80, 80, 64, 64, mode=mode)
        pr.q *= 64.0; pr.dev[0] = pr.send(pr.q)                               # scores of several hundred: the running maximum carries them
        check(talos, ctx, pr)


def test_nothing_to_do(talos, ctx):
    p, L = talos.ptr, talos.lib
    L.talos_attention_lse_fwd(ctx.handle, None, None, None, None, None, None, 0, 2, 1, 8, 8, 16, 16, 1.0, 0, 0, 0)
    out, lse, q = blank((1, 2, 20, 16)), blank((1, 2, 20)), put(np.ones((1, 2, 20, 16)))
    L.talos_attention_lse_fwd(ctx.handle, p(q), None, None, None, p(out), p(lse), 1, 2, 1, 20, 0, 16, 16, 1.0, 0, 0, 0)
    assert (get(out) == 0).all() and (get(lse) == -np.inf).all()
    dq, dk, dv = blank((1, 2, 20, 16)), blank((1, 1, 6, 16)), blank((1, 1, 6, 16))
    L.talos_attention_lse_bwd(ctx.handle, p(q), None, None, None, p(out), p(lse), p(q), p(dq), None, None, 1, 2, 1, 20, 0, 16, 16, 1.0, 0, 0, 0)
    assert (get(dq) == 0).all()
    k = put(np.ones((1, 1, 6, 16)))
    L.talos_attention_lse_bwd(ctx.handle, None, p(k), p(k), None, None, None, None, None, p(dk), p(dv), 1, 2, 1, 0, 6, 16, 16, 1.0, 0, 0, 0)
    assert (get(dk) == 0).all() and (get(dv) == 0).all()


@pytest.mark.parametrize("mode", [0, 1])
def test_agrees_with_attention_from_saved_probabilities(talos, ctx, mode):
    import torch
    pr = Problem(2, 4, 4, 64, 64, 32, 32, causal=True, mode=mode)
    pr.forward(talos, ctx); pr.backward(talos, ctx)
    p, L = talos.ptr, talos.lib
    out, probs, grads = blank((8, 64, 32)), blank((8, 64, 64)), [blank((8, 64, 32)) for _ in range(3)]
    L.talos_attention_fwd(ctx.handle, p(pr.dev[0]), p(pr.dev[1]), p(pr.dev[2]), p(out), p(probs), 8, 64, 32, 32, pr.scale, 1, mode)
    L.talos_attention_bwd(ctx.handle, p(pr.dev[0]), p(pr.dev[1]), p(pr.dev[2]), p(probs), p(pr.dev[3]), *(p(t) for t in grads), 8, 64, 32, 32, pr.scale, mode)
    ctx.synchronize()
    for a, b in zip([pr.out, *pr.grads], [out, *grads]):
        assert float((a.view(8, 64, 32) - b).norm() / b.norm()) <= 1e-5       # the framework's fp32 tolerance of each
