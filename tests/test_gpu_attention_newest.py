"""Long attention whose queries are the newest of each sequence's own keys (TALOS_ATTN_CAUSAL_NEWEST): several new tokens of each sequence over caches that are filled
to different lengths.  Each sequence is compared with itself alone, cut to its own keys, in 64 bits."""
import numpy as np
import pytest

import lm_reference as ref
from test_gpu_attention_long import Problem, ctx, lens, near, route  # noqa: F401
from test_gpu_norm_dropout import get

pytestmark = pytest.mark.gpu

NEWEST = 3


def newest(*shape, key_len, **more):
    pr = Problem(*shape, causal=True, key_len=key_len, **more)
    pr.tail = (*pr.tail[:8], NEWEST, *pr.tail[9:])
    return pr


def check_alone(talos, ctx, pr):  # noqa: F811
    results = [a.copy() for a in pr.forward(talos, ctx)]
    results += [a.copy() for a in pr.backward(talos, ctx)]
    scale, sk = float(np.float32(pr.scale)), pr.k.shape[2]
    for b, n in enumerate(pr.key_len):
        n = min(max(n, 0), sk)
        w = ref.attention(pr.q[b:b + 1], pr.k[b:b + 1, :, :n], pr.v[b:b + 1, :, :n], None, scale, True, pr.do[b:b + 1], pr.tail[-1])
        for got, want, bound, what in zip(results, w[:5], w[5:], ("out", "lse", "dq", "dk", "dv")):
            if what in ("dk", "dv"):
                assert (got[b, :, n:] == 0).all(), (b, what)
                near(got[b:b + 1, :, :n], want, bound, (b, what))
            else: near(got[b:b + 1], want, bound, (b, what))
    again = [*pr.forward(talos, ctx), *pr.backward(talos, ctx)]
    assert all((a == b).all() for a, b in zip(results, again))
    ctx.synchronize()


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("sq", [1, 2, 5, 8])
@pytest.mark.parametrize("heads,kv_heads,sk,d,dv,key_len", [(4, 2, 300, 64, 64, [300, 17, 0, 150]), (4, 1, 1000, 32, 32, [999, 3]), (2, 2, 40, 96, 64, [40, 8, 9, 1]), (8, 2, 4097, 128, 128, [4097, 2000]),
                                                            (3, 1, 70, 9, 5, [12, 70])])
def test_a_few_new_tokens(talos, ctx, heads, kv_heads, sk, d, dv, key_len, sq, layout):  # noqa: F811
    check_alone(talos, ctx, newest(len(key_len), heads, kv_heads, sq, sk, d, dv, key_len=key_len, layout=layout, mode=1))


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("shape,key_len", [((3, 4, 2, 70, 300, 64, 64), [300, 71, 190]), ((4, 2, 1, 70, 130, 32, 32), [64, 0, 130, 5]), ((3, 2, 2, 20, 50, 64, 64), [50, 20, 31]),
                                           ((3, 4, 2, 70, 300, 128, 128), [300, 71, 190]), ((3, 2, 2, 130, 200, 96, 64), [200, 129, 1]), ((2, 7, 1, 99, 93, 1, 1), [93, 50]),
                                           ((2, 2, 1, 200, 777, 64, 64), [500, 777])])
def test_many_new_tokens(talos, ctx, shape, key_len, mode, route):  # noqa: F811
    for layout, off in ((0, 0), (1, 3)): check_alone(talos, ctx, newest(*shape, key_len=key_len, layout=layout, off=off, mode=mode))


@pytest.mark.parametrize("shape", [(24, 8, 4, 140, 270, 32, 32), (16, 8, 8, 200, 200, 96, 128)])
def test_more_tiles_than_the_gpu_has_places(talos, ctx, shape):  # noqa: F811
    rng = np.random.RandomState(4)
    check_alone(talos, ctx, newest(*shape, key_len=list(rng.randint(0, shape[4] + 1, shape[0])), mode=1))


@pytest.mark.parametrize("shape", [(2, 4, 2, 5, 300, 64, 64), (2, 4, 2, 70, 300, 64, 64), (2, 2, 2, 100, 130, 128, 128), (2, 2, 1, 30, 60, 40, 40)])
def test_full_caches_are_the_other_mask(talos, ctx, shape):  # noqa: F811
    """Without key counts, and where all are sk, the two masks are one: the same bits."""
    for counts in (None, [shape[4]] * 2):
        pr = Problem(*shape, causal=True, key_len=counts, mode=1)
        first = [a.copy() for a in (*pr.forward(talos, ctx), *pr.backward(talos, ctx))]
        pr.tail = (*pr.tail[:8], NEWEST, *pr.tail[9:])
        assert all((a == b).all() for a, b in zip(first, (*pr.forward(talos, ctx), *pr.backward(talos, ctx))))


def test_new_tokens_do_not_see_each_others_future(talos, ctx):  # noqa: F811
    """Six new tokens a sequence; the last row of each cache is changed: only the last token's answer may change."""
    pr = newest(3, 4, 2, 6, 200, 64, 64, key_len=[200, 31, 100], mode=1)
    before = pr.forward(talos, ctx)[0].copy()
    for b, n in enumerate(pr.key_len): pr.k[b, :, n - 1] += 1.0; pr.v[b, :, n - 1] -= 2.0
    pr.dev[1], pr.dev[2] = pr.send(pr.k), pr.send(pr.v)
    after = pr.forward(talos, ctx)[0]
    assert (before[:, :, :5] == after[:, :, :5]).all() and (before[:, :, 5] != after[:, :, 5]).any(-1).all()
    assert get(pr.out).shape == pr.do.shape and lens(None) is None
