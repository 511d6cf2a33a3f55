"""A query that is NaN answers NaN, in its own row and in no other, on every route of long attention: up to eight queries (the decode step: one part, a cluster
of parts, parts joined by a kernel of their own), the CUDA cores, the tensor cores."""
import numpy as np
import pytest

from test_gpu_attention_long import Problem, ctx, route  # noqa: F401
from test_gpu_norm_dropout import get

pytestmark = pytest.mark.gpu


def check_nan_query(talos, ctx, pr, rows, empty=()):  # noqa: F811
    """rows: (sequence, head, query) whose q is set to NaN."""
    first, first_lse = (a.copy() for a in pr.forward(talos, ctx))
    for b, h, i in rows: pr.q[b, h, i, 0] = np.nan
    pr.dev[0] = pr.send(pr.q)
    out, lse = pr.forward(talos, ctx)
    hit = np.zeros(lse.shape, dtype=bool)
    for at in rows: hit[at] = at[0] not in empty
    assert np.isnan(out[hit]).all() and np.isnan(lse[hit]).all()
    assert (out[~hit] == first[~hit]).all() and (lse[~hit] == first_lse[~hit]).all()
    ctx.synchronize()


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("sq", [1, 2, 4, 8])
@pytest.mark.parametrize("sk", [3, 40, 1000, 9000])
@pytest.mark.parametrize("heads,kv_heads,d,dv", [(4, 1, 64, 64), (2, 2, 32, 32), (2, 1, 128, 128), (3, 1, 9, 5), (2, 2, 96, 64)])
def test_decode(talos, ctx, heads, kv_heads, d, dv, sk, sq, layout):  # noqa: F811
    pr = Problem(2, heads, kv_heads, sq, sk, d, dv, layout=layout, mode=1)
    check_nan_query(talos, ctx, pr, [(0, 1, sq - 1), (1, heads - 1, 0)])


@pytest.mark.parametrize("sk", [40, 9000])
def test_decode_of_all_queries_and_of_an_empty_sequence(talos, ctx, sk):  # noqa: F811
    """(A sequence without keys answers 0 whatever its query is.)"""
    pr = Problem(3, 4, 2, 1, sk, 64, 64, key_len=[sk, 0, 7], mode=1)
    check_nan_query(talos, ctx, pr, [(b, h, 0) for b in range(3) for h in range(4)], empty=(1,))


@pytest.mark.parametrize("shape", [(2, 4, 2, 9, 40, 64, 64), (1, 2, 1, 100, 130, 64, 64), (1, 2, 2, 140, 300, 96, 128)])
def test_more_queries(talos, ctx, shape, route):  # noqa: F811
    pr = Problem(*shape, mode=1)
    check_nan_query(talos, ctx, pr, [(0, 1, shape[3] - 1), (0, 0, 3)])


def test_causal_queries_in_front_of_the_first_key(talos, ctx):  # noqa: F811
    """Of eight queries over three keys the first five see none."""
    pr = Problem(1, 2, 1, 8, 3, 64, 64, causal=True, mode=1)
    first = pr.forward(talos, ctx)[0].copy()
    pr.q[0, 0, 2] = np.nan; pr.q[0, 1, 7] = np.nan
    pr.dev[0] = pr.send(pr.q)
    out, lse = pr.forward(talos, ctx)
    assert (out[0, 0] == first[0, 0]).all() and (lse[0, 0, :5] == -np.inf).all()
    assert np.isnan(out[0, 1, 7]).all() and np.isnan(lse[0, 1, 7]) and (out[0, 1, :7] == first[0, 1, :7]).all()
    assert get(pr.lse).shape == lse.shape
