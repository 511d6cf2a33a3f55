"""Layer norm and its junction of rows wider than 8 192 values, and of more rows than there are CTAs: the column sums that a CTA carries over its rows in shared memory."""
import numpy as np
import pytest

import lm_reference as ref
from lm_reference import U
from test_gpu_norm_dropout import blank, ctx, data, get, near, put, rounded  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("rows,dim", [(700, 9001), (700, 9004), (600, 16383), (500, 16384), (900, 8193)])
def test_backward(talos, ctx, rows, dim, off):  # noqa: F811
    rng, x, gamma, beta = data(rows, dim, rows + dim)
    dy, dh = rounded(rng, rows, dim), rounded(rng, rows, dim)
    _, mean, inv = ref.layernorm(x, gamma, beta, 1e-5)
    m, i, xd, gd, dyd, dhd = put(mean), put(inv), put(x, off), put(gamma), put(dy, off), put(dh, off)
    p, want, bound = talos.ptr, ref.layernorm_bwd(dy, x, gamma, mean, inv), ref.layernorm_bwd_bound(dy, x, gamma, mean, inv)
    out = blank(x.shape, off), blank(dim), blank(dim)
    talos.lib.talos_layernorm_bwd(ctx.handle, p(dyd), p(xd), p(gd), p(m), p(i), rows, dim, *(p(t) for t in out), 0)
    for got, w, b, what in zip(out, want, bound, ("dx", "dgamma", "dbeta")): near(got, w, b, what)
    # the junction's, from the same h = x: dresidual = dh + dx, dx dropped
    drop = blank(x.shape, off), blank(x.shape, off), blank(dim), blank(dim)
    talos.lib.talos_dropout_add_layernorm_bwd(ctx.handle, p(dyd), p(dhd), p(xd), p(gd), p(m), p(i), 0.3, 77, 9, None, rows, dim, *(p(t) for t in drop), 0)
    keep, scale = ref.keep(x.size, 0.3, 77, 9).reshape(x.shape), 1.0 / (1.0 - float(np.float32(0.3)))
    total, b_total = want[0] + dh, bound[0] + U * (np.abs(want[0]) + np.abs(dh))
    near(drop[1], total, b_total, "dresidual")
    near(drop[0], np.where(keep, total, 0.0) * scale, np.where(keep, b_total + 2 * U * np.abs(total), 0.0) * scale, "dropped dx")
    near(drop[2], want[1], bound[1], "junction's dgamma"); near(drop[3], want[2], bound[2], "junction's dbeta")
    assert (get(drop[2]) == get(out[1])).all()


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("rows,dim", [(700, 9001), (500, 16384)])
def test_forward(talos, ctx, rows, dim, off):  # noqa: F811
    _, x, gamma, beta = data(rows, dim, rows + dim)
    p, eps = talos.ptr, float(np.float32(1e-5))
    xd, gd, bd, y, mean, inv = put(x, off), put(gamma), put(beta), blank(x.shape, off), blank(rows), blank(rows)
    talos.lib.talos_layernorm_fwd(ctx.handle, p(xd), p(gd), p(bd), 1e-5, rows, dim, p(y), p(mean), p(inv))
    for got, w, b, what in zip((y, mean, inv), ref.layernorm(x, gamma, beta, eps), ref.layernorm_bound(x, gamma, beta, eps), ("y", "mean", "inv_std")): near(got, w, b, what)
