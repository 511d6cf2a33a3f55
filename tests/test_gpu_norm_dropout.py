"""Layer norm, dropout and their junction on the GPU against their 64-bit forms, with bounds counted from roundings."""
import numpy as np
import pytest

import lm_reference as ref
from lm_reference import U

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (3, 2), (5, 4), (33, 7), (1, 64), (70, 32), (64, 60), (257, 64), (9, 65), (31, 128), (40, 131), (1000, 256), (17, 300), (6, 512), (25, 516), (12, 771), (3, 1000),
          (300, 1024), (4, 1028), (5, 1500), (2, 2048), (700, 4096), (3, 4100), (3, 4099), (2, 8192), (2, 8196), (3, 9001), (2, 16383), (5, 16384)]


@pytest.fixture(scope="module")
def ctx(talos):
    c = talos.torch_context(0)
    yield c
    c.synchronize()


def put(a, off=0):
    """A device copy; `off` floats past an aligned address."""
    import torch
    t = torch.empty(a.size + off, device="cuda:0")[off:].view(a.shape)
    t.copy_(torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)))
    return t


def blank(shape, off=0, value=float("nan")):
    return put(np.full(shape, value), off)


def get(t):
    return t.double().cpu().numpy()


def rounded(rng, *shape):
    return rng.randn(*shape).astype(np.float32).astype(np.float64)


def data(rows, dim, seed, affine=True):
    rng = np.random.RandomState(seed)
    x = (rounded(rng, rows, dim) * np.float32(3) + np.float32(1.5)).astype(np.float32).astype(np.float64)
    gamma, beta = (rounded(rng, dim) + 1, rounded(rng, dim)) if affine else (None, None)
    if affine: gamma, beta = gamma.astype(np.float32).astype(np.float64), beta
    return rng, x, gamma, beta


def near(got, want, bound, what):
    err = np.abs(get(got) - want)
    assert np.isfinite(get(got)).all(), what
    assert (err <= bound).all(), "%s: off by %.3g, %.2f of the bound" % (what, err.max(), (err / np.maximum(bound, 1e-300)).max())


@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_layernorm_fwd(talos, ctx, rows, dim, off, affine):
    rng, x, gamma, beta = data(rows, dim, rows + dim, affine)
    xd, gd, bd = put(x, off), put(gamma) if affine else None, put(beta) if affine else None
    y, mean, inv = blank(x.shape, off), blank(rows), blank(rows)
    talos.lib.talos_layernorm_fwd(ctx.handle, talos.ptr(xd), talos.ptr(gd), talos.ptr(bd), 1e-5, rows, dim, talos.ptr(y), talos.ptr(mean), talos.ptr(inv))
    eps = float(np.float32(1e-5))
    want = ref.layernorm(x, gamma, beta, eps)
    for got, w, b, what in zip((y, mean, inv), want, ref.layernorm_bound(x, gamma, beta, eps), ("y", "mean", "inv_std")): near(got, w, b, what)
    talos.lib.talos_layernorm_fwd(ctx.handle, talos.ptr(xd), talos.ptr(gd), talos.ptr(bd), 1e-5, rows, dim, talos.ptr(xd), None, None)      # over its input
    assert (get(xd) == get(y)).all()


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_layernorm_bwd(talos, ctx, rows, dim, off):
    rng, x, gamma, _ = data(rows, dim, rows + 2 * dim)
    dy = rounded(rng, rows, dim)
    _, mean, inv = ref.layernorm(x, gamma, None, 1e-5)
    m, i = put(mean), put(inv)
    want = ref.layernorm_bwd(dy, x, gamma, mean, inv)
    bound = ref.layernorm_bwd_bound(dy, x, gamma, mean, inv)
    xd, gd, dyd = put(x, off), put(gamma), put(dy, off)

    def call(acc, start=float("nan")):
        out = blank(x.shape, off, start), blank(dim, 0, start), blank(dim, 0, start)
        talos.lib.talos_layernorm_bwd(ctx.handle, talos.ptr(dyd), talos.ptr(xd), talos.ptr(gd), talos.ptr(m), talos.ptr(i), rows, dim, *(talos.ptr(t) for t in out), acc)
        return out
    first = call(0)
    for got, w, b, what in zip(first, want, bound, ("dx", "dgamma", "dbeta")): near(got, w, b, what)
    for got, again in zip(first, call(0)): assert (get(got) == get(again)).all()       # the same bits
    for got, w, b, what in zip(call(7, 2.0), want, bound, ("dx", "dgamma", "dbeta")): near(got, w + 2.0, b + U * (np.abs(w) + 2), what + " accumulated")
    only = blank(dim)                                                                  # one result alone, the others not asked for
    talos.lib.talos_layernorm_bwd(ctx.handle, talos.ptr(dyd), talos.ptr(xd), talos.ptr(gd), talos.ptr(m), talos.ptr(i), rows, dim, None, None, talos.ptr(only), 0)
    assert (get(only) == get(first[2])).all()
    talos.lib.talos_layernorm_bwd(ctx.handle, talos.ptr(dyd), talos.ptr(xd), talos.ptr(gd), talos.ptr(m), talos.ptr(i), rows, dim, talos.ptr(dyd), None, None, 0)
    assert (get(dyd) == get(first[0])).all()                                           # dx over dy


def test_layernorm_no_rows_and_constant_rows(talos, ctx):
    a, b = blank(8), blank(8, 0, 3.0)
    talos.lib.talos_layernorm_bwd(ctx.handle, None, None, None, None, None, 0, 8, None, talos.ptr(a), talos.ptr(b), 4)
    assert (get(a) == 0).all() and (get(b) == 3).all()                                 # sums over nothing: overwritten, and added to
    talos.lib.talos_layernorm_fwd(ctx.handle, None, None, None, 1e-5, 0, 8, None, None, None)
    x, y = put(np.full((3, 96), 7.25)), blank((3, 96))
    talos.lib.talos_layernorm_fwd(ctx.handle, talos.ptr(x), None, None, 1e-5, 3, 96, talos.ptr(y), None, None)
    assert (get(y) == 0).all()                                                         # 96 x 7.25 is exact in fp32, whatever the order


def test_layernorm_far_mean(talos, ctx):
    # values of 4 096 +- 1: the variance comes from centred values, not from a difference of squares
    rng = np.random.RandomState(3)
    x = (4096.0 + rng.randn(50, 384)).astype(np.float32).astype(np.float64)
    y, mean, inv = blank(x.shape), blank(50), blank(50)
    xd = put(x)
    talos.lib.talos_layernorm_fwd(ctx.handle, talos.ptr(xd), None, None, 1e-5, 50, 384, talos.ptr(y), talos.ptr(mean), talos.ptr(inv))
    eps = float(np.float32(1e-5))
    for got, w, b, what in zip((y, mean, inv), ref.layernorm(x, None, None, eps), ref.layernorm_bound(x, None, None, eps), ("y", "mean", "inv_std")): near(got, w, b, what)


DROPS = [(0.0, 5, 0), (0.1, 2 ** 63 + 11, 3), (0.5, 2 ** 64 - 1, 2 ** 64 - 1), (0.9, 0, 2 ** 33)]


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("p,seed,offset", DROPS)
@pytest.mark.parametrize("n", [1, 3, 4, 5, 1023, 65536, 300001])
def test_dropout(talos, ctx, n, p, seed, offset, off):
    rng = np.random.RandomState(n)
    x, res, dy = (rounded(rng, n) for _ in range(3))
    x[::7] = np.inf
    keep = ref.keep(n, p, seed, offset)
    scale = float(np.float32(1.0 / (1.0 - float(np.float32(p)))))
    kept = np.where(keep, x, 0.0) * scale
    xd, rd, dyd, y, dx = put(x, off), put(res, off), put(dy, off), blank(n, off), blank(n, off)
    talos.lib.talos_dropout_fwd(ctx.handle, talos.ptr(xd), None, talos.ptr(y), n, p, seed, offset, None)
    assert (get(y) == kept.astype(np.float32)).all()                                   # one product: exact to the bit; dropped infinities are 0
    talos.lib.talos_dropout_fwd(ctx.handle, talos.ptr(xd), talos.ptr(rd), talos.ptr(y), n, p, seed, offset, None)
    fine = np.isfinite(kept)
    assert (np.abs(get(y) - (res + kept))[fine] <= 2 * U * (np.abs(kept) + np.abs(res))[fine]).all() and (get(y)[~fine] == np.inf).all()
    talos.lib.talos_dropout_bwd(ctx.handle, talos.ptr(dyd), talos.ptr(dx), n, p, seed, offset, None, 0)
    want = (np.where(keep, dy, 0.0) * scale)
    assert (get(dx) == want.astype(np.float32)).all()
    talos.lib.talos_dropout_bwd(ctx.handle, talos.ptr(dyd), talos.ptr(dx), n, p, seed, offset, None, 1)
    assert (np.abs(get(dx) - 2 * want) <= 4 * U * np.abs(want)).all()
    talos.lib.talos_dropout_bwd(ctx.handle, talos.ptr(dyd), talos.ptr(dyd), n, p, seed, offset, None, 0)
    assert (get(dyd) == want.astype(np.float32)).all()


def test_dropout_far_elements_and_device_offset(talos, ctx):
    import torch
    n = 3 * 2 ** 20 + 2
    x = put(np.ones(n)); y = blank(n)
    count = torch.tensor([2 ** 40 + 5], dtype=torch.int64, device="cuda:0")
    talos.lib.talos_dropout_fwd(ctx.handle, talos.ptr(x), None, talos.ptr(y), n, 0.25, 77, 2, talos.ptr(count))
    assert ((get(y) != 0) == ref.keep(n, 0.25, 77, 2 ** 40 + 7)).all()


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("p,seed,offset", DROPS[:3])
@pytest.mark.parametrize("rows,dim", [s for s in SHAPES if s[0] * s[1] < 300000])
def test_dropout_add_layernorm(talos, ctx, rows, dim, p, seed, offset, off):
    rng, x, gamma, beta = data(rows, dim, 3 * rows + dim)
    res, dy, dh = (rounded(rng, rows, dim) for _ in range(3))
    xd, rd, gd, bd = put(x, off), put(res, off), put(gamma), put(beta)
    h, y, mean, inv = blank(x.shape, off), blank(x.shape, off), blank(rows), blank(rows)
    talos.lib.talos_dropout_add_layernorm_fwd(ctx.handle, talos.ptr(xd), talos.ptr(rd), talos.ptr(gd), talos.ptr(bd), 1e-5, p, seed, offset, None, rows, dim, talos.ptr(h),
                                              talos.ptr(y), talos.ptr(mean), talos.ptr(inv))
    drop = ref.dropout(x, p, seed, offset)
    near(h, res + drop, 3 * U * (np.abs(drop) + np.abs(res)), "h")
    hh, eps = get(h), float(np.float32(1e-5))
    for got, w, b, what in zip((y, mean, inv), ref.layernorm(hh, gamma, beta, eps), ref.layernorm_bound(hh, gamma, beta, eps), ("y", "mean", "inv_std")): near(got, w, b, what)
    # backward, from statistics rounded once
    _, mu, iv = ref.layernorm(hh, gamma, beta, eps)
    m, i = put(mu), put(iv)
    dn, dgamma, dbeta = ref.layernorm_bwd(dy, hh, gamma, mu, iv)
    b_dn, b_g, b_b = ref.layernorm_bwd_bound(dy, hh, gamma, mu, iv)
    b_dn = b_dn + U * (np.abs(dn) + np.abs(dh))
    keep = ref.keep(x.size, p, seed, offset).reshape(x.shape)
    scale = 1.0 / (1.0 - float(np.float32(p)))
    dyd, dhd = put(dy, off), put(dh, off)

    def call(acc, with_dh, start=float("nan"), dx=True, dres=True):
        out = blank(x.shape, off, start) if dx else None, blank(x.shape, off, start) if dres else None, blank(dim, 0, start), blank(dim, 0, start)
        talos.lib.talos_dropout_add_layernorm_bwd(ctx.handle, talos.ptr(dyd), talos.ptr(dhd) if with_dh else None, talos.ptr(h), talos.ptr(gd), talos.ptr(m), talos.ptr(i), p, seed,
                                                  offset, None, rows, dim, *(talos.ptr(t) for t in out), acc)
        return out
    for with_dh in (True, False):
        total = dn + dh if with_dh else dn
        first = call(0, with_dh)
        near(first[1], total, b_dn, "dresidual")
        near(first[0], np.where(keep, total, 0.0) * scale, np.where(keep, b_dn + 2 * U * np.abs(total), 0.0) * scale, "dx")
        near(first[2], dgamma, b_g, "dgamma"); near(first[3], dbeta, b_b, "dbeta")
        assert (get(call(0, with_dh, dres=False)[0]) == get(first[0])).all() and (get(call(0, with_dh, dx=False)[1]) == get(first[1])).all()
    acc = call(15, False, 2.0)
    near(acc[1], dn + 2, b_dn + U * (np.abs(dn) + 2), "dresidual accumulated")
    near(acc[0], np.where(keep, dn, 0.0) * scale + 2, np.where(keep, b_dn + 2 * U * np.abs(dn), 0.0) * scale + U * (np.abs(dn) * scale + 2), "dx accumulated")
    near(acc[2], dgamma + 2, b_g + U * (np.abs(dgamma) + 2), "dgamma accumulated"); near(acc[3], dbeta + 2, b_b + U * (np.abs(dbeta) + 2), "dbeta accumulated")
    # the results over their inputs: h over x, dresidual over dh, dx over dy
    talos.lib.talos_dropout_add_layernorm_fwd(ctx.handle, talos.ptr(xd), talos.ptr(rd), talos.ptr(gd), talos.ptr(bd), 1e-5, p, seed, offset, None, rows, dim, talos.ptr(xd),
                                              talos.ptr(y), None, None)
    assert (get(xd) == hh).all()
    whole = call(0, True)
    talos.lib.talos_dropout_add_layernorm_bwd(ctx.handle, talos.ptr(dyd), talos.ptr(dhd), talos.ptr(h), talos.ptr(gd), talos.ptr(m), talos.ptr(i), p, seed, offset, None, rows, dim,
                                              talos.ptr(dyd), talos.ptr(dhd), None, None, 0)
    assert (get(dyd) == get(whole[0])).all() and (get(dhd) == get(whole[1])).all()


def test_junction_without_residual(talos, ctx):
    rng, x, gamma, beta = data(11, 52, 8)
    xd, h, y = put(x), blank(x.shape), blank(x.shape)
    talos.lib.talos_dropout_add_layernorm_fwd(ctx.handle, talos.ptr(xd), None, None, None, 1e-5, 0.4, 9, 1, None, 11, 52, talos.ptr(h), talos.ptr(y), None, None)
    near(h, ref.dropout(x, 0.4, 9, 1), 2 * U * np.abs(x) / 0.6, "h")


def test_captured_dropout_draws_anew(talos):
    import torch
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        own = talos.torch_context(0)
        n, x, y, step = 4099, put(np.ones(4099)), blank(4099), torch.zeros(1, dtype=torch.int64, device="cuda:0")
        talos.lib.talos_dropout_fwd(own.handle, talos.ptr(x), None, talos.ptr(y), n, 0.5, 21, 0, talos.ptr(step))
        own.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            talos.lib.talos_dropout_fwd(own.handle, talos.ptr(x), None, talos.ptr(y), n, 0.5, 21, 0, talos.ptr(step))
            step += 1
        for k in range(3):
            graph.replay()
            stream.synchronize()
            assert ((get(y) != 0) == ref.keep(n, 0.5, 21, k)).all(), k
    del graph
