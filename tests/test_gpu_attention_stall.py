"""Bounded waits of long attention's tensor-core kernels: a load that never arrives makes the waits for it run out; the kernel raises the error word and returns by
itself, with its results shared over a cluster and not, and the next call is right again."""
import pytest

from test_gpu_attention_long import Problem, ctx  # noqa: F401

pytestmark = pytest.mark.gpu


# (tiles shared by the CTAs of a cluster, and more tiles than the GPU has places), widths to 64 and above
@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("shape", [(1, 2, 1, 300, 600, 64, 64), (24, 8, 8, 200, 200, 32, 32), (1, 2, 1, 300, 600, 128, 96), (16, 8, 8, 200, 200, 96, 128)])
def test_a_load_that_never_arrives(talos, ctx, shape, mode):  # noqa: F811
    pr = Problem(*shape, causal=False, mode=mode)
    want = [a.copy() for a in (*pr.forward(talos, ctx), *pr.backward(talos, ctx))]
    ctx.synchronize()
    for load in (0, 1, 3):
        for call in (lambda: pr.forward(talos, ctx), lambda: pr.backward(talos, ctx)):
            try:
                talos.lib.talos_debug_gemm_stall(ctx.handle, load, 20000)
                call()
                with pytest.raises(talos.TalosError) as e: ctx.synchronize()
                assert e.value.status == talos.ERR_TIMEOUT
            finally:
                talos.lib.talos_debug_gemm_stall(ctx.handle, -1, 0)
            for a, b in zip(want, (*pr.forward(talos, ctx), *pr.backward(talos, ctx))): assert (a == b).all()
            ctx.synchronize()
