"""Which causal values long attention takes."""
import pytest

P = 4096     # an address that is never read: the call is refused first, or fails for want of a context


@pytest.mark.parametrize("causal,text", [(0, "null context"), (1, "null context"), (3, "null context"), (2, "causal"), (4, "causal"), (-1, "causal")])
def test_causal_values(talos, causal, text):
    tail = (2, 4, 2, 16, 32, 64, 64, 0.125, causal, 0, 1)
    for call in (lambda: talos.lib.talos_attention_lse_fwd(None, P, P, P, P, P, P, *tail), lambda: talos.lib.talos_attention_lse_bwd(None, P, P, P, P, P, P, P, P, P, P, *tail)):
        with pytest.raises(talos.TalosError) as e: call()
        assert e.value.status == talos.ERR_ARG and text in str(e.value)
