"""Long attention's tensor-memory kernels let the next kernel start (talos_pdl) only behind the block barrier that follows their allocation: otherwise two
dependent kernels could wait in their allocations at the same time, each for the other."""
import os
import re

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "talos-xii_b200", "csrc", "attention_long_tc.cu")


def test_next_kernel_starts_behind_the_allocation():
    text = re.sub(r"//[^\n]*", "", open(PATH).read())
    seen = list(re.finditer(r"\btmem_alloc\(", text))
    assert seen
    for m in seen:
        body = text[m.end():]
        assert body.index("__syncthreads()") < body.index("talos_pdl(")
        assert "talos_pdl(" not in text[text.rindex("__shared__", 0, m.start()):m.start()]
    # every kernel of the file makes the call
    kernels = re.split(r"__global__", text)[1:]
    assert all("talos_pdl(" in k or "TC_SETUP" in k for k in kernels), [k[:120] for k in kernels if "talos_pdl(" not in k]
