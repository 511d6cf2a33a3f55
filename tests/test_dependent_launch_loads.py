"""A kernel that reads through the read-only or streaming load functions (__ldg, __ldcs) passes its pointers through the wait for the kernel before it: the compiler
takes such a load for one of memory that nobody writes, and may otherwise move it above the wait.  What such a load then reads is what the kernel before it has
not written yet; no result on the GPU shows it reliably, so the sources are looked at."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "talos-xii_b200", "csrc")
FILES = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))
LOADS = r"\b__ld(?:g|cs|cg|ca)\("


def functions(text):
    """(is a kernel, name, body) of every device function, in order."""
    text = re.sub(r"//[^\n]*", "", text)
    marks = list(re.finditer(r"__global__|__device__", text))
    for m, following in zip(marks, marks[1:] + [None]):
        part = text[m.end():following.start() if following else len(text)]
        head = re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", part)
        name = re.search(r"(\w+)\s*\(", head)
        if name: yield m.group() == "__global__", name.group(1), head[name.end():]


def loading(funcs):
    """Names of the functions that make such a load, themselves or through others of the file."""
    names = {n for _, n, body in funcs if re.search(LOADS, body)}
    while True:
        more = {n for _, n, body in funcs if n not in names and any(re.search(r"\b%s\s*(?:<[^()]*>)?\(" % m, body) for m in names)}
        if not more: return names
        names |= more


@pytest.mark.parametrize("name", FILES)
def test_pointers_pass_through_the_wait(name):
    funcs = list(functions(open(os.path.join(CSRC, name)).read()))
    names = loading(funcs)
    bare = [n for kernel, n, body in funcs if kernel and n in names and not re.search(r"\b(?:talos_pdl|pdl_late)\(\s*[\w.\[\]]+", body)]
    assert not bare, bare


def test_the_kernels_are_found():
    seen = {}
    for name in FILES:
        funcs = list(functions(open(os.path.join(CSRC, name)).read()))
        names = loading(funcs)
        seen[name] = {n for kernel, n, _ in funcs if kernel and n in names}
    assert "attn_split_kernel" in seen["attention_long_tc.cu"] and "attn_decode_kernel" in seen["attention_long.cu"]
    assert {"norm_fwd_kernel", "norm_bwd_kernel", "dropout_kernel"} <= seen["norm.cu"] and "policy_loss_kernel" in seen["policy_loss.cu"]
