"""The header lets results of the norm lie on its operands, so the kernels may not promise the compiler that they do not: a result that is
right in place under one compiler says nothing of the next."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _text(*path):
    with open(os.path.join(ROOT, *path)) as f:
        return f.read()


def test_the_header_lets_them_coincide():
    text = " ".join(_text("include", "moe_fused_linear.h").split())
    assert "y may be x, s may be x or residual" in text and "dx may be dy, ds or s" in text


@pytest.mark.parametrize("kernel,together", [("norm_fwd_kernel", {"x", "residual", "y", "s"}),
                                             ("norm_bwd_kernel", {"dy", "ds", "s", "dx"})])
def test_no_promise_about_pointers_that_may_coincide(kernel, together):
    (parameters,) = re.findall(kernel + r"\(([^{]*?)\) \{", _text("transformers-qwen3-moe-fused_amd", "csrc", "norm.hip"))
    pointers = {}
    for p in parameters.split(","):
        found = re.search(r"\*\s*(__restrict__\s+)?(\w+)\s*$", p)
        if found:
            pointers[found.group(2)] = bool(found.group(1))
    assert together <= set(pointers)
    assert not {name for name in together if pointers[name]}
