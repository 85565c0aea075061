"""The Julia methods of the layer calls, read as text (there is no Julia to run
them with): every array whose pointer goes into a ccall has been through
operand(), which checks element type, size and contiguity, before it; and the
module names nothing that older Julia versions lack when it is loaded."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = open(os.path.join(ROOT, "cutile-triton_b200", "julia", "TileTritonB200.jl")).read()
CODE = re.sub(r'"""(?:.|\n)*?"""', '""', SOURCE)

ARRAYS = {
    "dense!": ["A", "B", "C", "bias", "R", "Z"],
    "dense_bwd!": ["dC", "A", "B", "Z", "dA", "dB", "dbias"],
    "moe_route": ["logits", "bias"],
    "moe_route_bwd": ["logits", "ids", "dweights"],
    "moe_combine!": ["out", "y", "weights", "ids", "R"],
    "moe_combine_bwd": ["dout", "ys", "weights", "ids"],
}


def body(name):
    m = re.search(r"^function %s\((.|\n)*?^end$" % re.escape(name), CODE, re.M)
    assert m, name
    return m.group(0)


@pytest.mark.parametrize("name", sorted(ARRAYS))
def test_arrays_are_checked_before_their_pointers_are_used(name):
    text = body(name)
    first = text.index("ccall(")
    for array in ARRAYS[name]:
        checks = [m.start() for m in re.finditer(r"\boperand\(%s, \"%s: \w+\", \w+" % (array, re.escape(name)), text)]
        if array == "bias" and name == "dense!":  # of either of two types
            checks = [m.start() for m in re.finditer(r"\boperand\(bias, \"dense!: bias\", bias isa", text)]
        assert checks and checks[0] < first, array
    # nothing else becomes a pointer
    used = set(re.findall(r"\borC\((\w+)\)|\bpointer\((\w+)\)", text))
    made = {"dweights"} if name == "moe_combine_bwd" else set()
    assert {a or b for a, b in used} <= set(ARRAYS[name]) | made
    for array in ("weights", "ids", "dweights"):
        if array in ARRAYS[name]:
            assert re.search(r"operand\(%s, [^\n]*packed=true\)" % array, text)


def test_no_names_that_older_versions_lack():
    assert "Core.BFloat16" not in CODE


def test_brackets_close():
    """A slip of the pen that would keep the module from loading."""
    bare = re.sub(r'"(?:\\.|[^"\\])*"', '""', CODE)
    bare = re.sub(r"#[^\n]*", "", bare)
    for o, c in ("()", "[]", "{}"):
        assert bare.count(o) == bare.count(c), o
