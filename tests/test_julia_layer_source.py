"""The Julia methods of the layer calls, read as text (there is no Julia to run
them with): the module names nothing that older Julia versions lack when it is
loaded."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = open(os.path.join(ROOT, "cutile-triton_b200", "julia", "TileTritonB200.jl")).read()
CODE = re.sub(r'"""(?:.|\n)*?"""', '""', SOURCE)


def test_no_names_that_older_versions_lack():
    assert "Core.BFloat16" not in CODE


def test_brackets_close():
    """A slip of the pen that would keep the module from loading."""
    bare = re.sub(r'"(?:\\.|[^"\\])*"', '""', CODE)
    bare = re.sub(r"#[^\n]*", "", bare)
    for o, c in ("()", "[]", "{}"):
        assert bare.count(o) == bare.count(c), o
