"""What the library shares between its translation units stays its own: a host
that has a symbol of the same name, or another build of the library in the same
process, must not take its place."""
import re
import subprocess

import pytest

from siphon_amd.build import HIP_SO, PKG


def exported():
    out = subprocess.run(["nm", "-D", "--defined-only", HIP_SO], check=True, text=True, capture_output=True).stdout
    return {line.split()[-1] for line in out.splitlines()}


def shared_names():
    """Functions and variables that context.h defines."""
    text = re.sub(r"//[^\n]*|\\\n", "", open(f"{PKG}/csrc/context.h").read())
    names = re.findall(r"^inline [\w ]+?\**(\w+)[(\[]", text, flags=re.M)
    assert {"set_err", "ensure", "order_before", "g_init_err"} <= set(names)
    return names


@pytest.mark.parametrize("name", shared_names())
def test_shared_state_is_not_exported(name):
    # as it is (variables), or with its length and arguments (functions)
    bad = [s for s in exported() if s == name or re.match(rf"_Z\w*?{len(name)}{name}", s)]
    assert not bad, bad
