"""Every kernel launch of dropout and of the gated unit is followed by a check
of its error in the function that made it: a refused launch must not pass for
a result."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "distributed_vgg_f_amd", "csrc")
LAUNCH, CHECK = "hipLaunchKernelGGL(", "HIP_CHECK(hipGetLastError())"


def unchecked(source):
    """Lines of launches with no check between them and the end of their
    function (a closing brace in the first column)."""
    pending, bad = [], []
    for number, line in enumerate(source.splitlines(), 1):
        if LAUNCH in line:
            pending.append(number)
        if CHECK in line:
            pending = []
        if line.startswith("}"):
            bad += pending
            pending = []
    return bad


def test_the_scan_sees_a_missing_check():
    checked = "void f() {\n  %sk);\n  %s;\n}\n" % (LAUNCH, CHECK)
    assert unchecked(checked) == []
    assert unchecked("void f() {\n  %sk);\n}\n%s" % (LAUNCH, checked)) == [2]


@pytest.mark.parametrize("name", ["dropout.hip", "gated.hip"])
def test_launches_are_checked(name):
    with open(os.path.join(CSRC, name)) as f:
        source = f.read()
    assert len(re.findall(re.escape(LAUNCH), source)) >= 3
    assert unchecked(source) == []
