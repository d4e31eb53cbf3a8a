"""The device sources share one namespace: an inline function defined in two of
them, perhaps with two bodies, is one function to the linker."""

import collections
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "distributed_vgg_f_amd", "csrc")
HEAD = re.compile(r"^DEV (?!static)[\w:<>]+ (\w+)\(([^)]*)\)", re.M)


def inline_functions(source):
    """(name, types of the arguments) of the file's inline device functions."""
    for name, args in HEAD.findall(source):
        types = [re.sub(r"\s*\w+$", "", a.strip()) if " " in a.strip() else
                 a.strip() for a in args.split(",")]
        yield name, tuple(types)


def test_the_scan_reads_names_and_types():
    source = "DEV float to_f(u16 v, __bf16) { }\nDEV u32 g() {\n"
    assert list(inline_functions(source)) == [("to_f", ("u16", "__bf16")),
                                              ("g", ("",))]


def test_no_inline_function_twice():
    where = collections.defaultdict(set)
    for name in os.listdir(CSRC):
        with open(os.path.join(CSRC, name)) as f:
            for function in inline_functions(f.read()):
                where[function].add(name)
    assert len(where) > 20
    assert {f: n for f, n in where.items() if len(n) > 1} == {}
