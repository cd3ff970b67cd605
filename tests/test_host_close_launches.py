"""Kernels that begin under the end of the one before read its results by plain loads.

A read-only load (``__ldg``) is defined for memory that nobody writes in the kernel's lifetime, and the compiler
may move it above the wait for the previous kernel.  In a kernel of ``launch_behind`` it may therefore read only
the inputs of the call, which were complete before the call's first kernel began.
"""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "tynx_b200" / "csrc"
# functions that run in kernels of launch_behind, and the inputs of the call that they read by __ldg
FUNCTIONS = {
    "diff_attn.cuh": {"sum_dlam": (), "lam_exponent": ("s.lam",), "length": ("len",), "report_length": ("s.len",)},
    "diff_attn.cu": {"k_diff_join": ("s.lam",)},
    "diff_attn_fwd.cu": {"k_diff_fwd": ("s.lam",), "item_at": ()},
    "diff_attn_bwd.cu": {"body": ("s.lam",), "k_diff_bwd": (), "k_diff_group_sum": ()},
    "rotary.cu": {"k_qk_norm_dw": ()},
}


def body_of(source, name):
    """The text between a function definition's braces."""
    for match in re.finditer(rf"\b{name}\(", source):
        depth, at = 0, match.end() - 1
        while True:  # the parameter list
            depth += {"(": 1, ")": -1}.get(source[at], 0)
            at += 1
            if depth == 0:
                break
        rest = re.match(r"\s*(const\s*)?\{", source[at:])
        if not rest:
            continue
        begin = at = at + rest.end()
        depth = 1
        while depth:
            depth += {"{": 1, "}": -1}.get(source[at], 0)
            at += 1
        return source[begin:at]
    raise AssertionError(f"no definition of {name}")


@pytest.mark.parametrize("file", sorted(FUNCTIONS))
def test_results_of_the_previous_kernel_are_read_by_plain_loads(file):
    source = re.sub(r"//[^\n]*", "", (CSRC / file).read_text())
    for name, inputs in FUNCTIONS[file].items():
        read = [m.split()[0].split("[")[0] for m in re.findall(r"__ldg\(([^)]*)", body_of(source, name))]
        assert set(read) <= set(inputs), (name, read)


def test_every_such_kernel_is_listed():
    listed = {name for functions in FUNCTIONS.values() for name in functions}
    for path in sorted(CSRC.glob("*.cu")):
        for name in re.findall(r"launch_behind\(\s*ctx,\s*\"[a-z_0-9]+\",\s*([a-z_0-9]+)", path.read_text()):
            assert name in listed, (path.name, name)
