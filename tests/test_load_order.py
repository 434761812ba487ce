"""CPU, the sources: a kernel that waits for the kernel before it (griddepcontrol.wait) reads nothing by a non-coherent
load.  Such a load is for data that nothing writes while the kernel runs, and under programmatic dependent launch it runs
before its inputs are written."""

from __future__ import annotations

import re

from conftest import REPO

CSRC = REPO / "vllm-qdq-plugin_b200" / "csrc"


def _code(path) -> str:
    return re.sub(r"//[^\n]*", "", path.read_text())


def _functions(text: str):
    """(name, body) of the outermost braces that follow a parameter list."""
    for m in re.finditer(r"\b(\w+)\((?:[^(){}]|\([^()]*\))*\)\s*(?:const\s*)?\{", text):
        depth, i = 1, m.end()
        while depth and i < len(text):
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        yield m.group(1), text[m.end():i]


def test_kernels_that_start_early_load_in_order():
    waiting = [(path.name, name, body) for path in sorted(CSRC.glob("*.cu")) for name, body in _functions(_code(path))
               if re.search(r"pdl_wait\(\)|griddepcontrol\.wait", body)]
    names = {name for _, name, _ in waiting}
    assert {"rmsnorm_mxfp8_kernel", "rows_mxfp8_kernel", "nvfp4_vec_kernel", "mxf8_few_rows_kernel", "amax_gs_small_kernel"} <= names
    for file, name, body in waiting:
        assert not re.search(r"\b(__ldg|ld_stream)\(|\.nc\b", body), f"{file}: {name}"


def test_row_kernels_of_mxfp8_have_no_other_load():
    """All of them wait, and so do the helpers that they read by."""
    text = _code(CSRC / "rows_mxfp8.cu")
    assert not re.search(r"\b(__ldg|ld_stream)\(|ld\.global\.nc", text) and "ld_stream_ordered(" in text
