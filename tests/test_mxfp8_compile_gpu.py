"""GPU: the MXFP8 operators under torch.compile, in processes whose first call of them is the traced one."""

from __future__ import annotations

import subprocess
import sys

import pytest

from conftest import REPO

pytestmark = pytest.mark.gpu

SCRIPT = """
import sys
sys.path[:0] = {path!r}
import torch
from mxfp8_cases import activation, random_weight, routing
from vllm_qdq_plugin.gemm import mxfp8_linear, mxfp8_moe_linear, prepare_mxfp8_moe_weight, prepare_mxfp8_weight
from vllm_qdq_plugin.qdq import rmsnorm_mxfp8, silu_mul_mxfp8
backend, part = {backend!r}, {part!r}
dev = torch.device("cuda", 0)
m, k = 40, 96  # 3 scales a row, stored 16 apart
x = activation(m, k, torch.bfloat16, 1, dev)
g = torch.ones(k, dtype=torch.bfloat16, device=dev)
if part != "rows":
    w = prepare_mxfp8_weight(*random_weight(128, k, seed=1, dev=dev))
    wm = prepare_mxfp8_moe_weight(*random_weight(2, 128, k, seed=1, dev=dev))
    _, sid, eid, ntp, tw = routing(m, 2, 1, 16, 1, dev)

def layer(x, r):
    rows, h, y = rmsnorm_mxfp8(x, g, r, norm_out=True)
    if part == "break":
        torch._dynamo.graph_break()  # rows leave one graph and enter the next
    if part == "rows":
        act = silu_mul_mxfp8(torch.cat([y, h], 1))
        return rows.codes, rows.scales, act.codes, act.scales
    up = mxfp8_linear(rows, w)
    act = silu_mul_mxfp8(up + 1)
    out = torch.zeros(m, 128, dtype=torch.bfloat16, device=dev)
    down = mxfp8_moe_linear(x, wm, sid, eid, ntp, tw, 16, 1, True, out=out)
    return act.codes, act.scales, h, up, down + mxfp8_moe_linear(rows, wm, sid, eid, ntp, tw, 16, 1, True)

compiled = torch.compile(layer, backend=backend, fullgraph=part != "break")
first = compiled(x, x)
graphs = torch._dynamo.utils.counters["stats"]["unique_graphs"]
second = compiled(x, x)
assert torch._dynamo.utils.counters["stats"]["unique_graphs"] == graphs, "compiled again"
want = layer(x, x)
assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(first, want, second))
print("ok")
"""


@pytest.mark.parametrize("backend,part", [("eager", "rows"), ("eager", "layer"), ("inductor", "rows"), ("inductor", "layer"),
                                          ("inductor", "break")])
def test_first_call_of_a_process_is_traced(tmp_path, backend, part):
    script = tmp_path / "first.py"
    path = [str(REPO / "vllm-qdq-plugin_b200"), str(REPO), str(REPO / "tests")]
    script.write_text(SCRIPT.format(path=path, backend=backend, part=part))
    done = subprocess.run([sys.executable, str(script)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "ok" in done.stdout, done.stderr[-3000:]
