"""Attention over graphs with hubs, as the library's other kernels meet them: rows and columns from none to a thousand edges, a graph
used as its own transpose, serving rows over hub rows."""
import numpy as np
import pytest

from attn_run import Case
from attn_tight import tight
from fusedmm_amd import synth
from test_gpu_attention import check_backward, check_forward
from test_gpu_attention_rows import check_rows

pytestmark = pytest.mark.gpu


def graph(name):
    if name == "rmat":
        g = synth.rmat_graph(11, 8, seed=5)
    else:
        g = synth.zipf_graph(1500, 1.8, 1400, 12000, seed=5)
    return g, len(g["pntrb"])


@pytest.mark.parametrize("kind,maps,d,dv", [("f32", 1, 32, 32), ("bf16", 2, 32, 64), ("f16", 1, 64, 64), ("bf16", 1, 100, 40)])
@pytest.mark.parametrize("name", ["rmat", "zipf"])
def test_graphs_with_hubs(name, kind, maps, d, dv):
    import torch
    g, n = graph(name)
    degree = g["pntre"] - g["pntrb"]
    assert degree.max() > 300 and np.median(degree) < 20
    c = Case(kind, maps, n, n, 4, 2, d, dv, g["indx"], g["pntrb"], g["pntre"], seed=3)
    c.make_plans(True)
    c.gradients()
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    e = tight(c, do=True)
    check_forward(c, e)
    check_backward(c, e)
    assert c.rows() == 0
    torch.cuda.synchronize()
    check_rows(c, e)
