"""The planner's view of MUL_MAT nodes of 4-bit weights on the CPU: the chains,
redirects and the gated GELU after them, as after nodes of FP16 weights."""

import pytest
import torch

import graph_lib as gl
import q4_lib
import sdhip
from helpers import rng

KINDS = ["q4_0", "q4_1"]


def weights(g, kind, n, k):
    return g.leaf(torch.from_numpy(q4_lib.random_blocks(rng(n + k), kind, n, k)))


def zeros(g, *shape):
    return g.leaf(torch.zeros(shape))


def planned(g, out, node):
    order, arr = g.build(out)
    status, p = gl.plan(sdhip.load(), arr, len(order), order.index(node))
    assert status == sdhip.OK and p.taken == gl.OP["MUL_MAT"]
    return order, p


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 15, 200])
def test_gated_gelu(kind, rows):
    g = gl.Graph("cpu")
    y = g.mul_mat(weights(g, kind, 2 * 96, 320), zeros(g, rows, 320))
    p = g.add_inplace(y, zeros(g, 2 * 96))
    gate = g.gelu_inplace(g.cont(g.view_columns(p, 96, 96)))
    # Dense, as ggml makes it: torch's own would have the view's stride for a single row.
    out = gl.T(torch.zeros((rows, 96)), "MUL", [g.view_columns(p, 0, 96), gate])
    order, plan = planned(g, out, y)
    assert plan.count == 7 == len(order) and plan.chain.count == 1
    assert plan.gated_out and plan.gated_out.contents.tensor.data == out.data.data_ptr()
    # With the gate read by a later node, the halves must be written: no fusion.
    order, plan = planned(g, g.add(gate, gate), y)
    assert not plan.gated_out and plan.count == 2


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 15, 200])
def test_redirects(kind, rows):
    g = gl.Graph("cpu")
    y = g.mul_mat(weights(g, kind, 70, 96), zeros(g, rows, 96))
    out = g.add(g.add_inplace(y, zeros(g, 70)), zeros(g, rows, 70))
    order, plan = planned(g, out, y)
    assert plan.count == 3 and plan.chain.redirect.contents.data == out.data.data_ptr() and not plan.chain.from_redirect
    # The residual in its own memory begins the sum.
    g = gl.Graph("cpu")
    y = g.mul_mat(weights(g, kind, 70, 96), zeros(g, rows, 96))
    d = g.dup(zeros(g, rows, 70))
    out = g.add_inplace(d, g.add_inplace(y, zeros(g, 70)))
    order, plan = planned(g, out, y)
    assert plan.chain.redirect.contents.data == d.data.data_ptr() and plan.chain.from_redirect
    # Not where that memory is what the product reads.
    g = gl.Graph("cpu")
    x = g.dup(zeros(g, rows, 96))
    y = g.mul_mat(weights(g, kind, 96, 96), x)
    order, plan = planned(g, g.add_inplace(x, y), y)
    assert not plan.chain.redirect and plan.count == 1
