"""Graphs with MUL_MAT nodes of 4-bit weights through sdhip_compute_nodes on
the device: the chain, the redirect and the gated GELU within the product, and
node by node (fuse=0), each against float64."""

import numpy as np
import pytest
import torch

import graph_lib as gl
import q4_lib
import sdhip
from helpers import rng, uniform
from test_gpu_q4 import gelu64

KINDS = ["q4_0", "q4_1"]
K, N = 352, 140


class Case:
    """A graph, its exact output, how far a right one may lie from it and the
    nodes the library computes of it, fused and apart."""

    def __init__(self, gpu, kind, rows, end):
        r = rng(rows)
        self.graph = g = gl.Graph(gpu)
        blocks, x = q4_lib.random_blocks(r, kind, N, K), uniform(r, (rows, K), 1.0)
        bias, res = uniform(r, (N,), 1.0), uniform(r, (rows, N), 1.0)
        leaf = lambda a: g.leaf(torch.from_numpy(a))
        p = g.add_inplace(g.mul_mat(leaf(blocks), leaf(x)), leaf(bias))
        exact, mag = q4_lib.exact(blocks, x)
        exact, mag = exact + bias, mag + np.abs(bias)
        if end == "gated":
            gate = g.gelu_inplace(g.cont(g.view_columns(p, N // 2, N // 2)))
            # Dense, as ggml makes it: torch's own would have the view's stride for a single row.
            self.out = gl.T(torch.full((rows, N // 2), float("nan"), device=gpu), "MUL", [g.view_columns(p, 0, N // 2), gate])
            self.fused = 7
            a, b = exact[:, :N // 2], exact[:, N // 2:]
            # d(a gelu(b)) <= |gelu| da + |a| 1.13 db; gelu's own exponential and division, and the product, add 2^-20.
            err = q4_lib.bound(K, 1)
            da, db = err * mag[:, :N // 2], err * mag[:, N // 2:]
            self.exact = a * gelu64(b)
            self.allowed = (np.abs(gelu64(b)) * da + 1.13 * np.abs(a) * db) * (1 + 1e-3) + 2.0 ** -20 * np.abs(a * b) + da * db
        elif end == "redirect":
            self.out = g.add(p, leaf(res))
            self.fused = 3
            self.exact, self.allowed = exact + res, q4_lib.bound(K, 2) * (mag + np.abs(res))
        else:
            self.out = g.add_inplace(g.dup(leaf(res)), p)
            self.fused = 3
            self.exact, self.allowed = exact + res, q4_lib.bound(K, 2) * (mag + np.abs(res))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 16, 40, 300])
@pytest.mark.parametrize("end", ["gated", "redirect", "own memory"])
@pytest.mark.parametrize("tuning", ["", "fuse=0", "fuse_residual=0"])
def test_graph(gpu, kind, rows, end, tuning):
    case = Case(gpu, kind, rows, end)
    order, arr = case.graph.build(case.out)
    sdhip.set_tuning(tuning)
    try:
        by_library = gl.run(sdhip.load(), order, arr)
        torch.cuda.synchronize()
    finally:
        sdhip.set_tuning("")
    if tuning == "":
        assert by_library == case.fused
    elif tuning == "fuse=0":
        assert by_library == 1
    got = case.out.data.cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all() and (np.abs(got - case.exact) <= case.allowed).all()
