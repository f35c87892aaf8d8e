"""A workspace's status outlives the scratch that it was first written to (needs a B200)."""

import pytest
import torch

from refinekv_b200 import paged_append
from refinekv_b200.attention import device_status
from test_gpu_paged_attention import Served

pytestmark = pytest.mark.gpu


def _flag(ws):
    small = Served([40], 2, 2, 64, 32, seed=1, spare=0)
    small.table[0, 0] = -1
    small.call(workspace=ws)


def test_status_survives_a_call_of_a_wider_shape():
    ws = {}
    _flag(ws)
    wide = Served([40, 300], 32, 2, 256, 32, seed=2)
    out, lse = wide.call(workspace=ws)
    wide.check(out, lse)
    assert device_status(ws) == 2


def test_status_survives_a_wider_shape_captured_in_a_graph():
    wide = Served([40, 300], 32, 2, 256, 32, seed=3)
    wide.call(workspace={})
    ws = {}
    _flag(ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = wide.call(workspace=ws)
    graph.replay()
    wide.check(out, lse)
    assert device_status(ws) == 2


def test_append_status_is_sticky():
    s = Served([40], 2, 2, 64, 32, seed=4)
    k = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    ws = {}
    for position, status in ((3, 0), (10 ** 6, 2), (3, 2)):
        at = torch.tensor([position], device="cuda")
        paged_append(k, k, s.kp, s.vp, s.table, at, workspace=ws)
        assert device_status(ws) == status
