"""The model graph on a stream of its own, on the CPU: the ops are stand-ins that write down the stream they run on."""
import torch

from lnsb200 import model
import test_serve_decoder as stand_in


class Ops(stand_in.Ops):
    """the stand-in with the graph's own cache and attention"""

    def rope(self, x, T, nh, hd, pos0):
        return self._op("rope", x.clone())

    def kv_store(self, il, k, v, pos0, T):
        self._op("kv", None)

    def attention(self, il, q, T, H, HKV, D, pos0):
        return self._op("attention", torch.zeros(T, H * D))

    def last_row(self, x):
        return x[-1:]


def _ran(ops):
    return {e[1] for e in ops.log if e[0] != "wait"}


def test_the_graph_runs_on_the_ops_stream():
    ops = Ops("side")
    assert model.forward(ops, stand_in.CFG, [1, 2, 3], 0).shape == (1, stand_in.CFG["vocab"])
    assert _ran(ops) == {"side"}
    assert ops.log[0] == ("wait", "side", "current") and ops.log[-1] == ("wait", "current", "side")
    assert ops.torch.cuda.now.name == "current"


def test_without_one_on_the_current():
    ops = Ops()
    model.forward(ops, stand_in.CFG, [1, 2, 3], 0)
    assert _ran(ops) == {"current"} and not [e for e in ops.log if e[0] == "wait"]


def test_ops_that_know_no_streams():
    """the CPU checker's ops have none"""
    ops = Ops()
    del ops.stream
    assert model.forward(ops, stand_in.CFG, [1, 2], 0).shape == (1, stand_in.CFG["vocab"])
