"""Tracers, torch.func transforms and forward-mode tangents: the dense attention entry points refuse what they cannot answer.

No GPU: the library is replaced by one whose calls succeed and write nothing, so that only the Python side is at work.
"""
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from sparseattention_b200 import _lib
from sparseattention_b200.ops import cross_attention, paged_attention_decode


class Silent:
    def __getattr__(self, name):
        return lambda *args: 1 if name.endswith("splits") else 0


@pytest.fixture(autouse=True)
def silent_library(monkeypatch):
    monkeypatch.setattr(_lib, "load", lambda: Silent())
    monkeypatch.setattr(_lib, "require_cuda", lambda *tensors: tensors[0].device)
    monkeypatch.setattr(_lib, "stream_ptr", lambda dev: None)
    monkeypatch.setattr(_lib, "on_device", lambda dev: _lib._NO_SWITCH)


def dense(q, k):
    return cross_attention(q, k, k)


def paged(q, k):
    return paged_attention_decode(q[:, 0], k, k, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32))


def inputs():
    return torch.randn(1, 3, 2, 8), torch.randn(1, 5, 2, 8)


OPS = pytest.mark.parametrize("op", [dense, paged])


@OPS
def test_plain_calls_pass(op):
    q, k = inputs()
    assert op(q, k).shape == (q.shape if op is dense else q[:, 0].shape)


@OPS
def test_tracing_is_refused(op):
    q, k = inputs()
    with torch.no_grad(), pytest.raises(_lib.HsaError, match="traced"):
        torch.jit.trace(op, (q, k), check_trace=False)
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(_lib.HsaError, match="traced"):
            make_fx(op, tracing_mode=mode)(q, k)

    class Holder(torch.nn.Module):
        def forward(self, q, k):
            return op(q, k)

    with pytest.raises(_lib.HsaError, match="traced"):
        torch.export.export(Holder(), (q, k), strict=False)


@OPS
@pytest.mark.parametrize("which", [0, 1])
def test_forward_mode_tangents_are_refused(op, which):
    args = list(inputs())
    with forward_ad.dual_level():
        op(*args)                                            # a level alone changes nothing
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with torch.no_grad(), pytest.raises(_lib.HsaError, match="forward-mode"):
            op(*args)


@OPS
def test_functional_transforms_are_refused(op):
    q, k = inputs()
    many = q.expand(4, *q.shape)
    for call in (lambda: torch.vmap(op, (0, None))(many, k), lambda: torch.func.jvp(op, (q, k), (q, k)),
                 lambda: torch.func.grad(lambda q: op(q, k).sum())(q), lambda: torch.func.functionalize(op)(q, k)):
        with torch.no_grad(), pytest.raises(_lib.HsaError, match="torch.func"):
            call()


@OPS
def test_compiled_callers_break_their_graph_at_the_call(op):
    q, k = inputs()
    graphs = []

    def backend(graph, example):
        graphs.append([str(n.target) for n in graph.graph.nodes if n.op == "call_function"])
        return graph.forward

    torch._dynamo.reset()
    got = torch.compile(lambda q, k: op(q * 2, k) + 1, backend=backend)(q, k)
    assert got.shape == op(q, k).shape
    assert len(graphs) >= 2 and len(graphs[-1]) == 1 and "add" in graphs[-1][0]
    assert not any("empty" in name for names in graphs for name in names)
    torch._dynamo.reset()
    with pytest.raises(Exception):
        torch.compile(lambda q, k: op(q * 2, k) + 1, backend=backend, fullgraph=True)(q, k)
    torch._dynamo.reset()
