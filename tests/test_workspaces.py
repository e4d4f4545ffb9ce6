"""CPU tests of who holds workspaces: the library's sizes and clears are made up, memory is the host's."""

import contextlib
from importlib import import_module
from types import SimpleNamespace

import pytest
import torch


class FakeLib:
    """Answers every size with ``need`` and every other call with success."""

    def __init__(self):
        self.need, self.cleared = 4096, []

    def __getattr__(self, name):
        if name.endswith("_workspace_bytes"):
            return lambda *a: self.need
        if name == "b200l_clear_status":
            return lambda ptr, stream: self.cleared.append(ptr) or 0
        return lambda *a: 0


@pytest.fixture
def fake(pkg, monkeypatch):
    lib = FakeLib()
    monkeypatch.setattr(pkg._lib, "lib", lambda: lib)
    monkeypatch.setattr(torch.cuda, "device", lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: SimpleNamespace(cuda_stream=0))
    return lib


def grow(layer, fake, need):
    fake.need = need
    desc = import_module(type(layer).__module__)._lib.LayerDesc()
    layer._ensure_workspace(desc, torch.device("cpu"), stepwise=True)
    return layer._ws


def test_a_replaced_workspace_takes_the_layers_graph_with_it(pkg, fake):
    layer = pkg.B200TransformerLayer(32, 1)
    first = grow(layer, fake, 4096)
    graph = layer._graph = object()
    assert grow(layer, fake, 4096) is first and layer._graph is graph
    assert grow(layer, fake, 1024) is first and layer._graph is graph
    assert grow(layer, fake, 8192) is not first and layer._graph is None
