"""CPU tests of who holds workspaces: the library's sizes and clears are made up, memory is the host's."""

import contextlib
import threading
import time
from importlib import import_module
from types import SimpleNamespace
from weakref import ref

import pytest
import torch


class FakeLib:
    """Answers every size with ``need`` and every other call with success."""

    def __init__(self):
        self.need, self.cleared, self.capturing, self.aside = 4096, [], False, False

    @contextlib.contextmanager
    def on_another_stream(self, stream):
        self.aside = True
        yield
        self.aside = False

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
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: lib.capturing and not lib.aside)
    monkeypatch.setattr(torch.cuda, "Stream", lambda *a: SimpleNamespace(cuda_stream=99, synchronize=lambda: None))
    monkeypatch.setattr(torch.cuda, "stream", lib.on_another_stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: SimpleNamespace(cuda_stream=0))
    return lib


def grow(module, fake, need):
    fake.need = need
    lib = import_module(type(module).__module__)._lib
    if hasattr(module, "layers"):
        module._ensure_workspace(lib.BlockDesc(), torch.device("cpu"))
    else:
        module._ensure_workspace(lib.LayerDesc(), torch.device("cpu"), stepwise=True)
    return module._ws


def test_a_replaced_workspace_takes_the_layers_graph_with_it(pkg, fake):
    layer = pkg.B200TransformerLayer(32, 1)
    first = grow(layer, fake, 4096)
    graph = layer._graph = object()
    assert grow(layer, fake, 4096) is first and layer._graph is graph
    assert grow(layer, fake, 1024) is first and layer._graph is graph
    assert grow(layer, fake, 8192) is not first and layer._graph is None


@pytest.mark.parametrize("stack", [False, True])
def test_an_outgrown_workspace_is_kept_if_a_capture_used_it(pkg, fake, stack):
    """A caller's captured step goes on using the workspace of its capture; others are freed as before."""
    cfg = pkg.TransformerConfig(1, 8, 32, 1, ffn_dim=64, num_layers=1, causal=True)
    module = pkg.B200Transformer(cfg) if stack else pkg.B200TransformerLayer(32, 1)
    held = []
    for need, capturing in ((4096, False), (8192, False), (8192, True), (4096, False), (16384, False), (32768, True), (65536, False)):
        fake.capturing = capturing
        buf = grow(module, fake, need)
        if not held or held[-1]() is not buf:
            held.append(ref(buf))
        del buf
        assert module.workspace_ptr % 1024 == 0 and fake.cleared[-1] == module.workspace_ptr
    assert [r() is not None for r in held] == [False, True, False, True, True]     # 4, 8, 16, 32, 64 KB
    assert len(fake.cleared) == 5


def test_no_stream_beside_the_captured_ones(pkg, fake, monkeypatch):
    """An error and not an endless search, and the thread's capture mode is put back."""
    layer = pkg.B200TransformerLayer(32, 1)
    modes = []
    fake.b200l_exchange_capture_mode = lambda mode: modes.append(mode) or 0
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        grow(layer, fake, 4096)
    assert len(modes) == 2 and layer._ws is None


def test_threads_take_turns_at_a_streams_workspace(pkg, monkeypatch):
    """A call's launches pass numbers through the workspace: no other thread's call on the
    same stream comes between them, nor between the choice of a buffer and its use; calls
    on different streams do not wait for one another."""
    kv = import_module(pkg.__name__ + ".kvcache")
    inside, most, made = {}, {}, []
    meet = threading.Barrier(2)

    class Lib:
        def b200l_kv_attention(self, c, desc, ws, size, stream):
            if stream != 5:
                meet.wait(10)               # both streams' calls at once, or the barrier breaks
            inside[stream] = inside.get(stream, 0) + 1
            most[stream] = max(most.get(stream, 0), inside[stream])
            time.sleep(0.01)
            inside[stream] -= 1
            return 0 if size else -4

        def b200l_kv_attention_workspace_bytes(self, c, desc):
            return 4096

    lib = Lib()
    monkeypatch.setattr(pkg._lib, "lib", lambda: lib)
    held = kv._Workspace()
    held.grow = lambda index, stream, need: made.append(stream) or held._held.setdefault((index, stream), [(1024, need, None)])[-1][:2]
    monkeypatch.setattr(kv, "_workspace", held)
    bad = []

    def run(stream):
        try:
            kv._attention(stream, 0, b"", b"")
        except Exception as e:              # (a thread's exception is seen below)
            bad.append(e)

    for streams in ([5] * 8, [6, 7]):
        threads = [threading.Thread(target=run, args=(s,)) for s in streams]
        for t in threads:
            t.start()
        for t in threads:
            t.join(30)
    assert not bad and most == {5: 1, 6: 1, 7: 1} and sorted(made) == [5, 6, 7]
