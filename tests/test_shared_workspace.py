"""The 16-bit GEMM's calls from several threads on one stream: they share the stream's workspace (tickets, partial tiles, repacked
operands), so what a call does between asking for it and its last launch is one step. Without a GPU: the library is a stand-in."""
import contextlib
import ctypes as C
import threading

import pytest
import torch

from flydsl_examples_b200 import _lib, gemm_a16w16 as module


class OnGpu(torch.Tensor):
    is_cuda = True


class Stream:
    cuda_stream = 0


class Library:
    """Records what is called; the first launch of two operands waits a while for another thread to go past it."""

    def __init__(self):
        self.events, self.others, self.launching = [], threading.Event(), threading.Event()

    def b200_gemm_workspace_bytes(self, args):
        return _lib.COUNTER_BYTES + args._obj.m * (1 << 20)

    def b200_gemm_prepare(self, args, handle):
        m = args._obj.m
        self.events.append(("prepare", m, args._obj.workspace))
        if len(self.events) > 1:
            self.others.set()
        handle._obj.value = m
        return 0

    def b200_gemm_launch(self, handle, stream):
        self.events.append(("launch", handle.value))
        if not self.launching.is_set():
            self.launching.set()
            self.others.wait(0.5)
        self.events.append(("launched", handle.value))
        return 0

    def b200_gemm_release(self, handle):
        pass


@pytest.mark.parametrize("entry", ["gemm_a16w16", "gemm_a16w16_to_pointer"])
def test_first_calls_of_two_threads_do_not_share_the_workspace_at_once(monkeypatch, entry):
    lib, ws = Library(), module._Workspace(torch.device("cpu"))
    monkeypatch.setattr(module._lib, "load", lambda: lib)
    monkeypatch.setattr(module, "_workspace_for", lambda device, stream: ws)
    monkeypatch.setattr(module, "_num_sms", lambda device: 148)
    monkeypatch.setattr(module, "_prepared", type(module._prepared)())
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    errors = []

    def call(m):
        try:
            a, b = (torch.zeros(r, 64, dtype=torch.bfloat16).as_subclass(OnGpu) for r in (m, 32))
            if entry == "gemm_a16w16":
                module.gemm_a16w16(a, b.t(), torch.zeros(m, 32, dtype=torch.bfloat16).as_subclass(OnGpu), stream=Stream())
            else:
                module.gemm_a16w16_to_pointer(a, b.t(), 4096, torch.bfloat16, stream=Stream())
        except Exception as e:
            errors.append(e)
    first = threading.Thread(target=call, args=(8,))
    first.start()
    assert lib.launching.wait(60)
    second = threading.Thread(target=call, args=(16,))  # needs a larger workspace, which replaces the first call's
    second.start()
    first.join()
    second.join()
    assert not errors
    assert [e[:2] for e in lib.events] == [("prepare", 8), ("launch", 8), ("launched", 8), ("prepare", 16), ("launch", 16), ("launched", 16)]
    assert lib.events[0][2] != lib.events[3][2] == ws.buf.data_ptr()
    # the first call's launch points into the buffer that is gone; it is not repeated as it was
    old, new = module._prepared.values()
    assert old.ws_gen != ws.generation == new.ws_gen
    assert isinstance(old.handle, C.c_void_p)


def test_captured_calls_have_workspaces_of_their_own(monkeypatch):
    # Graphs replay in any order and at once: no two may share tickets, partial tiles or repacked operands, nor may a graph keep the
    # stream's buffer, which a larger call replaces
    capturing, spans = [False], []

    class Recorder(Library):
        def b200_gemm_prepare(self, args, handle):
            at = args._obj.workspace
            spans.append((at, at + args._obj.workspace_bytes))
            assert not any((C.c_uint8 * (4 * 30)).from_address(at))
            handle._obj.value = 1
            return 0

        def b200_gemm_plan_query(self, args, plan):
            plan._obj.tiles_p, plan._obj.tiles_q, plan._obj.cta_group, plan._obj.partial_bytes = 3, 5, 2, 1
            return 0

        def b200_gemm_launch(self, handle, stream):
            self.launches = getattr(self, "launches", 0) + 1
            return 0
    lib, ws, held = Recorder(), module._Workspace(torch.device("cpu")), []
    empty = torch.empty
    monkeypatch.setattr(module._lib, "load", lambda: lib)
    monkeypatch.setattr(module, "_workspace_for", lambda device, stream: ws)
    monkeypatch.setattr(module, "_num_sms", lambda device: 148)
    monkeypatch.setattr(module, "_prepared", type(module._prepared)())
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", lambda stream: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    # the memory of a graph's pool: neither cleared nor given out twice here
    monkeypatch.setattr(torch, "empty", lambda *a, **k: held.append(empty(*a, **k).fill_(77)) or held[-1])
    a, b = (torch.zeros(r, 64, dtype=torch.bfloat16).as_subclass(OnGpu) for r in (8, 32))
    out = torch.zeros(8, 32, dtype=torch.bfloat16).as_subclass(OnGpu)

    def calls():
        module.gemm_a16w16(a, b.t(), out, stream=Stream())
        module.gemm_a16w16_to_pointer(a, b.t(), 4096, torch.bfloat16, stream=Stream())
    calls()
    calls()  # repeats: resolved launches
    assert len(spans) == 2 and spans[0] == spans[1] == (ws.buf.data_ptr(), ws.buf.data_ptr() + ws.buf.numel()) and lib.launches == 4
    capturing[0] = True
    calls()
    calls()
    captured = spans[2:]
    assert len(captured) == 4 and lib.launches == 8
    for i, (lo, hi) in enumerate(captured):
        assert hi - lo >= _lib.COUNTER_BYTES + (8 << 20)
        assert all(hi <= lo2 or hi2 <= lo for lo2, hi2 in captured[i + 1:] + spans[:1])
    capturing[0] = False
    calls()  # the stream's launches as they were
    assert len(spans) == 6 and lib.launches == 10
