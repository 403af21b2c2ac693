"""device_status() and the delta-rule kernels' error word, with a stand-in for the library's reading of it (no GPU)."""

import contextlib
import ctypes

import torch


def test_device_status_reads_the_delta_kernels_word(monkeypatch):
    """A wait that ran out on any device that launched them shows, and is cleared when asked."""
    from kernels import _lib
    words, seen = {0: 0, 1: 2}, []

    def read(word, clear, stream):
        dev = stream - 100
        word._obj.value = words[dev]
        seen.append((dev, clear))
        if clear:
            words[dev] = 0
        return 0

    class Library:
        delta_device_status = staticmethod(read)

    monkeypatch.setattr(_lib, "lib", Library())
    monkeypatch.setattr(_lib, "_launched", {0, 1})
    monkeypatch.setattr(_lib, "_ws", {})
    monkeypatch.setattr(_lib, "stream_ptr", lambda d: 100 + d.index)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda d: None)
    assert isinstance(ctypes.byref(ctypes.c_uint32(0))._obj, ctypes.c_uint32)
    assert _lib.device_status() == 2 and seen == [(0, 0), (1, 0)]
    assert _lib.device_status(clear=True) == 2 and _lib.device_status() == 0


def test_a_launch_marks_its_device(monkeypatch):
    from kernels import _lib
    launch = _lib.Launcher("delta_step_launch", _lib.DeltaStepArgs, "7qif" + "P3q" * 3 + "3P2qP" + "P3q")
    monkeypatch.setattr(launch, "_fn", lambda args, stream: 0)
    monkeypatch.setattr(_lib, "_launched", set())
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 3, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)
    launch(3, *[0] * 7, 0, 1.0, *[0] * 4 * 3, *[0] * 6, *[0] * 4)
    assert _lib._launched == {3}
