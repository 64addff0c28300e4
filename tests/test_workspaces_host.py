"""CPU: no two calls share a workspace. (An entry point launches several kernels over its workspace
without the interpreter's lock, so calls of two threads on one stream interleave.)"""
import threading

import torch

from muxi_race_b200.fused import _workspace


def test_two_calls_at_once_have_two_buffers():
    cpu = torch.device("cpu")
    held = []

    def call():
        held.append(_workspace(4096, cpu))

    call()
    t = threading.Thread(target=call)
    t.start()
    t.join()
    a, b = held
    assert a.numel() >= 4096 and b.numel() >= 4096 and a.dtype == torch.uint8
    assert a.data_ptr() + a.numel() <= b.data_ptr() or b.data_ptr() + b.numel() <= a.data_ptr()


def test_a_call_keeps_nothing():
    import gc
    import weakref

    ws = _workspace(1, torch.device("cpu"))
    assert ws.numel() >= 256
    seen = weakref.ref(ws)
    del ws
    gc.collect()
    assert seen() is None
