"""Which stream the Python faces launch on, without a device."""
import threading
from types import SimpleNamespace

import torch

from purhie_b200.csrc import fp8, ops


def test_a_scope_is_its_thread_s_own(monkeypatch):
    """Another thread's launches go to its own current stream, whatever scope this one is in, and the other way round."""
    main = threading.get_ident()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: SimpleNamespace(cuda_stream=5 if threading.get_ident() == main else 7))
    seen = {}

    def other():
        seen["beside"] = ops._stream(), fp8._scope()
        with ops.on_current_stream():
            seen["inside"] = ops._stream(), fp8._scope()
            entered.set()
            left.wait(10)

    assert fp8._scope() == -1
    entered, left = threading.Event(), threading.Event()
    with ops.on_current_stream():
        t = threading.Thread(target=other)
        t.start()
        assert entered.wait(10)
        assert ops._stream() == 5 and fp8._scope() == 5
    assert fp8._scope() == -1                    # (the other thread is still in its scope)
    left.set()
    t.join()
    assert seen == {"beside": (7, -1), "inside": (7, 7)}
