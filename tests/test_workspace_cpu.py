"""The per-stream workspaces of ``_lib``: what they keep, and who may use one at a
time.  The device and the library are stood in for, nothing is launched."""
import contextlib
import gc
import threading
import time
import weakref

import pytest
import torch

from adakv_b200 import _lib


@pytest.fixture
def host(monkeypatch):
    """Workspaces in host memory, with a library that accepts every sink."""

    class Library:
        @staticmethod
        def adakv_set_status_sink(ws, word, stream):
            return _lib.OK

    monkeypatch.setattr(_lib, "_workspaces", {})
    monkeypatch.setattr(_lib, "_sinks", {})
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 7)
    monkeypatch.setattr(_lib, "lib", lambda: Library)
    monkeypatch.setattr(_lib, "_get_device", lambda: None)  # (a CPU device has no index)
    monkeypatch.setattr(_lib, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)


def test_outgrown_workspace_is_kept(host):
    """A graph that was captured with the smaller buffer still writes there."""
    small = weakref.ref(_lib.workspace(300, "cpu", "pages"))
    at = small().data_ptr()
    large = _lib.workspace(4096, "cpu", "pages")
    gc.collect()
    assert large.numel() >= 4096 and large.data_ptr() != at
    assert small() is not None and small().data_ptr() == at
    assert _lib.workspace(300, "cpu", "pages") is large


def test_outgrown_workspaces_stay_small(host):
    """Calls that each need a little more do not pile up buffers."""
    sizes = {}
    for n in range(256, 200000, 64):
        ws = _lib.workspace(n, "cpu", "plan")
        sizes[ws.data_ptr()] = ws.numel()
    assert ws.numel() < 2 * 200000
    assert sum(sizes.values()) < 2 * ws.numel()


def test_unread_error_outlives_growth(host):
    """What an earlier call reported raises on the next call, also when that call
    needs a larger workspace."""
    small = _lib.workspace(300, "cpu", "pages")
    _lib._sinks[small.data_ptr()]._view[0] = _lib.ST_NO_PAGES
    large = _lib.workspace(4096, "cpu", "pages")
    assert large is not small
    with pytest.raises(RuntimeError, match="free pages"):
        _lib.raise_if_failed(large)


@pytest.mark.parametrize("sizes", [(256, 256, 256, 256), (256, 700, 5000, 40000)])
def test_calls_of_threads_on_one_stream_stay_together(host, sizes):
    """A call is several launches over one workspace: those of another thread on the
    same stream do not come between."""
    launches = []

    def call(who, at, nbytes, stream):
        for step in ("plan", "move"):
            launches.append((who, step))
            time.sleep(0.002)
        return _lib.OK

    def work(who):
        for _ in range(8):
            _lib.run(call, torch.device("cpu"), "pages", sizes[who], who)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(launches) == 64 and len(_lib._workspaces) == 1
    for plan, move in zip(launches[::2], launches[1::2]):
        assert plan == (plan[0], "plan") and move == (plan[0], "move")
    assert len(set(map(id, _lib._sinks.values()))) == 1  # one lock, whatever was outgrown


def test_a_failed_call_gives_the_workspace_back(host, monkeypatch):
    def refuse(rc):
        raise ValueError("refused")

    monkeypatch.setattr(_lib, "check", refuse)
    for _ in range(2):
        with pytest.raises(ValueError, match="refused"):
            _lib.run(lambda *a: _lib.ERR_INVALID, torch.device("cpu"), "pages", 256)


def test_reading_the_status_loses_no_report(host):
    """A call of another thread does not report between the reading and the clearing."""
    reports, seen = [], []
    ws = _lib.workspace(256, "cpu", "pages")

    def call(at, nbytes, stream):
        _lib._sinks[at]._view[0] = _lib.ST_NO_PAGES
        ws.view(torch.int32)[0] |= _lib.ST_NO_PAGES
        reports.append(1)
        return _lib.OK

    def read(at, out, stream):
        out._obj.value = int(ws.view(torch.int32)[0])
        time.sleep(0.001)
        ws.view(torch.int32)[0] = 0
        return _lib.OK

    _lib.lib().adakv_read_status = read
    done = threading.Event()

    def report():
        while not done.is_set():
            try:
                _lib.run(call, torch.device("cpu"), "pages", 256)
            except RuntimeError:
                time.sleep(0.0002)

    t = threading.Thread(target=report)
    t.start()
    for _ in range(100):
        before = len(reports)
        seen.append(_lib.read_status(ws))
        if len(reports) == before:
            time.sleep(0.0005)
    done.set()
    t.join()
    seen.append(_lib.read_status(ws))
    # each report was read once: at most one between two readings, and none lost
    assert sum(b != 0 for b in seen) == len(reports) > 1
