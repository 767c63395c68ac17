"""Captures of the engines: what is left of an earlier engine is not destroyed while another one captures (a captured graph that goes
during a capture ends the process)."""
import contextlib
import gc
import threading
import weakref

import pytest
import torch

from p2pfl_amd.runtime import engine as E
from test_layers_federation import Dropping, adapted, engine


@pytest.mark.parametrize("factory", [adapted, Dropping])
@pytest.mark.parametrize("batched", [True, False])
def test_a_module_engine_goes_with_its_last_reference(batched, factory):
    eng = engine(factory, batched=batched)
    eng.evaluate()
    gone = weakref.ref(eng)
    on = gc.isenabled()
    gc.disable()
    try:
        del eng
        assert gone() is None                    # (no cycle that would wait for the collector)
    finally:
        if on:
            gc.enable()


class Node:
    pass


def test_nothing_is_collected_during_a_capture(monkeypatch):
    @contextlib.contextmanager
    def graph(g, **kw):
        assert kw == {"capture_error_mode": "thread_local"}
        yield
    monkeypatch.setattr(torch.cuda, "graph", graph)
    assert gc.isenabled()
    old, new = Node(), Node()
    old.self, new.self = old, new                # garbage of before and of during the capture
    old_ref, new_ref = weakref.ref(old), weakref.ref(new)
    del old
    with E.capture(None):
        assert old_ref() is None and not gc.isenabled()
        del new
        for _ in range(100000):
            [[]]
        assert new_ref() is not None
    assert gc.isenabled()
    with pytest.raises(RuntimeError, match="declined"):
        with E.capture(None):
            raise RuntimeError("declined")
    assert gc.isenabled()
    gc.disable()                                 # a caller who has it off keeps it off
    try:
        with E.capture(None):
            pass
        assert not gc.isenabled()
    finally:
        gc.enable()


def test_two_captures_at_once_hold_the_collector_until_both_are_done(monkeypatch):
    monkeypatch.setattr(torch.cuda, "graph", lambda g, **kw: contextlib.nullcontext())
    inside, leave = threading.Event(), threading.Event()

    def other():
        with E.capture(None):
            inside.set()
            leave.wait(30)
    t = threading.Thread(target=other)
    t.start()
    assert inside.wait(30)
    with E.capture(None):
        assert not gc.isenabled()
    assert not gc.isenabled()                    # the other one captures yet
    leave.set()
    t.join(30)
    assert gc.isenabled() and not t.is_alive()
