"""The order in which native objects are freed, with a library that only writes the calls down: everything on a context
goes before the context, whatever order the garbage collector or the interpreter's end takes them in."""
import ctypes as C
import gc
import itertools

import numpy as np
import pytest

from pssa_amd import HipDevice, ModelWeights, PSSAConfig, PSSALayer, _abi


class Calls:
    """Stands for the loaded library: entry points succeed, handles are whole numbers."""

    def __init__(self):
        self.log, self.next = [], itertools.count(0x1000, 0x10)

    def __getattr__(self, name):
        def call(*args):
            self.log.append((name, args[0].value if hasattr(args[0], "value") else args[0]))
            for a in args:  # output handles are passed by reference, still empty
                out = getattr(a, "_obj", None)
                if isinstance(out, C.c_void_p) and not out.value:
                    out.value = next(self.next)
            return _abi.OK

        return call

    def freed(self):
        return [name for name, _ in self.log if name.endswith("_free") or name == "pssa_hip_destroy"]


def make(monkeypatch):
    cfg = PSSAConfig(depth=1, d_vocab=20, d_latent=16, d_state=8, d_mem_key=8, mem_capacity=10)
    weights = ModelWeights.init(cfg, 1, "baseline")
    calls = Calls()
    monkeypatch.setattr(_abi, "lib", lambda: calls)
    dev = HipDevice(0)
    layer = PSSALayer(dev, weights, lanes=1)
    buf = dev.empty((4,), np.float32)
    mat = dev.w4_matrix(np.zeros((2, 32), np.uint8), np.ones((2, 1), np.float32), 32)
    return calls, dev, layer, buf, mat


EVERYTHING = ["pssa_hip_device_free", "pssa_hip_lanes_free", "pssa_hip_model_free", "pssa_hip_w4_free"]


@pytest.mark.parametrize("order", list(itertools.permutations(range(4))))
def test_the_context_goes_last_in_any_order(monkeypatch, order):
    calls, *made = make(monkeypatch)
    made[0]._children.clear()  # as weak references are when a whole ring goes
    for i in order:
        made[i].__del__()
    assert calls.freed()[-1] == "pssa_hip_destroy" and sorted(calls.freed()[:-1]) == EVERYTHING
    assert calls.freed().index("pssa_hip_lanes_free") < calls.freed().index("pssa_hip_model_free")
    made.clear()
    gc.collect()
    assert len(calls.freed()) == 5  # nothing twice


def test_garbage_collection_of_a_ring(monkeypatch):
    calls, dev, layer, buf, mat = make(monkeypatch)
    dev.ring = [dev, layer, buf, mat]
    del dev, layer, buf, mat
    gc.collect()
    assert calls.freed()[-1] == "pssa_hip_destroy" and sorted(calls.freed()[:-1]) == EVERYTHING


def test_closing_the_device_closes_what_is_on_it(monkeypatch):
    calls, dev, layer, buf, mat = make(monkeypatch)
    mat.close()
    mat.close()
    dev.close()
    assert dev.handle is None and layer.handle is None and layer.model is None and buf.ptr is None and mat.handle is None
    assert calls.freed()[0] == "pssa_hip_w4_free" and calls.freed()[-1] == "pssa_hip_destroy"
    assert sorted(calls.freed()[:-1]) == EVERYTHING
    del dev, layer, buf, mat
    gc.collect()
    assert len(calls.freed()) == 5
