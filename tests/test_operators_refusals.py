"""What the language-model operators refuse: every argument is checked before the context is looked at, so nothing
here needs a GPU.  The pointers are never followed."""
import ctypes as C

import numpy as np
import pytest

from pssa_amd import _abi

P = 0x10000  # stands for a device array


def refused(fn, args, message):
    buf = C.create_string_buffer(512)
    rc = fn(*args, buf, C.sizeof(buf))
    assert rc in (_abi.EINVAL, _abi.EUNSUPPORTED) and message in buf.value.decode(), (rc, buf.value)


def changed(base, **change):
    return list({**base, **change}.values())


LOGPROBS = dict(ctx=None, logits=P, dtype=_abi.F32, rows=4, vocab=100, ld=100, targets=P, temperature=1.0, top_k=5,
                logprobs=P, entropy=P, top_ids=P, top_logprobs=P)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"logits": None}, "null buffer"), ({"dtype": 7}, "unknown dtype"), ({"rows": 0}, "positive"),
    ({"vocab": 0}, "positive"), ({"ld": 99}, "row stride"), ({"temperature": 0.0}, "temperature"),
    ({"temperature": float("nan")}, "temperature"), ({"temperature": float("inf")}, "temperature"),
    ({"top_k": 65}, "at most 64"), ({"top_ids": None}, "both of its outputs"), ({"targets": None}, "need targets"),
    ({"top_k": 0, "logprobs": None, "entropy": None}, "no output"), ({"logits": P + 2}, "misaligned"),
    ({"logits": P + 1, "dtype": _abi.BF16}, "misaligned"), ({"entropy": P + 2}, "misaligned"),
    ({"rows": 1 << 31, "vocab": 1 << 20, "ld": 1 << 20}, "too large"), ({"vocab": 1 << 25, "ld": 1 << 25}, "too large"),
    ({"rows": 1 << 20, "ld": 1 << 60}, "overflow")])
def test_token_logprobs_refuses(change, message):
    refused(_abi.lib().pssa_hip_token_logprobs_resident, changed(LOGPROBS, **change), message)


DISTILL = dict(ctx=None, logits=P, dtype=_abi.F32, rows=4, vocab=100, ld=100, ids=P, teacher=P, k=8, temperature=1.0,
               weights=None, losses=P, grad=P + 4096, ld_grad=100)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"ids": None}, "null buffer"), ({"losses": None}, "null buffer"), ({"k": 0}, "1..=1024"),
    ({"k": 1025}, "1..=1024"), ({"dtype": 2}, "unknown dtype"), ({"ld_grad": 99}, "row stride"),
    ({"temperature": -1.0}, "temperature"), ({"grad": P, "ld_grad": 101}, "in place"), ({"grad": P + 400}, "overlaps"),
    ({"grad": P - 400}, "overlaps"), ({"grad": P + 4098}, "misaligned"), ({"teacher": P + 1}, "misaligned"),
    ({"grad": None, "ld_grad": 0}, "null context"), ({"grad": P}, "null context")])
def test_distill_refuses(change, message):
    refused(_abi.lib().pssa_hip_distill_resident, changed(DISTILL, **change), message)


def test_batch_forms_refuse_null_lanes_and_python_forms_refuse_types():
    lib = _abi.lib()
    refused(lib.pssa_hip_batch_token_logprobs, [None, None, 1, 1.0, 0, None, None, None, None], "null lanes")
    refused(lib.pssa_hip_batch_distill, [None, None, None, 1, 1, 1.0, None, None, None], "null buffer")
    from pssa_amd.device import _dtype

    with pytest.raises(ValueError, match="f32"):
        _dtype("f64")
    assert np.uint32(_abi.NO_TOKEN) == 0xFFFFFFFF
