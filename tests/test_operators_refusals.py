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


def codes_of(w, group, zeros):
    from pssa_amd import quantize_w4

    return quantize_w4(w, group, zeros)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 31, 32), (2, 64, 64), (5, 129, 128), (4, 200, 64)])
def test_w4_quantize_rounds_to_the_nearest_code(n, k, group, zeros):
    """Every weight is within half a step of the code it got (the zero point's rounding can push one end past the last
    code: another half step there)."""
    rng = np.random.default_rng(n * k)
    w = rng.normal(0, 1, (n, k)).astype(np.float32)
    w[0] = np.abs(w[0])  # a row on one side of zero
    codes, scales, zp = codes_of(w, group, zeros)
    assert codes.max() <= 15 and scales.shape == (n, -(-k // group))
    at = np.arange(k) // group
    z = zp[:, at].astype(np.float64) if zeros else 8.0
    back = (codes - z) * scales[:, at].astype(np.float64)
    assert np.all(np.abs(back - w) <= scales[:, at] * (1.0 if zeros else 0.5) * (1 + 1e-6))
    if not zeros:
        assert codes.min() >= 1  # symmetric: -7..7


def test_w4_quantize_zero_rows_and_refusals():
    codes, scales, _ = codes_of(np.zeros((2, 40), np.float32), 32, False)
    assert not scales.any() and np.all(codes == 8)
    codes, scales, zp = codes_of(np.zeros((2, 40), np.float32), 32, True)
    assert not scales.any() and np.all(codes == zp[0, 0])
    for bad, group in ((np.full((1, 4), np.nan, np.float32), 32), (np.ones((1, 4), np.float32), 48)):
        with pytest.raises(_abi.HipError):
            codes_of(bad, group, False)


W4 = dict(ctx=None, codes=P, scales=P, zeros=None, n=16, k=64, group=32)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"codes": None}, "null buffer"), ({"n": 0}, "positive"), ({"k": 0}, "positive"),
    ({"group": 16}, "32, 64 or 128"), ({"group": 0}, "32, 64 or 128"), ({"scales": P + 2}, "misaligned"),
    ({"n": 1 << 31}, "too large"), ({"n": 1 << 30, "k": 1}, "too large"), ({"k": 1 << 25}, "too large"), ({"n": 1 << 30, "k": 1 << 20}, "too large")])
def test_w4_load_refuses(change, message):
    out = C.c_void_p(1)
    refused(_abi.lib().pssa_hip_w4_load_resident, changed(W4, **change) + [C.byref(out)], message)
    assert not out.value


def test_w4_products_refuse_null_weights():
    refused(_abi.lib().pssa_hip_matvec_w4_resident, [None, P, 0, 1, 64, P, 16], "null weights")
    refused(_abi.lib().pssa_hip_matvec_w4, [None, None, 0, 1, None, 0], "null weights")
    refused(_abi.lib().pssa_hip_w4_load, [None, None, 0, None, 0, None, 1, 1, 32, C.byref(C.c_void_p())], "null buffer")


LINEAR = dict(ctx=None, dtype=_abi.F32, q=P, ld_q=64, k=P + 0x10000, ld_k=32, v=P + 0x20000, ld_v=48, decay=P,
              state_in=None, lens=None, n_seqs=2, seq_len=8, heads=4, kv_heads=2, d_key=16, d_val=24, scale=1.0,
              out=P + 0x30000, ld_out=96, state_out=P + 0x40000)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"v": None}, "null buffer"), ({"decay": None}, "null buffer"), ({"dtype": 3}, "unknown dtype"),
    ({"heads": 0}, "positive"), ({"d_val": 0}, "positive"), ({"kv_heads": 0}, "divide"), ({"kv_heads": 3}, "divide"),
    ({"d_key": 129}, "128"), ({"d_val": 4097}, "4096"), ({"heads": 65536, "kv_heads": 65536}, "65535"),
    ({"n_seqs": 0}, "sequences"), ({"n_seqs": 65536}, "sequences"), ({"seq_len": 1 << 31}, "too many tokens"),
    ({"n_seqs": 60000, "seq_len": 1 << 20}, "too many tokens"), ({"ld_q": 63}, "row stride"), ({"ld_out": 95}, "row stride"), ({"ld_k": 1 << 24}, "2^24"),
    ({"scale": float("inf")}, "scale"), ({"q": P + 2}, "misaligned"), ({"state_out": P + 0x40002}, "misaligned"),
    ({"out": P}, "overlaps"), ({"out": P + 0x10000 + 4, "ld_out": 96}, "overlaps"), ({"state_out": P + 0x30000}, "states"),
    ({"state_in": P + 0x40004}, "states"), ({"state_in": P + 0x40000}, "null context"), ({"seq_len": 0}, "null context"),
    # One row buffer of q | k | v | out: the columns are apart; one element less and they are not.
    ({"ld_q": 240, "k": P + 256, "ld_k": 240, "v": P + 384, "ld_v": 240, "out": P + 576, "ld_out": 240}, "null context"),
    ({"ld_q": 240, "k": P + 256, "ld_k": 240, "v": P + 384, "ld_v": 240, "out": P + 572, "ld_out": 240}, "overlaps"),
    ({"ld_q": 239, "k": P + 256, "ld_k": 239, "v": P + 384, "ld_v": 239, "out": P + 576, "ld_out": 239}, "overlaps")])
def test_linear_attention_refuses(change, message):
    refused(_abi.lib().pssa_hip_linear_attention_resident, changed(LINEAR, **change), message)


def test_linear_attention_reserve_and_lens_refuse():
    fn = _abi.lib().pssa_hip_linear_attention_reserve
    refused(fn, [None, 0, None, 2, 8, 4, 16, 24], "null context")
    refused(fn, [None, 5, None, 2, 8, 4, 16, 24], "unknown dtype")
    refused(fn, [None, 0, None, 2, 8, 4, 130, 24], "128")
    from pssa_amd.device import _lens

    assert list(_lens([3, 0, 5])) == [3, 0, 5]
    with pytest.raises(ValueError, match="negative"):
        _lens([3, -1])


@pytest.mark.parametrize("change,message", [
    ({"state_in": P + 0x30000}, "the output overlaps the states"), ({"state_in": P + 0x30000 + 15 * 384 + 380}, "overlaps the states"),
    ({"state_in": P + 0x30000 + 15 * 384 + 384}, "null context"), ({"state_in": P + 0x30000 - 12288}, "null context"),
    ({"state_in": P + 0x30000 - 12284}, "overlaps the states"),
    ({"decay": P + 0x30000 - 12}, "overlaps its inputs"), ({"decay": P + 0x30000 - 16}, "null context"),
    ({"decay": P + 0x40000 + 12284}, "states overlap"), ({"decay": P + 0x40000 + 12288}, "null context"),
    ({"decay": P + 0x30000, "seq_len": 0}, "null context")])
def test_linear_attention_refuses_outputs_over_what_it_still_reads(change, message):
    """Heads of a token are written while other workgroups read the entry states and the decays: 16 tokens of 384 bytes
    out, 2 x 4 states of 16 x 24 values (12288 bytes), 4 decays."""
    refused(_abi.lib().pssa_hip_linear_attention_resident, changed(LINEAR, **change), message)
