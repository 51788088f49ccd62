"""What the operators of a serving step refuse (norms with 8-bit rows, 8-bit products, the gated delta rule, beam
search): every argument is checked before the context is looked at, so nothing here needs a GPU.  The pointers are never
followed."""
import ctypes as C

import numpy as np
import pytest

from pssa_amd import _abi

P = 0x100000  # stands for a device array


def refused(fn, args, message):
    buf = C.create_string_buffer(512)
    rc = fn(*args, buf, C.sizeof(buf))
    assert rc in (_abi.EINVAL, _abi.EUNSUPPORTED) and message in buf.value.decode(), (rc, buf.value)


def changed(base, **change):
    return list({**base, **change}.values())


NORM = dict(ctx=None, dtype=_abi.F32, x=P, ld_x=100, residual=P + 0x10000, ld_residual=100, gamma=P + 0x20000, eps=1e-5,
            rows=8, width=100, sum=P + 0x30000, ld_sum=100, out=P + 0x40000, ld_out=100, codes=P + 0x50000, ld_codes=100,
            scales=P + 0x60000)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"x": None}, "null buffer"), ({"gamma": None}, "null buffer"), ({"dtype": 2}, "unknown dtype"),
    ({"eps": 0.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"eps": 2.0}, "eps"), ({"rows": 0}, "positive"),
    ({"width": 0}, "positive"), ({"width": 65537, "ld_x": 65537}, "65536"), ({"ld_x": 99}, "row stride"),
    ({"ld_residual": 99}, "row stride"), ({"ld_codes": 99}, "row stride"), ({"ld_sum": 99}, "row stride"),
    ({"ld_out": 99}, "row stride"), ({"codes": None}, "together"), ({"scales": None}, "together"),
    ({"sum": None, "out": None, "codes": None, "scales": None}, "no output"), ({"x": P + 2}, "misaligned"),
    ({"gamma": P + 0x20002}, "misaligned"), ({"scales": P + 0x60002}, "misaligned"), ({"out": P + 0x40001, "dtype": 1}, "misaligned"),
    ({"codes": P + 0x50001}, "null context"), ({"residual": None, "ld_residual": 0}, "null context"),
    ({"rows": 1 << 32}, "too large"), ({"ld_x": 1 << 32}, "too large"),
    # In place: over an input with its stride; nothing else may touch one.
    ({"sum": P}, "null context"), ({"sum": P + 0x10000, "out": P}, "null context"), ({"sum": P, "out": P}, "outputs overlap"),
    ({"sum": P, "ld_sum": 101}, "overlaps an input"), ({"sum": P + 4}, "overlaps an input"), ({"codes": P}, "overlaps an input"),
    ({"out": P + 0x20000}, "overlaps an input"), ({"scales": P + 0x20000}, "overlaps an input"),
    ({"codes": P + 0x30000}, "outputs overlap"), ({"scales": P + 0x50000}, "outputs overlap"),
    # Other columns of the same rows are apart.
    ({"ld_x": 200, "sum": P + 400, "ld_sum": 200}, "null context"), ({"ld_x": 200, "sum": P + 396, "ld_sum": 200}, "overlaps an input")])
def test_rms_norm_refuses(change, message):
    refused(_abi.lib().pssa_hip_rms_norm_resident, changed(NORM, **change), message)


QUANT = dict(ctx=None, dtype=_abi.BF16, x=P, ld_x=64, rows=4, width=64, codes=P + 0x10000, ld_codes=64, scales=P + 0x20000)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"codes": None}, "null buffer"), ({"scales": None}, "null buffer"), ({"dtype": 9}, "unknown dtype"),
    ({"rows": 0}, "positive"), ({"width": 65537, "ld_x": 70000}, "65536"), ({"ld_codes": 63}, "row stride"),
    ({"x": P + 1}, "misaligned"), ({"codes": P + 8}, "overlap"), ({"scales": P + 0x10000}, "overlap"), ({"scales": P}, "overlap")])
def test_quantize_i8_refuses(change, message):
    refused(_abi.lib().pssa_hip_quantize_i8_resident, changed(QUANT, **change), message)


I8 = dict(ctx=None, x=P, ld_x=96, x_scales=P + 0x10000, w=P + 0x20000, ld_w=96, w_scales=P + 0x30000, m=4, n=50, k=96,
          y=P + 0x40000, y_dtype=_abi.F32, ld_y=50)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"x": None}, "null buffer"), ({"w_scales": None}, "null buffer"), ({"y": None}, "null buffer"),
    ({"y_dtype": 5}, "unknown dtype"), ({"m": 0}, "positive"), ({"n": 0}, "positive"), ({"k": 0}, "positive"),
    ({"k": 131072, "ld_x": 131072, "ld_w": 131072}, "131071"), ({"m": (1 << 20) + 1}, "too large"), ({"n": (1 << 24) + 1}, "too large"),
    ({"ld_x": 95}, "row stride"), ({"ld_w": 95}, "row stride"), ({"ld_y": 49}, "row stride"), ({"ld_w": 1 << 31}, "too large"),
    ({"y": P + 0x40002}, "misaligned"), ({"x_scales": P + 0x10001}, "misaligned"), ({"x": P + 1, "w": P + 0x20003}, "null context"),
    ({"y": P}, "overlaps"), ({"y": P + 0x20000 + 4796}, "overlaps"), ({"y": P + 0x10000}, "overlaps"), ({"y": P + 0x30000}, "overlaps")])
def test_matmul_i8_refuses(change, message):
    refused(_abi.lib().pssa_hip_matmul_i8_resident, changed(I8, **change), message)


def test_matmul_i8_reserve_refuses():
    fn = _abi.lib().pssa_hip_matmul_i8_reserve
    refused(fn, [None, 4, 4, 4], "null context")
    refused(fn, [None, 4, 0, 4], "positive")
    refused(fn, [None, 4, 4, 131072], "131071")


DELTA = dict(ctx=None, dtype=_abi.F32, q=P, ld_q=32, k=P + 0x10000, ld_k=32, v=P + 0x20000, ld_v=96, log_decay=P + 0x30000,
             beta=P + 0x38000, ld_gates=4, state_in=None, lens=None, n_seqs=2, seq_len=8, heads=4, key_heads=2, d_key=16,
             d_val=24, scale=1.0, out=P + 0x40000, ld_out=96, state_out=P + 0x50000)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"v": None}, "null buffer"), ({"beta": None}, "null buffer"), ({"log_decay": None}, "null buffer"),
    ({"dtype": 3}, "unknown dtype"), ({"heads": 0}, "positive"), ({"d_val": 0}, "positive"), ({"key_heads": 0}, "divide"),
    ({"key_heads": 3}, "divide"), ({"d_key": 129}, "128"), ({"d_val": 4097}, "4096"), ({"heads": 65536, "key_heads": 1}, "65535"),
    ({"n_seqs": 0}, "sequences"), ({"n_seqs": 65536}, "sequences"), ({"seq_len": 1 << 31}, "too many tokens"),
    ({"n_seqs": 60000, "seq_len": 1 << 20}, "too many tokens"), ({"n_seqs": 1, "seq_len": 1 << 30}, "too many tokens"), ({"ld_q": 31}, "row stride"), ({"ld_k": 31}, "row stride"),
    ({"ld_v": 95}, "row stride"), ({"ld_out": 95}, "row stride"), ({"ld_gates": 3}, "row stride"), ({"ld_k": 1 << 24}, "2^24"),
    ({"scale": float("nan")}, "scale"), ({"q": P + 2}, "misaligned"), ({"beta": P + 0x38002}, "misaligned"),
    ({"state_out": P + 0x50002}, "misaligned"), ({"out": P}, "overlaps its inputs"), ({"out": P + 0x30000}, "overlaps its inputs"),
    ({"out": P + 0x38000 + 200}, "overlaps its inputs"), ({"state_out": P + 0x40000}, "states"), ({"state_out": P + 0x30000}, "states"),
    ({"state_in": P + 0x50004}, "states"), ({"state_in": P + 0x50000}, "null context"), ({"state_in": P + 0x40000}, "states"),
    ({"seq_len": 0}, "null context"),
    # One row buffer of q | k | v | out: the columns are apart; one element less and they are not.
    ({"ld_q": 256, "k": P + 128, "ld_k": 256, "v": P + 256, "ld_v": 256, "out": P + 640, "ld_out": 256}, "null context"),
    ({"ld_q": 256, "k": P + 128, "ld_k": 256, "v": P + 256, "ld_v": 256, "out": P + 636, "ld_out": 256}, "overlaps its inputs"),
    # Gates side by side in one buffer, read by other workgroups while outputs are written.
    ({"beta": P + 0x30010, "ld_gates": 8}, "null context"), ({"beta": P + 0x30010, "ld_gates": 8, "out": P + 0x30100}, "overlaps its inputs")])
def test_delta_rule_refuses(change, message):
    refused(_abi.lib().pssa_hip_delta_rule_resident, changed(DELTA, **change), message)


def test_delta_rule_reserve_refuses():
    fn = _abi.lib().pssa_hip_delta_rule_reserve
    refused(fn, [None, 0, None, 2, 8, 4, 16, 24], "null context")
    refused(fn, [None, 5, None, 2, 8, 4, 16, 24], "unknown dtype")
    refused(fn, [None, 0, None, 2, 8, 4, 130, 24], "128")
    refused(fn, [None, 0, None, 0, 8, 4, 16, 24], "sequences")


BEAM = dict(ctx=None, logits=P, dtype=_abi.F32, groups=2, beams=4, vocab=100, ld=100, scores=P + 0x10000, last=P + 0x10100,
            eos=2, keep=4, parents=P + 0x10200, tokens=P + 0x10300, out_scores=P + 0x10400)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"logits": None}, "null buffer"), ({"scores": None}, "null buffer"), ({"tokens": None}, "null buffer"),
    ({"last": None}, "null context"), ({"dtype": 4}, "unknown dtype"), ({"groups": 0}, "positive"), ({"vocab": 0}, "positive"),
    ({"beams": 0}, "1..=64"), ({"beams": 65}, "1..=64"), ({"keep": 0}, "1..=64"), ({"keep": 65}, "1..=64"),
    ({"ld": 99}, "row stride"), ({"vocab": (1 << 24) + 1, "ld": 1 << 25}, "too large"), ({"groups": 1 << 40}, "too large"),
    ({"groups": 1 << 22}, "too large"), ({"logits": P + 2}, "misaligned"), ({"parents": P + 0x10202}, "misaligned"),
    ({"out_scores": P + 0x10000, "tokens": P + 0x10100}, "null context"), ({"out_scores": P + 0x10000, "keep": 3}, "overlaps an input"),
    ({"out_scores": P + 0x10004}, "overlaps an input"), ({"tokens": P + 0x10000}, "overlaps an input"),
    ({"parents": P + 0x10100}, "overlaps an input"), ({"parents": P}, "overlaps an input"), ({"tokens": P + 0x10200}, "outputs overlap")])
def test_beam_select_refuses(change, message):
    refused(_abi.lib().pssa_hip_beam_select_resident, changed(BEAM, **change), message)


GATHER = dict(ctx=None, src=P, ld_src=256, dst=P + 0x10000, ld_dst=256, row_bytes=256, groups=2, n_in=4, parents=P + 0x20000,
              n_out=8)


@pytest.mark.parametrize("change,message", [
    ({}, "null context"), ({"src": None}, "null buffer"), ({"row_bytes": 0}, "positive"), ({"groups": 0}, "positive"),
    ({"n_in": 0}, "1..=64"), ({"n_out": 65}, "1..=64"), ({"ld_src": 255}, "row stride"), ({"ld_dst": 255}, "row stride"),
    ({"parents": P + 0x20002}, "misaligned"), ({"dst": P}, "rows overlap"), ({"dst": P, "n_out": 4}, "null context"),
    ({"dst": P, "n_out": 4, "ld_dst": 260}, "rows overlap"), ({"dst": P + 0x700}, "rows overlap"),
    ({"parents": P + 0x10ffc}, "overlap the parents"), ({"ld_src": 1 << 60}, "too large"), ({"row_bytes": 1 << 39, "ld_src": 1 << 39, "ld_dst": 1 << 39}, "too large")])
def test_beam_gather_refuses(change, message):
    refused(_abi.lib().pssa_hip_beam_gather_resident, changed(GATHER, **change), message)


def test_beam_reserve_and_search_refuse():
    fn = _abi.lib().pssa_hip_beam_select_reserve
    refused(fn, [None, 2, 4, 100, 4], "null context")
    refused(fn, [None, 2, 65, 100, 4], "1..=64")
    ids, scores = np.empty(8, np.uint32), np.empty(4, np.float32)
    refused(_abi.lib().pssa_hip_beam_search, [None, 1, 4, 2, 2, _abi.ptr(ids, C.c_uint32), 8, _abi.ptr(scores), 4], "null argument")


@pytest.mark.parametrize("width", [1, 2, 16])
def test_norms_of_too_many_rows_refuse(width):
    """A workgroup steps up to 4096 rows on from its last one, in 31 bits."""
    most, far = 2 ** 31 - 4096, 1 << 44
    norm = dict(NORM, dtype=_abi.BF16, width=width, residual=None, ld_x=width, ld_sum=width, sum=far, out=None, codes=None,
                scales=None)
    quant = dict(QUANT, width=width, ld_x=width, ld_codes=width, codes=far, scales=2 * far)
    for fn, base in ((_abi.lib().pssa_hip_rms_norm_resident, norm), (_abi.lib().pssa_hip_quantize_i8_resident, quant)):
        base = dict(base, x=4 * far)
        refused(fn, changed(base, rows=most), "null context")
        for rows in (most + 1, 2 ** 31 - 2048, 2 ** 31 - 1):
            refused(fn, changed(base, rows=rows), "too large")


def test_launches_past_32_bits_refuse():
    """A thread moves a piece of a row or copies 16 bytes of it: what 2^32 threads would not hold is refused ahead."""
    most = 2 ** 32 - 256
    apart, place = dict(dst=1 << 50, n_in=2, n_out=2), dict(dst=P, n_in=17, n_out=17)
    for size, where, message in ((16 * most, apart, "null context"), (16 * (most + 1), apart, "too large"),
                                 (4 * (most - 1), apart, "null context"), (4 * (most + 1), apart, "too large"),
                                 (4 * most, place, "null context"), (4 * (most + 4), place, "too large"),
                                 (most - 1, apart, "null context"), (most + 1, apart, "too large")):
        base = dict(GATHER, parents=1 << 56, groups=1, row_bytes=size, ld_src=size, ld_dst=size)
        refused(_abi.lib().pssa_hip_beam_gather_resident, changed(base, **where), message)
    far = dict(I8, x=P + 1, w=1 << 50, y=1 << 55, m=100, k=131071, ld_x=131071, ld_w=131071, ld_y=1 << 24)
    most = (2 ** 32 - 256) // 8192 - 100  # channels, beside 100 rows
    for n, message in ((most, "null context"), (most + 1, "units of 16 bytes")):
        refused(_abi.lib().pssa_hip_matmul_i8_resident, changed(far, n=n, x_scales=1 << 57, w_scales=1 << 58), message)
    refused(_abi.lib().pssa_hip_matmul_i8_resident,
            changed(far, n=most + 1, k=131056, ld_x=131072, ld_w=131072, x=P, x_scales=1 << 57, w_scales=1 << 58), "null context")
    rows = dict(DELTA, dtype=_abi.BF16, q=1 << 50, k=1 << 51, v=1 << 52, out=1 << 53, log_decay=1 << 54, beta=1 << 55, state_out=None,
                heads=64, key_heads=1, d_key=16, d_val=4096, ld_q=16, ld_k=16, ld_v=64 * 4096, ld_out=64 * 4096, ld_gates=64, n_seqs=1)
    most = (2 ** 32 - 256) // (64 * 512)
    refused(_abi.lib().pssa_hip_delta_rule_resident, changed(rows, seq_len=most + 1), "null context")
    refused(_abi.lib().pssa_hip_delta_rule_resident, changed(rows, seq_len=most, v=(1 << 52) + 2), "null context")
    refused(_abi.lib().pssa_hip_delta_rule_resident, changed(rows, seq_len=most + 1, v=(1 << 52) + 2), "units of 16 bytes")
