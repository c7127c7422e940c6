"""Calls of the quantised decoder-layer operators that no launch has room for are refused as wrong arguments (status 1), in front
of anything on the device: the addresses are made up."""
import ctypes

import pytest

from test_quantized_host import FAKE, LINEAR, LOAD, PA, WRITE, _load, _run


@pytest.mark.parametrize("call,good,bad", [
    ("atbmi_linear_int8", LINEAR, dict(m=1, n=0x7fffff00, out_stride=0x7fffff00)),            # few tokens
    ("atbmi_linear_int8", LINEAR, dict(m=0x7fffff00, n=1000, k=16, out_stride=1000)),         # tiles, rows in 16-byte pieces
    ("atbmi_linear_int8", LINEAR, dict(m=0x7fffff00, n=1000, k=17, out_stride=1000)),         # tiles, any rows
    ("atbmi_reshape_and_cache_int4", WRITE, dict(tokens=1023, heads=1 << 20, ks=1 << 27, vs=1 << 27)),
    ("atbmi_reshape_and_cache_int4", WRITE, dict(tokens=1 << 30, heads=64, ks=1 << 13, vs=1 << 13)),
    ("atbmi_paged_cache_load_int4", LOAD, dict(d=256, reach=(1 << 26) - 1, rows=1 << 30, longest=1 << 30)),
])
def test_calls_past_a_launch_are_refused(binding, call, good, bad):
    lib = binding.kernels()
    assert getattr(lib, call)(*{**good, **bad}.values()) == 1
    assert b"one launch" in lib.atbmi_last_error()


def test_attention_past_a_launch_is_refused(binding):
    lib = binding.kernels()
    for bad in (dict(batch=1 << 24, maxBlocksPerSeq=1), dict(batch=1 << 20, numHeads=1 << 10, numKvHeads=1 << 5, maxBlocksPerSeq=1),
                dict(batch=1 << 21, numHeads=16, numKvHeads=16, maxBlocksPerSeq=300)):
        call = binding.AtbmiPaInt4Call(**{**PA, **bad})
        assert lib.atbmi_pa_int4_decode(ctypes.byref(call), FAKE, 1 << 62, None) == 1
        assert b"one launch" in lib.atbmi_last_error()


@pytest.mark.parametrize("call,good,bad", [
    ("atbmi_paged_cache_load_int4", LOAD, dict(reach=1 << 60)), ("atbmi_paged_cache_load_int4", LOAD, dict(reach=(1 << 60) + 3)),
    ("atbmi_paged_cache_load_int4", LOAD, dict(reach=1 << 26)), ("atbmi_reshape_and_cache_int4", WRITE, dict(tokens=1 << 31)),
    ("atbmi_reshape_and_cache_int4", WRITE, dict(tokens=(1 << 63) - 1, heads=64, ks=1 << 13, vs=1 << 13))])
def test_counts_whose_products_overflow_are_refused(binding, call, good, bad):
    lib = binding.kernels()
    assert getattr(lib, call)(*{**good, **bad}.values()) == 1


@pytest.mark.parametrize("change", [{4: [70000, 4], 5: [70000], 8: [70000]}, {4: [3, 1 << 25]}])
def test_load_operation_refuses_what_its_launch_would(binding, change):
    """In InferShape and Setup, not only when it is executed."""
    name, param, ins, outs, alias = _load(binding)
    assert _run(binding, (name, param, ins, outs, alias)) == ("S", "NO_ERROR")
    ins = [(t, change.get(i, shape)) for i, (t, shape) in enumerate(ins)]
    assert _run(binding, (name, param, ins, outs, alias)) == ("I", "ERROR_INVALID_TENSOR_DIM")
