"""The C-ABI library loads and exports every symbol the public header declares (no GPU needed)."""

import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "kfa.h")
LIB = os.path.join(ROOT, "kohakufa-cute_b200", "kohakufa_cute", "libkfa.so")


def declared_symbols():
    text = open(HEADER).read()
    return sorted(set(re.findall(r"KFA_API[^;(]*?\b(kfa_\w+)\s*\(", text)))


def test_header_declares_the_expected_entry_points():
    names = declared_symbols()
    for required in ("kfa_forward", "kfa_backward", "kfa_neighborhood_forward", "kfa_neighborhood_backward",
                     "kfa_center_keys", "kfa_merge_partial", "kfa_last_error"):
        assert required in names


@pytest.mark.skipif(not os.path.exists(LIB), reason="libkfa.so has not been built")
def test_library_exports_every_declared_symbol():
    lib = ctypes.CDLL(LIB)
    for name in declared_symbols():
        assert hasattr(lib, name), name
    lib.kfa_version.restype = ctypes.c_int
    assert lib.kfa_version() >= 1
    lib.kfa_last_error.restype = ctypes.c_char_p
    assert lib.kfa_last_error() == b""


@pytest.mark.skipif(not os.path.exists(LIB), reason="libkfa.so has not been built")
def test_python_binding_lists_every_declared_symbol():
    from kohakufa_cute import native

    assert sorted(native.SIGNATURES) == declared_symbols()
    native.library()


@pytest.mark.skipif(not os.path.exists(LIB), reason="libkfa.so has not been built")
def test_argument_errors_are_reported_without_a_gpu():
    from kohakufa_cute import native

    lib = native.library()
    record = native.KfaTensor()
    record.data = 16
    record.dtype = native.KFA_F32
    record.ndim = 4
    for i in range(4):
        record.sizes[i] = 2
        record.strides[i] = 1
    code = lib.kfa_forward(ctypes.byref(record), ctypes.byref(record), ctypes.byref(record), None, None, None, None,
                           None, 1.0, 0, None)
    assert code == 1
    assert b"FP16/BF16" in lib.kfa_last_error()


def test_records_packed_in_c_equal_those_packed_in_python():
    import torch

    from kohakufa_cute import native

    tensors = [torch.zeros(2, 3, 4, 8, dtype=t).transpose(1, 2) for t in native._DTYPES]
    tensors += [None, torch.zeros(5, dtype=torch.int32), torch.zeros(1, 2, 3, 4, 2, dtype=torch.float16)[:, 1:],
                torch.zeros(1, 2, 3, 4, 5, 6, dtype=torch.uint8), torch.zeros(3, dtype=torch.float64)]
    for pack in {native._packed_records, native._records}:
        buffer, addresses = pack(*tensors)
        assert len(addresses) == len(tensors)
        for address, t in zip(addresses, tensors):
            if t is None:
                assert address is None
                continue
            record = native.KfaTensor.from_address(address)
            assert record.data == t.data_ptr() and record.dtype == native._DTYPES.get(t.dtype, -1)
            assert record.ndim == t.dim()
            assert list(record.sizes) == list(t.shape) + [0] * (6 - t.dim())
            assert list(record.strides) == list(t.stride()) + [0] * (6 - t.dim())
        del buffer
    rows = torch.zeros(2, 3, 4, 16, dtype=torch.float16)
    for ok, t in ((True, rows), (True, rows.transpose(1, 2)), (False, rows[..., 1:9]), (False, rows[..., ::2]),
                  (True, rows[:, :, :1, :8]), (False, rows.expand(2, 3, 4, 16)[:1, :1, :1].expand(2, 3, 4, 16)),
                  (True, torch.zeros(1, 1, 1, 3, dtype=torch.float16))):
        assert native._rows_16_byte_addressable(t) is ok and native._all_rows_16_byte_addressable(t) is ok
        assert native._all_rows_16_byte_addressable(rows, t) is ok
    for bad in (3, object()):
        if native._fast_records is not None:
            with pytest.raises(AttributeError):
                native._fast_records.records(bad)
            with pytest.raises(AttributeError):
                native._fast_records.addressable(bad)
