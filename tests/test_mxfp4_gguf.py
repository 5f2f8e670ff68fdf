"""MXFP4 tensors in a GGUF file (no GPU needed): their payload is 17 bytes for
every 32 values of a row and reads back; a row that no block divides has no
known size; a payload cut short is refused."""
from __future__ import annotations

import numpy as np
import pytest

import gguf_io as gi

MXFP4 = 39


def writer(raw, ne):
    w = gi.GgufWriter()
    w.tensors.append(("w", MXFP4, ne, raw.tobytes()))
    return w


@pytest.fixture(scope="module")
def lib(wx):
    return wx.load()


@pytest.mark.parametrize("ne", [(32,), (64, 3), (96, 2, 5), (32, 1, 2, 3)])
def test_payload_reads_back(lib, wx, tmp_path, ne):
    n = int(np.prod(ne)) // 32 * 17
    raw = np.random.default_rng(n).integers(0, 256, n, dtype=np.uint8)
    after = np.arange(5, dtype=np.float32)
    p = writer(raw, ne).tensor("x", after, gi.GGML_F32, (5,)).write(tmp_path / "w.gguf")
    g = lib.wamx_gguf_open(str(p).encode())
    assert g, wx.last_error()
    try:
        assert lib.wamx_gguf_tensor_type(g, 0) == MXFP4 and lib.wamx_gguf_tensor_bytes(g, 0) == n
        for i, a in enumerate((raw, after)):
            out = np.zeros_like(a)
            wx.check(lib.wamx_gguf_read_tensor(g, i, out.ctypes.data, out.nbytes))
            assert np.array_equal(out, a)
        assert lib.wamx_gguf_read_tensor(g, 0, out.ctypes.data, n - 17) != 0 and "bytes" in wx.last_error()
    finally:
        lib.wamx_gguf_close(g)


def test_rows_that_no_block_divides_have_no_size(lib, wx, tmp_path):
    p = writer(np.zeros(34, np.uint8), (33, 2)).write(tmp_path / "w.gguf")
    g = lib.wamx_gguf_open(str(p).encode())
    assert g, wx.last_error()
    try:
        out = np.zeros(34, np.uint8)
        assert lib.wamx_gguf_tensor_bytes(g, 0) == 0
        assert lib.wamx_gguf_read_tensor(g, 0, out.ctypes.data, 34) != 0 and "39" in wx.last_error()
    finally:
        lib.wamx_gguf_close(g)


def test_cut_payload_is_refused(lib, wx, tmp_path):
    p = writer(np.zeros(2 * 17, np.uint8), (32, 8)).write(tmp_path / "w.gguf")
    assert not lib.wamx_gguf_open(str(p).encode()) and "outside" in wx.last_error()
