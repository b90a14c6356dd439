"""What the chunk operators refuse, before any launch (no GPU)."""

import numpy as np
import pytest

ONE = 0x1000  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def abi(built_library):
    from qwencore_b200 import abi as module

    return module


def refused(abi, name, good, changes):
    function = getattr(abi.lib, name)
    for index, value in changes:
        arguments = list(good)
        arguments[index] = value
        assert function(*arguments) == abi.CUDA_ERROR_INVALID_VALUE, (name, index, value)


def test_attention_chunk(abi):
    size = abi.lib.qwc_paged_attention_chunk_workspace_bytes()
    #       query gate keys values tables contexts begins ks vs out  ws  bytes tokens seqs blocks page pool stride scale stream
    good = [ONE, ONE, ONE, ONE, ONE, ONE, ONE, 0, 0, ONE, ONE, size, 4, 1, 8, 16, 9, 0, 0.0625, 0]
    refused(abi, "qwc_paged_attention_chunk_fp8", good, [
        (0, 0), (2, 0), (3, 0), (4, 0), (5, 0), (6, 0), (9, 0), (0, ONE + 8), (1, ONE + 8), (2, ONE + 4), (3, ONE + 4),
        (9, ONE + 8), (12, 0), (12, -1), (12, 65537), (13, 0), (13, 129), (14, 0), (14, 1 << 28), (15, 32), (15, 0),
        (16, 0), (16, 1 << 27), (17, 24 * 512 - 8), (17, 24 * 512 + 4), (18, 0.0), (18, float("nan")), (18, -1.0)])
    if size:
        refused(abi, "qwc_paged_attention_chunk_fp8", good, [(11, size - 1), (10, 0), (10, ONE + 8)])


def test_delta_chunk(abi):
    before = abi.get_shape()
    abi.configure(32, 64)
    size = abi.lib.qwc_delta_chunk_workspace_bytes(4, 2)
    #       state scales slots continues begins qkv alpha beta out cap tokens seqs gate stride weight eps ws bytes stream
    good = [ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, 3, 4, 2, ONE, 0, ONE, 1e-6, ONE, size, 0]
    try:
        refused(abi, "qwc_delta_chunk_int8", good, [
            (0, 0), (1, 0), (2, 0), (4, 0), (5, 0), (6, 0), (7, 0), (8, 0), (0, ONE + 4), (1, ONE + 4), (5, ONE + 2),
            (8, ONE + 2), (9, 1), (10, 0), (10, 65537), (11, 0), (11, 129), (12, 0), (14, 0), (12, ONE + 2),
            (13, 32 * 128 - 8), (13, 32 * 128 + 4), (15, 0.0), (15, float("inf"))])
        if size:
            refused(abi, "qwc_delta_chunk_int8", good, [(17, size - 1), (16, 0), (16, ONE + 8)])
    finally:
        abi.configure(*before)


def test_delta_prepare_chunk(abi):
    before = abi.get_shape()
    abi.configure(32, 64)
    width = (2 * 16 + 32) * 128 + 64
    #       mixed a b conv a_log dt history slots continues begins qkv alpha beta cap tokens seqs stride gate_stride stream
    good = [ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, 3, 4, 2, width, width, 0]
    try:
        refused(abi, "qwc_delta_prepare_chunk", good, [
            *[(i, 0) for i in (0, 1, 2, 3, 4, 5, 6, 7, 9, 10, 11, 12)], (0, ONE + 2), (3, ONE + 8), (10, ONE + 8), (13, 1),
            (14, 0), (14, 65537), (15, 0), (15, 129), (16, width - 65), (16, width + 4), (17, 31)])
    finally:
        abi.configure(*before)


def test_cache_copy(abi):
    def call(rows, pairs=ONE, count=1, arrays=None):
        table = np.array(rows, dtype=np.uint64)
        return abi.lib.qwc_cache_copy(table.ctypes.data, len(rows) if arrays is None else arrays, pairs, count, 0)

    good = (ONE, 64, 4)
    for bad in [(0, 64, 4), (ONE + 8, 64, 4), (ONE, 0, 4), (ONE, 24, 4), (ONE, 64, 0), (ONE, 64, 1 << 32),
                (ONE, 1 << 40, 4), (ONE, 1 << 20, 1 << 31)]:
        assert call([good, bad]) == abi.CUDA_ERROR_INVALID_VALUE, bad
    assert call([good], arrays=0) == abi.CUDA_ERROR_INVALID_VALUE
    assert call([good], pairs=0) == abi.CUDA_ERROR_INVALID_VALUE
    assert call([good], pairs=ONE + 4) == abi.CUDA_ERROR_INVALID_VALUE
    assert call([good], count=-1) == abi.CUDA_ERROR_INVALID_VALUE
    assert abi.lib.qwc_cache_copy(0, 1, ONE, 1, 0) == abi.CUDA_ERROR_INVALID_VALUE
    assert call([good], count=0) == 0 and call([good], pairs=0, count=0) == 0
