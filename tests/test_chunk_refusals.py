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


def test_wrappers_refuse_what_does_not_fit(abi):
    """Types and sizes are looked at before anything that needs a GPU."""
    import torch

    from qwencore_b200 import ops

    bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    zeros = lambda n, dtype: torch.zeros(n, dtype=dtype)  # noqa: E731

    def attention(**other):
        given = dict(query=zeros(2 * 6144, bf16), query_gate_projection=zeros(2 * 12288, bf16), key_cache=zeros(3 * 16384, torch.uint8),
                     value_cache=zeros(3 * 16384, torch.uint8), block_tables=zeros(4, i32), context_lengths=zeros(1, i32),
                     chunk_begins=zeros(2, i32), max_blocks_per_sequence=4, output=zeros(2 * 6144, bf16), tokens=2, sequences=1,
                     workspace=zeros(16, torch.uint8), page_size=16, num_blocks=3)
        ops.paged_attention_chunk(**{**given, **other})

    for other in (dict(query=zeros(2 * 6144 - 1, bf16)), dict(query=zeros(2 * 6144, torch.float16)), dict(output=zeros(2 * 6144, f32)),
                  dict(context_lengths=zeros(0, i32)), dict(chunk_begins=zeros(1, i32)), dict(block_tables=zeros(3, i32)),
                  dict(num_blocks=4), dict(query_gate_projection=zeros(2 * 12288 - 1, bf16)), dict(gate_stride=20000),
                  dict(query_gate_projection=zeros(2 * 12288, f32)), dict(key_scales=zeros(3, f32)), dict(value_scales=zeros(4, bf16))):
        with pytest.raises(AssertionError):
            attention(**other)

    before = abi.get_shape()
    abi.configure(32, 64)
    channels, width = 8192, 8192 + 4096 + 64

    def prepare(**other):
        given = dict(mixed=zeros(2 * width, bf16), a_offset=width - 64, b_offset=width - 32, conv_weight=zeros(channels * 4, bf16),
                     a_log=zeros(32, bf16), dt_bias=zeros(32, bf16), conv_state=zeros(2 * channels * 3, f32), state_slots=zeros(1, i32),
                     continues=None, chunk_begins=zeros(2, i32), qkv=zeros(2 * channels, bf16), alpha=zeros(64, f32),
                     beta=zeros(64, f32), state_capacity=2, tokens=2, sequences=1, mixed_stride=width)
        ops.delta_prepare_chunk(**{**given, **other})

    def delta(**other):
        given = dict(state=zeros(2 * 32 * 16384, torch.int8), state_scales=zeros(2 * 32 * 128, f32), state_slots=zeros(1, i32),
                     continues=zeros(1, i32), chunk_begins=zeros(2, i32), qkv=zeros(2 * channels, bf16), alpha=zeros(64, f32),
                     beta=zeros(64, f32), out=zeros(2 * 4096, bf16), state_capacity=2, tokens=2, sequences=1,
                     workspace=zeros(16, torch.uint8), gate=zeros(2 * 4096, bf16), norm_weight=zeros(128, bf16))
        ops.delta_chunk(**{**given, **other})

    try:
        for other in (dict(mixed=zeros(2 * width - 1, bf16)), dict(mixed=zeros(2 * width, f32)), dict(qkv=zeros(2 * channels - 1, bf16)),
                      dict(alpha=zeros(63, f32)), dict(beta=zeros(64, bf16)), dict(conv_state=zeros(2 * channels * 3, bf16)),
                      dict(state_capacity=3), dict(chunk_begins=zeros(1, i32)), dict(conv_weight=zeros(channels * 4, f32)),
                      dict(continues=zeros(0, i32))):
            with pytest.raises(AssertionError):
                prepare(**other)
        for other in (dict(state=zeros(2 * 32 * 16384, torch.uint8)), dict(state_capacity=3), dict(state_scales=zeros(8192, bf16)),
                      dict(qkv=zeros(2 * channels, f32)), dict(alpha=zeros(63, f32)), dict(out=zeros(2 * 4096, f32)),
                      dict(out=zeros(4096, bf16)), dict(gate=zeros(2 * 4096, f32)), dict(gate_offset=8), dict(gate_stride=4104),
                      dict(norm_weight=zeros(127, bf16)), dict(sequences=2)):
            with pytest.raises(AssertionError):
                delta(**other)
    finally:
        abi.configure(*before)

    with pytest.raises(AssertionError):
        ops.copy_table([zeros(7, f32)], 2)
    with pytest.raises(AssertionError):
        ops.copy_table([zeros((4, 4), f32).T], 2)
    with pytest.raises(AssertionError):
        ops.cache_copy(np.zeros((1, 3), dtype=np.int64), zeros(2, i32), 1)
    with pytest.raises(AssertionError):
        ops.cache_copy(np.zeros((1, 3), dtype=np.uint64), zeros(2, i32), 2)


def test_wrappers_refuse_other_types(abi):
    """Lists of anything but 32 bits would be read behind their ends or misread, weights of another type misread."""
    import torch

    from qwencore_b200 import ops

    bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    zeros = lambda n, dtype: torch.zeros(n, dtype=dtype)  # noqa: E731
    before = abi.get_shape()
    abi.configure(32, 64)
    channels, width = 8192, 8192 + 4096 + 64

    def attention(**other):
        given = dict(query=zeros(2 * 6144, bf16), query_gate_projection=zeros(2 * 12288, bf16), key_cache=zeros(3 * 16384, torch.uint8),
                     value_cache=zeros(3 * 16384, torch.uint8), block_tables=zeros(4, i32), context_lengths=zeros(1, i32),
                     chunk_begins=zeros(2, i32), max_blocks_per_sequence=4, output=zeros(2 * 6144, bf16), tokens=2, sequences=1,
                     workspace=zeros(16, torch.uint8), page_size=16, num_blocks=3)
        ops.paged_attention_chunk(**{**given, **other})

    def prepare(**other):
        given = dict(mixed=zeros(2 * width, bf16), a_offset=width - 64, b_offset=width - 32, conv_weight=zeros(channels * 4, bf16),
                     a_log=zeros(32, bf16), dt_bias=zeros(32, bf16), conv_state=zeros(2 * channels * 3, f32), state_slots=zeros(1, i32),
                     continues=zeros(1, i32), chunk_begins=zeros(2, i32), qkv=zeros(2 * channels, bf16), alpha=zeros(64, f32),
                     beta=zeros(64, f32), state_capacity=2, tokens=2, sequences=1, mixed_stride=width)
        ops.delta_prepare_chunk(**{**given, **other})

    def delta(**other):
        given = dict(state=zeros(2 * 32 * 16384, torch.int8), state_scales=zeros(2 * 32 * 128, f32), state_slots=zeros(1, i32),
                     continues=zeros(1, i32), chunk_begins=zeros(2, i32), qkv=zeros(2 * channels, bf16), alpha=zeros(64, f32),
                     beta=zeros(64, f32), out=zeros(2 * 4096, bf16), state_capacity=2, tokens=2, sequences=1,
                     workspace=zeros(16, torch.uint8), gate=zeros(2 * 4096, bf16), norm_weight=zeros(128, bf16))
        ops.delta_chunk(**{**given, **other})

    lists = {attention: dict(block_tables=4, context_lengths=1, chunk_begins=2),
             prepare: dict(state_slots=1, continues=1, chunk_begins=2), delta: dict(state_slots=1, continues=1, chunk_begins=2)}
    try:
        for call, names in lists.items():
            for name, count in names.items():
                for dtype in (torch.int64, torch.bool, torch.uint8, torch.int16, f32):
                    with pytest.raises(AssertionError):
                        call(**{name: zeros(2 * count, dtype)})
        for dtype in (torch.int64, f32):
            with pytest.raises(AssertionError):
                ops.cache_copy(np.zeros((1, 3), dtype=np.uint64), zeros(4, dtype), 1)
        for other in (dict(key_cache=zeros(3 * 16384, bf16)), dict(value_cache=zeros(3 * 16384, torch.float8_e5m2)),
                      dict(value_cache=zeros(3 * 16384, f32))):
            with pytest.raises(AssertionError):
                attention(**other)
        for other in (dict(a_log=zeros(32, f32)), dict(a_log=zeros(31, bf16)), dict(dt_bias=zeros(32, f32)),
                      dict(dt_bias=zeros(31, bf16)), dict(a_offset=-8), dict(b_offset=-8)):
            with pytest.raises(AssertionError):
                prepare(**other)
        for other in (dict(norm_weight=zeros(128, f32)), dict(norm_weight=zeros(128, torch.float16)), dict(gate_offset=-8)):
            with pytest.raises(AssertionError):
                delta(**other)
    finally:
        abi.configure(*before)


def test_copy_table_refuses_memory_of_the_host(built_library):
    import torch

    from qwencore_b200 import ops

    with pytest.raises(AssertionError):
        ops.copy_table([torch.zeros((4, 16))], 4)
