"""The ops of the 16-bit cache refuse bad arguments, with the same text from C++ (CPU key) and at trace time (meta tensors),
and the C ABI names the field.  No device is touched."""
import ctypes

import numpy as np
import pytest
import torch

from pth_flash_attn_b200 import capi, kv16, ops

BF16, F16, F32, I32, I64, U8 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64, torch.uint8


def _tables_args(device):
    z = lambda n, t: torch.zeros(n, dtype=t, device=device)
    return dict(context_lens=z(3, I32), query_lens=z(3, I32), free_blocks=z(9, I32), block_table=z((4, 5), I32), seq_lens=z(3, I32),
                query_start_loc=z(4, I32), slot_mapping=z(7, I64), positions=z(7, I64), pages_taken=z(1, I32), block_size=16)


def _write_args(device):
    z = lambda n, t: torch.zeros(n, dtype=t, device=device)
    return dict(key=z((3, 2, 64), F32), value=z((3, 2, 64), F32), k_cache=z((4, 16, 2, 64), BF16), v_cache=z((4, 16, 2, 64), BF16),
                slot_mapping=z(3, I64))


def _decode_args(device):
    z = lambda n, t: torch.zeros(n, dtype=t, device=device)
    return dict(out=z((3, 8, 64), BF16), lse=z((3, 8), F32), q=z((3, 8, 64), BF16), k_cache=z((4, 16, 2, 64), BF16),
                v_cache=z((4, 16, 2, 64), BF16), block_table=z((3, 2), I32), seq_lens=z(3, I32), softmax_scale=0.5, workspace=z(1 << 10, U8),
                window=0)


def _cross_args(device):
    a = _decode_args(device)
    a.pop("window")
    a["context_lens"] = a.pop("seq_lens")[:2]
    workspace, scale = a.pop("workspace"), a.pop("softmax_scale")
    return dict(a, query_start_loc=torch.zeros(3, dtype=I32, device=device), max_query_len=2, softmax_scale=scale, workspace=workspace)


_ARGS = {"page_tables": _tables_args, "kv16_write": _write_args, "kv16_decode_attention": _decode_args, "kv16_cross_attention": _cross_args}


def _t(shape, dtype):
    return lambda device: torch.zeros(shape, dtype=dtype, device=device)


BAD = [
    ("page_tables", "context_lens", _t((3, 1), I32), "context_lens must be 1-D, got 2-D"),
    ("page_tables", "query_lens", _t(3, I64), "query_lens must be int32, got int64"),
    ("page_tables", "query_lens", _t(2, I32), r"query_lens.size\(0\) must equal num_reqs = 3, got 2"),
    ("page_tables", "block_table", _t((2, 5), I32), "block_table has 2 rows, fewer than num_reqs = 3"),
    ("page_tables", "query_start_loc", _t(3, I32), r"query_start_loc.size\(0\) must equal num_reqs \+ 1 = 4, got 3"),
    ("page_tables", "slot_mapping", _t(7, I32), "slot_mapping must be int64, got int32"),
    ("page_tables", "slot_mapping", lambda d: torch.zeros(14, dtype=I64, device=d)[::2], "slot_mapping must have stride 1"),
    ("page_tables", "positions", _t(6, I64), r"positions.size\(0\) must equal slot_mapping.size\(0\) = 7, got 6"),
    ("page_tables", "pages_taken", _t(2, I32), r"pages_taken.size\(0\) must equal 1 = 1, got 2"),
    ("page_tables", "block_size", lambda d: 0, "block_size must be >= 1, got 0"),
    ("kv16_write", "k_cache", _t((4, 16, 2, 64), F32), "k_cache must be bfloat16 or float16, got float32"),
    ("kv16_write", "v_cache", _t((4, 16, 2, 64), F16), r"v_cache \(same dtype as k_cache\) must be bfloat16, got float16"),
    ("kv16_write", "v_cache", _t((5, 16, 2, 64), BF16), r"v_cache.size\(0\) must equal NB = 4, got 5"),
    ("kv16_write", "k_cache", _t((4, 16, 2, 96), BF16), "must be 64, 128 or 256, got 96"),
    ("kv16_write", "k_cache", _t((0, 16, 2, 64), BF16), "k_cache must not be empty"),
    ("kv16_write", "key", _t((3, 2, 64), I32), "key must be float32, bfloat16 or float16, got int32"),
    ("kv16_write", "key", _t((3, 4, 64), F32), r"key.size\(1\) must equal Hkv = 2, got 4"),
    ("kv16_write", "value", _t((4, 2, 64), F32), r"value.size\(0\) must equal T = 3, got 4"),
    ("kv16_write", "key", lambda d: torch.zeros((3, 2, 128), device=d)[..., ::2], "key must have stride 1 in its last dimension, got 2"),
    ("kv16_write", "slot_mapping", _t(2, I64), r"slot_mapping.size\(0\) must equal T = 3, got 2"),
    ("kv16_decode_attention", "q", _t((3, 8, 64), F16), r"q \(same dtype as k_cache\) must be bfloat16, got float16"),
    ("kv16_decode_attention", "q", _t((3, 64), BF16), "q must be 3-D, got 2-D"),
    ("kv16_decode_attention", "out", _t((3, 8, 64), F32), r"out \(same dtype as q\) must be bfloat16, got float32"),
    ("kv16_decode_attention", "lse", _t((3, 7), F32), r"lse.size\(1\) must equal Hq = 8, got 7"),
    ("kv16_decode_attention", "lse", lambda d: torch.zeros((8, 3), device=d).t(), "lse must be contiguous"),
    ("kv16_decode_attention", "seq_lens", _t(2, I32), r"q.size\(0\) must equal num_reqs = 2, got 3"),
    ("kv16_decode_attention", "seq_lens", _t(3, I64), "seq_lens must be int32, got int64"),
    ("kv16_decode_attention", "block_table", _t((2, 2), I32), "block_table has 2 rows, fewer than num_reqs = 3"),
    ("kv16_decode_attention", "softmax_scale", lambda d: 0.0, "softmax_scale must be finite and > 0, got 0"),
    ("kv16_decode_attention", "softmax_scale", lambda d: float("nan"), "softmax_scale must be finite and > 0, got nan"),
    ("kv16_decode_attention", "workspace", _t(8, F32), "workspace must be uint8, got float32"),
    ("kv16_decode_attention", "window", lambda d: -1, "window must be >= 0, got -1"),
    ("kv16_cross_attention", "query_start_loc", _t(4, I32), r"query_start_loc.size\(0\) must equal num_reqs \+ 1 = 3, got 4"),
    ("kv16_cross_attention", "max_query_len", lambda d: 4, r"max_query_len must be in \[0, T = 3\], got 4"),
]


@pytest.mark.parametrize("device", ["cpu", "meta"])
@pytest.mark.parametrize("op,name,value,message", BAD)
def test_refusals(op, name, value, message, device):
    args = _ARGS[op](device)
    args[name] = value(device)
    with pytest.raises(RuntimeError, match=f"{op}: .*{message}"):
        getattr(ops, op)(*args.values())


@pytest.mark.parametrize("Hq,message", [(7, "Hq = 7 must be a positive multiple of Hkv = 2"), (130, "G = Hq/Hkv = 65 exceeds the supported maximum 64")])
@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_head_counts(Hq, message, device):
    args = _decode_args(device)
    args.update(q=torch.zeros((3, Hq, 64), dtype=BF16, device=device), out=torch.zeros((3, Hq, 64), dtype=BF16, device=device))
    with pytest.raises(RuntimeError, match=message):
        ops.kv16_decode_attention(*args.values())


@pytest.mark.parametrize("op", sorted(_ARGS))
def test_valid_calls(op):
    getattr(ops, op)(*_ARGS[op]("meta").values())      # traces
    with pytest.raises(RuntimeError, match=f"{op}: arguments are valid, but the op computes on CUDA tensors only"):
        getattr(ops, op)(*_ARGS[op]("cpu").values())


@pytest.mark.parametrize("op", sorted(_ARGS))
def test_schemas_are_the_registered_ones(op):
    registered = getattr(torch.ops.pth_flash_attn, op).default._schema
    declared = torch._C.parse_schema("pth_flash_attn::" + kv16.SCHEMAS[op])
    assert [(a.name, str(a.type)) for a in registered.arguments] == [(a.name, str(a.type)) for a in declared.arguments]
    assert [a.alias_info is not None for a in registered.arguments] == [a.alias_info is not None for a in declared.arguments]


# ---- C ABI -----------------------------------------------------------------------
@pytest.fixture(autouse=True)
def _leave_no_error_behind():
    yield
    capi.load_library().kv16_check(_kv16_args(False))


_BUF = np.zeros(1 << 16, dtype=np.uint8)
_BASE = (_BUF.ctypes.data + 255) & ~255


def _kv16_args(cross):
    a = capi.new_args(capi.PthB200Kv16Args)
    a.q, a.q_stride_token, a.q_stride_head = _BASE, 8 * 128, 128
    a.out, a.out_stride_token, a.out_stride_head = _BASE + 4096, 8 * 128, 128
    for s in (a.k_cache, a.v_cache):
        s.data, s.stride_block, s.stride_slot, s.stride_head = _BASE + 8192, 4096, 256, 128
    a.block_table, a.block_table_row_stride, a.seq_lens = _BASE + 256, 2, _BASE + 512
    a.workspace, a.workspace_bytes = _BASE, 1 << 10
    a.dtype, a.num_blocks, a.block_size, a.num_kv_heads, a.num_q_heads, a.head_size = capi.BF16, 4, 16, 2, 8, 64
    a.num_reqs = a.num_tokens = 3
    a.num_pages = 2
    a.max_query_len, a.softmax_scale = 1, 0.5
    if cross:
        a.query_start_loc = _BASE + 768
    return a


@pytest.mark.parametrize("cross", [False, True])
@pytest.mark.parametrize("field,value,message", [
    ("abi_version", 1, "abi_version"), ("struct_bytes", 8, "struct_bytes"), ("dtype", capi.F32, "dtype must be F16 or BF16"),
    ("head_size", 96, "head_size must be"), ("num_q_heads", 7, "num_q_heads must be a positive multiple"), ("num_q_heads", 130, "must be <= 64"),
    ("block_size", 0, "block_size"), ("num_blocks", 0, "num_blocks"), ("softmax_scale", float("inf"), "softmax_scale"), ("window", -1, "window"),
    ("q", None, "q is NULL"), ("q", _BASE + 8, "q must be 16-byte aligned"), ("out_stride_head", 8, "out byte strides"), ("lse", _BASE + 2, "lse must be"),
    ("block_table", None, "block_table"), ("workspace", _BASE + 16, "workspace"), ("num_tokens", -1, "num_tokens"),
    ("num_pages", -1, "num_pages must be >= 0")])
def test_c_abi_refusals(field, value, message, cross):
    lib = capi.load_library()
    a = _kv16_args(cross)
    assert lib.kv16_check(a) == capi.OK, lib.last_error()
    setattr(a, field, value)
    assert lib.kv16_check(a) == capi.EINVAL and message in lib.last_error()


@pytest.mark.parametrize("field,value,message", [("data", _BASE + 4, "k_cache.data must be 16-byte aligned"), ("stride_slot", 264, "multiples of 16"),
                                                 ("stride_block", 8192, "same strides"), ("data", None, "k_cache.data is NULL")])
def test_c_abi_cache_refusals(field, value, message):
    lib, a = capi.load_library(), _kv16_args(False)
    setattr(a.k_cache, field, value)
    assert lib.kv16_check(a) == capi.EINVAL and message in lib.last_error()


def test_c_abi_calls_have_their_own_forms():
    lib = capi.load_library()
    assert lib.kv16_decode(_kv16_args(True)) == capi.EINVAL and "query_start_loc must be NULL" in lib.last_error()
    assert lib.kv16_cross(_kv16_args(False)) == capi.EINVAL and "query_start_loc is NULL" in lib.last_error()
    a = _kv16_args(True)
    a.window = 5
    assert lib.kv16_check(a) == capi.EINVAL and "window must be 0" in lib.last_error()
    a = _kv16_args(False)
    a.num_tokens = 4
    assert lib.kv16_check(a) == capi.EINVAL and "num_tokens must equal num_reqs" in lib.last_error()
    a = _kv16_args(True)
    a.max_query_len = 4
    assert lib.kv16_check(a) == capi.EINVAL and "max_query_len" in lib.last_error()


@pytest.mark.parametrize("field,value,message", [("num_reqs", 16385, "num_reqs must be in"), ("num_tokens", -1, "num_tokens"), ("block_size", 0, "block_size"),
                                                 ("query_start_loc", None, "query_start_loc"), ("context_lens", None, "context_lens"),
                                                 ("free_blocks", None, "free_blocks is NULL"), ("slot_mapping", None, "slot_mapping is NULL"),
                                                 ("positions", _BASE + 4, "8-byte aligned"), ("block_table", None, "block_table is NULL")])
def test_c_abi_tables_refusals(field, value, message):
    lib, a = capi.load_library(), capi.new_args(capi.PthB200TablesArgs)
    for name in ("context_lens", "query_lens", "free_blocks", "block_table", "seq_lens", "query_start_loc", "slot_mapping", "positions", "pages_taken"):
        setattr(a, name, _BASE)
    a.num_reqs, a.num_tokens, a.num_free, a.num_pages, a.block_size, a.block_table_row_stride = 2, 3, 4, 5, 16, 5
    setattr(a, field, value)
    assert lib.page_tables(a) == capi.EINVAL and message in lib.last_error()


@pytest.mark.parametrize("field,value,message", [("head_size", 32, "head_size"), ("src_dtype", 5, "src_dtype"), ("cache_dtype", capi.F32, "cache_dtype"),
                                                 ("key", None, "key is NULL"), ("value", _BASE + 1, "value must be 2-byte aligned"),
                                                 ("slot_mapping", None, "slot_mapping"), ("num_tokens", -1, "num_tokens")])
def test_c_abi_write_refusals(field, value, message):
    lib, a = capi.load_library(), capi.new_args(capi.PthB200Kv16WriteArgs)
    a.key = a.value = a.slot_mapping = _BASE
    a.src_dtype = a.cache_dtype = capi.BF16
    for s in (a.k_cache, a.v_cache):
        s.data, s.stride_block, s.stride_slot, s.stride_head = _BASE + 8192, 4096, 256, 128
    a.num_blocks, a.block_size, a.num_kv_heads, a.head_size, a.num_tokens = 4, 16, 2, 64, 1
    setattr(a, field, value)
    assert lib.kv16_write(a) == capi.EINVAL and message in lib.last_error()


def test_struct_sizes():
    assert ctypes.sizeof(capi.PthB200Kv16Args) == capi.load_library().lib.pthb200_kv16_args_bytes()


def test_workspace_bytes():
    for D in (64, 128, 256):
        assert kv16.workspace_bytes(D=D, num_sms=148) <= 64 << 20
    with pytest.raises(ValueError):
        kv16.workspace_bytes(D=96, num_sms=148)
    with pytest.raises(ValueError):
        kv16.workspace_bytes(D=64, num_sms=0)
