"""Argument checks of the 8-bit cache's operators and of rotary positions, through the ops, their fake kernels and the C ABI; and
the frequencies.  No device is touched."""
import ctypes
import math

import numpy as np
import pytest
import torch

from pth_flash_attn_b200 import capi, kv8, ops

F32, F64, BF16, F16, I32, I64, U8, F8 = (torch.float32, torch.float64, torch.bfloat16, torch.float16, torch.int32, torch.int64, torch.uint8,
                                         torch.float8_e4m3fn)


def _cache(device):
    z = lambda n, t: torch.zeros(n, dtype=t, device=device)
    return dict(k_cache=z((4, 32, 2, 64), F8), v_cache=z((4, 32, 2, 64), F8), k_scale=z((4, 2, 2), F32), v_scale=z((4, 2, 2), F32))


def _rotary_args(device):
    z = lambda n, t: torch.zeros(n, dtype=t, device=device)
    return dict(q_out=z((3, 4, 64), BF16), k_out=z((3, 2, 64), BF16), q=z((3, 4, 64), BF16), k=z((3, 2, 64), BF16), positions=z(3, I64),
                frequencies=z(32, F64), scale=1.0, interleaved=False, inverse=False)


def _write_args(device):
    z = lambda n, t: torch.zeros(n, dtype=t, device=device)
    return dict(key=z((3, 2, 64), F32), value=z((3, 2, 64), F32), **_cache(device), block_table=z((2, 3), I32), seq_lens=z(2, I32),
                query_start_loc=z(3, I32), max_query_len=2)


def _read_args(device):
    a = _write_args(device)
    return dict(key=a["key"], value=a["value"], **_cache(device), block_table=a["block_table"], first=a["seq_lens"],
                row_start_loc=a["query_start_loc"], max_rows=2)


def _decode_args(device):
    z = lambda n, t: torch.zeros(n, dtype=t, device=device)
    return dict(out=z((3, 8, 64), BF16), lse=z((3, 8), F32), q=z((3, 8, 64), BF16), **_cache(device), block_table=z((3, 2), I32), seq_lens=z(3, I32),
                softmax_scale=0.5, workspace=z(1 << 10, U8), window=0)


def _attend_args(device):
    a = _decode_args(device)
    tail = {n: a.pop(n) for n in ("softmax_scale", "workspace", "window")}
    a["seq_lens"] = a["seq_lens"][:2]
    return dict(a, query_start_loc=torch.zeros(3, dtype=I32, device=device), max_query_len=2, **tail, causal=True)


_ARGS = {"rotary": _rotary_args, "kv8_write": _write_args, "kv8_read": _read_args, "kv8_decode_attention": _decode_args,
         "kv8_attention": _attend_args}


def _t(shape, dtype):
    return lambda device: torch.zeros(shape, dtype=dtype, device=device)


_CACHE_BAD = [
    ("k_cache", _t((4, 32, 2, 64), U8), "k_cache must be float8_e4m3fn, got uint8"),
    ("v_cache", _t((4, 32, 2, 64), BF16), "v_cache must be float8_e4m3fn, got bfloat16"),
    ("k_scale", _t((4, 2, 2), F64), "k_scale must be float32, got float64"),
    ("k_cache", _t((4, 32, 2, 96), F8), "must be 64, 128 or 256, got 96"),
    ("k_cache", _t((0, 32, 2, 64), F8), "k_cache must not be empty"),
    ("v_cache", _t((4, 16, 2, 64), F8), r"v_cache.size\(1\) must equal BS = 32, got 16"),
    ("k_scale", _t((4, 4, 2), F32), "the tokens of a scale, must be a multiple of 16, got 32 / 4"),
    ("k_scale", _t((4, 0, 2), F32), "the tokens of a scale, must be a multiple of 16, got 32 / 0"),
    ("v_scale", _t((4, 1, 2), F32), r"v_scale.size\(1\) must equal k_scale.size\(1\) = 2, got 1"),
    ("v_scale", _t((4, 2, 3), F32), r"v_scale.size\(2\) must equal Hkv = 2, got 3"),
    ("k_scale", _t((4, 2), F32), "k_scale must be 3-D, got 2-D"),
]
BAD = [(op, *bad) for op in _ARGS if op != "rotary" for bad in _CACHE_BAD] + [
    ("kv8_write", "key", _t((3, 2, 64), I32), "key must be float32, bfloat16 or float16, got int32"),
    ("kv8_write", "key", _t((3, 4, 64), F32), r"key.size\(1\) must equal Hkv = 2, got 4"),
    ("kv8_write", "value", _t((4, 2, 64), F32), r"value.size\(0\) must equal T = 3, got 4"),
    ("kv8_write", "value", _t((3, 2, 64), F16), r"value \(same dtype as key\) must be float32, got float16"),
    ("kv8_write", "key", lambda d: torch.zeros((3, 2, 128), device=d)[..., ::2], "key must have stride 1 in its last dimension, got 2"),
    ("kv8_write", "block_table", _t((1, 3), I32), "block_table has 1 rows, fewer than num_reqs = 2"),
    ("kv8_write", "seq_lens", _t(2, I64), "seq_lens must be int32, got int64"),
    ("kv8_write", "query_start_loc", _t(4, I32), r"query_start_loc.size\(0\) must equal num_reqs \+ 1 = 3, got 4"),
    ("kv8_write", "max_query_len", lambda d: 4, r"max_query_len must be in \[0, T = 3\], got 4"),
    ("kv8_read", "first", _t(2, F32), "first must be int32, got float32"),
    ("kv8_read", "row_start_loc", _t(2, I32), r"row_start_loc.size\(0\) must equal num_reqs \+ 1 = 3, got 2"),
    ("kv8_read", "max_rows", lambda d: -1, r"max_rows must be in \[0, T = 3\], got -1"),
    ("kv8_decode_attention", "q", _t((3, 8, 64), F32), "q must be bfloat16 or float16, got float32"),
    ("kv8_decode_attention", "out", _t((3, 8, 64), F16), r"out \(same dtype as q\) must be bfloat16, got float16"),
    ("kv8_decode_attention", "lse", lambda d: torch.zeros((8, 3), device=d).t(), "lse must be contiguous"),
    ("kv8_decode_attention", "seq_lens", _t(2, I32), r"q.size\(0\) must equal num_reqs = 2, got 3"),
    ("kv8_decode_attention", "softmax_scale", lambda d: float("nan"), "softmax_scale must be finite and > 0, got nan"),
    ("kv8_decode_attention", "window", lambda d: -1, "window must be >= 0, got -1"),
    ("kv8_decode_attention", "workspace", _t(8, F32), "workspace must be uint8, got float32"),
    ("kv8_attention", "query_start_loc", _t(4, I32), r"query_start_loc.size\(0\) must equal num_reqs \+ 1 = 3, got 4"),
    ("kv8_attention", "max_query_len", lambda d: 4, r"max_query_len must be in \[0, T = 3\], got 4"),
    ("rotary", "q", _t((3, 4, 64), F64), "q must be float32, bfloat16 or float16, got float64"),
    ("rotary", "k", _t((3, 2, 64), F16), r"k \(same dtype as q\) must be bfloat16, got float16"),
    ("rotary", "k", _t((3, 2, 32), BF16), r"k.size\(2\) must equal D = 64, got 32"),
    ("rotary", "q_out", _t((3, 3, 64), BF16), r"q_out.size\(1\) must equal q.size\(1\) = 4, got 3"),
    ("rotary", "k_out", _t((3, 2, 64), F32), r"k_out \(same dtype as q\) must be bfloat16, got float32"),
    ("rotary", "positions", _t(3, I32), "positions must be int64, got int32"),
    ("rotary", "positions", _t(2, I64), r"positions.size\(0\) must equal T = 3, got 2"),
    ("rotary", "frequencies", _t(33, F64), r"frequencies.size\(0\) must be in \[1, D / 2 = 32\], got 33"),
    ("rotary", "frequencies", _t(0, F64), r"frequencies.size\(0\) must be in \[1, D / 2 = 32\], got 0"),
    ("rotary", "frequencies", _t(32, BF16), "frequencies must be float64 or float32, got bfloat16"),
    ("rotary", "scale", lambda d: float("inf"), "scale must be finite, got inf"),
    ("rotary", "k_out", lambda d: torch.zeros((3, 1, 64), dtype=BF16, device=d).expand(3, 2, 64), "k_out is written and must not have stride 0, as in dimension 1"),
    ("kv8_write", "k_cache", lambda d: torch.zeros((1, 32, 2, 64), dtype=F8, device=d).expand(4, 32, 2, 64), "k_cache is written and must not have stride 0"),
    ("kv8_write", "v_scale", lambda d: torch.zeros((4, 2, 1), device=d).expand(4, 2, 2), "v_scale is written and must not have stride 0, as in dimension 2"),
    ("kv8_read", "value", lambda d: torch.zeros((1, 2, 64), device=d).expand(3, 2, 64), "value is written and must not have stride 0, as in dimension 0"),
    ("kv8_decode_attention", "out", lambda d: torch.zeros((3, 1, 64), dtype=BF16, device=d).expand(3, 8, 64), "out is written and must not have stride 0"),
]


@pytest.mark.parametrize("device", ["cpu", "meta"])
@pytest.mark.parametrize("op,name,value,message", BAD)
def test_refusals(op, name, value, message, device):
    args = _ARGS[op](device)
    args[name] = value(device)
    with pytest.raises(RuntimeError, match=f"{op}: .*{message}"):
        getattr(ops, op)(*args.values())


def test_rotary_in_place_needs_the_same_strides():
    args = _rotary_args("cpu")
    args["q_out"] = args["q"].view(-1).as_strided((3, 4, 64), (64, 192, 1))
    with pytest.raises(RuntimeError, match="rotary: q_out in the place of q must have its strides"):
        ops.rotary(*args.values())


@pytest.mark.parametrize("Hq,message", [(7, "Hq = 7 must be a positive multiple of Hkv = 2"), (130, "G = Hq/Hkv = 65 exceeds the supported maximum 64")])
@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_head_counts(Hq, message, device):
    args = _decode_args(device)
    args.update(q=torch.zeros((3, Hq, 64), dtype=BF16, device=device), out=torch.zeros((3, Hq, 64), dtype=BF16, device=device))
    with pytest.raises(RuntimeError, match=message):
        ops.kv8_decode_attention(*args.values())


@pytest.mark.parametrize("op", sorted(_ARGS))
def test_valid_calls(op):
    getattr(ops, op)(*_ARGS[op]("meta").values())      # traces
    with pytest.raises(RuntimeError, match=f"{op}: arguments are valid, but the op computes on CUDA tensors only"):
        getattr(ops, op)(*_ARGS[op]("cpu").values())


@pytest.mark.parametrize("op", sorted(_ARGS))
def test_schemas_are_the_registered_ones(op):
    registered = getattr(torch.ops.pth_flash_attn, op).default._schema
    declared = torch._C.parse_schema("pth_flash_attn::" + kv8.SCHEMAS[op])
    assert [(a.name, str(a.type), a.default_value) for a in registered.arguments] == \
        [(a.name, str(a.type), a.default_value) for a in declared.arguments]
    assert [a.alias_info is not None for a in registered.arguments] == [a.alias_info is not None for a in declared.arguments]


# ---- C ABI -----------------------------------------------------------------------
@pytest.fixture(autouse=True)
def _leave_no_error_behind():
    yield
    capi.load_library().kv8_check(_kv8_args(False))


_BUF = np.zeros(1 << 16, dtype=np.uint8)
_BASE = (_BUF.ctypes.data + 255) & ~255


def _fill_cache(a):
    for s in (a.k_cache, a.v_cache):
        s.data, s.stride_block, s.stride_slot, s.stride_head = _BASE + 8192, 4096, 128, 64
    for s in (a.k_scale, a.v_scale):
        s.data, s.stride_block, s.stride_slot, s.stride_head = _BASE + 4096, 16, 8, 4
    a.block_table, a.block_table_row_stride = _BASE + 256, 2
    a.num_blocks, a.block_size, a.scale_tokens, a.num_kv_heads, a.head_size, a.num_pages = 4, 32, 16, 2, 64, 2
    return a


def _kv8_args(attend):
    a = _fill_cache(capi.new_args(capi.PthB200Kv8Args))
    a.q, a.q_stride_token, a.q_stride_head = _BASE, 8 * 128, 128
    a.out, a.out_stride_token, a.out_stride_head = _BASE + 4096, 8 * 128, 128
    a.seq_lens = _BASE + 512
    a.workspace, a.workspace_bytes = _BASE, 1 << 10
    a.dtype, a.num_q_heads = capi.BF16, 8
    a.num_reqs = a.num_tokens = 3
    a.max_query_len, a.softmax_scale, a.causal = 1, 0.5, 1
    if attend:
        a.query_start_loc = _BASE + 768
    return a


def _write_struct():
    a = _fill_cache(capi.new_args(capi.PthB200Kv8WriteArgs))
    a.key = a.value = a.seq_lens = a.query_start_loc = _BASE
    a.src_dtype, a.num_reqs, a.num_tokens, a.max_query_len = capi.BF16, 1, 2, 2
    return a


def _read_struct():
    a = _fill_cache(capi.new_args(capi.PthB200Kv8ReadArgs))
    a.key = a.value = a.first = a.row_start_loc = _BASE
    a.dst_dtype, a.num_reqs, a.num_rows, a.max_rows = capi.BF16, 1, 2, 2
    return a


def _rotary_struct():
    a = capi.new_args(capi.PthB200RotaryArgs)
    a.q = a.k = a.q_out = a.k_out = a.positions = a.frequencies = _BASE
    a.dtype, a.num_tokens, a.num_q_heads, a.num_k_heads, a.head_size, a.num_frequencies, a.scale = capi.BF16, 1, 2, 1, 64, 32, 1.0
    return a


_SHAPE_BAD = [
    ("abi_version", 1, "abi_version"), ("struct_bytes", 8, "struct_bytes"), ("head_size", 96, "head_size must be"), ("block_size", 0, "block_size"),
    ("num_blocks", 0, "num_blocks"), ("num_kv_heads", 0, "num_kv_heads"), ("num_kv_heads", 1 << 17, "num_kv_heads must be <= 65536"), ("scale_tokens", 24, "scale_tokens must be a multiple of 16"),
    ("scale_tokens", 48, "that divides block_size"), ("scale_tokens", 0, "scale_tokens"), ("num_pages", -1, "num_pages"), ("num_reqs", -1, "num_reqs"),
    ("block_table", None, "block_table is NULL")]


@pytest.mark.parametrize("attend", [False, True])
@pytest.mark.parametrize("field,value,message", _SHAPE_BAD + [
    ("dtype", capi.F32, "dtype must be F16 or BF16"), ("num_q_heads", 7, "num_q_heads must be a positive multiple"), ("num_q_heads", 130, "must be <= 64"),
    ("softmax_scale", float("inf"), "softmax_scale"), ("window", -1, "window"), ("q", None, "q is NULL"), ("q", _BASE + 8, "q must be 16-byte aligned"),
    ("out_stride_head", 8, "out byte strides"), ("lse", _BASE + 2, "lse must be"), ("workspace", _BASE + 16, "workspace"), ("num_tokens", -1, "num_tokens"),
    ("seq_lens", None, "seq_lens is NULL")])
def test_c_abi_refusals(field, value, message, attend):
    lib = capi.load_library()
    a = _kv8_args(attend)
    assert lib.kv8_check(a) == capi.OK, lib.last_error()
    setattr(a, field, value)
    assert lib.kv8_check(a) == capi.EINVAL and message in lib.last_error()


@pytest.mark.parametrize("stream,field,value,message", [
    ("k_cache", "data", _BASE + 8, "k_cache.data must be 16-byte aligned"), ("k_cache", "stride_slot", 136, "multiples of 16"),
    ("k_cache", "stride_block", 8192, "k_cache and v_cache must have the same strides"), ("v_scale", "data", _BASE + 2, "v_scale.data must be 4-byte aligned"),
    ("k_scale", "stride_head", 6, "multiples of 4"), ("k_scale", "stride_block", 32, "k_scale and v_scale must have the same strides"),
    ("v_scale", "data", None, "v_scale.data is NULL")])
def test_c_abi_cache_refusals(stream, field, value, message):
    lib, a = capi.load_library(), _kv8_args(False)
    setattr(getattr(a, stream), field, value)
    assert lib.kv8_check(a) == capi.EINVAL and message in lib.last_error()


def test_c_abi_calls_have_their_own_forms():
    lib = capi.load_library()
    assert lib.kv8_decode(_kv8_args(True)) == capi.EINVAL and "query_start_loc must be NULL" in lib.last_error()
    assert lib.kv8_attend(_kv8_args(False)) == capi.EINVAL and "query_start_loc is NULL" in lib.last_error()
    a = _kv8_args(False)
    a.num_tokens = 4
    assert lib.kv8_check(a) == capi.EINVAL and "num_tokens must equal num_reqs" in lib.last_error()
    a = _kv8_args(False)
    a.causal = 0
    assert lib.kv8_check(a) == capi.EINVAL and "causal must be 1" in lib.last_error()
    a = _kv8_args(True)
    a.max_query_len = 4
    assert lib.kv8_check(a) == capi.EINVAL and "max_query_len" in lib.last_error()


@pytest.mark.parametrize("field,value,message", _SHAPE_BAD + [
    ("src_dtype", 9, "src_dtype"), ("key", None, "key is NULL"), ("value", _BASE + 1, "value must be 2-byte aligned"), ("num_tokens", -1, "max_query_len must be"),
    ("max_query_len", 3, "max_query_len must be"), ("seq_lens", None, "seq_lens"), ("query_start_loc", None, "query_start_loc")])
def test_c_abi_write_refusals(field, value, message):
    lib, a = capi.load_library(), _write_struct()
    setattr(a, field, value)
    assert lib.kv8_write(a) == capi.EINVAL and message in lib.last_error()


@pytest.mark.parametrize("field,value,message", _SHAPE_BAD + [
    ("dst_dtype", 9, "dst_dtype"), ("key", _BASE + 8, "key must be 16-byte aligned"), ("value", None, "value is NULL"), ("max_rows", 3, "max_rows must be"),
    ("first", None, "first"), ("row_start_loc", None, "row_start_loc"), ("key_stride_head", 8, "key byte strides")])
def test_c_abi_read_refusals(field, value, message):
    lib, a = capi.load_library(), _read_struct()
    setattr(a, field, value)
    assert lib.kv8_read(a) == capi.EINVAL and message in lib.last_error()


@pytest.mark.parametrize("field,value,message", [
    ("abi_version", 1, "abi_version"), ("dtype", 9, "dtype"), ("head_size", 0, "head_size"), ("head_size", 1025, "head_size"),
    ("num_frequencies", 0, "num_frequencies"), ("num_frequencies", 33, "num_frequencies"), ("num_k_heads", -1, "num_k_heads"), ("q", None, "q is NULL"),
    ("k_out", _BASE + 1, "k_out must be 2-byte aligned"), ("positions", _BASE + 4, "positions"), ("frequencies", None, "frequencies"),
    ("scale", float("nan"), "scale must be finite"), ("num_q_heads", 1 << 30, "fewer than 2^28")])
def test_c_abi_rotary_refusals(field, value, message):
    lib, a = capi.load_library(), _rotary_struct()
    setattr(a, field, value)
    assert lib.rotary(a) == capi.EINVAL and message in lib.last_error()


def test_struct_sizes():
    lib = capi.load_library().lib
    assert ctypes.sizeof(capi.PthB200Kv8Args) == lib.pthb200_kv8_args_bytes()
    assert ctypes.sizeof(capi.PthB200RotaryArgs) == lib.pthb200_rotary_args_bytes()


def test_workspace_bytes():
    for D in (64, 128, 256):
        assert 0 < kv8.workspace_bytes(D=D, num_sms=148) <= 128 << 20
    with pytest.raises(ValueError):
        kv8.workspace_bytes(D=96, num_sms=148)
    with pytest.raises(ValueError):
        kv8.workspace_bytes(D=64, num_sms=0)


# ---- frequencies -------------------------------------------------------------------
def test_frequencies():
    f, scale = ops.rotary_frequencies(8, 10000.0)
    assert scale == 1.0 and f.dtype == F64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=F64), rtol=1e-14)
    linear, _ = ops.rotary_frequencies(8, 10000.0, scaling="linear", factor=4.0)
    assert torch.equal(linear, f / 4)
    ntk, _ = ops.rotary_frequencies(8, 10000.0, scaling="ntk", factor=4.0)
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-12)


def test_yarn_frequencies_keep_fast_pairs_and_stretch_slow_ones():
    plain, _ = ops.rotary_frequencies(128, 10000.0)
    f, scale = ops.rotary_frequencies(128, 10000.0, scaling="yarn", factor=16.0, trained=4096)
    assert math.isclose(scale, 0.1 * math.log(16.0) + 1.0)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(f[turns > 40], plain[turns > 40])
    assert torch.allclose(f[turns < 0.8], plain[turns < 0.8] / 16, rtol=1e-14)
    assert bool((f <= plain).all()) and bool((f >= plain / 16 * (1 - 1e-14)).all()) and bool((f[1:] <= f[:-1]).all())


@pytest.mark.parametrize("kw", [dict(dims=7), dict(dims=0), dict(dims=8, scaling="other"), dict(dims=8, base=1.0), dict(dims=8, factor=0.5),
                                dict(dims=8, trained=0), dict(dims=8, fast=1.0)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(**kw)
