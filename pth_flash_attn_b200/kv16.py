"""The operators of a 16-bit paged cache: schemas, fake kernels and typed wrappers.

Layers whose cache is not quantised, and the encoder's states of an encoder-decoder model, live in the same
pages as the int8 cache, as bf16 or fp16 cells.  Four ops serve them (``csrc/torch_kv16.cpp``, over the C ABI
``pthb200_page_tables`` / ``pthb200_kv16_*``):

* :func:`page_tables` makes a step's block table, slot map, positions and start offsets from the requests' lengths;
* :func:`kv16_write` stores the keys and values of new tokens at their slots;
* :func:`kv16_decode_attention` attends from one new token of each request over its cache;
* :func:`kv16_cross_attention` attends from any number of tokens of a request over its encoder's states.

All are out-variants that allocate nothing, read no device data on the host and do not synchronise; they run on
the current stream of their tensors' device and can be captured in a CUDA graph.  ``ops`` loads the library and
re-exports them.
"""

from __future__ import annotations

import math

import torch

SCHEMAS = {
    "page_tables":
        "page_tables(Tensor context_lens, Tensor query_lens, Tensor free_blocks, Tensor! block_table, Tensor! seq_lens, "
        "Tensor! query_start_loc, Tensor! slot_mapping, Tensor! positions, Tensor! pages_taken, int block_size) -> ()",
    "kv16_write":
        "kv16_write(Tensor key, Tensor value, Tensor! k_cache, Tensor! v_cache, Tensor slot_mapping) -> ()",
    "kv16_decode_attention":
        "kv16_decode_attention(Tensor! out, Tensor! lse, Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
        "Tensor seq_lens, float softmax_scale, Tensor! workspace, int window=0) -> ()",
    "kv16_cross_attention":
        "kv16_cross_attention(Tensor! out, Tensor! lse, Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
        "Tensor context_lens, Tensor query_start_loc, int max_query_len, float softmax_scale, Tensor! workspace) -> ()",
}
_NAMES = {torch.bfloat16: "bfloat16", torch.float16: "float16", torch.float32: "float32", torch.uint8: "uint8",
          torch.int8: "int8", torch.int32: "int32", torch.int64: "int64"}
_HEAD_SIZES = (64, 128, 256)
_16BIT = (torch.bfloat16, torch.float16)


class _Check:
    """The C++ checks of one op, raising the same text."""

    def __init__(self, op: str) -> None:
        self.op = op

    def fail(self, *parts: object) -> None:
        raise RuntimeError(self.op + ": " + "".join(str(x) for x in parts))

    @staticmethod
    def name(dtype: torch.dtype) -> str:
        return _NAMES.get(dtype, "an unsupported dtype")

    def rank(self, t, want: int, name: str) -> None:
        if t.dim() != want:
            self.fail(name, " must be ", want, "-D, got ", t.dim(), "-D")

    def dtype(self, t, want: torch.dtype, name: str) -> None:
        if t.dtype != want:
            self.fail(name, " must be ", self.name(want), ", got ", self.name(t.dtype))

    def size(self, t, dim: int, want: int, name: str, what: str) -> None:
        if t.size(dim) != want:
            self.fail(name, ".size(", dim, ") must equal ", what, " = ", want, ", got ", t.size(dim))

    def inner(self, t, name: str) -> None:
        if t.numel() != 0 and t.stride(-1) != 1:
            self.fail(name, " must have stride 1 in its last dimension, got ", t.stride(-1))

    def vector(self, t, dtype: torch.dtype, name: str) -> None:
        self.rank(t, 1, name)
        self.dtype(t, dtype, name)
        self.inner(t, name)

    def device(self, t, as_, name: str, of: str) -> None:
        if t.device != as_.device:
            self.fail(name, " must be on the same device as ", of)

    def caches(self, k_cache, v_cache) -> None:
        self.rank(k_cache, 4, "k_cache")
        self.rank(v_cache, 4, "v_cache")
        if k_cache.dtype not in _16BIT:
            self.fail("k_cache must be bfloat16 or float16, got ", self.name(k_cache.dtype))
        self.dtype(v_cache, k_cache.dtype, "v_cache (same dtype as k_cache)")
        D = k_cache.size(3)
        if D not in _HEAD_SIZES:
            self.fail("head size D = k_cache.size(3) must be 64, 128 or 256, got ", D)
        if k_cache.size(0) < 1 or k_cache.size(1) < 1 or k_cache.size(2) < 1:
            self.fail("k_cache must not be empty")
        for dim, what in enumerate(("NB", "BS", "Hkv", "D")):
            self.size(v_cache, dim, k_cache.size(dim), "v_cache", what)
        self.inner(k_cache, "k_cache")
        self.inner(v_cache, "v_cache")


def _page_tables_fake(context_lens, query_lens, free_blocks, block_table, seq_lens, query_start_loc, slot_mapping,
                      positions, pages_taken, block_size) -> None:
    c = _Check("page_tables")
    c.vector(context_lens, torch.int32, "context_lens")
    c.vector(query_lens, torch.int32, "query_lens")
    c.vector(free_blocks, torch.int32, "free_blocks")
    c.rank(block_table, 2, "block_table")
    c.dtype(block_table, torch.int32, "block_table")
    c.inner(block_table, "block_table")
    c.vector(seq_lens, torch.int32, "seq_lens")
    c.vector(query_start_loc, torch.int32, "query_start_loc")
    c.vector(slot_mapping, torch.int64, "slot_mapping")
    c.vector(positions, torch.int64, "positions")
    c.vector(pages_taken, torch.int32, "pages_taken")
    R = context_lens.size(0)
    c.size(query_lens, 0, R, "query_lens", "num_reqs")
    c.size(seq_lens, 0, R, "seq_lens", "num_reqs")
    c.size(query_start_loc, 0, R + 1, "query_start_loc", "num_reqs + 1")
    c.size(pages_taken, 0, 1, "pages_taken", "1")
    if block_table.size(0) < R:
        c.fail("block_table has ", block_table.size(0), " rows, fewer than num_reqs = ", R)
    if positions.size(0) != 0:
        c.size(positions, 0, slot_mapping.size(0), "positions", "slot_mapping.size(0)")
    if block_size < 1:
        c.fail("block_size must be >= 1, got ", block_size)
    for t, name in ((query_lens, "query_lens"), (free_blocks, "free_blocks"), (block_table, "block_table"),
                    (seq_lens, "seq_lens"), (query_start_loc, "query_start_loc"), (slot_mapping, "slot_mapping"),
                    (positions, "positions"), (pages_taken, "pages_taken")):
        c.device(t, context_lens, name, "context_lens")


def _kv16_write_fake(key, value, k_cache, v_cache, slot_mapping) -> None:
    c = _Check("kv16_write")
    c.caches(k_cache, v_cache)
    c.rank(key, 3, "key")
    c.rank(value, 3, "value")
    if key.dtype not in (torch.float32, *_16BIT):
        c.fail("key must be float32, bfloat16 or float16, got ", c.name(key.dtype))
    c.dtype(value, key.dtype, "value (same dtype as key)")
    T, Hkv, D = key.size(0), k_cache.size(2), k_cache.size(3)
    c.size(key, 1, Hkv, "key", "Hkv")
    c.size(key, 2, D, "key", "D")
    c.size(value, 0, T, "value", "T")
    c.size(value, 1, Hkv, "value", "Hkv")
    c.size(value, 2, D, "value", "D")
    c.inner(key, "key")
    c.inner(value, "value")
    c.vector(slot_mapping, torch.int64, "slot_mapping")
    c.size(slot_mapping, 0, T, "slot_mapping", "T")
    for t, name in ((value, "value"), (k_cache, "k_cache"), (v_cache, "v_cache"), (slot_mapping, "slot_mapping")):
        c.device(t, key, name, "key")


def _check_attention(c, out, lse, q, k_cache, v_cache, block_table, seq_lens, softmax_scale, workspace) -> None:
    c.rank(q, 3, "q")
    c.caches(k_cache, v_cache)
    c.dtype(q, k_cache.dtype, "q (same dtype as k_cache)")
    T, Hq, Hkv, D = q.size(0), q.size(1), k_cache.size(2), k_cache.size(3)
    c.size(q, 2, D, "q", "D")
    c.inner(q, "q")
    c.rank(out, 3, "out")
    c.dtype(out, q.dtype, "out (same dtype as q)")
    c.size(out, 0, T, "out", "T")
    c.size(out, 1, Hq, "out", "Hq")
    c.size(out, 2, D, "out", "D")
    c.inner(out, "out")
    if Hq < 1 or Hq % Hkv != 0:
        c.fail("Hq = ", Hq, " must be a positive multiple of Hkv = ", Hkv)
    if Hq // Hkv > 64:
        c.fail("G = Hq/Hkv = ", Hq // Hkv, " exceeds the supported maximum 64")
    c.dtype(lse, torch.float32, "lse")
    if lse.numel() != 0:
        c.rank(lse, 2, "lse")
        c.size(lse, 0, T, "lse", "T")
        c.size(lse, 1, Hq, "lse", "Hq")
        if lse.stride(1) != 1 or lse.stride(0) != Hq:
            c.fail("lse must be contiguous")
    c.rank(block_table, 2, "block_table")
    c.dtype(block_table, torch.int32, "block_table")
    c.inner(block_table, "block_table")
    c.vector(seq_lens, torch.int32, "seq_lens")
    if block_table.size(0) < seq_lens.size(0):
        c.fail("block_table has ", block_table.size(0), " rows, fewer than num_reqs = ", seq_lens.size(0))
    if not (math.isfinite(softmax_scale) and softmax_scale > 0.0):
        c.fail("softmax_scale must be finite and > 0, got ", f"{softmax_scale:g}")
    c.vector(workspace, torch.uint8, "workspace")
    for t, name in ((out, "out"), (lse, "lse"), (k_cache, "k_cache"), (v_cache, "v_cache"), (block_table, "block_table"),
                    (seq_lens, "seq_lens"), (workspace, "workspace")):
        c.device(t, q, name, "q")


def _kv16_decode_attention_fake(out, lse, q, k_cache, v_cache, block_table, seq_lens, softmax_scale, workspace,
                                window=0) -> None:
    c = _Check("kv16_decode_attention")
    _check_attention(c, out, lse, q, k_cache, v_cache, block_table, seq_lens, softmax_scale, workspace)
    c.size(q, 0, seq_lens.size(0), "q", "num_reqs")
    if window < 0:
        c.fail("window must be >= 0, got ", window)


def _kv16_cross_attention_fake(out, lse, q, k_cache, v_cache, block_table, context_lens, query_start_loc,
                               max_query_len, softmax_scale, workspace) -> None:
    c = _Check("kv16_cross_attention")
    _check_attention(c, out, lse, q, k_cache, v_cache, block_table, context_lens, softmax_scale, workspace)
    c.vector(query_start_loc, torch.int32, "query_start_loc")
    c.size(query_start_loc, 0, context_lens.size(0) + 1, "query_start_loc", "num_reqs + 1")
    if not 0 <= max_query_len <= q.size(0):
        c.fail("max_query_len must be in [0, T = ", q.size(0), "], got ", max_query_len)
    c.device(query_start_loc, q, "query_start_loc", "q")


_FAKES = {"page_tables": _page_tables_fake, "kv16_write": _kv16_write_fake,
          "kv16_decode_attention": _kv16_decode_attention_fake, "kv16_cross_attention": _kv16_cross_attention_fake}
_OPS: dict = {}


def register() -> None:
    """Binds the loaded library's ops and their fake kernels (``ops`` calls it behind ``load_library``)."""
    for name, fake in _FAKES.items():
        torch.library.register_fake(f"pth_flash_attn::{name}")(fake)
        _OPS[name] = getattr(torch.ops.pth_flash_attn, name).default


def _op(name: str):
    try:
        return _OPS[name]
    except KeyError:
        raise RuntimeError(f"{name}: the op library is not built; run `python -m pth_flash_attn_b200.build` "
                           "(there is no fallback implementation)") from None


def workspace_bytes(*, D: int, num_sms: int) -> int:
    """Bytes of the ``workspace`` of the attention ops: enough for any call of head size ``D`` on a device of ``num_sms`` SMs."""
    from . import capi

    n = capi.load_library().kv16_workspace_bytes(D, num_sms)
    if n < 0:
        raise ValueError(f"D must be one of {_HEAD_SIZES} and num_sms >= 1, got {D} and {num_sms}")
    return n


def page_tables(context_lens, query_lens, free_blocks, block_table, seq_lens, query_start_loc, slot_mapping, positions,
                pages_taken, block_size: int) -> None:
    """The tables of a step, from its requests' lengths.

    ``context_lens`` / ``query_lens`` int32 ``[R]``: tokens that a request has, and new ones.  Its new pages are taken off
    ``free_blocks`` (int32) in the order of requests, and entered in ``block_table`` (int32 ``[>= R, pages]``) behind
    those it has.  Written as well: ``seq_lens [R]``, ``query_start_loc [R + 1]`` (int32), ``slot_mapping`` and ``positions``
    (int64 ``[T]``; ``positions`` may be empty), ``pages_taken`` (int32 ``[1]``).  Padding tokens get slot -1.  If
    ``pages_taken`` exceeds the list, the pages past it are entered as -1 and their tokens get slot -1.
    """
    _op("page_tables")(context_lens, query_lens, free_blocks, block_table, seq_lens, query_start_loc, slot_mapping,
                       positions, pages_taken, block_size)


def kv16_write(key, value, k_cache, v_cache, slot_mapping) -> None:
    """Stores ``key`` / ``value`` ``[T, Hkv, D]`` (fp32, bf16 or fp16) at ``slot_mapping`` (int64 ``[T]``), rounded to the type of
    ``k_cache`` / ``v_cache`` ``[blocks, block_size, Hkv, D]`` (bf16 or fp16).  A slot outside the cache skips the token."""
    _op("kv16_write")(key, value, k_cache, v_cache, slot_mapping)


def kv16_decode_attention(out, lse, q, k_cache, v_cache, block_table, seq_lens, softmax_scale: float, workspace,
                          window: int = 0) -> None:
    """Attention of one new token of each request over its cache.

    ``q``, ``out`` ``[R, Hq, D]`` and the cache have one 16-bit type; ``lse`` fp32 ``[R, Hq]`` (natural logarithm) may be empty.
    ``window > 0`` limits a token to the newest ``window`` keys.  ``workspace`` (uint8, at least
    :func:`workspace_bytes`) is zeroed once by its owner, and left ready for the next call; calls that may
    overlap need one each.
    """
    _op("kv16_decode_attention")(out, lse, q, k_cache, v_cache, block_table, seq_lens, softmax_scale, workspace, window)


def kv16_cross_attention(out, lse, q, k_cache, v_cache, block_table, context_lens, query_start_loc, max_query_len: int,
                         softmax_scale: float, workspace) -> None:
    """Attention of the tokens ``query_start_loc[r] .. query_start_loc[r + 1)`` of request ``r`` over all
    ``context_lens[r]`` states of its encoder, which lie in pages of the cache.

    ``q``, ``out`` ``[T, Hq, D]``; ``max_query_len`` bounds the tokens of a request (1 for a decoding step); ``lse`` and
    ``workspace`` as in :func:`kv16_decode_attention`.  Where a request has more than one token and ``max_query_len`` times
    ``Hq / Hkv`` is 17 or more, probabilities are rounded to the cache's type (1.4 times the error of the output's own rounding);
    below, and in :func:`kv16_decode_attention`, they are kept in two such parts.
    """
    _op("kv16_cross_attention")(out, lse, q, k_cache, v_cache, block_table, context_lens, query_start_loc, max_query_len,
                                softmax_scale, workspace)
