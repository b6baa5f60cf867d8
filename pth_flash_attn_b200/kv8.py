"""The operators of an 8-bit paged cache with a scale per block of tokens and head, and rotary positions: schemas, fake
kernels and typed wrappers.

Cells are e4m3 numbers ``c`` (``float8_e4m3fn``) in views ``[blocks, slots, heads, D]`` of the pages that the other caches use too;
``k_scale`` / ``v_scale`` (fp32 ``[blocks, slots / g, heads]``) hold a scale for every ``g`` slots of a page and head, ``g`` a multiple of
16 that divides the page.  An element is ``c * scale``.  Five ops serve a layer (``csrc/torch_kv8.cpp``, over the C ABI
``pthb200_rotary`` / ``pthb200_kv8_*``):

* :func:`rotary` turns queries and keys by their positions (``positions`` of :func:`.kv16.page_tables`);
* :func:`kv8_write` quantises the keys and values of new tokens into their blocks;
* :func:`kv8_read` brings runs of positions back into 16- or 32-bit rows;
* :func:`kv8_decode_attention` attends from one new token of each request over its cache;
* :func:`kv8_attention` attends from any number of new tokens of each request over its cache, causally.

All are out-variants that allocate nothing, read no device data on the host and do not synchronise; they run on
the current stream of their tensors' device and can be captured in a CUDA graph.  ``ops`` loads the library and
re-exports them.
"""

from __future__ import annotations

import math

import torch

from .kv16 import _Check as _Check16

SCHEMAS = {
    "rotary":
        "rotary(Tensor! q_out, Tensor! k_out, Tensor q, Tensor k, Tensor positions, Tensor frequencies, float scale=1.0, "
        "bool interleaved=False, bool inverse=False) -> ()",
    "kv8_write":
        "kv8_write(Tensor key, Tensor value, Tensor! k_cache, Tensor! v_cache, Tensor! k_scale, Tensor! v_scale, Tensor block_table, "
        "Tensor seq_lens, Tensor query_start_loc, int max_query_len) -> ()",
    "kv8_read":
        "kv8_read(Tensor! key, Tensor! value, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor block_table, "
        "Tensor first, Tensor row_start_loc, int max_rows) -> ()",
    "kv8_decode_attention":
        "kv8_decode_attention(Tensor! out, Tensor! lse, Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
        "Tensor block_table, Tensor seq_lens, float softmax_scale, Tensor! workspace, int window=0) -> ()",
    "kv8_attention":
        "kv8_attention(Tensor! out, Tensor! lse, Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
        "Tensor block_table, Tensor seq_lens, Tensor query_start_loc, int max_query_len, float softmax_scale, Tensor! workspace, "
        "int window=0, bool causal=True) -> ()",
}
_HEAD_SIZES = (64, 128, 256)
_16BIT = (torch.bfloat16, torch.float16)
_FLOATS = (torch.float32, *_16BIT)
_MORE_NAMES = {torch.float64: "float64", torch.float8_e4m3fn: "float8_e4m3fn"}


class _Check(_Check16):
    """The C++ checks of one op, raising the same text."""

    @staticmethod
    def name(dtype: torch.dtype) -> str:
        return _MORE_NAMES.get(dtype) or _Check16.name(dtype)

    def written(self, **tensors) -> None:
        for name, t in tensors.items():
            for d in range(t.dim()):
                if t.size(d) > 1 and t.stride(d) == 0 and t.numel() != 0:
                    self.fail(name, " is written and must not have stride 0, as in dimension ", d)

    def caches8(self, k_cache, v_cache, k_scale, v_scale) -> None:
        self.rank(k_cache, 4, "k_cache")
        self.rank(v_cache, 4, "v_cache")
        self.rank(k_scale, 3, "k_scale")
        self.rank(v_scale, 3, "v_scale")
        self.dtype(k_cache, torch.float8_e4m3fn, "k_cache")
        self.dtype(v_cache, torch.float8_e4m3fn, "v_cache")
        self.dtype(k_scale, torch.float32, "k_scale")
        self.dtype(v_scale, torch.float32, "v_scale")
        NB, BS, Hkv, D = k_cache.shape
        groups = k_scale.size(1)
        if D not in _HEAD_SIZES:
            self.fail("head size D = k_cache.size(3) must be 64, 128 or 256, got ", D)
        if NB < 1 or BS < 1 or Hkv < 1:
            self.fail("k_cache must not be empty")
        for dim, (want, what) in enumerate(((NB, "NB"), (BS, "BS"), (Hkv, "Hkv"), (D, "D"))):
            self.size(v_cache, dim, want, "v_cache", what)
        self.size(k_scale, 0, NB, "k_scale", "NB")
        if groups < 1 or BS % groups or BS // groups % 16:
            self.fail("BS / k_scale.size(1), the tokens of a scale, must be a multiple of 16, got ", BS, " / ", groups)
        self.size(k_scale, 2, Hkv, "k_scale", "Hkv")
        self.size(v_scale, 0, NB, "v_scale", "NB")
        self.size(v_scale, 1, groups, "v_scale", "k_scale.size(1)")
        self.size(v_scale, 2, Hkv, "v_scale", "Hkv")
        self.inner(k_cache, "k_cache")
        self.inner(v_cache, "v_cache")

    def rows(self, key, value, k_cache) -> None:
        self.rank(key, 3, "key")
        self.rank(value, 3, "value")
        if key.dtype not in _FLOATS:
            self.fail("key must be float32, bfloat16 or float16, got ", self.name(key.dtype))
        self.dtype(value, key.dtype, "value (same dtype as key)")
        Hkv, D = k_cache.size(2), k_cache.size(3)
        self.size(key, 1, Hkv, "key", "Hkv")
        self.size(key, 2, D, "key", "D")
        self.size(value, 0, key.size(0), "value", "T")
        self.size(value, 1, Hkv, "value", "Hkv")
        self.size(value, 2, D, "value", "D")
        self.inner(key, "key")
        self.inner(value, "value")

    def table(self, block_table, lens, name: str) -> None:
        self.rank(block_table, 2, "block_table")
        self.dtype(block_table, torch.int32, "block_table")
        self.inner(block_table, "block_table")
        self.vector(lens, torch.int32, name)
        if block_table.size(0) < lens.size(0):
            self.fail("block_table has ", block_table.size(0), " rows, fewer than num_reqs = ", lens.size(0))

    def starts(self, starts, R: int, longest: int, T: int, name: str, bound: str) -> None:
        self.vector(starts, torch.int32, name)
        self.size(starts, 0, R + 1, name, "num_reqs + 1")
        if not 0 <= longest <= T:
            self.fail(bound, " must be in [0, T = ", T, "], got ", longest)

    def devices(self, as_, of: str, **others) -> None:
        for name, t in others.items():
            self.device(t, as_, name, of)


def _kv8_write_fake(key, value, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, max_query_len) -> None:
    c = _Check("kv8_write")
    c.caches8(k_cache, v_cache, k_scale, v_scale)
    c.rows(key, value, k_cache)
    c.table(block_table, seq_lens, "seq_lens")
    c.starts(query_start_loc, seq_lens.size(0), max_query_len, key.size(0), "query_start_loc", "max_query_len")
    c.written(k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale)
    c.devices(key, "key", value=value, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, block_table=block_table,
              seq_lens=seq_lens, query_start_loc=query_start_loc)


def _kv8_read_fake(key, value, k_cache, v_cache, k_scale, v_scale, block_table, first, row_start_loc, max_rows) -> None:
    c = _Check("kv8_read")
    c.caches8(k_cache, v_cache, k_scale, v_scale)
    c.rows(key, value, k_cache)
    c.table(block_table, first, "first")
    c.starts(row_start_loc, first.size(0), max_rows, key.size(0), "row_start_loc", "max_rows")
    c.written(key=key, value=value)
    c.devices(key, "key", value=value, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, block_table=block_table,
              first=first, row_start_loc=row_start_loc)


def _check_attention(c, out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale, workspace, window) -> None:
    c.rank(q, 3, "q")
    c.caches8(k_cache, v_cache, k_scale, v_scale)
    if q.dtype not in _16BIT:
        c.fail("q must be bfloat16 or float16, got ", c.name(q.dtype))
    T, Hq, Hkv, D = q.size(0), q.size(1), k_cache.size(2), k_cache.size(3)
    c.size(q, 2, D, "q", "D")
    c.inner(q, "q")
    c.rank(out, 3, "out")
    c.dtype(out, q.dtype, "out (same dtype as q)")
    c.size(out, 0, T, "out", "T")
    c.size(out, 1, Hq, "out", "Hq")
    c.size(out, 2, D, "out", "D")
    c.inner(out, "out")
    c.written(out=out)
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
    c.table(block_table, seq_lens, "seq_lens")
    if not (math.isfinite(softmax_scale) and softmax_scale > 0.0):
        c.fail("softmax_scale must be finite and > 0, got ", f"{softmax_scale:g}")
    if window < 0:
        c.fail("window must be >= 0, got ", window)
    c.vector(workspace, torch.uint8, "workspace")
    c.devices(q, "q", out=out, lse=lse, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, block_table=block_table,
              seq_lens=seq_lens, workspace=workspace)


def _kv8_decode_attention_fake(out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale, workspace,
                               window=0) -> None:
    c = _Check("kv8_decode_attention")
    _check_attention(c, out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale, workspace, window)
    c.size(q, 0, seq_lens.size(0), "q", "num_reqs")


def _kv8_attention_fake(out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, max_query_len,
                        softmax_scale, workspace, window=0, causal=True) -> None:
    c = _Check("kv8_attention")
    _check_attention(c, out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale, workspace, window)
    c.starts(query_start_loc, seq_lens.size(0), max_query_len, q.size(0), "query_start_loc", "max_query_len")
    c.device(query_start_loc, q, "query_start_loc", "q")


def _rotary_fake(q_out, k_out, q, k, positions, frequencies, scale=1.0, interleaved=False, inverse=False) -> None:
    c = _Check("rotary")
    c.rank(q, 3, "q")
    c.rank(k, 3, "k")
    if q.dtype not in _FLOATS:
        c.fail("q must be float32, bfloat16 or float16, got ", c.name(q.dtype))
    c.dtype(k, q.dtype, "k (same dtype as q)")
    T, D, half = q.size(0), q.size(2), frequencies.numel()
    if not 1 <= D <= 1024:
        c.fail("head size D = q.size(2) must be in [1, 1024], got ", D)
    c.size(k, 0, T, "k", "T")
    c.size(k, 2, D, "k", "D")
    for x, y, name in ((q, q_out, "q"), (k, k_out, "k")):
        c.inner(x, name)
        c.rank(y, 3, f"{name}_out")
        c.dtype(y, q.dtype, f"{name}_out (same dtype as q)")
        c.size(y, 0, T, f"{name}_out", "T")
        c.size(y, 1, x.size(1), f"{name}_out", f"{name}.size(1)")
        c.size(y, 2, D, f"{name}_out", "D")
        c.inner(y, f"{name}_out")
        c.written(**{f"{name}_out": y})
    c.vector(positions, torch.int64, "positions")
    c.size(positions, 0, T, "positions", "T")
    c.rank(frequencies, 1, "frequencies")
    if frequencies.dtype not in (torch.float64, torch.float32):
        c.fail("frequencies must be float64 or float32, got ", c.name(frequencies.dtype))
    c.inner(frequencies, "frequencies")
    if not 1 <= half <= D // 2:
        c.fail("frequencies.size(0) must be in [1, D / 2 = ", D // 2, "], got ", half)
    if not abs(scale) <= torch.finfo(torch.float32).max:
        c.fail("scale must be finite, got ", f"{scale:g}")
    c.devices(q, "q", k=k, q_out=q_out, k_out=k_out, positions=positions, frequencies=frequencies)


_FAKES = {"rotary": _rotary_fake, "kv8_write": _kv8_write_fake, "kv8_read": _kv8_read_fake,
          "kv8_decode_attention": _kv8_decode_attention_fake, "kv8_attention": _kv8_attention_fake}
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

    n = capi.load_library().kv8_workspace_bytes(D, num_sms)
    if n < 0:
        raise ValueError(f"D must be one of {_HEAD_SIZES} and num_sms >= 1, got {D} and {num_sms}")
    return n


def rotary_frequencies(dims: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0, trained: int = 4096,
                       fast: float = 32.0, slow: float = 1.0, device=None):
    """``frequencies`` (float64 ``[dims / 2]``, radians per position) and ``scale`` for :func:`rotary`.

    ``base ** (-2 i / dims)``, for contexts ``factor`` times the ``trained`` length by one of: ``"linear"``, positions divided by
    ``factor``; ``"ntk"``, a base enlarged so that the slowest pair turns ``factor`` times slower and the fastest as before;
    ``"yarn"``, pairs that turn more than ``fast`` times over the trained length as they are, those that turn less than
    ``slow`` times ``factor`` times slower, a blend between them, linear in the pair's index, and a scale of ``0.1 ln(factor) + 1``.
    """
    if dims < 2 or dims % 2:
        raise ValueError(f"dims must be even and >= 2, got {dims}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be none, linear, ntk or yarn, got {scaling!r}")
    if not (base > 1.0 and factor >= 1.0 and trained >= 1 and fast > slow > 0.0):
        raise ValueError("base must be above 1, factor and trained at least 1, and fast above slow above 0")
    if scaling == "ntk" and dims > 2:
        base *= factor ** (dims / (dims - 2))
    i = torch.arange(dims // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / dims)
    if scaling == "linear":
        return (f / factor).to(device), 1.0
    if scaling != "yarn":
        return f.to(device), 1.0

    def index(turns: float) -> float:   # of the pair that turns so many times
        return dims * math.log(trained / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), dims - 1)
    slower = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    return (f * (1.0 - slower) + f / factor * slower).to(device), 0.1 * math.log(factor) + 1.0


def rotary(q_out, k_out, q, k, positions, frequencies, scale: float = 1.0, interleaved: bool = False, inverse: bool = False) -> None:
    """Turns queries and keys by their positions.

    ``q`` ``[T, Hq, D]`` and ``k`` ``[T, Hk, D]`` (fp32, bf16 or fp16; either may have no heads), ``positions`` int64 ``[T]``,
    ``frequencies`` (float64 or float32 ``[n]``, radians per position; :func:`rotary_frequencies`).  The first ``2 n`` dimensions of a
    head turn, pair ``i`` by ``position * frequencies[i]``: pairs are ``(i, i + n)``, or ``(2 i, 2 i + 1)`` if ``interleaved``.  Turned pairs
    are multiplied by ``scale``, the other dimensions copied.  Angles have 64 bits, so far positions turn as
    exactly as near ones.  ``inverse`` turns back, which is also the gradient of turning.  ``q_out`` / ``k_out`` may be ``q`` / ``k``
    themselves, and must not overlap them otherwise.
    """
    _op("rotary")(q_out, k_out, q, k, positions, frequencies, scale, interleaved, inverse)


def kv8_write(key, value, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, max_query_len: int) -> None:
    """Quantises the keys and values of new tokens into the 8-bit cache.

    ``key`` / ``value`` ``[T, Hkv, D]`` (fp32, bf16 or fp16).  The tokens ``query_start_loc[r] .. query_start_loc[r + 1)`` of request ``r``
    are the last of its ``seq_lens[r]`` tokens; their slots come from ``block_table`` (int32 ``[>= R, pages]``).  ``max_query_len`` bounds the
    tokens of a request.  A block of tokens whose first position is written gets the smallest power of two as its scale with
    which its values fit; one that goes on keeps its scale, or gets the one that its new values need if that is larger, and
    its older cells are rounded again.  Values are rounded to nearest even; infinities become the largest number.  Tokens without a
    block (ids outside the cache, positions past the table) are skipped.  Two requests must not write to one block of tokens.
    """
    _op("kv8_write")(key, value, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, max_query_len)


def kv8_read(key, value, k_cache, v_cache, k_scale, v_scale, block_table, first, row_start_loc, max_rows: int) -> None:
    """Reads runs of positions back: row ``row_start_loc[r] + i`` of ``key`` / ``value`` ``[T, Hkv, D]`` (fp32, bf16 or fp16) becomes position
    ``first[r] + i`` of request ``r``, rounded once, zero where there is no such cell.  ``max_rows`` bounds the rows of a request; rows
    that belong to none are left as they are."""
    _op("kv8_read")(key, value, k_cache, v_cache, k_scale, v_scale, block_table, first, row_start_loc, max_rows)


def kv8_decode_attention(out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale: float, workspace,
                         window: int = 0) -> None:
    """Attention of one new token of each request over its cache.

    ``q``, ``out`` ``[R, Hq, D]`` bf16 or fp16; ``lse`` fp32 ``[R, Hq]`` (natural logarithm) may be empty.  ``window > 0`` limits a
    token to the newest ``window`` keys.  Scales are positive finite numbers, and may be broadcast; ``out`` must not overlap the
    inputs.  ``workspace`` (uint8, at least :func:`workspace_bytes`) is zeroed once by its owner, and
    left ready for the next call; calls that may overlap need one each.
    """
    _op("kv8_decode_attention")(out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, softmax_scale, workspace, window)


def kv8_attention(out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, max_query_len: int,
                  softmax_scale: float, workspace, window: int = 0, causal: bool = True) -> None:
    """Attention of the tokens ``query_start_loc[r] .. query_start_loc[r + 1)`` of request ``r``, the last of its ``seq_lens[r]``
    tokens, over its cache.

    A token at position ``p`` sees the keys ``max(0, p - window + 1) .. p`` (all up to ``p`` with a window of 0; up to the request's end
    without ``causal``).  ``q``, ``out`` ``[T, Hq, D]``; ``max_query_len`` bounds the tokens of a request; ``lse`` and ``workspace`` as in
    :func:`kv8_decode_attention`.  ``max_query_len`` also chooses the kernel, for all of the call's requests: tokens of prompts and single
    ones are served best by a call each.
    """
    _op("kv8_attention")(out, lse, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_start_loc, max_query_len,
                         softmax_scale, workspace, window, causal)
