"""The paged KV cache in 8 bits and the attention that reads it.

Layout and mathematics: ``csrc/kernels/kv8.cuh``.  Codes are int8 or e4m3, [num_blocks, kv_heads, 16, head_dim], with one
fp32 scale for each (block, head), a power of two; keys and values have scales of their own.  A block begins when its slot
0 is written; tokens that join it later can raise its scale, and then the codes below them are rounded once more.  A token
with a value that is not finite makes its block and head read as NaN until the block begins again.

Page numbers, slots, table rows and lengths come from device memory.  What lies outside the cache or its tables is not accessed:
the keys that a page, a table row, or columns behind the table's last stand for are left out, the kernel sets the device's status
word, and ``check_status`` raises.
"""
from __future__ import annotations

import ctypes
import math
import struct
from decimal import Decimal, localcontext
from functools import lru_cache
from typing import Optional, Tuple

import torch

from .. import _native
from . import checks as _checks
from .kernels import OperandError, _check, _run_check, status_word

_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_PRECISIONS = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_BLOCK = 16
_TILE = 16                                   # query rows of an attention tile


# the launchers' call records (kv8_attention.cu, kv8_cache.cu, kv8_chunk.cu), packed: a decode step is made of calls of a few microseconds, and
# three dozen arguments one by one cost as much as the kernel
_APPEND_CALL = struct.Struct("=10Q4q8i")
_READ_CALL = struct.Struct("=8Q2q4i")
_ATTENTION_CALL = struct.Struct("=16Q6q13if")
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")
_raw_stream = torch._C._cuda_getCurrentRawStream


class KV8Cache:
    """Codes and scales of one layer's keys and values, or of one rank's share of them."""
    __slots__ = ("k", "v", "k_scale", "v_scale", "num_blocks", "kv_heads", "head_dim", "code", "_index", "_status")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if k.dtype not in _CODES or v.dtype != k.dtype:
            raise OperandError(f"cache codes must be int8 or float8_e4m3fn, keys and values alike, got {k.dtype} and {v.dtype}")
        if k.dim() != 4 or k.shape != v.shape or k.shape[2] != _BLOCK or k.shape[3] not in (64, 128) or 0 in k.shape:
            raise OperandError(f"cache codes must be [blocks, kv_heads, 16, 64 or 128], got {tuple(k.shape)} and {tuple(v.shape)}")
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or s.shape != k.shape[:2] or not s.is_contiguous() or s.device != k.device:
                raise OperandError(f"cache scales must be contiguous fp32 {tuple(k.shape[:2])} on {k.device}, got {s.dtype} "
                                   f"{tuple(s.shape)} on {s.device}")
        for c in (k, v):
            if not c.is_contiguous() or c.data_ptr() % 16 or c.device != k.device:
                raise OperandError("cache codes must be contiguous from a 16-byte boundary, keys and values on one device")
        if k.shape[0] * _BLOCK > 2 ** 31 - 1:
            raise OperandError(f"cache slots are 32-bit numbers; {k.shape[0]} blocks have more")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_blocks, self.kv_heads, _, self.head_dim = k.shape
        self.code = _CODES[k.dtype]
        self._index = k.get_device()                        # -1 on the host
        # made here, not in a call: a call may be the first of a graph's capture, whose memory goes with the graph
        self._status = status_word(k.device).data_ptr() if self._index >= 0 else 0

    @classmethod
    def alloc(cls, num_blocks: int, kv_heads: int, head_dim: int, precision: str = "int8", device="cuda") -> "KV8Cache":
        """An empty cache: every block reads as zeros."""
        if precision not in _PRECISIONS:
            raise OperandError(f"cache precision is 'int8' or 'fp8', got '{precision}'")
        shape = (num_blocks, kv_heads, _BLOCK, head_dim)
        mk = lambda: torch.zeros(shape, dtype=torch.uint8, device=device).view(_PRECISIONS[precision])
        return cls(mk(), mk(), torch.zeros(shape[:2], device=device), torch.zeros(shape[:2], device=device))

    def _pointers(self) -> Tuple[int, int, int, int]:
        return self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr()

    @property
    def device(self) -> torch.device:
        return self.k.device

    @property
    def dtype(self) -> torch.dtype:
        return self.k.dtype


class _On:
    """The cache's device for a call made while another is current."""
    __slots__ = ("_ctx",)

    def __init__(self, index: int):
        if index < 0:
            raise OperandError("the 8-bit cache kernels run on a CUDA device, got a cache on the host")
        self._ctx = torch.cuda.device(index) if index != torch._C._cuda_getDevice() else None

    def __enter__(self):
        if self._ctx is not None:
            self._ctx.__enter__()

    def __exit__(self, *error):
        if self._ctx is not None:
            self._ctx.__exit__(*error)


def _rows16(what: str, t: torch.Tensor, cols: int, index: int, dtype: Optional[torch.dtype] = None) -> int:
    """Row stride of a 16-bit matrix whose rows the kernels read or write in 16-byte pieces."""
    if t.dim() != 2 or t.get_device() != index or (t.dtype not in _DTYPES if dtype is None else t.dtype is not dtype):
        raise OperandError(f"{what} must be a matrix of {dtype or 'bf16 or fp16'} on device {index}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    rows, width = t.shape
    if width < cols:
        raise OperandError(f"{what} has {width} columns, {cols} are read or written")
    ld, unit = t.stride()
    if rows <= 1:
        ld = -(-width // 8) * 8
    if unit != 1 and width > 1 or ld % 8 or ld < cols or t.data_ptr() % 16:
        raise OperandError(f"{what} must have unit column stride and rows that start on 16-byte boundaries and do not overlap, got "
                           f"strides {t.stride()}")
    return ld


def _apart(at: int, ld: int, cols: int, at2: int, ld2: int, cols2: int, rows: int) -> bool:
    """Whether two matrices of 16-bit values (address, row stride, columns) have no element in common.  Of two row strides, only
    matrices that lie one behind the other count as apart."""
    gap = (at2 - at) // 2
    if gap >= (rows - 1) * ld + cols or -gap >= (rows - 1) * ld2 + cols2:
        return True
    return ld == ld2 and gap % ld >= cols and gap % ld + cols2 <= ld


def _ints(what: str, t: torch.Tensor, n: int, index: int) -> int:
    """Address of n int32 values."""
    if t.dtype is not torch.int32 or t.get_device() != index or t.dim() != 1 or t.numel() < n or not t.is_contiguous():
        raise OperandError(f"{what} must be {n} contiguous int32 values on device {index}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _table(t: torch.Tensor, rows: int, index: int) -> Tuple[int, int, int]:
    """(row stride, rows, columns) of block tables that need ``rows`` rows (0: are indexed by a vector)."""
    if t.dim() != 2 or t.dtype is not torch.int32 or t.get_device() != index:
        raise OperandError(f"block_tables must be an int32 matrix on device {index}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    (n, width), (ld, unit) = t.shape, t.stride()
    if n <= 1:
        ld = max(ld, width)
    if not 1 <= width <= 1 << 26 or (unit != 1 and width > 1) or ld < width:
        raise OperandError(f"block_tables must have columns (up to 2^26), in unit stride, and rows that do not overlap, got {tuple(t.shape)}, strides {t.stride()}")
    if n < rows:
        raise OperandError(f"block_tables has {n} rows for {rows}")
    return ld, n, width


def _heads(heads: int, cache: KV8Cache) -> None:
    if heads <= 0 or heads % cache.kv_heads or heads > 65535:
        raise OperandError(f"{heads} heads do not divide into {cache.kv_heads} cached heads")


def _offset(what: str, off: int) -> None:
    if off < 0 or off % 8:
        raise OperandError(f"{what} is {off}; heads must start at a multiple of 8 columns")


@lru_cache(maxsize=64)
def _turns(head_dim: int, base: float):
    """base^(-2j/d) / (2 pi) for each channel pair, as the nearest 64-bit fractions of a turn: the array, which must live, and its address."""
    if not (base > 0.0 and math.isfinite(base)):
        raise OperandError(f"rotary base must be a positive number, got {base}")
    with localcontext() as ctx:                              # 64 bits behind the point, and what stands in front of it where base < 1
        ctx.prec = 40 + max(0, -math.floor(math.log10(base)))
        log, unit = Decimal(base).ln(), 2 ** 64 / (2 * _PI)
        f = [int(((log * (-2 * j) / head_dim).exp() * unit).to_integral_value()) & (2 ** 64 - 1) for j in range(head_dim // 2)]
    arr = (ctypes.c_ulonglong * len(f))(*f)
    return arr, ctypes.addressof(arr)


def kv8_append(qkv: torch.Tensor, k_off: int, v_off: int, slots: torch.Tensor, cache: KV8Cache, heads: int,
               positions: Optional[torch.Tensor] = None, rope_base: float = 0.0, rotated: Optional[torch.Tensor] = None) -> None:
    """Put the K and V columns of a fused QKV activation [tokens, ld] into their cache slots (int32 [tokens], -1: not cached).
    The tokens of one block stand in consecutive rows with rising slots, as a scheduler lists them.  With ``positions`` and
    ``rope_base`` > 0, q and k are rotated first; the rotated columns go to ``rotated`` (laid out as qkv; default: qkv
    itself, with which another buffer shares no element)."""
    d, kvh, index = cache.head_dim, cache.kv_heads, cache._index
    _heads(heads, cache)
    rope = positions is not None and rope_base > 0
    if not rope and rotated is not None:
        raise OperandError("rotated needs positions and a rotary base")
    _offset("k_off", k_off)
    _offset("v_off", v_off)
    ld = _rows16("qkv", qkv, max(k_off, v_off) + kvh * d, index)
    tokens, rot, ld_rot, pos, turns = qkv.shape[0], 0, 0, 0, 0
    slot_ptr = _ints("slots", slots, tokens, index)
    if rope:
        if k_off < heads * d:
            raise OperandError(f"k_off {k_off} lies inside the {heads} heads of q")
        to = qkv if rotated is None else rotated
        ld_rot = _rows16("rotated", to, k_off + kvh * d, index, qkv.dtype)
        if to.shape[0] < tokens:
            raise OperandError(f"rotated has {to.shape[0]} rows for {tokens} tokens")
        if to.data_ptr() == qkv.data_ptr() and (ld_rot == ld or tokens <= 1):
            if v_off < heads * d or abs(v_off - k_off) < kvh * d:
                raise OperandError(f"v_off {v_off} lies inside the columns that are rotated in place")
        elif tokens and not _apart(qkv.data_ptr(), ld, max(k_off, v_off) + kvh * d, to.data_ptr(), ld_rot, k_off + kvh * d, tokens):
            raise OperandError("rotated overlaps qkv; it is qkv itself, or apart from it")
        angles = _turns(d, float(rope_base))                 # kept while the launcher copies it
        rot, pos, turns = to.data_ptr(), _ints("positions", positions, tokens, index), angles[1]

    with _On(index):
        if _checks.enabled():
            _run_check(_checks.kv8_append, qkv, slots, cache.k, positions)
        rc = _native.cuda().ronn_kv8_append(_APPEND_CALL.pack(qkv.data_ptr(), rot, slot_ptr, pos, turns, *cache._pointers(), cache._status, ld,
                                                              ld_rot, cache.num_blocks, tokens, k_off, v_off, heads, kvh, d,
                                                              _DTYPES[qkv.dtype], cache.code, 0), _raw_stream(index))
    _check(rc, "kv8_append")


def kv8_read(cache: KV8Cache, blocks: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of whole cache blocks (int32 [n]) as two [n, kv_heads, 16, head_dim] tensors."""
    if dtype not in _DTYPES:
        raise OperandError(f"kv8_read gives bf16 or fp16, not {dtype}")
    n, index = blocks.numel(), cache._index
    ptr = _ints("blocks", blocks, n, index)
    with _On(index):
        if _checks.enabled():
            _run_check(_checks._in_range, "blocks", blocks, 0, cache.num_blocks, "cache blocks")
        shape = (n, cache.kv_heads, _BLOCK, cache.head_dim)
        k, v = blocks.new_empty(shape, dtype=dtype), blocks.new_empty(shape, dtype=dtype)
        rc = _native.cuda().ronn_kv8_read(_READ_CALL.pack(*cache._pointers(), ptr, k.data_ptr(), v.data_ptr(), cache._status, n, cache.num_blocks,
                                                          cache.kv_heads, cache.head_dim, _DTYPES[dtype], cache.code), _raw_stream(index))
    _check(rc, "kv8_read")
    return k, v


def _out(out: Optional[torch.Tensor], q: torch.Tensor, q_off: int, ld_q: int, read: int, rows: int, cols: int, index: int) -> int:
    """Row stride of the result, 0 where it is still to be made.  ``read``: columns of q from q_off on that the call reads."""
    if out is None:
        return 0
    ld = _rows16("out", out, cols, index, q.dtype)
    if out.shape[0] < rows:
        raise OperandError(f"out has {out.shape[0]} rows for {rows} of q")
    if rows and not _apart(q.data_ptr() + 2 * q_off, ld_q, read, out.data_ptr(), ld, cols, rows):
        raise OperandError("out overlaps the columns of q that are read")
    return ld


def _scale(scale: Optional[float], d: int) -> float:
    if scale is None:
        return d ** -0.5
    if not math.isfinite(scale):
        raise OperandError(f"scale must be finite, got {scale}")
    return float(scale)


def _attention(what, cache, q, q_off, ld, tables, table, bt_row, seq_start, q_len, kv_len, out, ld_o, n_seq, max_q, max_ctx, heads, causal,
               scale, check, k_off=0, v_off=0, slots=0, positions=0, turns=0, form=None) -> torch.Tensor:
    table_ld, table_rows, width = table
    kvh, d, index, longest = cache.kv_heads, cache.head_dim, cache._index, min(max_ctx, width * _BLOCK)
    with _On(index):
        if _checks.enabled():
            check()
        lib = _native.cuda()
        if out is None:
            out = q.new_empty((q.shape[0], heads * d))
        chunked = seq_start != 0 and scale > 0 and longest > 0 and (lib.ronn_kv8_chunk_form(n_seq, max_q, longest, heads, kvh, d) if form is None
                                                                    else form == "expanded")
        need = (lib.ronn_kv8_chunk_scratch(n_seq, longest, kvh, d) if chunked else
                lib.ronn_kv8_attention_scratch(n_seq, max_q, longest, heads, kvh, d))
        # this call's own: captured graphs and other streams share none
        scratch = q.new_empty((need,), dtype=torch.uint8) if need else None
        call = lib.ronn_kv8_chunk_attention if chunked else lib.ronn_kv8_attention
        rc = call(_ATTENTION_CALL.pack(
            q.data_ptr() + 2 * q_off, *cache._pointers(), tables.data_ptr(), bt_row, seq_start, q_len, kv_len, out.data_ptr(), slots, positions,
            turns, scratch.data_ptr() if need else 0, cache._status, ld, q.shape[0], cache.num_blocks, table_ld, ld_o or heads * d, need,
            table_rows, width, n_seq, max_q, longest, heads, kvh, d, causal, _DTYPES[q.dtype], cache.code, k_off, v_off, scale), _raw_stream(index))
    _check(rc, what)
    return out


def kv8_attention(q: torch.Tensor, cache: KV8Cache, block_tables: torch.Tensor, ctx_len: torch.Tensor, heads: int, max_ctx: int,
                  bt_row: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  append=None, rope=None) -> torch.Tensor:
    """Attention of single rows: row r of q ([rows, ld], head h at column h * head_dim) attends to the first ``ctx_len[r]`` keys
    that row ``bt_row[r]`` (default r) of the block tables lists.  Returns [rows, heads * head_dim], in ``out`` if given
    (which must not overlap q); a row with no keys gives zeros.  ``max_ctx``, the longest context, sizes the launch.
    ``append=(k_off, v_off, slots)`` (decode, one row per sequence): q is the fused QKV activation, and each row's new K and V
    first join the cache at the row's slot, which is that of key ``ctx_len[r] - 1``.  ``rope=(positions, base)`` with
    ``append``: q and the new k are rotated (q in memory stays as it is).  Where more than 16 heads share a cached head, the
    append is a launch of its own."""
    d, index = cache.head_dim, cache._index
    _heads(heads, cache)
    more = {}
    cols = heads * d
    if append is not None:
        k_off, v_off, slots = append
        _offset("k_off", k_off)
        _offset("v_off", v_off)
        cols = max(cols, max(k_off, v_off) + cache.kv_heads * d)
    elif rope is not None:
        raise OperandError("rope needs append: without it q is taken as it is")
    ld = _rows16("q", q, cols, index)
    rows = q.shape[0]
    table = _table(block_tables, rows if bt_row is None else 0, index)
    ctx = _ints("ctx_len", ctx_len, rows, index)
    at = 0 if bt_row is None else _ints("bt_row", bt_row, rows, index)
    if append is not None:
        more = dict(k_off=k_off, v_off=v_off, slots=_ints("slots", slots, rows, index))
        if rope is not None:
            angles = _turns(d, float(rope[1]))
            more.update(positions=_ints("positions", rope[0], rows, index), turns=angles[1])
    if max_ctx < 0:
        raise OperandError(f"max_ctx is {max_ctx}")
    if append is not None and heads // cache.kv_heads > _TILE:           # several tiles of a head's rows: one append before them
        factor = _scale(scale, d)
        _out(out, q, 0, ld, cols, rows, heads * d, index)
        turned = None if rope is None else q.new_empty((rows, k_off + cache.kv_heads * d))
        kv8_append(q, k_off, v_off, slots, cache, heads, *((rope[0], float(rope[1]), turned) if rope is not None else ()))
        return kv8_attention(q if rope is None else turned, cache, block_tables, ctx_len, heads, max_ctx, bt_row, out, factor)

    def check():
        _run_check(_checks.paged_attention, q, cache.k, block_tables, ctx_len, heads, d, int(max_ctx), bt_row,
                   append[2] if append else None, rope[0] if rope else None)
    return _attention("kv8_attention", cache, q, 0, ld, block_tables, table, at, 0, 0, ctx, out, _out(out, q, 0, ld, cols, rows, heads * d, index), rows,
                      1, int(max_ctx), heads, 0, _scale(scale, d), check, **more)


def kv8_prefill_attention(q: torch.Tensor, q_off: int, cache: KV8Cache, block_tables: torch.Tensor, seq_start: torch.Tensor,
                          q_len: torch.Tensor, kv_len: torch.Tensor, max_q_len: int, max_kv_len: int, heads: int,
                          causal: bool = True, bt_row: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                          scale: Optional[float] = None, form: Optional[str] = None) -> torch.Tensor:
    """Attention of query chunks (chunked prompts, prefix hits): sequence s has ``q_len[s]`` queries from row ``seq_start[s]`` of q
    on ([tokens, ld], head h at column q_off + h * head_dim) and attends to the ``kv_len[s]`` keys that row ``bt_row[s]``
    (default s) of the block tables lists; with ``causal`` its queries are the last positions of that context, and a query in
    front of the first key gives zeros.  The new tokens' K and V are in the cache already.  Returns [tokens, heads * head_dim], in
    ``out`` if given (which must not overlap these columns of q); rows that belong to no sequence are not written.  ``max_q_len``
    bounds the queries of a sequence, ``max_kv_len`` (in whole cache blocks) its keys; a sequence that passes them or the rows of q
    is left out and reported, its rows are not written.
    Few queries read the codes as they are ("direct"); for many the contexts are expanded to 16-bit values first and the
    tensor-core attention runs over those ("expanded", for a positive scale; fp16 keeps values within its range, and probabilities
    in the activations' type).  ``form`` names one, for measurements."""
    d, index = cache.head_dim, cache._index
    _heads(heads, cache)
    _offset("q_off", q_off)
    ld = _rows16("q", q, q_off + heads * d, index)
    tokens, n_seq = q.shape[0], seq_start.numel()
    table = _table(block_tables, n_seq if bt_row is None else 0, index)
    start, count, keys = (_ints(name, t, n_seq, index) for name, t in (("seq_start", seq_start), ("q_len", q_len), ("kv_len", kv_len)))
    at = 0 if bt_row is None else _ints("bt_row", bt_row, n_seq, index)
    if form not in (None, "direct", "expanded"):
        raise OperandError(f"form is 'direct' or 'expanded', not {form!r}")
    if max_q_len < 0 or max_kv_len < 0:
        raise OperandError(f"max_q_len is {max_q_len}, max_kv_len {max_kv_len}")

    def check():
        _run_check(_checks.sequences, tokens, seq_start, q_len, kv_len, False, block_tables.shape[1] * _BLOCK, True)
        rows_of = bt_row if bt_row is not None else torch.arange(n_seq, device=q.device, dtype=torch.int32)
        _run_check(_checks.paged_attention, kv_len[:n_seq, None], cache.k, block_tables, kv_len, 0, 0, block_tables.shape[1] * _BLOCK, rows_of)
    return _attention("kv8_prefill_attention", cache, q, q_off, ld, block_tables, table, at, start, count, keys, out,
                      _out(out, q, q_off, ld, heads * d, tokens, heads * d, index), n_seq, min(int(max_q_len), tokens), int(max_kv_len), heads, 1 if causal else 0,
                      _scale(scale, d), check, form=form)
