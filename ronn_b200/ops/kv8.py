"""The paged KV cache in 8 bits and the attention that reads it.

Layout and mathematics: ``csrc/kernels/kv8.cuh``.  Codes are int8 or e4m3, [num_blocks, kv_heads, 16, head_dim], with one
fp32 scale for each (block, head), a power of two; keys and values have scales of their own.  A block begins when its slot
0 is written; tokens that join it later can raise its scale, and then the codes below them are rounded once more.  A token
with a value that is not finite makes its block and head read as NaN until the block begins again.

Page numbers, slots and table rows come from device memory.  One that lies outside the cache is not accessed: the key it
stands for is left out, the kernel sets the device's status word, and ``check_status`` raises.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from functools import lru_cache
from typing import Optional, Tuple

import torch

from .. import _native
from . import checks as _checks
from .kernels import KernelError, OperandError, _DT, _check, _ptr, _run_check, status_word

_CODES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_PRECISIONS = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_BLOCK = 16


def _aligned(t: torch.Tensor) -> bool:
    return t.data_ptr() % 16 == 0


class KV8Cache:
    """Codes and scales of one layer's keys and values, or of one rank's share of them."""
    __slots__ = ("k", "v", "k_scale", "v_scale", "num_blocks", "kv_heads", "head_dim", "code")

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
            if not c.is_contiguous() or not _aligned(c) or c.device != k.device:
                raise OperandError("cache codes must be contiguous from a 16-byte boundary, keys and values on one device")
        if k.shape[0] * _BLOCK > 2 ** 31 - 1:
            raise OperandError(f"cache slots are 32-bit numbers; {k.shape[0]} blocks have more")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_blocks, self.kv_heads, _, self.head_dim = k.shape
        self.code = _CODES[k.dtype]

    @classmethod
    def alloc(cls, num_blocks: int, kv_heads: int, head_dim: int, precision: str = "int8", device="cuda") -> "KV8Cache":
        """An empty cache: every block reads as zeros."""
        if precision not in _PRECISIONS:
            raise OperandError(f"cache precision is 'int8' or 'fp8', got '{precision}'")
        shape = (num_blocks, kv_heads, _BLOCK, head_dim)
        mk = lambda: torch.zeros(shape, dtype=torch.uint8, device=device).view(_PRECISIONS[precision])
        return cls(mk(), mk(), torch.zeros(shape[:2], device=device), torch.zeros(shape[:2], device=device))

    @property
    def device(self) -> torch.device:
        return self.k.device

    @property
    def dtype(self) -> torch.dtype:
        return self.k.dtype


def _guard(device: torch.device):
    """The operands' device for the launch, where it is not the current one."""
    if device.type != "cuda":
        raise OperandError(f"the 8-bit cache kernels run on a CUDA device, got a cache on {device}")
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _rows16(what: str, t: torch.Tensor, cols: int, device: torch.device, dtype: Optional[torch.dtype] = None) -> int:
    """Row stride of a 16-bit matrix whose rows the kernels read or write in 16-byte pieces."""
    if t.dim() != 2 or t.dtype not in (torch.bfloat16, torch.float16) or t.device != device or (dtype is not None and t.dtype != dtype):
        raise OperandError(f"{what} must be a matrix of {dtype or 'bf16 or fp16'} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.shape[1] < cols:
        raise OperandError(f"{what} has {t.shape[1]} columns, {cols} are read or written")
    ld = t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8
    if t.stride(1) != 1 and t.shape[1] > 1 or ld % 8 or ld < cols or not _aligned(t):
        raise OperandError(f"{what} must have unit column stride and rows that start on 16-byte boundaries and do not overlap, got "
                           f"strides {t.stride()}")
    return ld


def _ints(what: str, t: Optional[torch.Tensor], n: int, device: torch.device) -> None:
    if t is not None and (t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or t.dim() != 1 or t.numel() < n):
        raise OperandError(f"{what} must be {n} contiguous int32 values on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _table(block_tables: torch.Tensor, device: torch.device) -> int:
    t = block_tables
    if t.dim() != 2 or t.dtype != torch.int32 or t.device != device or (t.stride(1) != 1 and t.shape[1] > 1) or t.shape[1] < 1:
        raise OperandError(f"block_tables must be an int32 matrix with unit column stride on {device}, got {t.dtype} {tuple(t.shape)}")
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if ld < t.shape[1]:
        raise OperandError(f"rows of block_tables overlap (strides {t.stride()})")
    return ld


def _heads(heads: int, cache: KV8Cache) -> None:
    if heads <= 0 or heads % cache.kv_heads or heads > 65535:
        raise OperandError(f"{heads} heads do not divide into {cache.kv_heads} cached heads")


def _offset(what: str, off: int) -> None:
    if off < 0 or off % 8:
        raise OperandError(f"{what} is {off}; heads must start at a multiple of 8 columns")


@lru_cache(maxsize=64)
def _turns(head_dim: int, base: float):
    """base^(-2j/d) / (2 pi) for each channel pair, as 64-bit fractions of a turn."""
    if not (base > 0.0 and math.isfinite(base)):
        raise OperandError(f"rotary base must be a positive number, got {base}")
    f = [int(base ** (-2.0 * j / head_dim) / (2.0 * math.pi) * 2.0 ** 64) & (2 ** 64 - 1) for j in range(head_dim // 2)]
    return (ctypes.c_ulonglong * len(f))(*f)


def kv8_append(qkv: torch.Tensor, k_off: int, v_off: int, slots: torch.Tensor, cache: KV8Cache, heads: int,
               positions: Optional[torch.Tensor] = None, rope_base: float = 0.0, rotated: Optional[torch.Tensor] = None) -> None:
    """Put the K and V columns of a fused QKV activation [tokens, ld] into their cache slots (int32 [tokens], -1: not cached).
    The tokens of one block stand in consecutive rows with rising slots, as a scheduler lists them.  With ``positions`` and
    ``rope_base`` > 0, q and k are rotated first; the rotated columns go to ``rotated`` (laid out as qkv; default: qkv itself)."""
    d, kvh, dev = cache.head_dim, cache.kv_heads, cache.device
    _heads(heads, cache)
    rope = positions is not None and rope_base > 0
    if not rope and rotated is not None:
        raise OperandError("rotated needs positions and a rotary base")
    _offset("k_off", k_off)
    _offset("v_off", v_off)
    ld = _rows16("qkv", qkv, max(k_off, v_off) + kvh * d, dev)
    rot = qkv if rotated is None else rotated
    ld_rot = _rows16("rotated", rot, max(heads * d, k_off + kvh * d), dev, qkv.dtype) if rope else 0
    if rope and k_off < heads * d:
        raise OperandError(f"k_off {k_off} lies inside the {heads} heads of q")
    tokens = qkv.shape[0]
    if rope and rot.shape[0] < tokens:
        raise OperandError(f"rotated has {rot.shape[0]} rows for {tokens} tokens")
    _ints("slots", slots, tokens, dev)
    if rope:
        _ints("positions", positions, tokens, dev)
    with _guard(dev):
        if _checks.enabled():
            _run_check(_checks.kv8_append, qkv, slots, cache.k, positions)
        rc = _native.cuda().ronn_kv8_append(qkv.data_ptr(), ld, rot.data_ptr() if rope else None, ld_rot, k_off, v_off,
                                            slots.data_ptr(), positions.data_ptr() if rope else None,
                                            _turns(d, float(rope_base)) if rope else None, cache.k.data_ptr(), cache.v.data_ptr(),
                                            cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), cache.num_blocks, tokens, heads, kvh,
                                            d, _DT[qkv.dtype], cache.code, status_word(dev).data_ptr(),
                                            torch.cuda.current_stream().cuda_stream)
    _check(rc, "kv8_append")


def kv8_read(cache: KV8Cache, blocks: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of whole cache blocks (int32 [n]) as two [n, kv_heads, 16, head_dim] tensors."""
    dev = cache.device
    if dtype not in (torch.bfloat16, torch.float16):
        raise OperandError(f"kv8_read gives bf16 or fp16, not {dtype}")
    n = blocks.numel()
    _ints("blocks", blocks, n, dev)
    with _guard(dev):
        if _checks.enabled():
            _run_check(_checks._in_range, "blocks", blocks, 0, cache.num_blocks, "cache blocks")
        k = torch.empty((n, cache.kv_heads, _BLOCK, cache.head_dim), dtype=dtype, device=dev)
        v = torch.empty_like(k)
        rc = _native.cuda().ronn_kv8_read(cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
                                          blocks.data_ptr(), k.data_ptr(), v.data_ptr(), n, cache.num_blocks, cache.kv_heads,
                                          cache.head_dim, _DT[dtype], cache.code, status_word(dev).data_ptr(),
                                          torch.cuda.current_stream().cuda_stream)
    _check(rc, "kv8_read")
    return k, v


def _out(out: Optional[torch.Tensor], q: torch.Tensor, rows: int, cols: int) -> Tuple[torch.Tensor, int]:
    if out is None:
        out = torch.empty((rows, cols), dtype=q.dtype, device=q.device)
        return out, cols
    ld = _rows16("out", out, cols, q.device, q.dtype)
    if out.shape[0] < rows:
        raise OperandError(f"out has {out.shape[0]} rows for {rows} of q")
    return out, ld


def _scale(scale: Optional[float], d: int) -> float:
    s = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not math.isfinite(s):
        raise OperandError(f"scale must be finite, got {s}")
    return s


def _attention(q_ptr, q, ld, rows, cache, tables, table_ld, bt_row, seq_start, q_len, kv_len, out, ld_o, n_seq, max_q, max_ctx, heads, causal,
               scale, append=None, rope=None) -> int:
    lib, dev, d = _native.cuda(), cache.device, cache.head_dim
    max_ctx = min(max_ctx, tables.shape[1] * _BLOCK)
    need = lib.ronn_kv8_attention_scratch(n_seq, max_q, max_ctx, heads, cache.kv_heads, d)
    scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None       # this call's own: graphs share none
    return lib.ronn_kv8_attention(q_ptr, ld, rows, cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
                                  cache.num_blocks, tables.data_ptr(), table_ld, tables.shape[0], tables.shape[1], _ptr(bt_row),
                                  _ptr(seq_start), _ptr(q_len), kv_len.data_ptr(), out.data_ptr(), ld_o, n_seq, max_q, max_ctx, heads,
                                  cache.kv_heads, d, causal, scale, _DT[q.dtype], cache.code, append[0] if append else 0,
                                  append[1] if append else 0, append[2].data_ptr() if append else None, rope[0].data_ptr() if rope else None,
                                  _turns(d, float(rope[1])) if rope else None, _ptr(scratch), need, status_word(dev).data_ptr(),
                                  torch.cuda.current_stream().cuda_stream)


def kv8_attention(q: torch.Tensor, cache: KV8Cache, block_tables: torch.Tensor, ctx_len: torch.Tensor, heads: int, max_ctx: int,
                  bt_row: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  append=None, rope=None) -> torch.Tensor:
    """Attention of single rows: row r of q ([rows, ld], head h at column h * head_dim) attends to the first ``ctx_len[r]`` keys
    that row ``bt_row[r]`` (default r) of the block tables lists.  Returns [rows, heads * head_dim]; a row with no keys gives
    zeros.  ``max_ctx``, the longest context, sizes the launch.
    ``append=(k_off, v_off, slots)`` (decode, one row per sequence): q is the fused QKV activation, and each row's new K and V
    first join the cache at the row's slot, which is that of key ``ctx_len[r] - 1``.  ``rope=(positions, base)`` with
    ``append``: q and the new k are rotated (q in memory stays as it is)."""
    d, dev, rows = cache.head_dim, cache.device, q.shape[0] if q.dim() else 0
    _heads(heads, cache)
    if rope is not None and append is None:
        raise OperandError("rope needs append: without it q is taken as it is")
    ld = _rows16("q", q, heads * d if append is None else max(heads * d, max(append[0], append[1]) + cache.kv_heads * d), dev)
    table_ld = _table(block_tables, dev)
    _ints("ctx_len", ctx_len, rows, dev)
    _ints("bt_row", bt_row, rows, dev)
    if bt_row is None and block_tables.shape[0] < rows:
        raise OperandError(f"block_tables has {block_tables.shape[0]} rows for {rows} of q")
    if append is not None:
        _ints("slots", append[2], rows, dev)
        _offset("k_off", append[0])
        _offset("v_off", append[1])
    if rope is not None:
        _ints("positions", rope[0], rows, dev)
        _turns(d, float(rope[1]))
    if int(max_ctx) < 0:
        raise OperandError(f"max_ctx is {max_ctx}")
    sc = _scale(scale, d)
    with _guard(dev):
        if _checks.enabled():
            _run_check(_checks.paged_attention, q, cache.k, block_tables, ctx_len, heads, d, int(max_ctx), bt_row,
                       append[2] if append else None, rope[0] if rope else None)
        out, ld_o = _out(out, q, rows, heads * d)
        rc = _attention(q.data_ptr(), q, ld, rows, cache, block_tables, table_ld, bt_row, None, None, ctx_len, out, ld_o, rows, 1,
                        int(max_ctx), heads, 0, sc, append, rope)
    _check(rc, "kv8_attention")
    return out


def kv8_prefill_attention(q: torch.Tensor, q_off: int, cache: KV8Cache, block_tables: torch.Tensor, seq_start: torch.Tensor,
                          q_len: torch.Tensor, kv_len: torch.Tensor, max_q_len: int, max_kv_len: int, heads: int,
                          causal: bool = True, bt_row: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                          scale: Optional[float] = None) -> torch.Tensor:
    """Attention of query chunks (chunked prompts, prefix hits): sequence s has ``q_len[s]`` queries from row ``seq_start[s]`` of q
    on ([tokens, ld], head h at column q_off + h * head_dim) and attends to the ``kv_len[s]`` keys that row ``bt_row[s]``
    (default s) of the block tables lists; with ``causal`` its queries are the last positions of that context, and a query in
    front of the first key gives zeros.  The new tokens' K and V are in the cache already.  Returns [tokens, heads * head_dim];
    rows that belong to no sequence are not written.  ``max_q_len`` and ``max_kv_len`` bound the lengths."""
    d, dev, tokens = cache.head_dim, cache.device, q.shape[0] if q.dim() else 0
    _heads(heads, cache)
    _offset("q_off", q_off)
    ld = _rows16("q", q, q_off + heads * d, dev)
    table_ld = _table(block_tables, dev)
    n_seq = seq_start.numel()
    for name, t in (("seq_start", seq_start), ("q_len", q_len), ("kv_len", kv_len), ("bt_row", bt_row)):
        _ints(name, t, n_seq, dev)
    if bt_row is None and block_tables.shape[0] < n_seq:
        raise OperandError(f"block_tables has {block_tables.shape[0]} rows for {n_seq} sequences")
    if int(max_q_len) < 0 or int(max_kv_len) < 0:
        raise OperandError(f"max_q_len is {max_q_len}, max_kv_len {max_kv_len}")
    sc = _scale(scale, d)
    with _guard(dev):
        if _checks.enabled():
            _run_check(_checks.sequences, tokens, seq_start, q_len, kv_len, False, block_tables.shape[1] * _BLOCK)
            rows_of = bt_row if bt_row is not None else torch.arange(n_seq, device=dev, dtype=torch.int32)
            _run_check(_checks.paged_attention, kv_len[:n_seq, None], cache.k, block_tables, kv_len, 0, 0,
                       block_tables.shape[1] * _BLOCK, rows_of)
        out, ld_o = _out(out, q, tokens, heads * d)
        rc = _attention(q.data_ptr() + 2 * q_off, q, ld, tokens, cache, block_tables, table_ld, bt_row, seq_start, q_len, kv_len, out, ld_o,
                        n_seq, int(max_q_len), int(max_kv_len), heads, 1 if causal else 0, sc)
    _check(rc, "kv8_prefill_attention")
    return out
