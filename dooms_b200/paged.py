"""Python face of the operators of a serving step over a key / value cache in pages (include/dooms_cuda.h: dooms_cuda_paged_cache): rotary positions with the cache
write, attention of single tokens and of packed prompts over the pages, and sampling. Tensors are device tensors (torch's); outputs are written in place and nothing is
allocated. `stream` is a cudaStream_t as an integer (0: the default stream); without one a call goes to torch's current stream, as the tensors' own work does."""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import torch

from . import _lib as L

_F32, _F16, _I32 = torch.float32, torch.float16, torch.int32
_DTYPES = {_F32: L.F32, _F16: L.F16}


def _pointer(name: str, t, dtype, shape: tuple) -> int:
    """The tensor's address, if it is contiguous and of that dtype and shape."""
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise L.DoomsError(L.INVALID_ARGUMENT, f"{name}: expected a contiguous {dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


_MOST = (1 << 31) - 1


def _int32(name: str, *values: int) -> None:
    """That the values fit the C arguments, which would take the low 32 bits of one that does not. (Rows of queries need no such check: 2^31 of them fit no GPU.)"""
    if not all(-_MOST <= v <= _MOST for v in values):
        raise L.DoomsError(L.INVALID_ARGUMENT, f"{name}: {values} does not fit 32 bits")


def _dtype(name: str, t) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise L.DoomsError(L.UNSUPPORTED, f"{name}: float32 or float16 expected, got {t.dtype}")
    return dt


def _scratch(t) -> tuple[int, int]:
    """The scratch tensor's address and bytes."""
    if not t.is_contiguous():
        raise L.DoomsError(L.INVALID_ARGUMENT, "scratch: expected a contiguous tensor")
    return t.data_ptr(), t.numel() * t.element_size()


def _stream(stream: int | None) -> int:
    if stream is None:      # (where torch has not begun to use a GPU there is no other stream than the default one)
        return torch.cuda.current_stream().cuda_stream if torch.cuda.is_initialized() else 0
    return stream


class PagedCache:
    """Pools of keys and values, f16 [n_pages][page_size][n_head_kv][head_dim], and the pages of every sequence, int32 [n_sequences][max_pages]. The object refers to the
    tensors' memory (and keeps them alive); their contents may change between calls, the page table's too."""

    def __init__(self, keys, values, page_table):
        if len(keys.shape) != 4 or len(page_table.shape) != 2:
            raise L.DoomsError(L.INVALID_ARGUMENT, "pools of four dimensions and a page table of two expected")
        n_pages, page_size, n_head_kv, head_dim = keys.shape
        _int32("pools and page table", *keys.shape, *page_table.shape)
        c = L.PagedCache()
        c.struct_size = C.sizeof(L.PagedCache)
        c.keys, c.values = _pointer("keys", keys, _F16, tuple(keys.shape)), _pointer("values", values, _F16, tuple(keys.shape))
        c.page_table = _pointer("page_table", page_table, _I32, tuple(page_table.shape))
        c.n_pages, c.page_size, c.n_head_kv, c.head_dim = n_pages, page_size, n_head_kv, head_dim
        c.n_sequences, c.max_pages = page_table.shape
        self._c, self._ref, self._keep, self._ropes = c, C.byref(c), (keys, values, page_table), {}

    def scratch_bytes(self, n_head: int) -> int:
        """Bytes of scratch memory that attention and attention_prompt take, for any number of rows."""
        _int32("n_head", n_head)
        n = L.lib().dooms_cuda_attention_paged_scratch_bytes(n_head, self._c.n_head_kv, self._c.head_dim)
        if n == 0:
            raise L.DoomsError(L.INVALID_ARGUMENT, f"{n_head} query heads on {self._c.n_head_kv} key / value heads of {self._c.head_dim}")
        return n

    def rope_store(self, qkv, sequence, at, positions, q, base: float, neox: bool, sections: Sequence[int] | None = None, stream: int | None = None) -> None:
        """Rows [n][(n_head + 2 n_head_kv) head_dim] of f32 (rows may be further apart): turned queries into q [n][n_head][head_dim] (f32 or f16), turned keys and the values
        into position at[r] of sequence[r] (negative: an idle row). positions: int32 [n_axes][n]; sections: rotary pairs per axis (one axis: all of them)."""
        c, (n, n_head, head_dim) = self._c, q.shape
        sections = (head_dim // 2,) if sections is None else tuple(sections)
        if not 1 <= len(sections) <= 4:
            raise L.DoomsError(L.INVALID_ARGUMENT, "sections: 1 to 4 axes")
        rope = self._ropes.get((base, neox, sections))      # (the argument struct: a program has one or two)
        if rope is None:
            _int32("sections", *sections)
            rope = self._ropes[base, neox, sections] = L.Rope(C.sizeof(L.Rope), base, int(neox), len(sections), (C.c_int32 * 4)(*sections))
        if qkv.dtype is not _F32 or tuple(qkv.shape) != (n, (n_head + 2 * c.n_head_kv) * head_dim) or qkv.stride(1) != 1:
            raise L.DoomsError(L.INVALID_ARGUMENT, f"qkv: float32 rows of {(n_head + 2 * c.n_head_kv) * head_dim} values expected, one for each of the {n} rows of q")
        stride = qkv.stride(0) if n > 1 else qkv.shape[1]
        L.check(L.lib().dooms_cuda_rope_store_paged(self._ref, C.byref(rope), qkv.data_ptr(), stride, n_head, n, _pointer("sequence", sequence, _I32, (n,)),
                                                    _pointer("at", at, _I32, (n,)), _pointer("positions", positions, _I32, (len(sections), n)),
                                                    _dtype("q", q), _pointer("q", q, q.dtype, (n, n_head, c.head_dim)), _stream(stream)))

    def attention(self, q, sequence, lengths, max_length: int, out, scratch, scale: float = 0.0, stream: int | None = None) -> None:
        """One new token per row: q, out [n][n_head][head_dim], both f32 or both f16; row r sees the first lengths[r] <= max_length positions of sequence[r]."""
        n, n_head = q.shape[0], q.shape[1]
        shape = (n, n_head, self._c.head_dim)
        if not 0 <= max_length <= _MOST:      # (no sequence is longer; a larger bound means the same)
            max_length = max(-1, min(max_length, _MOST))
        L.check(L.lib().dooms_cuda_attention_paged(self._ref, _dtype("q", q), _pointer("q", q, q.dtype, shape), _pointer("sequence", sequence, _I32, (n,)),
                                                   _pointer("lengths", lengths, _I32, (n,)), max_length, _pointer("out", out, q.dtype, shape), n_head, n, scale,
                                                   *_scratch(scratch), _stream(stream)))

    def attention_prompt(self, q, sequence, start, lengths, out, scratch, scale: float = 0.0, stream: int | None = None) -> None:
        """Packed prompts, causal: q, out f16 [rows][n_head][head_dim]; prompt i has rows start[i] .. start[i + 1] - 1, the last of lengths[i] positions of sequence[i]."""
        rows, n_head = q.shape[0], q.shape[1]
        shape, n = (rows, n_head, self._c.head_dim), sequence.shape[0]
        if n > _MOST:
            _int32("sequence", n)
        L.check(L.lib().dooms_cuda_attention_prompt_paged(self._ref, _pointer("q", q, _F16, shape), _pointer("sequence", sequence, _I32, (n,)),
                                                          _pointer("start", start, _I32, (n + 1,)), _pointer("lengths", lengths, _I32, (n,)),
                                                          _pointer("out", out, _F16, shape), n_head, n, rows, scale, *_scratch(scratch), _stream(stream)))


def sample_rows(logits, uniform, tokens, probability=None, temperature=None, top_k=None, top_p=None, min_p=None, stream: int | None = None) -> None:
    """tokens[r] (int32) from logits [rows][n] (f32; rows may be further apart) and uniform[r] in [0, 1); the filters are f32 (top_k: int32) tensors of one value per row, or
    None for off (temperature: 1). See dooms_cuda_sample_rows."""
    rows, n = logits.shape
    if rows > _MOST or n > _MOST:
        _int32("logits", rows, n)
    if logits.dtype is not _F32 or (n > 1 and logits.stride(1) != 1):
        raise L.DoomsError(L.INVALID_ARGUMENT, "logits: rows of float32 expected")

    def row(name, t, dtype=_F32):
        return None if t is None else _pointer(name, t, dtype, (rows,))
    L.check(L.lib().dooms_cuda_sample_rows(logits.data_ptr(), logits.stride(0) if rows > 1 else n, rows, n, row("temperature", temperature), row("top_k", top_k, _I32),
                                           row("top_p", top_p), row("min_p", min_p), row("uniform", uniform), row("tokens", tokens, _I32), row("probability", probability),
                                           _stream(stream)))
