"""A paged 8-bit KV cache of several sequences: int8 codes with a scale for each
block of 32 tokens and kv head, the append that fills it, the attention that
reads it, and its page operations (plh_kv8_*, include/picolm_hip.h).  Pointers
are device addresses; everything is queued on the library stream."""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._native import PlhKv8Cache, PlhKv8Seqs, check, lib
from .device import DeviceBuffer
from .rope import Tables

BLOCK = 32


class Cache:
    """Codes and scales of n_pages pages; its own zeroed memory where none is given."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int,
                 page_tokens: int, codes: int | None = None, scales: int | None = None):
        self.desc = PlhKv8Cache(n_layers, n_kv_heads, head_dim, n_pages, page_tokens, codes,
                                scales)
        self.ref = C.byref(self.desc)
        self.kv_dim = n_kv_heads * head_dim
        self.code_bytes = lib.plh_kv8_code_bytes(self.ref)
        self.scale_bytes = lib.plh_kv8_scale_bytes(self.ref)
        if not self.code_bytes:
            raise ValueError(f"no 8-bit cache of {n_layers} layers, {n_kv_heads} kv heads of "
                             f"{head_dim}, {n_pages} pages of {page_tokens} tokens")
        self._own = []
        for name, nbytes in (("codes", self.code_bytes), ("scales", self.scale_bytes)):
            if getattr(self.desc, name) is None:
                buf = DeviceBuffer(nbytes)
                buf.zero()
                self._own.append(buf)
                setattr(self.desc, name, buf.ptr)

    def free(self) -> None:
        for b in self._own:
            b.free()
        self._own = []


class Sequences:
    """Page table, lengths and page counts; its own memory (no sequence holds a
    page) where none is given, which then needs n_pages."""

    def __init__(self, n_seqs: int, max_pages: int, n_pages: int = 0, table: int | None = None,
                 lens: int | None = None, refs: int | None = None):
        if (None in (table, lens, refs)) and not (table is lens is refs is None and n_pages > 0):
            raise ValueError("table, lens and refs are given together, or n_pages")
        self._own = []
        if table is None:
            for a in (np.full(n_seqs * max_pages, -1, np.int32), np.zeros(n_seqs, np.int32),
                      np.zeros(n_pages, np.int32)):
                self._own.append(DeviceBuffer.from_numpy(a))
            table, lens, refs = (b.ptr for b in self._own)
        self.desc = PlhKv8Seqs(n_seqs, max_pages, table, lens, refs)
        self.ref = C.byref(self.desc)

    def free(self) -> None:
        for b in self._own:
            b.free()
        self._own = []


def trim(cache: Cache, seqs: Sequences, keep: int) -> None:
    """len[s] = keep[s] where 0 <= keep[s] < len[s]; the pages behind are given back."""
    check(lib.plh_kv8_trim(cache.ref, seqs.ref, keep), "plh_kv8_trim")


def fork(cache: Cache, seqs: Sequences, parent: int) -> None:
    """Sequence s becomes what parent[s] was, sharing its pages (-1: stays)."""
    check(lib.plh_kv8_fork(cache.ref, seqs.ref, parent), "plh_kv8_fork")


def extend(cache: Cache, seqs: Sequences, add: int, status: int) -> None:
    """Room for add[s] more tokens of every sequence; status int32 [2], {0, 0} when done."""
    check(lib.plh_kv8_extend(cache.ref, seqs.ref, add, status), "plh_kv8_extend")


def compact(cache: Cache, seqs: Sequences, status: int) -> None:
    """Live pages to the lowest numbers; status int32 [2]: live pages, pages moved."""
    check(lib.plh_kv8_compact(cache.ref, seqs.ref, status), "plh_kv8_compact")


def append(cache: Cache, seqs: Sequences, layer: int, n_rows: int, row_start: int, k: int, v: int,
           k_stride: int = 0, v_stride: int = 0, rope: Tables | None = None,
           q: int | None = None, n_heads: int = 0, q_stride: int = 0, q_out: int | None = None,
           q_out_stride: int = 0) -> None:
    """Stores a batch's k (rotated by `rope`) and v rows, and rotates its q rows into q_out.
    Strides are in floats, 0 for rows that lie next to each other."""
    qd = n_heads * cache.desc.head_dim
    check(lib.plh_kv8_append(cache.ref, seqs.ref, layer, n_rows, row_start,
                             None if rope is None else rope.ref, q, n_heads, q_stride or qd,
                             q_out, q_out_stride or qd, k, k_stride or cache.kv_dim, v,
                             v_stride or cache.kv_dim),
          "plh_kv8_append")


def attend(cache: Cache, seqs: Sequences, layer: int, n_heads: int, n_rows: int, row_start: int,
           q: int, out: int, q_stride: int = 0, out_stride: int = 0) -> None:
    """Causal attention of a batch's (rotated) q rows over their sequences."""
    qd = n_heads * cache.desc.head_dim
    check(lib.plh_kv8_attn(cache.ref, seqs.ref, layer, n_heads, n_rows, row_start, q,
                           q_stride or qd, out, out_stride or qd),
          "plh_kv8_attn")


def fetch(cache: Cache, seqs: Sequences, layer: int, n_rows: int, row_start: int, k: int, v: int,
          k_stride: int = 0, v_stride: int = 0) -> None:
    """The stored values of a batch's rows."""
    check(lib.plh_kv8_fetch(cache.ref, seqs.ref, layer, n_rows, row_start, k,
                            k_stride or cache.kv_dim, v, v_stride or cache.kv_dim),
          "plh_kv8_fetch")
