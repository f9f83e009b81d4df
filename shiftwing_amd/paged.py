"""A paged key-value cache on the device, driven through the C ABI
(coli_cuda_paged_{append,decode,prompt}, include/shiftwing_moe.h Part 3).

Arrays come and go as float32; `kind` is what the device holds ("f32", "f16",
"bf16").  Every step runs in libshiftwing_moe.so; nothing here computes but the
conversion of types.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from .abi import ColiPaged

__all__ = ["KINDS", "PagedCache", "from_kind", "shaped", "to_kind"]

KINDS = {"f32": 0, "f16": 1, "bf16": 2}


def to_kind(a, kind):
    """float32 values as the device holds them (bf16: rounded to nearest even, as 16-bit words)."""
    a = np.ascontiguousarray(a, np.float32)
    if kind == "f32":
        return a
    if kind == "f16":
        return a.astype(np.float16)
    u = a.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def from_kind(a, kind):
    if kind == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32)
    return a.astype(np.float32)


def shaped(what, a, shape):
    """ValueError unless array a has the shape; the C calls take the sizes on trust."""
    if np.shape(a) != tuple(shape):
        raise ValueError(f"{what} has shape {np.shape(a)}, not {tuple(shape)}")


def packed(start, sequences, rows):
    """ValueError unless start names rows of that many sequences within the tensors' rows."""
    if len(start) != sequences + 1 or (sequences and start[-1] > rows):
        raise ValueError(f"start of {len(start)} entries up to {start[-1] if len(start) else 0} for {sequences} sequences "
                         f"in {rows} rows")


def word(kind):
    """The numpy type of one element."""
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[kind]


def ints(a):
    """A host array of C ints; ValueError where the values are none, or not in a row."""
    given = np.asarray(a)
    with np.errstate(invalid="ignore"):
        a = np.ascontiguousarray(given.astype(np.int32))
    if given.ndim != 1 or not np.array_equal(given, a):
        raise ValueError(f"not a row of C ints: {given}")
    return a, C.c_void_p(a.ctypes.data)


class PagedCache:
    """Key and value pools of `pages` pages and the page table of `sequences` sequences."""

    def __init__(self, be, *, kind, query_heads, kv_heads, head_dim, page_size, pages, table_pages, sequences):
        self.be, self.kind, self.sequences = be, kind, sequences
        self.nh, self.nkv, self.hd, self.page_size = query_heads, kv_heads, head_dim, page_size
        self.shape = (pages, page_size, kv_heads, head_dim)
        self.c = ColiPaged(KINDS[kind], query_heads, kv_heads, head_dim, page_size, pages, table_pages,
                           page_size * kv_heads * head_dim)
        self.k_pool = be.upload(np.zeros(self.shape, word(kind)))
        self.v_pool = be.upload(np.zeros(self.shape, word(kind)))
        self.set_table(np.full((sequences, table_pages), -1, np.int32))

    def set_table(self, table):
        """Page ids [sequences][table_pages]; ids outside the pool name no page."""
        shaped("table", table, (self.sequences, self.c.table_pages))
        self.table = self.be.upload(np.ascontiguousarray(table, np.int32))

    def _put(self, a):
        return self.be.upload(to_kind(a, self.kind))

    def _rows(self, a, n):
        return from_kind(self.be.download(a, (n, self.nh, self.hd), word(self.kind)), self.kind)

    def append(self, start, length, k, v, q=None, *, q_norm=None, k_norm=None, eps=1e-6, rotary_dim=0, theta=1e4):
        """coli_cuda_paged_append: k and v [rows][kv_heads][head_dim] into their pages; the normalised and
        rotated queries come back where q [rows][query_heads][head_dim] is given."""
        be = self.be
        start, hs = ints(start)
        length, hl = ints(length)
        rows = np.shape(k)[0]
        self._fits(length)
        packed(start, len(length), rows)
        for what, x, heads in (("k", k, self.nkv), ("v", v, self.nkv), ("q", q, self.nh)):
            if x is not None:
                shaped(what, x, (rows, heads, self.hd))
        for what, x in (("q_norm", q_norm), ("k_norm", k_norm)):
            if x is not None:
                shaped(what, x, (self.hd,))
        dk, dv = self._put(k), self._put(v)
        dq = self._put(q) if q is not None else None
        out = be.upload(np.zeros(np.shape(q), word(self.kind))) if q is not None else None
        norms = [be.upload(np.asarray(w, np.float32)) if w is not None else None for w in (q_norm, k_norm)]
        row = self.nkv * self.hd
        be.check(be.lib.coli_cuda_paged_append(
            be.ctx, C.byref(self.c), self.k_pool.p, self.v_pool.p, self.table.p, hs, hl, len(length),
            out.p if out else None, dq.p if dq else None, self.nh * self.hd, self.hd, dk.p, row, dv.p, row,
            *[w.p if w else None for w in norms], eps, rotary_dim, theta), "coli_cuda_paged_append")
        if out is None:
            be.sync()
            return None
        return self._rows(out, np.shape(q)[0])

    def decode(self, q, length, scale, gate=None):
        """coli_cuda_paged_decode: one new token a sequence, q (and gate) [sequences][query_heads][head_dim]."""
        return self._attend("coli_cuda_paged_decode", q, (), length, scale, gate)

    def prompt(self, q, start, length, scale, gate=None):
        """coli_cuda_paged_prompt: packed rows, the last start[s + 1] - start[s] positions of each sequence.
        Rows of no sequence come back zero."""
        return self._attend("coli_cuda_paged_prompt", q, (start,), length, scale, gate)

    def _fits(self, length):
        if len(length) > self.sequences:
            raise ValueError(f"{len(length)} sequences, more than the table's {self.sequences}")

    def _attend(self, name, q, start, length, scale, gate):
        be = self.be
        rows = np.shape(q)[0]
        length, hl = ints(length)
        start = [ints(s) for s in start]
        self._fits(length)
        if start:
            packed(start[0][0], len(length), rows)
        shaped("q", q, (rows if start else len(length), self.nh, self.hd))
        if gate is not None:
            shaped("gate", gate, np.shape(q))
        dq, dg = self._put(q), self._put(gate) if gate is not None else None
        out = be.upload(np.zeros((rows, self.nh, self.hd), word(self.kind)))
        be.check(getattr(be.lib, name)(
            be.ctx, C.byref(self.c), out.p, dq.p, dg.p if dg else None, self.nh * self.hd, self.hd, self.k_pool.p,
            self.v_pool.p, self.table.p, *[p for _, p in start], hl, len(length), scale), name)
        return self._rows(out, rows)

    def read(self):
        """Both pools, [pages][page_size][kv_heads][head_dim]."""
        return tuple(from_kind(self.be.download(p, self.shape, word(self.kind)), self.kind) for p in (self.k_pool, self.v_pool))

    def write(self, k, v):
        """Both pools whole."""
        shaped("k", k, self.shape)
        shaped("v", v, self.shape)
        self.k_pool, self.v_pool = self._put(k), self._put(v)
