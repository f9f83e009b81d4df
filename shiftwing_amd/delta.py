"""The gated delta rule of the Gated DeltaNet layer on packed sequences, driven
through the C ABI (coli_cuda_delta_{prompt,step}, include/shiftwing_moe.h Part 3).

Arrays come and go as float32; `kind` is the element type of q, k, v and the output
on the device ("f32", "f16", "bf16"); states are fp32, laid out as DeviceGdn's.
Every step runs in libshiftwing_moe.so.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from .abi import ColiDelta
from .paged import KINDS, from_kind, ints, packed, shaped, to_kind, word

__all__ = ["DeltaRule"]


class DeltaRule:
    """The recurrent states of `slots` sequences and the gates' parameters of one layer."""

    def __init__(self, be, *, kind, key_heads, value_heads, key_dim, value_dim, slots, a_log, dt_bias):
        self.be, self.kind, self.slots = be, kind, slots
        self.kh, self.vh, self.dk, self.dv = key_heads, value_heads, key_dim, value_dim
        shaped("a_log", a_log, (value_heads,))
        shaped("dt_bias", dt_bias, (value_heads,))
        self.a_log, self.dt_bias = (be.upload(np.asarray(x, np.float32)) for x in (a_log, dt_bias))
        self.write(np.zeros((slots, value_heads, key_dim, value_dim), np.float32))

    def write(self, state):
        shaped("state", state, (self.slots, self.vh, self.dk, self.dv))
        self.state = self.be.upload(np.ascontiguousarray(state, np.float32))

    def read(self):
        return self.be.download(self.state, (self.slots, self.vh, self.dk, self.dv), np.float32)

    def prompt(self, mix, a, b, start, slot):
        """coli_cuda_delta_prompt on rows q | k | v (mix, as the layer's convolution leaves them).  Rows of no
        sequence come back zero."""
        return self._call("coli_cuda_delta_prompt", mix, a, b, (start,), slot)

    def step(self, mix, a, b, slot):
        """coli_cuda_delta_step: one token a row, row r in slot[r]."""
        return self._call("coli_cuda_delta_step", mix, a, b, (), slot)

    def _call(self, name, mix, a, b, start, slot):
        be = self.be
        rows, width = np.shape(mix)
        kd = self.kh * self.dk
        slot, hs = ints(slot)
        start = [ints(s) for s in start]
        if start:
            packed(start[0][0], len(slot), rows)
        shaped("mix", mix, (rows if start else len(slot), 2 * kd + self.vh * self.dv))
        shaped("a", a, (rows, self.vh))
        shaped("b", b, (rows, self.vh))
        d = ColiDelta(KINDS[self.kind], self.kh, self.vh, self.dk, self.dv, self.slots, width, width, width)
        x = be.upload(to_kind(mix, self.kind))
        size = np.dtype(word(self.kind)).itemsize
        da, db = (be.upload(np.asarray(y, np.float32)) for y in (a, b))
        out = be.upload(np.zeros((rows, self.vh, self.dv), word(self.kind)))
        be.check(getattr(be.lib, name)(
            be.ctx, C.byref(d), out.p, x.p, C.c_void_p(x.ptr + kd * size), C.c_void_p(x.ptr + 2 * kd * size), da.p, db.p,
            self.a_log.p, self.dt_bias.p, self.state.p, self.state.p, *[p for _, p in start], hs, len(slot)), name)
        return from_kind(be.download(out, (rows, self.vh, self.dv), word(self.kind)), self.kind)
