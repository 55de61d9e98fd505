"""Rotary positions beyond the reference's tables: scaled frequencies, rotation
of part of a head (plh_rope_*, include/picolm_hip.h).  Pointers are device
addresses; everything is queued on the library stream."""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._native import PlhRope, PlhRopeSpec, check, lib

SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "bands": 3, "ramp": 4}


class Spec:
    """How far a pair turns per position (plh_rope_spec)."""

    def __init__(self, rot_dim: int, freq_base: float = 10000.0, scaling: str = "none",
                 factor: float = 1.0, trained_len: float = 0.0, low: float = 0.0,
                 high: float = 0.0, magnitude: float = 0.0):
        if scaling not in SCALINGS:
            raise ValueError(f"scaling {scaling!r}: one of {', '.join(SCALINGS)}")
        self.desc = PlhRopeSpec(rot_dim, SCALINGS[scaling], freq_base, factor, trained_len, low,
                                high, magnitude)

    def frequencies(self):
        """(theta [rot_dim/2] float64, magnitude); needs no device."""
        freq = np.empty(max(self.desc.rot_dim // 2, 1), np.float64)
        mag = C.c_double(0.0)
        check(lib.plh_rope_frequencies_host(C.byref(self.desc), freq.ctypes.data, C.byref(mag)),
              "plh_rope_frequencies_host")
        return freq, float(mag.value)


def make_tables(spec: Spec, first_pos: int, n_pos: int, cos: int, sin: int) -> None:
    """cos and sin [n_pos][rot_dim/2] fp32 of positions first_pos.. into device memory."""
    check(lib.plh_rope_tables(C.byref(spec.desc), first_pos, n_pos, cos, sin), "plh_rope_tables")


class Tables:
    """Device tables [n_pos][rot_dim/2] and how a head's pairs lie (plh_rope)."""

    def __init__(self, rope_type: int, rot_dim: int, n_pos: int, cos: int, sin: int):
        self.desc = PlhRope(rope_type, rot_dim, n_pos, cos, sin)
        self.ref = C.byref(self.desc)


def rotate(tables: Tables, n_rows: int, pos: int, head_dim: int, q: int | None, n_heads: int,
           q_stride: int, q_out: int | None, q_out_stride: int, k: int | None = None,
           n_kv_heads: int = 0, k_stride: int = 0, k_out: int | None = None,
           k_out_stride: int = 0) -> None:
    """Rotates rows of q and k (either may have 0 heads) at positions pos[row] (int32)."""
    check(lib.plh_rope_rows(tables.ref, n_rows, pos, head_dim, q, n_heads, q_stride, q_out,
                            q_out_stride, k, n_kv_heads, k_stride, k_out, k_out_stride),
          "plh_rope_rows")
