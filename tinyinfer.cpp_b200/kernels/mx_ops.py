"""Bindings of the kernels in ``csrc/mx_*.cu`` (library ``mx``): rows and weights in the microscaled format, 4 or 8
bits an element and a power-of-two scale for every 32 of a row (the OCP MX formats MXFP4 and MXFP8 with e4m3).

``CudaOps`` inherits these methods; the library is built when one of them is first called, so an engine with bfloat16
weights never compiles it.

mx_quantize(x, bits, out=None)                       rows of float32 or bfloat16 into the format
mx_dequantize(q, dtype, out=None)                    the numbers it stands for
mx_rmsnorm(x, weight, eps, bits, delta, out=None)    x += delta; RMS norm of x in the format
mx_linear(a, w, out, accumulate=False)               out (+)= a @ w.T in float32, w of 4 bits
mx_linear_glu(a, w, cols, bits, out=None)            silu(a @ gate.T) * (a @ up.T) in the format
mx_pack_linear(w) / mx_pack_gate_up(gate, up)        weights of those products

Rows are padded with zeros to whole chunks of 128 elements.  ``MxRows.codes`` is ``[rows, padded * bits / 8]`` bytes (two
4-bit codes a byte, the even element low); ``MxRows.scales`` is ``[rows / 128 rounded up, padded / 128, 512]`` bytes, the
scales of 128 rows and one chunk as ``[row % 32][row / 32 % 4][block % 4]``, each ``s`` standing for 2^(s - 127), 255 for NaN.
A block's scale is the largest power of two in its largest magnitude, over the element type's own (4 or 256); elements round
to nearest even and saturate (at 6 or 448), and a block with an infinity or a NaN becomes NaN.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from .build import load_library

_CODE = {torch.float32: 0, torch.bfloat16: 1}
_vp, _i, _f, _ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong

BLOCK, CHUNK, TILE_ROWS, TILE_BYTES = 32, 128, 128, 512


class MxRows(NamedTuple):
    """Rows in the microscaled format.  ``settled``: the caller knows that whatever wrote them finished before the launch in
    front of the call they are handed to (weights made when a model was loaded), so that a product may fetch them while
    that launch still runs."""
    codes: torch.Tensor
    scales: torch.Tensor
    bits: int
    cols: int
    settled: bool = False

    @property
    def rows(self) -> int:
        return self.codes.shape[0]


def _padded(cols: int) -> int:
    return -(-cols // CHUNK) * CHUNK


class MxOps:
    _mx_lib = None

    @property
    def mx(self):
        """The kernels of the microscaled format, built and loaded when first needed."""
        if self._mx_lib is None:
            b = load_library("mx")
            b.ti_last_error.restype = ctypes.c_char_p
            b.ti_mx_quantize.argtypes = [_vp, _i, _ll, _i, _i, _i, _i, _vp, _vp, _vp]
            b.ti_mx_dequantize.argtypes = [_vp, _vp, _i, _i, _i, _i, _vp, _i, _ll, _vp]
            b.ti_mx_rmsnorm.argtypes = [_vp, _ll, _vp, _i, _ll, _vp, _i, _i, _i, _f, _i, _vp, _vp, _vp]
            b.ti_mx_gemm.argtypes = [_vp, _vp, _i, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp, _vp]
            b.ti_mx_gemm_glu.argtypes = [_vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp, _vp]
            self._mx_lib = b
        return self._mx_lib

    @staticmethod
    def _mx_need(cond: bool, msg: str) -> None:
        if not cond:
            from .cuda_ops import KernelError
            raise KernelError(msg)

    def _mx_check(self, q: MxRows, who: str) -> int:
        """The padded row length of rows that are laid out as they have to be."""
        codes, scales, kp = q.codes, q.scales, _padded(q.cols)
        if not (q.cols >= 1 and q.bits in (4, 8) and codes.dtype == scales.dtype == torch.uint8 and codes.dim() == 2
                and codes.shape[1] * 8 == kp * q.bits and codes.is_contiguous() and scales.is_contiguous()
                and scales.shape == (-(-codes.shape[0] // TILE_ROWS), kp // CHUNK, TILE_BYTES)
                and codes.device == self._mx_device and scales.device == self._mx_device):
            self._mx_need(False, f"{who}: not {q.cols} columns of {q.bits} bits with their scales on {self._mx_device}")
        return kp

    @property
    def _mx_device(self):
        found = self.__dict__.get("_mx_on")
        if found is None:
            found = self._mx_on = torch.device("cuda", self._device_index)
        return found

    def _mx_out(self, out, rows: int, cols: int, bits: int, who: str):
        """``out`` if it can hold the rows, or new rows."""
        if out is None:
            self._mx_need(bits in (4, 8), f"{who}: {bits} bits (4 and 8 are known)")
            kp = _padded(cols)
            return MxRows(torch.empty((rows, kp * bits // 8), dtype=torch.uint8, device=self._mx_device),
                          torch.empty((-(-rows // TILE_ROWS), kp // CHUNK, TILE_BYTES), dtype=torch.uint8,
                                      device=self._mx_device), bits, cols)
        self._mx_check(out, who)
        self._mx_need(out.rows == rows and out.cols == cols and out.bits == bits,
                      f"{who}: out holds {out.rows} x {out.cols} of {out.bits} bits, not {rows} x {cols} of {bits}")
        return out

    def mx_quantize(self, x, bits=8, out=None) -> MxRows:
        """Rows of float32 or bfloat16 (any distance between them) in the format."""
        self._mx_need(x.dim() == 2 and x.shape[1] >= 1 and x.stride(1) == 1 and x.dtype in _CODE
                      and x.device == self._mx_device,
                      "mx_quantize: x must be rows of float32 or bfloat16 on the kernel set's device")
        rows, cols = x.shape
        out = self._mx_out(out, rows, cols, bits, "mx_quantize")
        if rows:
            self._ok(self.mx.ti_mx_quantize(x.data_ptr(), _CODE[x.dtype], x.stride(0), rows, cols, _padded(cols), bits,
                                            out.codes.data_ptr(), out.scales.data_ptr(), self._stream()), self.mx)
        return out

    def mx_dequantize(self, q: MxRows, dtype=torch.bfloat16, out=None):
        """The numbers that rows in the format stand for (in bfloat16 exactly, unless below its range)."""
        kp = self._mx_check(q, "mx_dequantize")
        if out is None:
            out = torch.empty((q.rows, q.cols), dtype=dtype, device=self._mx_device)
        self._mx_need(out.dtype in _CODE and out.shape == (q.rows, q.cols) and out.stride(1) == 1
                      and out.device == self._mx_device, "mx_dequantize: out must be float32 or bfloat16 of the rows' shape")
        if q.rows:
            self._ok(self.mx.ti_mx_dequantize(q.codes.data_ptr(), q.scales.data_ptr(), q.rows, q.cols, kp, q.bits,
                                              out.data_ptr(), _CODE[out.dtype], out.stride(0), self._stream()), self.mx)
        return out

    def mx_rmsnorm(self, x, weight, eps, bits=8, delta=None, out=None) -> MxRows:
        """``x += delta`` (in place; float32 rows, delta float32 or bfloat16 or none), then the rows
        ``x / sqrt(mean(x^2) + eps) * weight`` in the format.  A row is at most 32,768 elements."""
        self._mx_need(x.dim() == 2 and x.shape[1] >= 1 and x.dtype == torch.float32 and x.stride(1) == 1
                      and x.device == self._mx_device, "mx_rmsnorm: x must be float32 rows on the kernel set's device")
        rows, cols = x.shape
        self._mx_need(weight.dtype == torch.float32 and weight.shape == (cols,) and weight.is_contiguous()
                      and weight.device == self._mx_device, "mx_rmsnorm: weight must be float32 of the row length")
        at, code, ld = None, 0, 0
        if delta is not None:
            self._mx_need(delta.shape == x.shape and delta.dtype in _CODE and delta.stride(1) == 1
                          and delta.device == self._mx_device, "mx_rmsnorm: delta must be float32 or bfloat16 of x's shape")
            at, code, ld = delta.data_ptr(), _CODE[delta.dtype], delta.stride(0)
        out = self._mx_out(out, rows, cols, bits, "mx_rmsnorm")
        if rows:
            self._ok(self.mx.ti_mx_rmsnorm(x.data_ptr(), x.stride(0), at, code, ld, weight.data_ptr(), rows, cols,
                                           _padded(cols), eps, bits, out.codes.data_ptr(), out.scales.data_ptr(),
                                           self._stream()), self.mx)
        return out

    def mx_linear(self, a: MxRows, w: MxRows, out, accumulate=False):
        """out (+)= a @ w.T, float32 sums; ``a`` of 8 or 4 bits, ``w`` of 4."""
        kp = self._mx_check(a, "mx_linear (rows)")
        self._mx_check(w, "mx_linear (weights)")
        self._mx_need(w.bits == 4 and w.cols == a.cols, "mx_linear: weights must have 4 bits and the rows' columns")
        m, n = a.rows, w.rows
        self._mx_need(out.dtype == torch.float32 and out.shape == (m, n) and out.stride(1) == 1
                      and out.device == self._mx_device, "mx_linear: out must be float32 of rows x weights")
        if m and n:
            self._ok(self.mx.ti_mx_gemm(a.codes.data_ptr(), a.scales.data_ptr(), a.bits, w.codes.data_ptr(),
                                        w.scales.data_ptr(), out.data_ptr(), m, n, kp, max(out.stride(0), n), int(accumulate),
                                        int(w.settled), self.status.data_ptr(), self._stream()), self.mx)
        return out

    def mx_linear_glu(self, a: MxRows, w: MxRows, cols: int, bits=8, out=None) -> MxRows:
        """``silu(a @ gate.T) * (a @ up.T)``, ``cols`` columns, in the format; ``w`` from ``mx_pack_gate_up``."""
        kp = self._mx_check(a, "mx_linear_glu (rows)")
        self._mx_check(w, "mx_linear_glu (weights)")
        out_kp = _padded(cols)
        self._mx_need(cols >= 1 and w.bits == 4 and w.cols == a.cols and w.rows == 2 * out_kp,
                      f"mx_linear_glu: weights must be packed gate and up rows of 4 bits for {cols} columns")
        out = self._mx_out(out, a.rows, cols, bits, "mx_linear_glu")
        if a.rows:
            self._ok(self.mx.ti_mx_gemm_glu(a.codes.data_ptr(), a.scales.data_ptr(), a.bits, w.codes.data_ptr(),
                                            w.scales.data_ptr(), out.codes.data_ptr(), out.scales.data_ptr(), bits, a.rows,
                                            out_kp, kp, int(w.settled), self.status.data_ptr(), self._stream()), self.mx)
        return out

    # ---- weights -------------------------------------------------------------------------
    def mx_pack_linear(self, w) -> MxRows:
        """A product's weight ``[n, k]`` in 4 bits.  Waits until it is made, and says so (``settled``)."""
        q = self.mx_quantize(w, 4)
        torch.cuda.current_stream(self._mx_device).synchronize()
        return q._replace(settled=True)

    def mx_pack_gate_up(self, gate, up) -> MxRows:
        """Gate and up rows ``[cols, k]`` as one weight of 4 bits: strips of 32 gate rows followed by their 32 up rows, with
        rows of zeros up to whole chunks of columns."""
        self._mx_need(gate.shape == up.shape and gate.dtype == up.dtype and gate.dim() == 2,
                      "mx_pack_gate_up: gate and up must be alike")
        pad = _padded(gate.shape[0]) - gate.shape[0]
        both = [torch.nn.functional.pad(t, (0, 0, 0, pad)).view(-1, BLOCK, t.shape[1]) for t in (gate, up)]
        return self.mx_pack_linear(torch.stack(both, dim=1).view(-1, gate.shape[1]))
