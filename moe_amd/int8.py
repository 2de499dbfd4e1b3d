"""Products in 8-bit integers with a scale for each token and channel
(include/moe_hip.h, "products in 8-bit integers").

The reference multiplies f32 activations by quantised rows (quant::matmul,
src/quant.rs:482-506), which model.Linear keeps at f32 precision.  Here both
sides are held in 8 bits, which the matrix cores multiply exactly at twice the
rate of 16-bit floats and a decode step reads as single bytes.
"""
from __future__ import annotations

import ctypes as C

from . import _lib as L
from .paged import _OnDevice, _fits, _need, _on_its_device, _refused, _rows

try:
    import torch
except ImportError:  # pragma: no cover - torch is part of the image
    torch = None

_DT = {} if torch is None else {torch.float32: L.DT_F32, torch.float16: L.DT_F16, torch.bfloat16: L.DT_BF16}


class Int8Linear(_OnDevice):
    """y = x W^T in 8 bits.  `weights`: tensors [channels, values] (float32,
    float16 or bfloat16, contiguous rows) or one of them; several over the same
    input become one product, their channels one behind the other.  They are
    quantised once, on torch's current stream of their device, and not kept; that
    is done when the object is made, so its calls may go to any stream."""

    def __init__(self, weights):
        ws = list(weights) if isinstance(weights, (list, tuple)) else [weights]
        _need(bool(ws), "a product without weights")
        for w in ws:
            _need(w.dim() == 2 and w.dtype in _DT and w.shape[0] >= 1 and w.shape[1] >= 1 and
                  (w.stride(1) == 1 or w.shape[1] == 1) and (w.shape[0] == 1 or w.stride(0) >= w.shape[1]),
                  "weights must be float32, float16 or bfloat16 [channels, values] with contiguous rows that do not overlap")
            _need(w.shape[1] == ws[0].shape[1] and w.device == ws[0].device,
                  "weights of one product have the same width and device")
        # (a single row may have any stride)
        self._pack([(w.data_ptr(), _DT[w.dtype], (w.stride(0) if w.shape[0] > 1 else w.shape[1]) * w.element_size(), w.shape[0])
                    for w in ws], ws[0].shape[1], ws[0].device)

    @classmethod
    def of_views(cls, ctx, views, device) -> "Int8Linear":
        """Of weight views (layer.View) of a context's regions, in any format
        that moe_int8_pack takes."""
        rows = []
        for v in views:
            p = C.c_void_p()
            L.check(L.lib().moe_region_ptr(ctx.handle, v.region, C.byref(p)), "moe_region_ptr")
            _need(v.cols == views[0].cols, "weights of one product have the same width")
            rows.append((p.value + v.offset, v.dt, v.nbytes // v.rows, v.rows))
        self = cls.__new__(cls)
        self._pack(rows, views[0].cols, torch.device(device))
        return self

    def _pack(self, rows, k, device) -> None:
        n = sum(r[3] for r in rows)
        _fits(channels=n, values=k)
        self.n, self.k = n, k
        b = C.c_uint64()
        _refused(L.lib().moe_int8_pack_size(n, k, C.byref(b)), "moe_int8_pack_size")
        _need(device.type == "cuda", f"weights on {device}: the kernels run on the GPU")
        self._index = device.index if device.index is not None else torch.cuda.current_device()
        self.device = device = torch.device("cuda", self._index)
        with torch.cuda.device(self._index):
            self.packed = torch.empty(b.value, dtype=torch.uint8, device=device)
            at = 0
            for ptr, dt, row_bytes, m in rows:
                _refused(L.lib().moe_int8_pack(ptr, dt, row_bytes, m, at, n, k, self.packed.data_ptr(), b.value,
                                               torch._C._cuda_getCurrentRawStream(self._index)), "moe_int8_pack")
                at += m
            torch.cuda.current_stream().synchronize()
        self._where, self._width = self.packed.data_ptr(), -(-k // 64) * 64
        self._sizes = {}

    def workspace_size(self, t: int) -> int:
        n = self._sizes.get(t)
        if n is None:
            _fits(rows=t)
            b = C.c_uint64()
            _refused(L.lib().moe_int8_linear_workspace_size(self.n, self.k, t, C.byref(b)), "moe_int8_linear_workspace_size")
            if len(self._sizes) > 256:
                self._sizes.clear()
            n = self._sizes[t] = b.value
        return n

    @_on_its_device
    def __call__(self, x, y, residual=None, stream=None):
        """y [rows, channels] = x [rows, values] W^T, float32 with contiguous
        rows; residual += y where it is given.  y and residual may each lie in
        x's memory, but not in each other's."""
        t = x.shape[0]
        xs, ys = _rows(x, t, self.k, "x"), _rows(y, t, self.n, "y")
        rs, r = 0, None
        if residual is None:
            self._check_device(x, y)
        else:
            rs, r = _rows(residual, t, self.n, "residual"), residual.data_ptr()
            self._check_device(x, y, residual)
        need = self.workspace_size(t)
        sp = self._on(stream)
        rc = 1
        if t * self._width <= 16384 and t <= 4:  # no workspace, unless results lie in x's memory
            rc = L.lib().moe_int8_linear(self._where, self.n, self.k, x.data_ptr(), xs, t, y.data_ptr(), ys, r, rs, None, 0, sp)
        if rc:
            ws = self._scratch(need, sp)
            rc = L.lib().moe_int8_linear(self._where, self.n, self.k, x.data_ptr(), xs, t, y.data_ptr(), ys, r, rs,
                                         ws.data_ptr(), need, sp)
        if rc:
            _refused(rc, "moe_int8_linear")
        return y
