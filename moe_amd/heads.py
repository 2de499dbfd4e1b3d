"""Biases, norms of queries and keys for each head and the rotation by position
in one pass (include/moe_hip.h, "biases, head norms and rotation in one pass").

What the reference's attention does to its projections before the cache write
(src/model.rs:707-730): every value is read and written once, with the results
that moe_add_bias, moe_rmsnorm and moe_rope give in turn, bit for bit.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _lib as L
from .paged import _OnDevice, _fits, _ids, _need, _on_its_device, _refused, _rows

try:
    import torch
except ImportError:  # pragma: no cover - torch is part of the image
    torch = None


class HeadRope(_OnDevice):
    """For rows of `heads` query heads and `n_kv` key heads of `width` values:
    biases q_bias, k_bias (and v_bias, for the values' rows), norms q_norm and
    k_norm (one weight for each value of a head, or of the whole projection),
    then the rotation of the `dim` values from `offset` on (None: to the head's
    end), pair (i, i + dim / 2) by pos * inv_freq[i]."""

    def __init__(self, heads: int, n_kv: int, width: int, inv_freq, *, offset: int = 0, dim: Optional[int] = None,
                 q_norm=None, k_norm=None, q_bias=None, k_bias=None, v_bias=None, eps: float = 1e-6):
        _fits(heads=heads, n_kv=n_kv, width=width, offset=offset)
        _need(heads >= 1 and n_kv >= 1 and width >= 1, f"{heads} heads over {n_kv} of {width} values")
        dim = width - offset if dim is None else dim
        _need(offset >= 0 and dim >= 0 and dim % 2 == 0 and offset + dim <= width,
              f"rotating {dim} values from {offset} on in heads of {width}")
        for t in (inv_freq, q_norm, k_norm, q_bias, k_bias, v_bias):
            _need(t is None or (t.dtype == torch.float32 and t.dim() == 1 and t.is_contiguous() and t.device == inv_freq.device),
                  "frequencies, norms and biases must be contiguous float32 vectors on one device")
        spans = []
        for name, t, h in (("q_norm", q_norm, heads), ("k_norm", k_norm, n_kv)):
            _need(t is None or t.numel() in (width, h * width), f"{name} must have {width} or {h * width} values")
            spans.append(h if t is not None and t.numel() != width else 1)
        for name, t, n in (("q_bias", q_bias, heads * width), ("k_bias", k_bias, n_kv * width)):
            _need(t is None or t.numel() == n, f"{name} must have {n} values")
        _need(v_bias is None or v_bias.numel() >= 1, "v_bias without values")
        self.heads, self.n_kv, self.width, self.inv_freq = heads, n_kv, width, inv_freq
        self.q_norm, self.k_norm, self.q_bias, self.k_bias, self.v_bias = q_norm, k_norm, q_bias, k_bias, v_bias
        self.device, self._index = inv_freq.device, inv_freq.get_device()
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.c = L.HeadRopeC(q_bias=at(q_bias), k_bias=at(k_bias), v_bias=at(v_bias), q_norm=at(q_norm), k_norm=at(k_norm),
                             inv_freq=at(inv_freq), heads=heads, n_kv=n_kv, width=width, q_span=spans[0], k_span=spans[1],
                             offset=offset, dim=dim, n_inv=inv_freq.numel(), eps=eps,
                             v_width=0 if v_bias is None else v_bias.numel())
        self._c = C.byref(self.c)

    @_on_its_device
    def __call__(self, q, k, pos, v=None, *, q_out=None, k_out=None, v_out=None, stream=None):
        """Rows q [rows, heads * width] and k [rows, n_kv * width] (float32,
        contiguous rows) at positions pos (int32 [rows]), in place or into
        q_out and k_out, which otherwise share no memory with them; v [rows,
        values] gets v_bias, where there is one."""
        n = q.shape[0]
        _fits(rows=n)
        q_out, k_out = q if q_out is None else q_out, k if k_out is None else k_out
        qw, kw = self.heads * self.width, self.n_kv * self.width
        qs, ks, qo, ko = _rows(q, n, qw, "q"), _rows(k, n, kw, "k"), _rows(q_out, n, qw, "q_out"), _rows(k_out, n, kw, "k_out")
        _ids(pos, torch.int32, n, "pos")
        va = (None, 0, None, 0)
        if v is None or self.v_bias is None:
            _need(v is None or v_out is None, "v_out without a v_bias")
            self._check_device(q, k, pos, q_out, k_out)
        else:
            v_out = v if v_out is None else v_out
            w = self.v_bias.numel()
            va = (v.data_ptr(), _rows(v, n, w, "v"), v_out.data_ptr(), _rows(v_out, n, w, "v_out"))
            self._check_device(q, k, pos, q_out, k_out, v, v_out)
        rc = L.lib().moe_head_rope_rows(self._c, q.data_ptr(), qs, k.data_ptr(), ks, va[0], va[1], n, pos.data_ptr(),
                                        q_out.data_ptr(), qo, k_out.data_ptr(), ko, va[2], va[3], self._on(stream))
        if rc:
            _refused(rc, "moe_head_rope_rows")
        return q_out, k_out
