"""A projection over GGUF weights shared by a batch of tokens, beside the low-rank adapters of
the requests they belong to: y_t = W x_t + s_a B_a (A_a x_t), a = the adapter of token t.

* ``SharedProjection`` — W [n_out][n_in] in Q8_0 or Q4_0 blocks, laid out once on the device
  (the batched counterpart of ``quant.matvec_col_major``, src/quant/mod.rs:939-970, for decode
  batches; the reference projects token by token).
* ``AdapterBank`` — the adapters that are loaded: A, B, rank and scale of each. A slot can be
  rewritten in place between calls (``bank.set``).
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from ._lib import (PI_ERR_ARG, PI_ERR_INDEX, PI_QT_BF16, PI_QT_F16, PI_QT_F32, Context,
                   PiError, PiLoraBank, lib, raw_stream)

_DTYPES = {torch.float32: PI_QT_F32, torch.float16: PI_QT_F16, torch.bfloat16: PI_QT_BF16}


class AdapterBank:
    """Adapters of one projection: a [n, R, n_in] and b [n, n_out, R] CUDA tensors of f32, f16 or
    bf16; ranks int32 [n] (default R each; what lies past an adapter's rank is not used) and
    scales f32 [n] (default 1). The bank keeps copies, the rank dimension padded to a multiple
    of 8."""

    def __init__(self, a, b, ranks=None, scales=None):
        if not (a.is_cuda and b.is_cuda and a.dim() == 3 and b.dim() == 3) or a.dtype not in _DTYPES or \
                b.dtype != a.dtype or b.device != a.device:
            raise PiError(PI_ERR_ARG, "adapters: a [n, R, n_in] and b [n, n_out, R] must be CUDA tensors of one "
                                      "type (f32, f16 or bf16) and device")
        n, R, n_in = a.shape
        if n < 1 or not 1 <= R <= 1024 or b.shape[0] != n or b.shape[2] != R:
            raise PiError(PI_ERR_ARG, "adapters: need a [n, R, n_in] and b [n, n_out, R], n >= 1, 1 <= R <= 1024")
        for v, dt, what in ((ranks, torch.int32, "ranks int32"), (scales, torch.float32, "scales f32")):
            if v is not None and (v.dtype != dt or v.shape != (n,) or v.device != a.device):
                raise PiError(PI_ERR_ARG, f"adapters: {what} [n] on the adapters' device")
        a, b = a.detach(), b.detach()  # copies of parameters; set() writes into them
        self.n, self.rank, self.n_in, self.n_out, self.device = n, R, n_in, b.shape[1], a.device
        pad = -R % 8
        self.a = torch.nn.functional.pad(a, (0, 0, 0, pad)) if pad else a.clone(memory_format=torch.contiguous_format)
        self.b = torch.nn.functional.pad(b, (0, pad)) if pad else b.clone(memory_format=torch.contiguous_format)
        full = torch.full((n,), R, dtype=torch.int32, device=a.device)
        self.ranks = full if ranks is None else torch.minimum(ranks, full)
        self.scales = torch.ones(n, dtype=torch.float32, device=a.device) if scales is None else scales.detach().clone()
        self.desc = PiLoraBank(self.a.data_ptr(), self.b.data_ptr(), self.ranks.data_ptr(), self.scales.data_ptr(),
                               _DTYPES[a.dtype], n, R + pad)
        self._desc = C.byref(self.desc)

    def set(self, i: int, a, b, scale: float = 1.0) -> None:
        """Replaces adapter i by a [r, n_in], b [n_out, r] with r <= R (stream-ordered)."""
        if not 0 <= i < self.n:
            raise PiError(PI_ERR_INDEX, f"adapters: no slot {i} among {self.n}")
        r = a.shape[0] if a.dim() == 2 else -1
        if not 0 <= r <= self.rank or tuple(a.shape) != (r, self.n_in) or tuple(b.shape) != (self.n_out, r):
            raise PiError(PI_ERR_ARG, f"adapters: need a [r, {self.n_in}] and b [{self.n_out}, r], r <= {self.rank}")
        self.a[i, :r].copy_(a.detach())
        self.b[i, :, :r].copy_(b.detach())
        self.ranks[i] = r
        self.scales[i] = scale


class SharedProjection:
    """W [n_out][n_in] from GGUF bytes (host bytes / numpy, or a CUDA uint8 tensor), Q8_0 or Q4_0."""

    def __init__(self, raw, qtype: int, n_out: int, n_in: int, device: int | None = None):
        self.qtype, self.n_out, self.n_in = int(qtype), n_out, n_in
        on_dev = hasattr(raw, "is_cuda") and raw.is_cuda
        if device is None:
            device = raw.device.index if on_dev else torch.cuda.current_device()
        self.device, self.index, self._ws_bytes = torch.device("cuda", device), device, {}
        self.ctx = Context.of(device)
        if on_dev:
            if raw.device != self.device or raw.dtype != torch.uint8 or not raw.is_contiguous():
                raise PiError(PI_ERR_ARG, "projection: device weights must be contiguous uint8 on its device")
            torch.cuda.current_stream(self.device).synchronize()
            src, nbytes = raw.data_ptr(), raw.numel()
        else:
            raw = np.frombuffer(raw, np.uint8) if isinstance(raw, (bytes, bytearray, memoryview)) else \
                np.ascontiguousarray(raw).reshape(-1).view(np.uint8)
            src, nbytes = raw.ctypes.data, raw.size
        h = C.c_void_p()
        self.ctx.check(lib().pi_proj_create(self.ctx.h, src, nbytes, self.qtype, n_in, n_out, 0 if on_dev else 1,
                                            C.byref(h)))
        self.h = h

    def __del__(self):
        try:
            if getattr(self, "h", None):
                lib().pi_proj_destroy(self.h)
        except Exception:
            pass

    def forward(self, x, bank: AdapterBank | None = None, adapter_ids=None, out=None):
        """y [T, n_out] for x [T, n_in] (CUDA f32) on torch's current stream.

        adapter_ids: int32 [T], the adapter of each token, negative for none; an id past the
        bank adds nothing and is reported by ``Context.sync_check`` (PI_ERR_INDEX)."""
        dev, n_in, n_out = self.index, self.n_in, self.n_out
        if x.dtype != torch.float32 or x.get_device() != dev or x.dim() != 2 or x.shape[1] != n_in or \
                not x.is_contiguous():
            raise PiError(PI_ERR_ARG, f"projection: x must be contiguous f32 [T, {n_in}] on {self.device}")
        T = x.shape[0]
        if (bank is None) != (adapter_ids is None):
            raise PiError(PI_ERR_ARG, "projection: a bank and adapter_ids come together")
        desc, ids, rank = None, None, 0
        if bank is not None:
            if bank.n_in != n_in or bank.n_out != n_out or bank.device != self.device:
                raise PiError(PI_ERR_ARG, f"projection: the bank is for [{bank.n_out}][{bank.n_in}] on {bank.device}")
            if adapter_ids.dtype != torch.int32 or adapter_ids.shape != (T,) or adapter_ids.get_device() != dev or \
                    not adapter_ids.is_contiguous():
                raise PiError(PI_ERR_ARG, f"projection: adapter_ids must be contiguous int32 [T] on {self.device}")
            desc, ids, rank = bank._desc, adapter_ids.data_ptr(), bank.rank
        if out is None:
            out = torch.empty(T, n_out, dtype=torch.float32, device=self.device)
        elif out.dtype != torch.float32 or out.shape != (T, n_out) or out.get_device() != dev or \
                not out.is_contiguous():
            raise PiError(PI_ERR_ARG, f"projection: out must be contiguous f32 [T, {n_out}] on {self.device}")
        if T == 0:
            return out
        L = lib()
        nbytes = self._ws_bytes.get((T, rank))
        if nbytes is None:
            nbytes = self._ws_bytes[(T, rank)] = L.pi_proj_workspace(self.h, T, desc)
        # the caching allocator's memory: one workspace per call and per captured graph
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        rc = L.pi_proj_forward(self.ctx.h, self.h, x.data_ptr(), T, desc, ids, out.data_ptr(), ws.data_ptr(), nbytes,
                               raw_stream(dev))
        if rc:
            self.ctx.check(rc)
        return out
