"""Linear layers with 4-bit weights and a scale for each group of columns.

``Linear4bit`` keeps one weight ``[N, K]`` resident and computes
``y = x @ W.T (+ bias)`` for 1 to 32 rows per pass over the weight with
``nsm_linear4bit`` (``csrc/nsm_linear4bit.cu``): the attention projections,
dense MLPs and heads of a 4-bit checkpoint, next to the block-sparse MLP
(the reference dequantises such a weight and calls ``F.linear``,
``streaming_llama_runtime.py:4765``).  Unlike ``Nf4LmHead`` it takes any even
``K``, integer weights, any group size that is a multiple of 32, and up to 32
rows in one pass whatever ``K`` is; it lays the weight out once, in tiles that
a warp streams.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._torch import dtype_code, ptr, require_cuda, stream_handle
from .nf4 import nf4_code, quantize_nf4


class Linear4bit:
    """``W[n, k] = (T[q[n, k]] - z[n, k // group_size]) * scales[n, k // group_size]``.

    ``packed`` uint8, ``N * K / 2`` bytes row by row, column ``2i`` in the high
    nibble of byte ``i``; ``scales`` fp32 / fp16 / bf16 ``[N, ceil(K /
    group_size)]`` (held in fp32).  With ``code`` (16 values) ``T`` is that
    codebook, as for NF4.  Without it the weights are integers and ``zeros``
    (uint8, the scales' shape) their zero points, 8 when it is ``None``.  The
    layer keeps copies in its own layout: the arguments may be freed.

    A codebook is held to 22 bits; ``fp16_code=True`` rounds it to fp16 (11 bits), which
    takes about two thirds of the time on large weights.

    Calls on different streams may overlap; a call inside a CUDA graph capture
    takes its scratch memory from the capture's own pool.
    """

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, *, out_features: int, in_features: int,
                 group_size: int = 64, code: torch.Tensor | None = None, zeros: torch.Tensor | None = None,
                 bias: torch.Tensor | None = None, fp16_code: bool = False):
        for name, t in (("packed", packed), ("scales", scales), ("zeros", zeros), ("code", code), ("bias", bias)):
            if t is None:
                continue
            require_cuda(t, name)
            if t.device != packed.device:
                raise RuntimeError(f"{name} is on {t.device} but packed is on {packed.device}")
        N, K, gs = int(out_features), int(in_features), int(group_size)
        if N <= 0 or K <= 0 or K % 2:
            raise RuntimeError(f"a [{N}, {K}] weight is not supported: in_features must be even")
        if gs <= 0 or gs % 32:
            raise RuntimeError(f"group_size ({gs}) must be a multiple of 32")
        groups = -(-K // gs)
        if packed.dtype != torch.uint8 or packed.numel() * 2 != N * K:
            raise RuntimeError(f"packed has {packed.numel()} values of {packed.dtype} for a [{N}, {K}] 4-bit weight")
        if scales.numel() != N * groups:
            raise RuntimeError(f"scales has {scales.numel()} values for a [{N}, {K}] weight with group_size {gs}")
        if code is not None and zeros is not None:
            raise RuntimeError("a weight with a codebook has no zero points")
        if fp16_code and code is None:
            raise RuntimeError("fp16_code is for weights with a codebook")
        if code is not None and code.numel() != 16:
            raise RuntimeError(f"code has {code.numel()} entries, expected 16")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.numel() != N * groups):
            raise RuntimeError(f"zeros must be uint8 with {N * groups} values")
        if bias is not None and bias.numel() != N:
            raise RuntimeError(f"bias has {bias.numel()} values for {N} outputs")
        self.out_features, self.in_features, self.group_size = N, K, gs
        self.device = packed.device
        self._lib = lib = _lib.load()
        with torch.cuda.device(self.device):
            def new(n, dt):
                return torch.empty(int(n), dtype=dt, device=self.device)

            count = int(lib.nsm_linear4bit_scale_count(N, K, gs))
            if count == 0:
                raise RuntimeError(f"a [{N}, {K}] weight is too large")
            self.packed = new(lib.nsm_linear4bit_packed_bytes(N, K), torch.uint8)
            self.scales = new(count, torch.float32)
            self.zeros = new(count, torch.uint8) if zeros is not None else None
            src, sc = packed.reshape(-1).contiguous(), scales.contiguous()
            zp = zeros.contiguous() if zeros is not None else None
            _lib.check(lib.nsm_linear4bit_pack(src.data_ptr(), K // 2, sc.data_ptr(), dtype_code(sc.dtype), ptr(zp), N, K,
                                               gs, int(code is not None), self.packed.data_ptr(), self.scales.data_ptr(),
                                               ptr(self.zeros), stream_handle(self.device)), "nsm_linear4bit_pack")
            self.code = code.reshape(-1).to(torch.float32, copy=True) if code is not None else None
            self.bias = bias.reshape(-1).clone(memory_format=torch.contiguous_format) if bias is not None else None
        self._c = _lib.Linear4bitWeightsC(ptr(self.packed), ptr(self.scales), ptr(self.zeros), ptr(self.code),
                                          ptr(self.bias), dtype_code(self.bias.dtype) if bias is not None else 0, N, K, gs)
        self._ref = ctypes.byref(self._c)
        self._fn = lib.nsm_linear4bit_code16 if fp16_code else lib.nsm_linear4bit
        self._ws_bytes: dict[tuple[int, int], int] = {}
        self._spare = torch.empty(256, dtype=torch.uint8, device=self.device)  # for calls that need no workspace

    # ---- construction
    @classmethod
    def from_param(cls, p, device: torch.device | str = "cuda", bias: torch.Tensor | None = None,
                   fp16_code: bool = False) -> "Linear4bit":
        """From a ``checkpoint.Nf4Param`` (host tensors)."""
        if p.in_features % p.blocksize:
            raise RuntimeError(f"{p.name}: quant blocks of {p.blocksize} do not divide the {p.in_features} columns of a row")
        dev = torch.device(device)
        return cls(p.packed.to(dev), p.absmax.to(dev), out_features=p.out_features, in_features=p.in_features,
                   group_size=p.blocksize, code=p.code.to(dev), bias=bias.to(dev) if bias is not None else None,
                   fp16_code=fp16_code)

    @classmethod
    def from_checkpoint(cls, ckpt, name: str, device: torch.device | str = "cuda",
                        bias: torch.Tensor | None = None, fp16_code: bool = False) -> "Linear4bit":
        """A quantised weight of an ``Nf4Checkpoint``."""
        return cls.from_param(ckpt.load_param(name), device, bias, fp16_code)

    @classmethod
    def from_dense(cls, weight: torch.Tensor, device: torch.device | str = "cuda", group_size: int = 64,
                   kind: str = "nf4", bias: torch.Tensor | None = None, fp16_code: bool = False) -> "Linear4bit":
        """A dense ``[N, K]`` weight quantised on the device: ``kind`` ``"nf4"``
        (nearest code value, absmax per group) or ``"int4"`` (round to -7..7,
        absmax / 7 per group).  ``group_size`` must divide ``K``."""
        if weight.dim() != 2:
            raise RuntimeError(f"Expected a rank-2 dense weight, got shape {tuple(weight.shape)}")
        N, K = (int(s) for s in weight.shape)
        if group_size <= 0 or K % group_size:
            raise RuntimeError(f"group_size ({group_size}) must divide in_features ({K})")
        dev = torch.device(device)
        w = weight.to(dev)
        code = None
        if kind == "nf4":
            code = nf4_code(dev)
            packed, scales = quantize_nf4(w, code, group_size)
        elif kind == "int4":
            grp = w.to(torch.float32).reshape(N, K // group_size, group_size)
            scales = grp.abs().amax(dim=-1) / 7.0
            q = torch.round(grp / torch.where(scales > 0, scales, torch.ones_like(scales))[..., None]).clamp_(-7, 7)
            q = (q + 8).to(torch.uint8).reshape(N, K)
            packed = (q[:, 0::2] << 4) | q[:, 1::2]
        else:
            raise RuntimeError(f"unknown kind of 4-bit weight {kind!r} (nf4 or int4)")
        return cls(packed, scales, out_features=N, in_features=K, group_size=group_size, code=code,
                   bias=bias.to(dev) if bias is not None else None, fp16_code=fp16_code)

    # ---- forward
    def max_rows_per_call(self, dtype: torch.dtype) -> int:
        return int(self._lib.nsm_linear4bit_max_rows(dtype_code(dtype)))

    def weight_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.packed, self.scales, self.zeros, self.code, self.bias)
                   if t is not None)

    def error(self) -> int:
        """Read and clear the error word of the layers on this device (``NSM_ERR_TIMEOUT``:
        a wait inside a kernel ran out and outputs of a call since the last check are NaN;
        0: all is well).  Synchronises the current stream; calls on others must be done."""
        code = ctypes.c_int32(0)
        with torch.cuda.device(self.device):
            _lib.check(self._lib.nsm_linear4bit_error(ctypes.byref(code), stream_handle(self.device)),
                       "nsm_linear4bit_error")
        return int(code.value)

    def __call__(self, x: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        return self.forward(x, out_dtype)

    def forward(self, x: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """``x [..., K]`` -> ``y [..., N]`` (``out_dtype``, default x's); rows are
        processed in groups of ``max_rows_per_call``, each group streaming the
        weight once."""
        dev, K = self.device, self.in_features
        if x.device != dev:
            require_cuda(x, "x")
            raise RuntimeError(f"x is on {x.device} but the weight is on {dev}")
        shape = x.shape
        if not shape or shape[-1] != K:
            raise RuntimeError(f"x has shape {tuple(shape)} but the layer expects {K} features")
        if out_dtype is None:
            out_dtype = x.dtype
        xc, oc = dtype_code(x.dtype), dtype_code(out_dtype)
        out = torch.empty(*shape[:-1], self.out_features, dtype=out_dtype, device=dev)
        if len(shape) != 2:
            x = x.reshape(-1, K)
        rows, (stride, inner) = x.shape[0], x.stride()
        if rows == 0:
            return out
        if inner != 1 or (rows > 1 and stride < K):
            x = x.contiguous()
            stride = K
        if torch.cuda.current_device() != dev.index:
            with torch.cuda.device(dev):
                self._run(x, xc, stride, rows, out, oc)
        else:
            self._run(x, xc, stride, rows, out, oc)
        return out

    def _run(self, x: torch.Tensor, xc: int, stride: int, rows: int, out: torch.Tensor, oc: int) -> None:
        lib, N, dev = self._lib, self.out_features, self.device
        per = 16 if xc == _lib.NSM_F32 else 32
        xp, op = x.data_ptr(), out.data_ptr()
        stream = stream_handle(dev)
        while True:
            n = rows if rows < per else per
            need = self._ws_bytes.get((n, xc))
            if need is None:
                need = self._ws_bytes[(n, xc)] = int(lib.nsm_linear4bit_workspace_bytes(n, xc, N, self.in_features))
            ws = self._spare if need == 256 else torch.empty(need, dtype=torch.uint8, device=dev)
            status = self._fn(xp, xc, n, stride, self._ref, op, oc, N, ws.data_ptr(), need, stream)
            if status:
                _lib.check(status, "nsm_linear4bit")
            rows -= n
            if rows == 0:
                return
            xp += n * stride * x.element_size()
            op += n * N * out.element_size()
