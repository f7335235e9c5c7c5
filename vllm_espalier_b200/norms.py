"""The norms before and after a block, fused with the block's gate and the scaled residual add.

Between two blocks of a decoder the residual stream and the next block's input come from one pass over the rows:

    v = x (+ x2)                                         the block's output; x2: a second one (routed + shared experts)
    p = post(v)                                          the norm after the block, if it has one
    r = residual_scale * residual + block_scale * act(gate) * p
    h = pre(r)                                           the norm before the next block

Everything is fp32 between the inputs and one rounding an output; h is the norm of the unrounded r. The kernel is
esp_block_norm (csrc/norms.cu); it allocates nothing but its outputs and captures into CUDA graphs.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import DTYPE, esp_block_norm_op_t, launch, lib

KINDS = {"rms": 1, "layer": 2}
ACTS = {"none": 0, "sigmoid": 1, "tanh": 2}
GATE_NONE, GATE_CHANNEL, GATE_ROW, GATE_ELEMENT = range(4)
MAX_D = 49152


class BlockNorm:
    """One place between two blocks of width d.

    pre, post: the norms' weight [d], True for a norm without a weight, None for no norm; pre_bias, post_bias: [d].
    kind: "rms" or "layer". weight_offset: a norm multiplies by weight_offset + weight (1.0 for weights stored around
    zero). gate_act: the activation of the gate that forward() is given: "none", "sigmoid" or "tanh"."""

    def __init__(self, d: int, pre=None, pre_bias=None, post=None, post_bias=None, kind: str = "rms",
                 eps: float = 1e-6, weight_offset: float = 0.0, gate_act: str = "none", residual_scale: float = 1.0,
                 block_scale: float = 1.0):
        if not 1 <= d <= MAX_D:
            raise ValueError(f"width {d} outside 1..{MAX_D}")
        if kind not in KINDS:
            raise ValueError(f"kind {kind!r}: expected one of {sorted(KINDS)}")
        if gate_act not in ACTS:
            raise ValueError(f"gate_act {gate_act!r}: expected one of {sorted(ACTS)}")
        on, tensors = {}, {}
        for name, w, b in (("pre", pre, pre_bias), ("post", post, post_bias)):
            if not (w is None or isinstance(w, (bool, torch.Tensor))) or not (b is None or isinstance(b, torch.Tensor)):
                raise ValueError(f"{name} must be a tensor, True or None and its bias a tensor or None, got "
                                 f"{type(w).__name__} and {type(b).__name__}")
            on[name] = w is not None and w is not False
            if b is not None and not on[name]:
                raise ValueError(f"{name}_bias without the {name} norm")
            for key, t in ((f"{name}_w", w if isinstance(w, torch.Tensor) else None), (f"{name}_b", b)):
                if t is not None:
                    if not t.is_cuda or t.shape != (d,) or t.dtype not in DTYPE:
                        raise ValueError(f"{name} weight and bias must be CUDA fp16/bf16/fp32 [{d}] tensors")
                    tensors[key] = t.contiguous()
        dtypes, devices = {t.dtype for t in tensors.values()}, {t.device for t in tensors.values()}
        if len(dtypes) > 1 or len(devices) > 1:
            raise ValueError(f"the weights and biases of one BlockNorm share a dtype and a device, got "
                             f"{sorted(map(str, dtypes))} on {sorted(map(str, devices))}")
        self.device = devices.pop() if devices else None        # of the weights; none without any
        self.d, self.kind, self.has_pre, self.tensors = d, kind, on["pre"], tensors
        at = {k: t.data_ptr() for k, t in tensors.items()}
        self._op = esp_block_norm_op_t(d, KINDS[kind] * on["post"], KINDS[kind] * on["pre"], ACTS[gate_act], eps,
                                       weight_offset, residual_scale, block_scale,
                                       DTYPE[dtypes.pop()] if dtypes else 2, at.get("post_w"), at.get("post_b"),
                                       at.get("pre_w"), at.get("pre_b"))
        self._ref = C.addressof(self._op)

    def _rows(self, t: torch.Tensor, name: str, x: torch.Tensor) -> torch.Tensor:
        if t.shape != x.shape or t.device != x.device or t.dtype not in DTYPE:
            raise ValueError(f"{name} must be fp16/bf16/fp32 {tuple(x.shape)} on {x.device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        return t if t.stride(1) == 1 else t.contiguous()

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, x2: torch.Tensor | None = None,
                gate: torch.Tensor | None = None, out: torch.Tensor | None = None,
                normed: torch.Tensor | None = None):
        """x, x2 [rows, d] of one dtype, residual [rows, d]; gate [d], [rows, 1] or [rows, d]. Returns (r, h): r in the
        residual's dtype (x's without one), h in x's, None without the pre norm. out / normed: tensors to write r / h
        to (out may be the residual or x, normed may be x)."""
        d, x_dtype = self.d, x.dtype
        x_code = DTYPE.get(x_dtype)
        if x.dim() != 2 or x.shape[1] != d or not x.is_cuda or x_code is None:
            raise ValueError(f"x must be a CUDA fp16/bf16/fp32 [rows, {d}] tensor, got {x_dtype} {tuple(x.shape)}")
        if self.device is not None and x.device != self.device:
            raise ValueError(f"x must be on the weights' {self.device}, got {x.device}")
        x_stride, step = x.stride()
        if step != 1:
            x = x.contiguous()
            x_stride = d
        rows = x.shape[0]
        x2_ptr = x2_stride = residual_ptr = residual_stride = gate_ptr = gate_stride = kind = gate_dtype = 0
        if x2 is not None:
            x2 = self._rows(x2, "x2", x)
            if x2.dtype != x_dtype:
                raise ValueError(f"x2 must have x's dtype {x_dtype}, got {x2.dtype}")
            x2_ptr, x2_stride = x2.data_ptr(), x2.stride(0)
        r_like, r_dtype, r_code = x, x_dtype, x_code
        if residual is not None:
            r_like = residual = self._rows(residual, "residual", x)
            residual_ptr, residual_stride, r_dtype = residual.data_ptr(), residual.stride(0), residual.dtype
            r_code = DTYPE[r_dtype]
        if gate is not None:
            if gate.device != x.device or gate.dtype not in DTYPE:
                raise ValueError(f"gate must be fp16/bf16/fp32 on {x.device}, got {gate.dtype} on {gate.device}")
            if gate.shape == (d,):
                kind, gate = GATE_CHANNEL, gate.contiguous()
            elif gate.shape == (rows, 1):
                kind, gate_stride = GATE_ROW, gate.stride(0)
            elif gate.shape == (rows, d):
                gate = gate if gate.stride(1) == 1 else gate.contiguous()
                kind, gate_stride = GATE_ELEMENT, gate.stride(0)
            else:
                raise ValueError(f"gate must be [{d}], [{rows}, 1] or [{rows}, {d}], got {tuple(gate.shape)}")
            gate_ptr, gate_dtype = gate.data_ptr(), DTYPE[gate.dtype]
        if out is None:
            out, r_stride = r_like.new_empty((rows, d)), d
        else:
            r_stride = self._given(out, "out", x, r_dtype)
        h_ptr = h_stride = 0
        if self.has_pre:
            if normed is None:
                normed, h_stride = x.new_empty((rows, d)), d
            else:
                h_stride = self._given(normed, "normed", x, x_dtype)
            h_ptr = normed.data_ptr()
        elif normed is not None:
            raise ValueError("normed given, but this BlockNorm has no pre norm")
        if rows:
            launch(x.device, lib().esp_block_norm, self._ref, x.data_ptr(), x_stride, x2_ptr, x2_stride, x_code,
                   residual_ptr, residual_stride, r_code, gate_ptr, kind, gate_dtype, gate_stride, out.data_ptr(), r_stride,
                   h_ptr, h_stride, rows)
        return out, normed

    @staticmethod
    def _given(t: torch.Tensor, name: str, x: torch.Tensor, dtype: torch.dtype) -> int:
        if t.shape != x.shape or t.dtype != dtype or t.device != x.device or t.stride(1) != 1:
            raise ValueError(f"{name} must be {dtype} {tuple(x.shape)} on {x.device} with unit column stride")
        return t.stride(0)

    __call__ = forward
