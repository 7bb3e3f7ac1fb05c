"""y = x @ W^T (+ b), W stored [out, in].

float32 runs: the product is the CUDA-core kernel with true 32-bit accumulation.
bfloat16 runs: the reference hands every bf16 dense product to cuBLAS through
``F.linear`` (acvram/kernels/__init__.py:1896-1899); so may this engine, and it
does for the shapes its own tensor-core kernel does not take.  Logits are the
exception in both: bfloat16 operands, accumulated and returned in float32
(acvram/engine/model.py:369-410), by a kernel of this package.

A bias is there when the weight file holds one, as in the reference
(acvram/engine/loader.py:269-270); it is kept in float32 and added to the float
accumulator in the tensor-core product's epilogue, or by a kernel of its own
after the products that have no such epilogue.
"""

from __future__ import annotations

import torch

from ..kernels import ops
from ..weights.needs import TensorNeed, WeightError


class Linear:
    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None) -> None:
        self.weight = weight.contiguous()
        self.out_features, self.in_features = self.weight.shape
        self.bias = None if bias is None else bias.to(device=weight.device, dtype=torch.float32).contiguous()

    @classmethod
    def stacked(cls, weights: list[torch.Tensor], biases: list | None = None) -> "Linear":
        """One product for several projections of the same input: rows concatenated
        (the reference stacks q,k,v and gate,up at load, acvram/engine/layers.py:1476-1560).
        ``biases``: one per projection or None; where some have one and others not, the others get zeros."""
        bias = None
        if biases is not None and any(b is not None for b in biases):
            bias = torch.cat([b.float() if b is not None else torch.zeros(w.shape[0], device=w.device)
                              for w, b in zip(weights, biases)])
        return cls(torch.cat(list(weights), dim=0), bias)

    @staticmethod
    def needs(prefix: str, out_features: int, in_features: int, bias: bool | None) -> dict[str, TensorNeed]:
        """``prefix + "weight"`` and, with ``bias`` True, ``prefix + "bias"``; None: the bias is read if the file has it."""
        needs = {prefix + "weight": TensorNeed((out_features, in_features))}
        if bias is not False:
            needs[prefix + "bias"] = TensorNeed((out_features,), "bias", optional=bias is None)
        return needs

    def weight_bytes(self) -> int:
        n = self.weight.numel() * self.weight.element_size()
        return n + (self.bias.numel() * 4 if self.bias is not None else 0)

    def flops(self, tokens: int) -> float:
        return 2.0 * tokens * self.out_features * self.in_features

    def __call__(self, x: torch.Tensor, out_dtype: torch.dtype | None = None, plan: tuple | None = None,
                 unary: str | None = None) -> torch.Tensor:
        """``plan``: how the tensor-core product tiles and splits this call (``ops.gemm_tc``), for a caller that knows
        its shape better than the general rules do.  ``unary``: an activation (a name of ``ops.ACTIVATIONS``) on every
        output: in the tensor-core product's epilogue where that product runs, by a kernel of its own otherwise."""
        w = self.weight
        out_dtype = out_dtype or x.dtype
        out = x.new_empty((x.shape[0], self.out_features), dtype=out_dtype)      # (0.5 us under torch.empty with a device)
        if x.shape[0] == 0:
            return out
        if x.dtype == torch.float32:
            ops.gemm_simt(x, w, out)
            if self.bias is not None:
                ops.add_bias(out, self.bias)
        elif out_dtype == torch.float32 and plan is not None and ops.gemm_tc_takes(x, w):
            ops.gemm_tc(x, w, out, plan=plan, static_weights=True, bias=self.bias)
        elif out_dtype == torch.float32:
            ops.linear_bf16_f32out(x, w, out, static_weights=True, bias=self.bias)
        else:
            # (the tensor-core product adds the bias, and applies the activation, itself)
            return ops.linear_bf16(x, w, out, static_weights=True, bias=self.bias, unary=unary)
        if unary is not None:
            ops.activation(out, out, unary)
        return out


class Fp8Rows:
    """Activations in 8 bits (``ops.fp8_rows``) on their way into an ``Fp8Linear``; ``dtype``: the element type of the run."""

    __slots__ = ("values", "scales", "dtype")

    def __init__(self, rows: int, columns: int, device, dtype: torch.dtype) -> None:
        self.values, self.scales = ops.fp8_rows(rows, columns, device)
        self.dtype = dtype

    @classmethod
    def of(cls, x: "torch.Tensor | Fp8Rows") -> "Fp8Rows":
        """x itself, or the quantised rows of a tensor."""
        if isinstance(x, Fp8Rows):
            return x
        rows = cls(x.shape[0], x.shape[1], x.device, x.dtype)
        ops.quantize_fp8(x, rows.values, rows.scales)
        return rows

    @property
    def shape(self):
        return self.values.shape

    @property
    def device(self):
        return self.values.device

    def new_empty(self, shape, dtype: torch.dtype | None = None) -> torch.Tensor:
        return torch.empty(shape, device=self.values.device, dtype=dtype or self.dtype)


class Fp8Linear:
    """y = x W^T with W in e4m3, a scale for each block of 128 x 128 of it, and x quantised in groups of 128 of a row
    (``ops.linear_fp8``).  Tensors behind ``prefix``: weight, and weight_scale_inv, the blocks' scales [out / 128, in / 128]; a weight
    in more bits (then without scales) is quantised when it is loaded.

    Several projections of the same input are one product where their rows are whole blocks, else one each, side by side in
    the output."""

    bias = None

    def __init__(self, matrices: list[tuple[torch.Tensor, torch.Tensor]]) -> None:
        merged: list[tuple[torch.Tensor, torch.Tensor]] = []
        for values, scales in matrices:
            if merged and merged[-1][0].shape[0] % ops.FP8_GROUP == 0:
                merged[-1] = (self._rows(torch.cat([merged[-1][0].view(torch.uint8), values.view(torch.uint8)])),
                              torch.cat([merged[-1][1], scales]))
            else:
                merged.append((values, scales))
        self.matrices = merged
        self.in_features = merged[0][0].shape[1]
        self.out_features = sum(v.shape[0] for v, _ in merged)

    @staticmethod
    def _rows(codes: torch.Tensor) -> torch.Tensor:
        """The codes (uint8) as e4m3 rows that start on 16 bytes."""
        values, _ = ops.fp8_rows(codes.shape[0], codes.shape[1], codes.device)
        values.view(torch.uint8).copy_(codes)
        return values

    @staticmethod
    def needs(name: str, out_features: int, in_features: int) -> dict[str, TensorNeed]:
        """The tensors of the weight called ``name`` (a bias beside it is known by name, and refused when the weight is loaded)."""
        blocks = tuple(-(-n // ops.FP8_GROUP) for n in (out_features, in_features))
        return {name: TensorNeed((out_features, in_features), "fp8"),
                name + "_scale_inv": TensorNeed(blocks, "scale", optional=True),
                Fp8Linear._bias_of(name): TensorNeed((out_features,), "bias", optional=True)}

    @staticmethod
    def _bias_of(name: str) -> str:
        return name.removesuffix("weight") + "bias"

    @staticmethod
    def matrix(tensors, name: str, device) -> tuple[torch.Tensor, torch.Tensor]:
        """(values, scales) on the device of the weight called ``name``."""
        w, scales = tensors[name], tensors.get(name + "_scale_inv")
        if tensors.get(Fp8Linear._bias_of(name)) is not None:
            raise WeightError(name, unexpected=[Fp8Linear._bias_of(name) + " (8-bit weights are built without biases)"])
        if w.dtype == ops.FP8:
            if scales is None:
                raise WeightError(name, missing=[name + "_scale_inv"])
            return Fp8Linear._rows(w.view(torch.uint8).to(device)), scales.to(device=device, dtype=torch.float32).contiguous()
        if scales is not None:
            raise WeightError(name, wrong_dtype=[(name, f"{w.dtype} beside block scales")])
        values, _ = ops.fp8_rows(w.shape[0], w.shape[1], device)
        scales = torch.empty(tuple(-(-n // ops.FP8_GROUP) for n in w.shape), device=device, dtype=torch.float32)
        return ops.quantize_fp8(w.to(device), values, scales, ops.FP8_GROUP)

    def weight_bytes(self) -> int:
        return sum(v.numel() + 4 * s.numel() for v, s in self.matrices)

    def flops(self, tokens: int) -> float:
        return 2.0 * tokens * self.out_features * self.in_features

    def __call__(self, x: torch.Tensor | Fp8Rows, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        x = Fp8Rows.of(x)
        out = x.new_empty((x.shape[0], self.out_features), dtype=out_dtype or x.dtype)
        if len(self.matrices) == 1:
            return ops.linear_fp8(x.values, x.scales, *self.matrices[0], out, static_weights=True)
        at = 0
        for values, scales in self.matrices:
            ops.linear_fp8(x.values, x.scales, values, scales, out[:, at:at + values.shape[0]], static_weights=True)
            at += values.shape[0]
        return out
