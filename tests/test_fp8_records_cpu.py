"""The records in which the 8-bit operators' arguments travel, against the C structs as the kernels' sources declare them: what a call
packs is read back field by field through a structure made from the declaration."""

from __future__ import annotations

import contextlib
import ctypes
import os
import re

import pytest
import torch

from acvram_b200.kernels import build, ops
from acvram_b200.kernels.ops import FP8

_C = {"int": ctypes.c_int, "long long": ctypes.c_longlong, "float": ctypes.c_float}


def declared(source: str, name: str) -> type:
    """A ctypes structure with the fields, in their order, of ``struct name`` in csrc/``source``."""
    with open(os.path.join(build.CSRC, source), encoding="utf-8") as fh:
        body = re.search(r"struct " + name + r" \{(.*?)\};", fh.read(), re.S).group(1)
    fields = []
    for line in filter(None, (part.strip() for part in re.sub(r"//[^\n]*", "", body).split(";"))):
        kind = next(k for k in ("const void", "long long", "int", "float") if line.startswith(k))
        for item in line[len(kind):].split(","):
            item = item.strip()
            assert item.startswith("*") == (kind == "const void"), line
            fields.append((item.lstrip("*"), ctypes.c_void_p if kind == "const void" else _C[kind]))
    return type(name, (ctypes.Structure,), {"_fields_": fields})


class Matrix:
    """As much of a tensor on a device as a call looks at; every one has an address and strides of its own."""
    made = 0

    def __init__(self, shape, dtype):
        Matrix.made += 1
        self.shape, self.dtype, self.ndim = torch.Size(shape), dtype, len(shape)
        self.at = Matrix.made << 12
        self.row = (shape[1] if len(shape) == 2 else 1) + 16 * Matrix.made

    def stride(self, i=None):
        s = (self.row, 1) if self.ndim == 2 else (1,)
        return s if i is None else s[i]

    def data_ptr(self):
        return self.at

    def get_device(self):
        return 0


@pytest.fixture
def sent(monkeypatch):
    """Calls go to a list of (entry, bytes) in place of the library."""
    got = []
    for name in ("quantize_fp8", "linear_fp8", "add_gated_norms"):
        monkeypatch.setitem(ops._entries, name, lambda packed, name=name: got.append((name, packed)) or 0)
    monkeypatch.setitem(ops._status_at, 0, 0x7770)
    monkeypatch.setitem(ops._sm_counts, 0, 148)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0x5550, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    return got


def record(sent, entry: str, struct: type):
    name, packed = sent.pop()
    assert name == entry and not sent
    # (the compiler rounds a struct up to its alignment; nothing is read from there)
    assert ctypes.sizeof(struct) - 7 <= len(packed) <= ctypes.sizeof(struct)
    r = struct.from_buffer_copy(packed + bytes(8))
    return {f: getattr(r, f) for f, _ in struct._fields_}


BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,code", [(F32, ops.dtype_code(F32)), (BF, ops.dtype_code(BF))])
def test_quantize(sent, dtype, code):
    x, q = Matrix((300, 200), dtype), Matrix((300, 200), FP8)
    for block, rows in ((1, 300), (128, 3)):
        s = Matrix((rows, 2), F32)
        ops.quantize_fp8(x, q, s, block)
        assert record(sent, "quantize_fp8", declared("quantize_fp8.cu", "QuantizeFp8Args")) == {
            "x": x.at, "q": q.at, "s": s.at, "stream": 0x5550, "ldx": x.row, "ldq": q.row, "lds": s.row, "dtype": code, "T": 300, "K": 200,
            "block_rows": block, "sms": 148}


@pytest.mark.parametrize("static", [False, True])
@pytest.mark.parametrize("out_dtype", [F32, BF])
def test_product(sent, out_dtype, static):
    x, xs, w, ws, out = Matrix((7, 300), FP8), Matrix((7, 3), F32), Matrix((200, 300), FP8), Matrix((2, 3), F32), Matrix((7, 200), out_dtype)
    ops.linear_fp8(x, xs, w, ws, out, static_weights=static, plan=(2, 128, 5))
    assert record(sent, "linear_fp8", declared("gemm_fp8_tc.cu", "Fp8LinearArgs")) == {
        "x": x.at, "sx": xs.at, "w": w.at, "sw": ws.at, "out": out.at, "w2": None, "sw2": None, "so": None, "status": 0x7770, "stream": 0x5550,
        "ldx": x.row, "ldsx": xs.row, "ldw": w.row, "ldsw": ws.row, "ldo": out.row, "ldw2": 0, "ldsw2": 0, "ldso": 0,
        "M": 7, "N": 200, "K": 300, "out_f32": int(out_dtype is F32), "flags": int(static), "plan": 2 | 128 << 4 | 5 << 16, "sms": 148}


def test_gated_product(sent):
    x, xs, g, gs, u, us = (Matrix((7, 300), FP8), Matrix((7, 3), F32), Matrix((200, 300), FP8), Matrix((2, 3), F32), Matrix((200, 300), FP8),
                           Matrix((2, 3), F32))
    out, so = Matrix((7, 200), FP8), Matrix((7, 2), F32)
    ops.linear_fp8_swiglu(x, xs, g, gs, u, us, out, so, static_weights=True)
    assert record(sent, "linear_fp8", declared("gemm_fp8_tc.cu", "Fp8LinearArgs")) == {
        "x": x.at, "sx": xs.at, "w": g.at, "sw": gs.at, "out": out.at, "w2": u.at, "sw2": us.at, "so": so.at, "status": 0x7770, "stream": 0x5550,
        "ldx": x.row, "ldsx": xs.row, "ldw": g.row, "ldsw": gs.row, "ldo": out.row, "ldw2": u.row, "ldsw2": us.row, "ldso": so.row,
        "M": 7, "N": 200, "K": 300, "out_f32": 0, "flags": 1, "plan": 0, "sms": 148}


@pytest.mark.parametrize("gate", [None, "channels", "rows"])
@pytest.mark.parametrize("stream,delta,out_dtype,kind", [(F32, BF, FP8, 2), (BF, F32, BF, 1), (F32, F32, F32, 0), (BF, BF, None, 3)])
def test_norms(sent, stream, delta, out_dtype, kind, gate):
    x, d, w1, w2 = Matrix((5, 300), stream), Matrix((5, 300), delta), Matrix((300,), F32), Matrix((300,), F32)
    g = None if gate is None else Matrix((300,), F32) if gate == "channels" else Matrix((5, 300), BF)
    out = None if out_dtype is None else Matrix((5, 300), out_dtype)
    s = Matrix((5, 3), F32) if kind == 2 else None
    ops.add_gated_norms(x, d, out, s, post_weight=w1, post_eps=0.25, gate=g, residual_scale=0.75, weight=w2 if out is not None else None, eps=0.5,
                        static_weights=gate is None)
    at = lambda m: None if m is None else m.at
    row = lambda m: 0 if m is None else m.row
    rows = g if gate == "rows" else None
    assert record(sent, "add_gated_norms", declared("gated_norms.cu", "GatedNormsArgs")) == {
        "x": x.at, "d": d.at, "g": at(rows), "gc": at(g if gate == "channels" else None), "w1": w1.at, "w2": at(w2 if out is not None else None),
        "out": at(out), "s": at(s), "stream": 0x5550, "ldx": x.row, "ldd": d.row, "ldg": row(rows), "ldo": row(out), "lds": row(s),
        "x_dtype": ops.dtype_code(stream), "d_dtype": ops.dtype_code(delta), "g_dtype": ops.dtype_code(BF) if gate == "rows" else 0,
        "out_kind": kind, "T": 5, "H": 300, "sms": 148, "early_w": int(gate is None), "c": 0.75, "e1": 0.25, "e2": 0.5}
