"""Weights from safetensors, by tensor name.

The model's parts declare what they need (``ParamSpec``); this module turns that
into the list of checkpoint tensors, reads them from every ``*.safetensors`` of the
folder (sorted, as serve.py:1389-1393 does; the index json is not needed), places
fused parameters row range by row range (q/k/v into qkv_proj, gate/up into
gate_up_proj: serve.py:72-74, 1352-1358) and hands every part its tensors.

Dtypes: matrices are kept in the engine's dtype; vectors too, except that a tensor
the file stores in 32-bit stays 32-bit; integer tables become int32.

Errors: one ``WeightError`` lists all missing tensors, all unexpected tensors and all
wrong shapes (tinyserve asserts on missing ones and warns on unused ones,
serve.py:1397-1403).  ``lm_head.weight`` in a checkpoint of a tied model is ignored,
as it has no home there either (serve.py:1385-1387)."""
from __future__ import annotations

import math
import os
import re
from dataclasses import dataclass

import torch
from safetensors import safe_open

from ..kernels import ops
from ..parts.base import ParamSpec, Source, interleave_halves


class WeightError(RuntimeError):
    """The checkpoint does not fit the model; the message lists every fault."""

    def __init__(self, missing, unexpected, wrong_shape, duplicates=()):
        self.missing, self.unexpected = list(missing), list(unexpected)
        self.wrong_shape, self.duplicates = list(wrong_shape), list(duplicates)
        lines = ["checkpoint does not match the model:"]
        if self.missing:
            lines.append(f"  missing tensors ({len(self.missing)}): " + ", ".join(self.missing))
        if self.unexpected:
            lines.append(f"  unexpected tensors ({len(self.unexpected)}): " + ", ".join(self.unexpected))
        for name, got, want in self.wrong_shape:
            lines.append(f"  wrong shape: {name} is {list(got)}, expected {list(want)}")
        if self.duplicates:
            lines.append(f"  stored twice ({len(self.duplicates)}): " + ", ".join(self.duplicates))
        super().__init__("\n".join(lines))


@dataclass(frozen=True)
class ExpectedTensor:
    name: str            # checkpoint tensor name
    shape: tuple
    part: object
    param: str           # local parameter name in the part
    spec: ParamSpec
    row_start: int
    row_end: int


def _sources(local_name: str, spec: ParamSpec):
    if spec.sources:
        return spec.sources
    rows = spec.shape[0] if spec.shape else 1
    return (Source(local_name, 0, rows),)


def expected_tensors(model) -> list:
    """Every checkpoint tensor the model reads, in a fixed order."""
    out = []
    rules = [(re.compile(pattern), repl) for pattern, repl in getattr(getattr(model, "spec", None), "name_rules", ())]
    for part in model.named_parts():
        for local, spec in part.param_specs().items():
            for src in _sources(local, spec):
                shape = (src.row_end - src.row_start,) + tuple(spec.shape[1:])
                name = f"{part.path}.{src.name}" if part.path else src.name
                for pattern, repl in rules:
                    name = pattern.sub(repl, name)
                out.append(ExpectedTensor(name, shape, part, local, spec, src.row_start, src.row_end))
    return out


def _param_dtype(spec: ParamSpec, engine_dtype, stored_dtypes):
    if spec.role == "int_table":
        return torch.int32
    if spec.role == "vector" and all(d == torch.float32 for d in stored_dtypes):
        return torch.float32
    return engine_dtype


def tensor_shapes(model_dir) -> dict:
    """{tensor name: shape} of every ``*.safetensors`` file of the folder (headers only)."""
    index, _ = _index_folder(model_dir)
    return {name: shape for name, (_, shape, _) in index.items()}


def _index_folder(model_dir):
    files = sorted(f for f in os.listdir(model_dir) if f.endswith(".safetensors"))
    if not files:
        raise FileNotFoundError(f"{model_dir!r} holds no *.safetensors file")
    index, duplicates = {}, []
    for fname in files:
        with safe_open(os.path.join(model_dir, fname), "pt", device="cpu") as fh:
            for key in fh.keys():
                if key in index:
                    duplicates.append(key)
                sl = fh.get_slice(key)
                index[key] = (fname, tuple(sl.get_shape()), sl.get_dtype())
    return index, duplicates


_ST_DTYPES = {"F32": torch.float32, "BF16": torch.bfloat16, "F16": torch.float16,
              "F64": torch.float64, "I32": torch.int32, "I64": torch.int64, "I16": torch.int16,
              "I8": torch.int8, "U8": torch.uint8, "BOOL": torch.bool}


def check_checkpoint(model, index, duplicates=()):
    """Compare the model's expected tensors with a {name: (file, shape, dtype)} index."""
    expected = expected_tensors(model)
    names = {e.name for e in expected}
    missing = [e.name for e in expected if e.name not in index]
    tied = model.lm_head is None if hasattr(model, "lm_head") else False
    unread = [re.compile(pattern) for pattern in getattr(getattr(model, "spec", None), "unread_names", ())]
    unexpected = [k for k in sorted(index) if k not in names
                  and not (tied and k == "lm_head.weight")
                  and not any(pattern.fullmatch(k) for pattern in unread)]
    wrong = [(e.name, index[e.name][1], e.shape) for e in expected
             if e.name in index and tuple(index[e.name][1]) != tuple(e.shape)]
    if missing or unexpected or wrong or duplicates:
        raise WeightError(missing, unexpected, wrong, duplicates)
    return expected


def check_weight_dtype(model, weight_dtype: str) -> float:
    """The share of the model's parameters that ``weight_dtype`` changes; one that changes nothing is refused."""
    sizes = [(math.prod(spec.shape), spec.int8) for part in model.named_parts() for spec in part.param_specs().values()]
    share = sum(n for n, int8 in sizes if int8) / max(1, sum(n for n, _ in sizes)) if weight_dtype == "int8" else 0.0
    if weight_dtype == "int8" and share == 0.0:
        raise ValueError("no matrix of the model can be held in 8 bits: only the projections of attention and of dense feed-forwards are, "
                         "and it has none")
    return share


def held(spec: ParamSpec, tensor, weight_dtype: str):
    """A parameter as the engine holds it: with ``weight_dtype`` "int8" the matrices that only products read are brought to 8
    bits, row by row.  Returns (what the part binds, its bytes)."""
    if weight_dtype == "int8" and spec.int8:
        rows = ops.quantize_rows(tensor)
        return rows, rows.codes.numel() + 4 * rows.scales.numel()
    return tensor, tensor.numel() * tensor.element_size()


def settle(device) -> None:
    """What was placed on ``device`` is complete when this returns: products fetch weights ahead of their wait for the kernels before
    them, and some weights are results of kernels (codes of 8 bits, interleaved rows)."""
    if torch.device(device).type == "cuda":
        torch.cuda.synchronize(device)


def load_weights(model, model_dir: str, dtype: torch.dtype, device, weight_dtype: str = "auto") -> int:
    """Fill every part of ``model`` from ``model_dir``; returns the bytes placed.  ``weight_dtype``: see ``held``."""
    check_weight_dtype(model, weight_dtype)
    index, duplicates = _index_folder(model_dir)
    expected = check_checkpoint(model, index, duplicates)
    by_param = {}
    for e in expected:
        by_param.setdefault((id(e.part), e.param), []).append(e)
    tensors, handles, total = {}, {}, 0
    try:
        for (_, local), entries in by_param.items():
            part, spec = entries[0].part, entries[0].spec
            stored = [_ST_DTYPES.get(index[e.name][2], torch.float32) for e in entries]
            pdtype = _param_dtype(spec, dtype, stored)
            param = torch.empty(spec.shape, dtype=pdtype, device=device)
            for e in entries:
                fname = index[e.name][0]
                if fname not in handles:
                    handles[fname] = safe_open(os.path.join(model_dir, fname), "pt", device="cpu")
                src = handles[fname].get_tensor(e.name)
                dst = param[e.row_start:e.row_end] if param.dim() else param
                dst.copy_(src.to(pdtype) if src.dtype != pdtype else src)
            if spec.interleave_halves:
                param = interleave_halves(param, spec.interleave_halves).contiguous()
            param, size = held(spec, param, weight_dtype)
            tensors.setdefault(id(part), (part, {}))[1][local] = param
            total += size
    finally:
        handles.clear()
    for part, bound in tensors.values():
        part.bind(bound)
    for part in model.named_parts():
        if id(part) not in tensors:
            part.bind({})
    settle(device)
    return total
