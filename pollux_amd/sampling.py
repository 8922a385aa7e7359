"""The next token of each row of logits: generate's sampling rules on the device (generate.py:286-336).

The reference samples on the host's side of every step: repetition penalty,
temperature, top-k, top-p and one multinomial draw as a dozen tensor
operations and a copy to the host.  ``sample_rows`` (plx_sample_rows,
up to four kernels) takes its uniform numbers from the caller, so a step
can be captured in a graph and repeated exactly; min-p is there beside the
reference's rules.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib

_X_TYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


@dataclass(frozen=True)
class Sampling:
    """The rules of a sampled generation: each a number, or a tensor with a value per sequence.

    The defaults draw from the plain distribution; the reference's generate
    uses repetition_penalty 1.1 (generate.py:286-336).
    """

    temperature: float | torch.Tensor = 1.0
    top_k: int | torch.Tensor = 0
    top_p: float | torch.Tensor = 1.0
    min_p: float | torch.Tensor = 0.0
    repetition_penalty: float | torch.Tensor = 1.0


def sample_rows(
    logits: torch.Tensor,
    u: torch.Tensor,
    *,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor = 0,
    top_p: float | torch.Tensor = 1.0,
    min_p: float | torch.Tensor = 0.0,
    repetition_penalty: float | torch.Tensor = 1.0,
    seen: torch.Tensor | None = None,
    seen_len: torch.Tensor | None = None,
    vocab: int | None = None,
    out: torch.Tensor | None = None,
    details: bool = False,
):
    """int64 [rows]: a token per row of logits [rows, width] (fp32, fp16 or bf16), drawn by u [rows] (fp32, in [0, 1)).

    In this order: the logits of tokens in ``seen`` (int64 [rows, n], of which
    the first seen_len -- an int64 tensor of rows values, or of one -- count) are divided by
    repetition_penalty where positive and multiplied by it elsewhere;
    temperature; top_k > 0 leaves the k largest (of equal ones the lowest
    indices); top_p < 1 the smallest set of the largest whose probability
    reaches it; min_p those with at least min_p of the largest's probability;
    the token is the first, by index, at which the summed probability of what
    is left passes u.  temperature 0 takes the largest logit.  Each rule is a
    number or a tensor [rows] (top_k int64, the others fp32).  Only the first
    ``vocab`` columns are tokens (the padded rows of a head are not).

    A row without a distribution (a NaN, nothing above -inf, settings that are
    none) gets -1.  ``out``: where to put the tokens.  With ``details``:
    (tokens, log-probability of each among what was left fp32, how many were
    left int64; logits of -inf never are).
    """
    _lib.require_device(logits, "sample_rows logits")
    if logits.dim() != 2 or logits.dtype not in _X_TYPES:
        raise ValueError("sample_rows: logits [rows, width] in float32, float16 or bfloat16")
    rows, width = logits.shape
    n = width if vocab is None else int(vocab)
    if not 1 <= n <= width:
        raise ValueError(f"sample_rows: a vocabulary of {n} in rows of {width}")
    dev, index = logits.device, logits.get_device()
    x = logits if logits.stride(1) == 1 and (rows <= 1 or logits.stride(0) >= width) else logits.contiguous()
    keep = [x]

    def per_row(name: str, t: torch.Tensor, dtype: torch.dtype) -> int:
        if t.dtype != dtype or t.numel() != rows or t.get_device() != index:
            raise ValueError(f"sample_rows: {name} must be {dtype} with {rows} values on {dev}")
        if not t.is_contiguous():
            t = t.contiguous()
            keep.append(t)
        return t.data_ptr()

    u_ptr = per_row("u", u, torch.float32)
    rules = _lib.SampleRules(1.0, 1.0, 0.0, 1.0)
    for name, value in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p), ("penalty", repetition_penalty)):
        if isinstance(value, torch.Tensor):
            setattr(rules, name + "_rows", per_row(name, value, torch.float32))
        else:
            setattr(rules, name, value)
    if isinstance(top_k, torch.Tensor):
        rules.top_k_rows = per_row("top_k", top_k, torch.int64)
    else:
        rules.top_k = int(top_k)
    if seen is not None:
        if seen.dim() != 2 or seen.shape[0] != rows or seen.dtype != torch.int64 or seen.get_device() != index:
            raise ValueError(f"sample_rows: seen must be int64 [{rows}, n] on {dev}")
        if seen.stride(1) != 1 and seen.shape[1] > 1:
            seen = seen.contiguous()
            keep.append(seen)
        rules.seen, rules.seen_stride, rules.seen_cols = seen.data_ptr(), seen.stride(0), seen.shape[1]
        if seen_len is not None:
            if seen_len.dtype != torch.int64 or seen_len.numel() not in (1, rows) or seen_len.get_device() != index:
                raise ValueError(f"sample_rows: seen_len must be int64 with 1 or {rows} values on {dev}")
            if not seen_len.is_contiguous():
                seen_len = seen_len.contiguous()
                keep.append(seen_len)
            rules.seen_len, rules.seen_len_stride = seen_len.data_ptr(), int(seen_len.numel() > 1)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=dev)
    elif out.dtype != torch.int64 or out.numel() != rows or not out.is_contiguous() or out.device != dev:
        raise ValueError("sample_rows: out must be a contiguous int64 tensor with one element per row")
    logp = torch.empty(rows, dtype=torch.float32, device=dev) if details else None
    kept = torch.empty(rows, dtype=torch.int64, device=dev) if details else None
    with _lib.on_device(dev):
        lib = _lib.lib()
        need = lib.plx_sample_rows_workspace_bytes(rows, n)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        st = lib.plx_sample_rows(_lib.ptr(x), _X_TYPES[x.dtype], rows, n, x.stride(0) if rows > 1 else width, u_ptr,
                                 ctypes.byref(rules), _lib.ptr(out), _lib.ptr(logp), _lib.ptr(kept), _lib.ptr(ws), need,
                                 _lib.stream_of(dev))
    _lib.check(st, "sample_rows")
    return (out, logp, kept) if details else out
