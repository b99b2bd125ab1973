"""Next tokens from logits and given uniform numbers, with the settings of each row on the device (csrc/sampling.cu): a decoding step that draws its tokens has no
host reads and can be replayed from a CUDA graph.

The CPU path states the same contract in plain PyTorch, in 64 bits, and is the oracle of the numerics tests."""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Union

import torch

from .._native import register_signatures
from ._common import check, cur_stream, lib

MAX_VOCAB = 16 * 40960                  # logits that a cluster's shared memory holds
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
# the kernel's argument block, as csrc/sampling.cu declares it
_ARGS = struct.Struct("@8q3d6i")

Setting = Union[float, torch.Tensor]


@register_signatures
def _sigs(lib_):
    if hasattr(lib_, "tyr_sample"):
        lib_.tyr_sample.argtypes, lib_.tyr_sample.restype = [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p], ctypes.c_int


def _setting(name: str, v, rows: int, dev: int, dtype: torch.dtype, least: float):
    """(address, number) of a setting: a tensor with one number a row, or one for all."""
    if isinstance(v, torch.Tensor):
        if v.shape != (rows,) or v.dtype != dtype or not v.is_contiguous() or v.get_device() != dev:
            raise ValueError(f"sample: {name} is a number or contiguous {dtype} [{rows}] beside the logits")
        return v.data_ptr(), 0
    if not v >= least:
        raise ValueError(f"sample: {name} must be at least {least}, got {v}")
    return 0, v


def _sample_ref(logits, draws, temperature, top_k, top_p, min_p):
    column = lambda v: (v.double() if isinstance(v, torch.Tensor) else torch.full((logits.shape[0],), float(v), dtype=torch.float64, device=logits.device))[:, None]
    t, k, p, m = column(temperature), column(top_k), column(top_p), column(min_p).nan_to_num(nan=0.0).clamp(max=1.0)
    x = logits.double() + 0.0                                       # -0 is 0
    x = torch.where(torch.isnan(x), -math.inf, x)
    infinite = (x == math.inf).any(-1, keepdim=True)
    x = torch.where(infinite, torch.where(x == math.inf, 0.0, -math.inf), x)
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    none, greedy = x[:, :1] == -math.inf, ~(t > 0)
    ago = torch.where(x == -math.inf, -math.inf, x - torch.where(none, 0.0, x[:, :1]))
    w = torch.where(ago == -math.inf, 0.0, torch.exp(ago / torch.where(greedy, 1.0, t)))
    rank = torch.arange(x.shape[1], device=x.device)
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = w.cumsum(-1) - w
    kept = (w > 0) & (w >= m) & (~(p < 1) | (before < p * w.sum(-1, keepdim=True)) | (rank == 0))
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))
    c = w.cumsum(-1)
    past = (w > 0) & (c > draws.double()[:, None] * c[:, -1:])
    last = (torch.where(w > 0, rank, -1)).amax(-1, keepdim=True)
    token = torch.where(past.any(-1, keepdim=True), past.to(torch.uint8).argmax(-1, keepdim=True), last)
    return torch.where(none, -1, torch.where(greedy, order[:, :1], token))[:, 0]


def sample(logits: torch.Tensor, draws: torch.Tensor, *, temperature: Setting = 1.0, top_k: Optional[Union[int, torch.Tensor]] = None, top_p: Setting = 1.0,
           min_p: Setting = 0.0) -> torch.Tensor:
    """logits [rows, V] (bf16, fp16 or fp32), draws [rows] uniform in [0, 1) (fp32 or fp64) -> int64 [rows].

    With w = exp((logit - the row's largest) / ``temperature``) and the tokens in the order of their logits, equal ones by index: the first ``top_k`` stay (0 or None:
    all), of these those whose predecessors hold less than ``top_p`` of their weight (1: all; the first always stays), of these those with w >= ``min_p``.  The token is
    the first one, by index, at which the weight of what stays exceeds the row's draw times the whole.  All of it is decided in 64 bits, and a
    setting given as a number counts as such; a draw of 0 takes the first index that stays, however little it weighs, unless that rounds to nothing.

    A temperature of 0 takes the largest logit, the lowest index among equals.  -inf and NaN are never chosen, infinite logits share the draw; a row with nothing to
    choose from gives -1.  Every setting is a number or holds one for each row (fp32; ``top_k`` int32), on the logits' device; NaN for a row filters nothing there, and as its temperature
    takes the largest logit."""
    shape, dev = logits.shape, logits.get_device()
    if len(shape) != 2 or shape[0] == 0 or shape[1] == 0:
        raise ValueError(f"sample: logits are [rows, vocabulary], got {tuple(shape)}")
    B, V = shape
    if draws.shape != (B,) or draws.dtype not in (torch.float32, torch.float64) or draws.get_device() != dev:
        raise ValueError(f"sample: draws are fp32 or fp64 [{B}] beside the logits")
    top_k = 0 if top_k is None else top_k
    if not isinstance(top_k, (int, torch.Tensor)):
        raise ValueError(f"sample: top_k is a whole number, got {top_k}")
    t_at, t = _setting("temperature", temperature, B, dev, torch.float32, 0.0)
    k_at, k = _setting("top_k", top_k, B, dev, torch.int32, 0)
    p_at, p = _setting("top_p", top_p, B, dev, torch.float32, 0.0)
    m_at, m = _setting("min_p", min_p, B, dev, torch.float32, 0.0)
    if dev < 0:
        if not logits.is_floating_point():
            raise ValueError(f"sample: logits in {logits.dtype} are not supported")
        return _sample_ref(logits, draws, temperature, top_k, top_p, min_p)
    number = _DTYPES.get(logits.dtype)
    if number is None or V > MAX_VOCAB:
        raise ValueError(f"sample: {V} logits in {logits.dtype} are not supported (bf16, fp16 or fp32, up to {MAX_VOCAB})")
    row, one = logits.stride()
    if one != 1 and V > 1:
        logits, row = logits.contiguous(), V
    draws, device = draws.contiguous(), logits.device
    token = torch.empty(B, dtype=torch.int64, device=device)
    packed = _ARGS.pack(logits.data_ptr(), draws.data_ptr(), t_at, p_at, m_at, k_at, token.data_ptr(), row, t, p, m, B, V, 0, draws.dtype == torch.float64,
                        min(k, V), 0)
    check(lib().tyr_sample(packed, number, cur_stream(device)), "sample")
    return token
