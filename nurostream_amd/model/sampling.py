"""Sampling the next token of each row of logits on the GPU, from given random numbers (the reference's api.py:179-191
samples one row on the host's side, by temperature and top-p)."""
from __future__ import annotations

import ctypes as C

import torch

from .. import _native as N
from .draft import _call, _check, _ptr


def _setting(name: str, x, dtype: torch.dtype, device, B: int):
    """(the host's value, None) or (0, the device array)."""
    if isinstance(x, torch.Tensor):
        _check(name, x, dtype, device, B)
        return 0, x
    return x, None


def sample(logits: torch.Tensor, uniforms: torch.Tensor | None = None, *, temperature: float | torch.Tensor = 1.0,
           top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0, min_p: float | torch.Tensor = 0.0,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """A token for each row of logits (B, vocab), fp32 / fp16 / bf16 -> (B,) int32.

    Weights e^((x - max) / temperature); of the tokens by descending logit (equal ones by their index) the first top_k (0:
    all), of those the ones before which less than top_p of their whole weight lies (1: all), of those the ones of at
    least min_p of the largest weight; then the first token, in index order, at which the running sum of the weights exceeds
    uniforms[row] ((B,) fp32 in [0, 1)) times their total. temperature 0: the largest logit, the lowest index of equals
    (uniforms may be None). A NaN logit counts as -infinity; a row without any weight gives -1. Each setting is a number, or
    a device tensor (B,) of one per row (fp32; top_k int32), where a temperature of 0 or less is greedy, a top_k below 1 and
    a top_p of 1 or more leave all, and a top_p of 0 or less or a min_p of 1 or more leaves the likeliest."""
    if logits.dim() != 2:
        raise ValueError(f"logits of shape {tuple(logits.shape)}: (rows, vocab)")
    N.require_device(logits)
    code = N.act_dtype_code(logits.dtype)
    B, V = logits.shape
    dev = logits.device
    if V and (logits.stride(1) != 1 or (B > 1 and logits.stride(0) < V)):
        logits = logits.contiguous()
    ld = logits.stride(0) if B > 1 else V
    _check("uniforms", uniforms, torch.float32, dev, B)
    t, ts = _setting("temperature", temperature, torch.float32, dev, B)
    p, ps = _setting("top_p", top_p, torch.float32, dev, B)
    m, ms = _setting("min_p", min_p, torch.float32, dev, B)
    k, ks = _setting("top_k", top_k, torch.int32, dev, B)
    _check("out", out, torch.int32, dev, B)
    token = torch.empty(B, dtype=torch.int32, device=dev) if out is None else out
    lib = N.load()
    nb = max(16, lib.nsx_sample_workspace_bytes(B, V))
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)  # stream-ordered scratch, as the output
    settings = N.SamplingC(float(t), float(p), float(m), max(-1, min(int(k), V)), _ptr(ts), _ptr(ps), _ptr(ms), _ptr(ks))
    _call("sample", lib.nsx_sample, dev, logits.data_ptr(), code, ld, B, V, _ptr(uniforms), C.byref(settings), token.data_ptr(),
          ws.data_ptr(), nb)
    return token


__all__ = ["sample"]
