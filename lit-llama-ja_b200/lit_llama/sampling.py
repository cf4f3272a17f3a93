"""What a step's logits are asked: one token a row from given random numbers, and how likely given tokens are.

    u = torch.rand(rows, device=logits.device)
    tokens = sample(logits, u, temperature=0.8, top_k=200, top_p=0.95, min_p=0.02)
    scores = token_logprobs(logits, tokens)

Settings are numbers, or one a row on the GPU: requests of a served batch have their own.  Nothing looks at them on the host, so that a captured step
serves any.  Both go to the current stream of the logits' device.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Tuple, Union

import torch

from . import _native as N

_NOTHING = contextlib.nullcontext()
_current_device = N._current_device or torch.cuda.current_device

Setting = Union[None, int, float, torch.Tensor]

LARGEST = 1 << 18                    # of a vocabulary whose weights' sum has 62 bits


_TYPES = {torch.float32: N.LL_F32, torch.bfloat16: N.LL_BF16, torch.float16: N.LL_F16}


def _rows(logits: torch.Tensor) -> Tuple[torch.Tensor, int, int, int, int]:
    """The logits as the kernels take them, their type's number, rows, vocabulary and device."""
    code = _TYPES.get(logits.dtype)
    if logits.dim() != 2 or code is None:
        raise RuntimeError(f"logits: [rows, vocabulary] of float32, bfloat16 or float16, not {logits.dtype} {tuple(logits.shape)}")
    N.require_cuda(logits)
    R, V = logits.shape
    if not 0 < V <= LARGEST:
        raise RuntimeError(f"logits of {V} tokens: 1 to {LARGEST}")
    if logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("logits: draws and scores of tokens have no gradient")
    return logits if V == 1 or logits.stride(1) == 1 else logits.contiguous(), code, R, V, logits.get_device()


def _vector(name: str, x: torch.Tensor, dtype: torch.dtype, R: int, device: int) -> torch.Tensor:
    if x.dtype is not dtype or x.get_device() != device or x.shape != (R,):
        raise RuntimeError(f"{name}: {R} numbers of {dtype} on cuda:{device}, one a row, not {x.dtype} {tuple(x.shape)} on {x.device}")
    return x if x.is_contiguous() else x.contiguous()


def _setting(name: str, x: Setting, R: int, device: int, off, low, high, dtype=torch.float32) -> Tuple[Optional[torch.Tensor], Union[int, float]]:
    """A row's numbers, or one of all."""
    if x is None:
        return None, off
    if isinstance(x, torch.Tensor):
        return _vector(name, x, dtype, R, device), off
    if not low <= x <= high or (dtype is torch.int32 and x != int(x)):      # (no numbers too)
        raise ValueError(f"{name} {x}: {low} to {high}")
    return None, x


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature: Setting = 1.0, top_k: Setting = None, top_p: Setting = None, min_p: Setting = None) -> torch.Tensor:
    """Draw a token a row of ``logits [rows, vocabulary]``, from ``u [rows]`` (float32, 0 to 1): int64 ``[rows]``.

    Kept are the ``top_k`` largest logits, of these the largest ones until their probabilities reach ``top_p`` of the kept ones', of these those of at
    least ``min_p`` of the largest probability; equal logits stay together, as ``generate``'s top_k keeps them.  The draw goes through the kept ones in the
    order of the vocabulary.  Weights are whole numbers of 2^-44 of the largest one, so that a draw depends on no order of sums; a token of less is not
    drawn.  ``temperature`` 0 (under 2^-100): the largest logit (of equal ones the first).

    Settings are numbers or one a row on the GPU, float32 (``top_k`` int32); there a ``top_k`` below 1, a ``top_p`` of 1 and a ``min_p`` of 0 change nothing.  A row that
    allows no draw gets -1: a logit or setting that is no number, no logit above -inf, a negative temperature, a ``u`` outside of 0 to 1."""
    logits, code, R, V, device = _rows(logits)
    t, t_all = _setting("temperature", temperature, R, device, 1.0, 0.0, 3.0e38)
    k, k_all = _setting("top_k", top_k, R, device, 0, 1, 2**31 - 1, torch.int32)
    p, p_all = _setting("top_p", top_p, R, device, 1.0, 0.0, 1.0)
    m, m_all = _setting("min_p", min_p, R, device, 0.0, 0.0, 1.0)
    u = _vector("u", u, torch.float32, R, device)
    out = u.new_empty(R, dtype=torch.int64)
    if R:
        with _NOTHING if _current_device() == device else torch.cuda.device(device):
            N.call("ll_sample_rows", logits.data_ptr(), code, R, V, logits.stride(0), u.data_ptr(), N.ptr(t), t_all, N.ptr(k), int(k_all), N.ptr(p), p_all, N.ptr(m), m_all,
                   out.data_ptr(), N.stream())
    return out


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: Setting = 1.0) -> torch.Tensor:
    """Logarithms of the probabilities that softmax(``logits [rows, vocabulary]`` / temperature) gives to ``tokens [rows]`` (int64): float32 ``[rows]``.  No number
    for a token that is not of the vocabulary, or a row of which there is no softmax.  Batches of vectors of 16 bytes are added up in 32 bits,
    and these in 64 for 32-bit rows that are not short: a row's last bits go with where it begins."""
    logits, code, R, V, device = _rows(logits)
    t, t_all = _setting("temperature", temperature, R, device, 1.0, 1.0e-30, 3.0e38)
    tokens = _vector("tokens", tokens, torch.int64, R, device)
    out = tokens.new_empty(R, dtype=torch.float32)
    if R:
        with _NOTHING if _current_device() == device else torch.cuda.device(device):
            N.call("ll_token_logprobs", logits.data_ptr(), code, R, V, logits.stride(0), tokens.data_ptr(), N.ptr(t), t_all, out.data_ptr(), N.stream())
    return out
