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


def _rows(logits: torch.Tensor) -> torch.Tensor:
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise RuntimeError(f"logits: [rows, vocabulary] of float32, bfloat16 or float16, not {logits.dtype} {tuple(logits.shape)}")
    N.require_cuda(logits)
    if logits.shape[1] < 1 or logits.shape[1] > LARGEST:
        raise RuntimeError(f"logits of {logits.shape[1]} tokens: 1 to {LARGEST}")
    if logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("logits: draws and scores of tokens have no gradient")
    return logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()


def _vector(name: str, x: torch.Tensor, dtype: torch.dtype, logits: torch.Tensor) -> torch.Tensor:
    if x.shape != logits.shape[:1] or x.dtype is not dtype or x.device != logits.device:
        raise RuntimeError(f"{name}: {logits.shape[0]} numbers of {dtype} on {logits.device}, one a row, not {x.dtype} {tuple(x.shape)} on {x.device}")
    return x.contiguous()


def _setting(name: str, x: Setting, logits: torch.Tensor, off, low, high, dtype=torch.float32) -> Tuple[Optional[torch.Tensor], Union[int, float]]:
    """A row's numbers, or one of all."""
    if isinstance(x, torch.Tensor):
        return _vector(name, x, dtype, logits), off
    if x is None:
        return None, off
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
    logits = _rows(logits)
    t, t_all = _setting("temperature", temperature, logits, 1.0, 0.0, 3.0e38)
    k, k_all = _setting("top_k", top_k, logits, 0, 1, 2**31 - 1, torch.int32)
    p, p_all = _setting("top_p", top_p, logits, 1.0, 0.0, 1.0)
    m, m_all = _setting("min_p", min_p, logits, 0.0, 0.0, 1.0)
    u = _vector("u", u, torch.float32, logits)
    R, V = logits.shape
    out = u.new_empty(R, dtype=torch.int64)
    if R:
        with _NOTHING if _current_device() == logits.get_device() else torch.cuda.device(logits.device):
            N.call("ll_sample_rows", N.ptr(logits), N.dtype_code(logits.dtype), R, V, logits.stride(0), N.ptr(u), N.ptr(t), t_all, N.ptr(k), int(k_all), N.ptr(p), p_all,
                   N.ptr(m), m_all, N.ptr(out), N.stream())
    return out


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: Setting = 1.0) -> torch.Tensor:
    """Logarithms of the probabilities that softmax(``logits [rows, vocabulary]`` / temperature) gives to ``tokens [rows]`` (int64): float32 ``[rows]``.  No number
    for a token that is not of the vocabulary, or a row of which there is no softmax.  Sums are of 32 bits, by vectors of 16 bytes: a row's last bits go with where it begins."""
    logits = _rows(logits)
    t, t_all = _setting("temperature", temperature, logits, 1.0, 1.0e-30, 3.0e38)
    tokens = _vector("tokens", tokens, torch.int64, logits)
    R, V = logits.shape
    out = tokens.new_empty(R, dtype=torch.float32)
    if R:
        with _NOTHING if _current_device() == logits.get_device() else torch.cuda.device(logits.device):
            N.call("ll_token_logprobs", N.ptr(logits), N.dtype_code(logits.dtype), R, V, logits.stride(0), N.ptr(tokens), N.ptr(t), t_all, N.ptr(out), N.stream())
    return out
