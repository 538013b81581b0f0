"""Attention of prompt chunks over the paged K/V cache (``pa_prompt`` in the C ABI).

The reference attends from one new token per sequence; its caches are filled by
test code (``tests/correctness.py:30-36``). A serving loop first runs the prompt:
it writes a chunk's K and V with ``write_kv_cache`` and attends from all of its
tokens at once, causally, over everything the sequence has cached, under the same
sliding window as the decode steps that follow (``paged_attention(window=...)``).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from ._native import PagedAttentionError
from .torch_kernel import DecodeWorkspace, default_workspace, window_args


def paged_prompt_attention(Q: torch.Tensor, K_Cache: torch.Tensor, V_Cache: torch.Tensor,
                           Block_Table: torch.Tensor, query_starts: torch.Tensor,
                           seq_lens: torch.Tensor, block_size: int, *,
                           window: Optional[int] = None, num_sinks: int = 0,
                           scale: Optional[float] = None, return_lse: bool = False,
                           num_splits: Optional[int] = None,
                           workspace: Optional[DecodeWorkspace] = None,
                           out: Optional[torch.Tensor] = None):
    """``O [T, Hq, D]`` for packed queries ``Q [T, Hq, D]`` of ``B`` sequences.

    Sequence ``b`` owns rows ``query_starts[b] .. query_starts[b + 1] - 1`` (int32
    ``[B + 1]``, ascending); they are its last tokens, ``seq_lens[b]`` (int32 ``[B]``)
    counting them in. The row at position p sees token t when ``t <= p`` and, with a
    ``window``, ``t < num_sinks or t > p - window``. Pages with no visible token are not
    read (entry -1 will do). Rows that see nothing get 0 and LSE -1e30; rows outside
    every sequence (padding) are left as they were in ``out``, their LSE is not set.
    Scores of NaN or +infinity make their row and its LSE NaN.

    Probabilities are rounded once to Q's type before the product with V (sums, maxima
    and outputs are held in 32 bits), where ``paged_attention`` keeps twice as many bits
    of them: one token through either differs by a rounding.

    ``return_lse=True`` adds ``LSE [T, Hq]`` (fp32, natural log). ``num_splits``: parts of
    the keys that separate CTAs take and a second kernel joins (default: chosen by the
    sizes). Asynchronous on the current stream; scratch comes from ``workspace``
    (default: the stream's), whose status word gets ``PA_STATUS_*`` bits; as with
    ``paged_attention``, calls that share one must be ordered, and a graph keeps the one
    it was captured with, grown by a call before. Inference only."""
    win, sinks = window_args("paged_prompt_attention", window, num_sinks)
    if num_splits is not None and int(num_splits) < 1:
        raise ValueError("paged_prompt_attention: num_splits must be at least 1")
    if scale is not None and not float(scale) > 0:
        raise ValueError("paged_prompt_attention: scale must be positive")
    if torch.is_grad_enabled() and (Q.requires_grad or K_Cache.requires_grad
                                    or V_Cache.requires_grad):
        raise RuntimeError("paged_prompt_attention is inference-only.")
    if not Q.is_cuda:
        raise ValueError("paged_prompt_attention: all tensors must be CUDA tensors")
    ws = workspace if workspace is not None else default_workspace(Q.device)
    ext = _native.ext()
    for _ in range(2):
        status, res, need = ext.prompt(
            Q, K_Cache, V_Cache, Block_Table, query_starts, seq_lens, int(block_size),
            0.0 if scale is None else float(scale), bool(return_lse), ws.buffer, ws.status, out,
            win, sinks, 0 if num_splits is None else int(num_splits))
        if status == 0:
            return res[0] if len(res) == 1 else tuple(res)
        ws.ensure(need, 0)
    raise PagedAttentionError("pa_prompt", _native.PA_ERR_WORKSPACE)
