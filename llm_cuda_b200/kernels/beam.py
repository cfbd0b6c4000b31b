"""Beam search over the paged cache (CUDA): selection and reordering.

``beam_select`` is to a beam search what ``argmax_rows`` is to the greedy loop
(``src/llm_cuda/models/llama3/model.py:214`` of llm-cuda): it picks the best continuations
of every prompt over its beams and the vocabulary.  ``beam_reorder`` then lets every beam
of the paged cache continue from its parent.  The reference decodes greedily and has no
counterpart of either.
"""

from __future__ import annotations

import torch

from .. import _native as N
from .decode_attention import default_status

MAX_BEAMS = 32
MAX_CANDIDATES = 64


def beam_select(
    logits: torch.Tensor,
    beam_scores: torch.Tensor,
    num_out: int | None = None,
    finished: torch.Tensor | None = None,
    eos_token_id: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``num_out`` (default: the number of beams) best of
    ``beam_scores[g, k] + log_softmax(logits[g, k])`` over the beams and the vocabulary.

    ``logits``: ``[G * K, V]`` or ``[G, K, V]``, the vocabulary contiguous (rows may be
    views into a wider buffer).  ``beam_scores`` fp32 ``[G, K]``.  ``finished`` bool
    ``[G, K]``: a finished beam offers ``eos_token_id`` at its own score and nothing else.
    A beam with a score or log-sum-exp that is not finite offers its tokens at ``-inf``.
    Returns ``(scores fp32, beams int32, tokens int64)``, each ``[G, num_out]``, best first,
    ties to the lowest (beam, token); beams of equal logits and scores tie wherever their rows
    begin.  A log-sum-exp is good to 2^-20: candidates of different beams that are closer come
    in either order.
    """
    lib = N.load()
    if not logits.is_cuda or not beam_scores.is_cuda:
        raise ValueError("beam_select needs CUDA tensors")
    if beam_scores.dim() != 2 or beam_scores.dtype != torch.float32:
        raise ValueError("beam_scores must be fp32 [prompts, beams]")
    G, K = beam_scores.shape
    if not 1 <= K <= MAX_BEAMS:
        raise ValueError(f"beam_select takes 1 to {MAX_BEAMS} beams")
    if logits.dim() == 3:
        if logits.shape[:2] != (G, K):
            raise ValueError("logits must be [prompts, beams, vocabulary]")
        if G > 1 and K > 1 and logits.stride(0) != K * logits.stride(1):
            logits = logits.contiguous()
        stride = logits.stride(1) if K > 1 else logits.stride(0)
    elif logits.dim() == 2:
        if logits.shape[0] != G * K:
            raise ValueError("logits must have one row per beam")
        stride = logits.stride(0)
    else:
        raise ValueError("logits must be [G * K, V] or [G, K, V]")
    V = logits.shape[-1]
    if V < 1:
        raise ValueError("the vocabulary is empty")
    if (V > 1 and logits.stride(-1) != 1) or (G * K > 1 and stride < V):
        logits = logits.contiguous()
        stride = V
    stride = max(stride, V)         # of a single row it says nothing
    n = K if num_out is None else int(num_out)
    if not 1 <= n <= min(MAX_CANDIDATES, K * V):
        raise ValueError(f"num_out must be 1 to {MAX_CANDIDATES} and at most beams * vocabulary")
    if logits.device != beam_scores.device:
        raise ValueError("logits and beam_scores must be on one device")
    eos = -1
    if finished is not None:
        if finished.shape != beam_scores.shape or finished.dtype not in (torch.bool, torch.uint8):
            raise ValueError("finished must be bool [prompts, beams]")
        if eos_token_id is None or not 0 <= int(eos_token_id) < V:
            raise ValueError("finished beams need an eos_token_id inside the vocabulary")
        if finished.device != logits.device:
            raise ValueError("finished must be on the device of the logits")
        eos = int(eos_token_id)
        finished = finished.contiguous()
    beam_scores = beam_scores.contiguous()
    dev = logits.device
    scores = torch.empty(G, n, dtype=torch.float32, device=dev)
    beams = torch.empty(G, n, dtype=torch.int32, device=dev)
    tokens = torch.empty(G, n, dtype=torch.int64, device=dev)
    with N.on_device(dev):
        rc = lib.llmc_beam_select(
            logits.data_ptr(), stride, beam_scores.data_ptr(), N.ptr(finished), scores.data_ptr(),
            beams.data_ptr(), tokens.data_ptr(), G, K, V, n, eos, N.dtype_code(logits.dtype),
            N.raw_stream(dev))
    N.check(rc, "llmc_beam_select")
    return scores, beams, tokens


def beam_reorder(
    pools: torch.Tensor,
    own_table: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    parents: torch.Tensor,
    status: torch.Tensor | None = None,
) -> None:
    """Beam ``i`` of every prompt becomes a continuation of beam ``parents[g, i]``, in place.

    ``pools`` ``[layers, 2, num_pages, Hkv, page_size, d]``: the K and V pools of all layers.
    ``own_table`` int32 ``[G * K, max_pages]``: the pages that each beam writes (constant,
    distinct behind the prompt); ``block_table``, the same shape: the pages that it reads,
    updated here.  ``seq_lens`` int32 ``[G * K]``: the tokens held, equal for the beams of a
    prompt.  ``parents`` int32 ``[G, K]``.  Full pages are shared between beams, the page in
    progress is copied.  A bad parent, page or length sets ``status`` and leaves its prompt
    as it was.
    """
    lib = N.load()
    if not pools.is_cuda:
        raise ValueError("beam_reorder needs CUDA tensors")
    if pools.dim() != 6 or pools.shape[1] != 2 or not pools.is_contiguous():
        raise ValueError("pools must be contiguous [layers, 2, num_pages, Hkv, page_size, d]")
    N.dtype_code(pools.dtype)
    if parents.dim() != 2 or parents.dtype != torch.int32:
        raise ValueError("parents must be int32 [prompts, beams]")
    G, K = parents.shape
    if not 1 <= K <= MAX_BEAMS:
        raise ValueError(f"beam_reorder takes 1 to {MAX_BEAMS} beams")
    for t, what in ((own_table, "own_table"), (block_table, "block_table")):
        if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != G * K or \
                not t.is_contiguous() or t.device != pools.device:
            raise ValueError(f"{what} must be contiguous int32 [prompts * beams, max_pages]")
    if own_table.shape != block_table.shape or (
            G * K > 0 and own_table.data_ptr() == block_table.data_ptr()):
        raise ValueError("own_table and block_table must be two tables of one shape")
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (G * K,) or \
            not seq_lens.is_contiguous() or seq_lens.device != pools.device:
        raise ValueError("seq_lens must be contiguous int32 [prompts * beams]")
    if parents.device != pools.device:
        raise ValueError("parents must be on the device of the pools")
    if G == 0:
        return
    parents = parents.contiguous()
    layers, _, num_pages, Hkv, P, d = pools.shape
    st = status if status is not None else default_status(pools.device)
    with N.on_device(pools.device):
        rc = lib.llmc_beam_reorder(
            pools.data_ptr(), own_table.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
            parents.data_ptr(), st.data_ptr(), G, K, layers, Hkv, d, P, own_table.shape[1],
            num_pages, pools.element_size(), N.raw_stream(pools.device))
    N.check(rc, "llmc_beam_reorder")
