"""Paged decode attention for a batch whose sequences share prefixes (CUDA).

Beams of one prompt, or requests behind one system prompt, hold the same first tokens.
``shared_prefix_decode`` computes what ``paged_decode`` computes, but reads the shared
tokens of a group of sequences once for all of them.  The reference decodes one sequence
(``src/llm_cuda/kernels/triton/decode_attention.py:204-287`` of llm-cuda) and has no
counterpart.

Scores, softmax statistics and partial sums are fp32 and the output is rounded once;
``paged_decode`` rounds 16-bit scores as the reference's torch path does, so the two agree
to the tensor type's accuracy, not bit for bit.
"""

from __future__ import annotations

import functools
import math

import torch

from .. import _native as N
from .decode_attention import default_status


def _check_index(t: torch.Tensor, what: str, dim: int, device: torch.device) -> None:
    if t.dtype != torch.int32 or t.dim() != dim:
        raise ValueError(f"{what} must be a {dim}-D int32 tensor")
    if t.device != device or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous on the device of q")


def shared_prefix_decode(
    q: torch.Tensor,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    group_starts: torch.Tensor,
    shared_lens: torch.Tensor,
    *,
    max_group: int | None = None,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
    force_generic: bool = False,
) -> torch.Tensor:
    """Decode attention of ``q [B, Hq, d]`` (or ``[B, Hq, 1, d]``) over paged K/V.

    ``group_starts`` int32 ``[G + 1]``: group ``g`` holds the sequences
    ``group_starts[g] .. group_starts[g + 1] - 1``.  ``shared_lens`` int32 ``[G]``: how many
    first tokens the group's sequences have in common (any number, 0 for none).  Every row
    of ``block_table`` names all pages of its sequence.  ``max_group`` bounds the sequences
    of a group (default: the batch); it sizes the workspace (512 sequences of 64/8 heads in as
    many groups: 104 MB with 1, 630 MB with the default), and sequences of a group beyond it
    are decoded by themselves.  Sequences of length 0 give zeros.  All lengths
    are read on the device, so the call can be captured in a CUDA graph.
    """
    lib = N.load()
    if not q.is_cuda:
        raise ValueError("shared_prefix_decode needs CUDA tensors")
    dev, dtype, q_shape = q.device, q.dtype, q.shape
    if len(q_shape) == 4:
        if q_shape[2] != 1:
            raise ValueError("q must be [B, Hq, d] or [B, Hq, 1, d]: one query token per sequence")
        q = q.reshape(q_shape[0], q_shape[1], q_shape[3])
    elif len(q_shape) != 3:
        raise ValueError("q must be [B, Hq, d] or [B, Hq, 1, d]: one query token per sequence")
    q = q.contiguous()
    B, Hq, d = q.shape
    pages = key_pages.shape
    if len(pages) != 4 or value_pages.shape != pages or pages[3] != d:
        raise ValueError("pages must be [num_pages, Hkv, page_size, d] with the head_dim of q")
    if key_pages.dtype != dtype or value_pages.dtype != dtype:
        raise ValueError("q and pages must share a dtype")
    if key_pages.device != dev or value_pages.device != dev:
        raise ValueError("q and pages must be on one device")
    if not (key_pages.is_contiguous() and value_pages.is_contiguous()):
        raise ValueError("pages must be contiguous")
    num_pages, Hkv, P, _ = pages
    if Hq % Hkv:
        raise ValueError("n_heads must be a multiple of n_kv_heads")
    _check_index(block_table, "block_table", 2, dev)
    _check_index(seq_lens, "seq_lens", 1, dev)
    _check_index(group_starts, "group_starts", 1, dev)
    _check_index(shared_lens, "shared_lens", 1, dev)
    G = shared_lens.shape[0]
    rows, max_pages = block_table.shape
    if rows != B or seq_lens.shape[0] != B:
        raise ValueError("block_table and seq_lens must have one row per sequence")
    if group_starts.shape[0] != G + 1:
        raise ValueError("group_starts must have one entry more than shared_lens")
    max_group = B if max_group is None else int(max_group)
    if max_group < 1 and B > 0:
        raise ValueError("max_group must be positive")
    max_group = max(1, min(max_group, B))
    if out is None:
        out = torch.empty(q_shape, dtype=dtype, device=dev)
    elif out.shape not in (q.shape, q_shape) or out.dtype != dtype or out.device != dev or \
            not out.is_contiguous():
        raise ValueError("out must be contiguous and match q")
    elif out.shape != q_shape:
        out = out.view(q_shape)
    if B == 0:
        return out
    dt = N.dtype_code(dtype)
    st = status if status is not None else default_status(dev)
    with N.on_device(dev):
        # From the caching allocator, per call: ordered with the stream, private to a graph
        # that captures it, never shared by two calls in flight.
        nbytes = _workspace_bytes(dev.index, B, Hq, Hkv, d, P, G, max_group, dt)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = lib.llmc_shared_prefix_decode(
            q.data_ptr(), key_pages.data_ptr(), value_pages.data_ptr(), block_table.data_ptr(),
            seq_lens.data_ptr(), group_starts.data_ptr(), shared_lens.data_ptr(), out.data_ptr(),
            ws.data_ptr(), nbytes, st.data_ptr(), B, Hq, Hkv, d, P, max_pages, num_pages, G,
            max_group, 1.0 / math.sqrt(d) if scale is None else float(scale), dt,
            N.LLMC_DECODE_FORCE_GENERIC if force_generic else 0, N.raw_stream(dev))
    N.check(rc, "llmc_shared_prefix_decode")
    return out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device_index: int, *sizes: int) -> int:
    return max(16, N.load().llmc_shared_prefix_workspace_bytes(*sizes))
