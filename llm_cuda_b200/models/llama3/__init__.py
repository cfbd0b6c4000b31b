"""Llama 3 decode-path modules mirroring ``llm_cuda.models.llama3``."""

from .kv_cache import (
    BeamKVCache,
    PagedKVCache,
    PagedKVLayerCache,
    SharedPrefix,
    make_beam_table,
    make_block_table,
)
from .rotary import RopeTable, build_inv_freq, build_rope_cache

__all__ = ["BeamKVCache", "PagedKVCache", "PagedKVLayerCache", "RopeTable", "SharedPrefix",
           "build_inv_freq", "build_rope_cache", "make_beam_table", "make_block_table"]
