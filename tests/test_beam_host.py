"""Refusals of the beam and shared-prefix entry points, before any launch (no GPU)."""

import pytest
import torch

import llm_cuda_b200._native as N
from llm_cuda_b200.kernels.beam import beam_reorder, beam_select
from llm_cuda_b200.kernels.shared_prefix import shared_prefix_decode


def _prefix(lib, q=16, ws=16, nbytes=1 << 40, B=4, Hq=8, Hkv=2, d=128, P=16, mp=4, np_=8, G=1,
            mg=4, dt=N.LLMC_BF16):
    return lib.llmc_shared_prefix_decode(q, 16, 16, 16, 16, 16, 16, 16, ws, nbytes, 16, B, Hq, Hkv,
                                         d, P, mp, np_, G, mg, 0.1, dt, 0, None)


def test_shared_prefix_refusals():
    lib = N.load()
    err = lib.llmc_last_error_string
    assert _prefix(lib, dt=9) == -1 and b"dtype" in err()
    assert _prefix(lib, Hkv=3) == -1 and b"multiple" in err()
    assert _prefix(lib, d=257) == -2
    assert _prefix(lib, q=None) == -1 and b"NULL" in err()
    assert _prefix(lib, ws=20) == -1 and b"aligned" in err()
    assert _prefix(lib, nbytes=16) == -1 and b"workspace" in err()
    assert _prefix(lib, mg=0) == -1
    assert _prefix(lib, G=5) == -1 and b"groups" in err()
    assert _prefix(lib, mp=1 << 28, P=16) == -1
    assert _prefix(lib, np_=1 << 28) == -2
    assert _prefix(lib, B=0) == 0
    need = lib.llmc_shared_prefix_workspace_bytes(4, 8, 2, 128, 16, 1, 4, N.LLMC_BF16)
    assert need > 0
    assert lib.llmc_shared_prefix_workspace_bytes(4, 8, 2, 128, 16, 1, 400, N.LLMC_BF16) == need
    assert lib.llmc_shared_prefix_workspace_bytes(4, 7, 2, 128, 16, 1, 4, N.LLMC_BF16) == 0


def _select(lib, logits=16, stride=100, G=1, K=4, V=100, n=4, eos=-1, fin=None, dt=N.LLMC_BF16):
    return lib.llmc_beam_select(logits, stride, 16, fin, 16, 16, 16, G, K, V, n, eos, dt, None)


def test_beam_select_refusals():
    lib = N.load()
    err = lib.llmc_last_error_string
    assert _select(lib, dt=5) == -1 and b"dtype" in err()
    assert _select(lib, K=33) == -1
    assert _select(lib, K=0) == -1
    assert _select(lib, n=65) == -1 and b"n <= 64" in err()
    assert _select(lib, V=1, stride=1, n=5) == -1
    assert _select(lib, stride=99) == -1 and b"row_stride" in err()
    assert _select(lib, fin=16) == -1 and b"eos" in err()
    assert _select(lib, fin=16, eos=100) == -1
    assert _select(lib, logits=17) == -1 and b"misaligned" in err()
    assert _select(lib, logits=18, dt=N.LLMC_F32) == -1
    assert _select(lib, logits=None) == -1
    assert _select(lib, G=0) == 0


def _reorder(lib, pools=16, own=16, bt=32, G=1, K=4, layers=2, Hkv=2, d=64, P=16, mp=4, np_=8, e=2):
    return lib.llmc_beam_reorder(pools, own, bt, 16, 16, 16, G, K, layers, Hkv, d, P, mp, np_, e,
                                 None)


def test_beam_reorder_refusals():
    lib = N.load()
    err = lib.llmc_last_error_string
    assert _reorder(lib, e=1) == -1 and b"elem_bytes" in err()
    assert _reorder(lib, K=33) == -1
    assert _reorder(lib, G=65536) == -1
    assert _reorder(lib, layers=0) == -1
    assert _reorder(lib, bt=16) == -1 and b"two tables" in err()
    assert _reorder(lib, pools=None) == -1
    assert _reorder(lib, P=1 << 20, d=1 << 10) == -2
    assert _reorder(lib, P=1 << 20, d=1, mp=1 << 12) == -1
    assert _reorder(lib, G=0) == 0


def test_python_entry_points_refuse_cpu_tensors():
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    kv = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        shared_prefix_decode(q, kv, kv, i.view(2, 1), i, i, i[:1])
    with pytest.raises(ValueError, match="CUDA"):
        beam_select(torch.zeros(2, 10), torch.zeros(1, 2))
    with pytest.raises(ValueError, match="CUDA"):
        beam_reorder(torch.zeros(1, 2, 4, 2, 16, 64), i.view(2, 1), i.view(2, 1), i, i.view(1, 2))


def test_beam_table_shares_the_prompts_full_pages():
    from llm_cuda_b200.models.llama3 import make_beam_table

    table, n = make_beam_table([33, 0, 48], beams=3, page_size=16, max_pages=4)
    assert table.shape == (9, 4) and n == (2 + 3 * 2) + 3 * 4 + (3 + 3 * 1)
    assert (table[0:3, :2] == table[0, :2]).all()            # 32 tokens shared
    assert (table[6:9, :3] == table[6, :3]).all()
    own = torch.cat([table[0:3, 2:].flatten(), table[3:6].flatten(), table[6:9, 3:].flatten()])
    names = torch.cat([own, table[0, :2], table[6, :3]]).tolist()
    assert sorted(names) == list(range(n))                   # every page once
    shuffled, m = make_beam_table([33, 0, 48], 3, 16, 4, torch.Generator().manual_seed(0))
    assert m == n and sorted(set(shuffled.flatten().tolist())) == list(range(n))
    with pytest.raises(ValueError, match="max_pages"):
        make_beam_table([65], 2, 16, 4 - 1)
    with pytest.raises(ValueError, match="beams"):
        make_beam_table([5], 0, 16, 4)


def test_beam_cache_layout_and_refusals():
    from llm_cuda_b200.models.llama3 import BeamKVCache, PagedKVLayerCache, SharedPrefix

    c = BeamKVCache(2, 2, 64, 40, 16, "cpu", torch.bfloat16, [20, 33], beams=4)
    assert c.pools.shape == (2, 2, 1 + 4 * 2 + 2 + 4 * 1, 2, 16, 64)
    for i, layer in enumerate(c.layer_caches):
        assert layer.batch_size == 8
        assert layer.key_pages.data_ptr() == c.pools[i, 0].data_ptr()
        assert layer.value_pages.data_ptr() == c.pools[i, 1].data_ptr()
        assert layer.block_table.data_ptr() == c.block_table.data_ptr()   # one table
    assert c.shared.max_group == 4 and c.shared.group_starts.tolist() == [0, 4, 8]
    lead = c.leaders().get_layer(1)
    assert lead.batch_size == 2 and lead.shared is None
    assert torch.equal(lead.block_table, c.own_table[::4])
    assert lead.key_pages.data_ptr() == c.pools[1, 0].data_ptr()
    with pytest.raises(ValueError, match="prompt"):
        BeamKVCache(1, 2, 64, 40, 16, "cpu", torch.bfloat16, [41], 2)
    with pytest.raises(ValueError, match="prompt"):
        BeamKVCache(1, 2, 64, 40, 16, "cpu", torch.bfloat16, [], 2)
    with pytest.raises(ValueError, match="ascending"):
        SharedPrefix([0, 3, 2], [1, 1], "cpu")
    with pytest.raises(ValueError, match="one entry more"):
        SharedPrefix([0, 3], [1, 1], "cpu")
    kv = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="go together"):
        PagedKVLayerCache(2, 64, 64, 16, "cpu", torch.bfloat16, key_pages=kv)
    with pytest.raises(ValueError, match="pools must be"):
        PagedKVLayerCache(2, 64, 64, 16, "cpu", torch.bfloat16, key_pages=kv[:3],
                          value_pages=kv[:3])


@pytest.mark.parametrize("beams", [0, 33])
def test_beam_cache_refuses_more_beams_than_the_kernels_take(beams):
    from llm_cuda_b200.models.llama3 import BeamKVCache

    with pytest.raises(ValueError, match="1 to 32 beams"):
        BeamKVCache(1, 2, 64, 40, 16, "cpu", torch.bfloat16, [20], beams)


def test_beam_select_refuses_a_vocabulary_past_its_ties():
    lib = N.load()
    assert _select(lib, V=(1 << 27) + 1, stride=1 << 28) == -2
    assert b"2^27" in lib.llmc_last_error_string()


def test_refused_step_over_shared_prefixes_appends_nothing():
    from llm_cuda_b200.models.llama3 import BeamKVCache

    c = BeamKVCache(1, 2, 64, 40, 16, "cpu", torch.bfloat16, [20], beams=2)
    lc = c.get_layer(0)
    lc.host_lengths = [20, 20]
    q, k = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="partition_tokens"):
        lc.rope_append_decode(q, k, k, None, partition_tokens=64)
    with pytest.raises(ValueError, match="out must"):
        lc.rope_append_decode(q, k, k, None, out=torch.zeros(2, 4, 1, 32, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="q must"):
        lc.rope_append_decode(q[:, :3], k, k, None)
    assert lc.host_lengths == [20, 20] and lc.seq_lens.tolist() == [0, 0]


def test_no_prompts_need_no_pointers():
    """An empty tensor's address is NULL."""
    lib = N.load()
    assert lib.llmc_beam_select(None, 100, None, None, None, None, None, 0, 4, 100, 4, -1,
                                N.LLMC_BF16, None) == 0


def test_cache_refuses_pools_and_groups_of_another_device():
    """A kernel would be given their addresses."""
    from llm_cuda_b200.models.llama3 import PagedKVLayerCache, SharedPrefix

    kv = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    far = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="meta")
    ok = PagedKVLayerCache(2, 64, 64, 16, "cpu", torch.bfloat16, key_pages=kv, value_pages=kv.clone(),
                           shared=SharedPrefix([0, 1], [5], "cpu"))
    assert ok.key_pages is kv
    for k, v in ((far, far), (kv, far), (far, kv)):
        with pytest.raises(ValueError, match="device"):
            PagedKVLayerCache(2, 64, 64, 16, "cpu", torch.bfloat16, key_pages=k, value_pages=v)
    with pytest.raises(ValueError, match="device"):
        PagedKVLayerCache(2, 64, 64, 16, "cpu", torch.bfloat16, key_pages=kv, value_pages=kv,
                          shared=SharedPrefix([0, 1], [5], "meta"))
