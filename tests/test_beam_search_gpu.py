"""The beam operators together, as a beam search uses them."""

import pytest
import torch

from llm_cuda_b200.kernels.beam import beam_select
from llm_cuda_b200.models.llama3 import BeamKVCache, RopeTable
from llm_cuda_b200.models.llama3.decode_model import DecodeConfig, Llama3DecodeModel

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def attend(q, k, v):
    """64-bit attention of q [Hq, d] over k, v [Hkv, L, d]."""
    r = q.shape[0] // k.shape[0]
    k, v = k.double().repeat_interleave(r, 0), v.double().repeat_interleave(r, 0)
    p = torch.softmax(torch.einsum("hd,htd->ht", q.double(), k) * q.shape[-1] ** -0.5, -1)
    return torch.einsum("ht,htd->hd", p, v), torch.einsum("ht,htd->hd", p, v.abs())


@pytest.mark.parametrize("prompts,beams,hq,hkv,d,P,dtype", [
    ([37, 16, 5], 4, 32, 8, 128, 16, torch.bfloat16),
    ([64, 33], 5, 8, 2, 64, 16, torch.float16),
    ([20, 9], 3, 4, 2, 64, 8, torch.float32),
    ([130], 8, 16, 4, 128, 128, torch.bfloat16)])
def test_cache_follows_its_beams(prompts, beams, hq, hkv, d, P, dtype):
    """Append, attend, reorder over many steps: every beam's cache equals the history of its
    own line of parents, bit for bit, and attention equals 64-bit attention over it."""
    g = torch.Generator().manual_seed(beams)
    steps, layers = 21, 2
    cache = BeamKVCache(layers, hkv, d, max(prompts) + steps + 1, P, DEV, dtype, prompts, beams,
                        generator=torch.Generator().manual_seed(1))
    cache.pools.fill_(float("nan"))
    rope = RopeTable(max(prompts) + steps + 1, d, 500000.0, DEV, dtype)
    G = len(prompts)

    def rand(*s):
        return torch.randn(*s, generator=g).to(dtype).to(DEV)

    hist = [[[None, None] for _ in range(G * beams)] for _ in range(layers)]
    # prompts of different lengths, one after the other through a one-row cache of the pages
    lead = cache.leaders()
    for li in range(layers):
        lc = lead.get_layer(li)
        for gi, n in enumerate(prompts):
            k, v = rand(1, hkv, n, d), rand(1, hkv, n, d)
            table = lc.block_table[gi:gi + 1].contiguous()
            from llm_cuda_b200.kernels.rope import rope_append

            rope_append(None, k, v, lc.key_pages, lc.value_pages, table,
                        torch.zeros(1, dtype=torch.int32, device=DEV), lc.status)
            for b in range(gi * beams, (gi + 1) * beams):
                hist[li][b] = [k[0], v[0]]
    cache.fork()
    u = torch.finfo(dtype).eps / 2
    for step in range(steps):
        for li in range(layers):
            lc = cache.get_layer(li)
            q, k, v = rand(G * beams, hq, 1, d), rand(G * beams, hkv, 1, d), rand(G * beams, hkv, 1, d)
            q_rot = torch.empty_like(q)
            out = lc.rope_append_decode(q, k, v, rope, q_out=q_rot)
            for b in range(G * beams):
                pos = hist[li][b][0].shape[1]
                page = int(lc.block_table[b, pos // P])
                k_rot = lc.key_pages[page, :, pos % P]          # rotated by the append
                hist[li][b] = [torch.cat([hist[li][b][0], k_rot[:, None]], 1),
                               torch.cat([hist[li][b][1], v[b]], 1)]
                assert torch.equal(lc.value_pages[page, :, pos % P], v[b, :, 0])
                if step % 5 == 0 or step == steps - 1:
                    o, A = attend(q_rot[b, :, 0], *hist[li][b])
                    # output and weights rounded to the type, scores and sums in fp32
                    tol = u * o.abs() + (u + 1e-4) * A if u > 2.0 ** -20 else 1e-4 * A
                    assert ((out[b, :, 0].double() - o).abs() <= tol).all()
        parents = torch.randint(0, beams, (G, beams), generator=g, dtype=torch.int32)
        cache.reorder(parents.to(DEV))
        for li in range(layers):
            old = list(hist[li])
            for gi in range(G):
                for i in range(beams):
                    hist[li][gi * beams + i] = old[gi * beams + int(parents[gi, i])]
    cache.check_status()
    for li in range(layers):
        lc = cache.get_layer(li)
        for b in range(G * beams):
            n = hist[li][b][0].shape[1]
            ids = lc.block_table[b, :-(-n // P)].long()
            for pages, want in ((lc.key_pages, hist[li][b][0]), (lc.value_pages, hist[li][b][1])):
                got = pages[ids].permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n]
                assert torch.equal(got, want)


def tiny(dtype, seed=3):
    cfg = DecodeConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                       num_attention_heads=4, num_key_value_heads=2, initializer_range=0.12)
    return Llama3DecodeModel.random_init(cfg, DEV, dtype, seed=seed, max_positions=128)


def plain_search(m, ids, beams, steps, eos):
    """Beam search that runs every hypothesis through the model from its first token."""
    G, S = ids.shape
    hyps = [[([], 0.0, False)] for _ in range(G)]
    for step in range(steps):
        for gi in range(G):
            cand = []
            full = torch.stack([torch.cat([ids[gi], torch.tensor(h, dtype=torch.long, device=DEV)])
                                for h, _, _ in hyps[gi]])
            lg = m.prefill(full, m.make_cache(len(full), full.shape[1])).double()
            lp = torch.log_softmax(lg, -1).cpu()
            for i, (h, s, done) in enumerate(hyps[gi]):
                if done:
                    cand.append((s, -i, -eos, h + [eos], True))
                    continue
                top = torch.topk(lp[i], beams)
                cand += [(s + float(v), -i, -int(t), h + [int(t)], int(t) == eos)
                         for v, t in zip(top.values, top.indices)]
            cand.sort(reverse=True)
            hyps[gi] = [(h, s, d) for s, _, _, h, d in cand[:beams]]
    return hyps


@pytest.mark.parametrize("eos_rank", [None, 1])
def test_beam_search_equals_plain_search(eos_rank):
    """fp32: the same hypotheses as a search that recomputes everything.  Scores: each of the
    steps' logits is within 1e-4 of the other computation (fp32 sums of 256 terms through two
    layers), and a log-probability moves by at most twice that."""
    m = tiny(torch.float32)
    ids = torch.randint(0, 512, (3, 19), generator=torch.Generator().manual_seed(1)).to(DEV)
    steps, beams = 7, 4
    eos = None
    if eos_rank is not None:     # a token that some beams reach: the second best first token
        lg = m.prefill(ids, m.make_cache(3, 19))
        eos = int(torch.topk(lg[0], 2).indices[eos_rank])
    toks, scores = m.beam_search(ids, beams, steps, eos_token_id=eos, shuffle_seed=4)
    want = plain_search(m, ids, beams, steps, -1 if eos is None else eos)
    for gi in range(3):
        assert toks[gi].tolist() == [h for h, _, _ in want[gi]]
        ref = torch.tensor([s for _, s, _ in want[gi]])
        assert (scores[gi].cpu() - ref).abs().max() <= steps * 2e-4
    if eos is not None:          # a finished beam repeats the token
        assert any(eos in h[:-1] for h in toks.view(-1, steps).tolist())
        for h in toks.view(-1, steps).tolist():
            if eos in h:
                assert set(h[h.index(eos):]) == {eos}


def test_beam_search_of_one_beam_starts_greedily():
    m = tiny(torch.bfloat16, seed=5)
    ids = torch.randint(0, 512, (2, 30), generator=torch.Generator().manual_seed(2)).to(DEV)
    toks, scores = m.beam_search(ids, 1, 6)
    first = m.prefill(ids, m.make_cache(2, 30)).argmax(-1)
    assert torch.equal(toks[:, 0, 0], first)
    assert torch.isfinite(scores).all() and (scores < 0).all()


def test_beam_step_in_a_graph():
    """Decode step, selection and reordering captured once and replayed: as eager steps."""
    m = tiny(torch.bfloat16, seed=7)
    ids = torch.randint(0, 512, (2, 21), generator=torch.Generator().manual_seed(3)).to(DEV)
    beams, steps = 4, 5

    def start():
        cache = m.make_beam_cache([21, 21], beams, 64, shuffle_seed=6)
        logits = m.prefill(ids, cache.leaders())
        cache.fork()
        sc, _, tok = beam_select(logits, torch.zeros(2, 1, device=DEV), num_out=beams)
        return cache, sc, tok.view(-1)

    def step(cache, sc, tok):
        lg = m.decode_step(tok, cache)
        s, par, t = beam_select(lg, sc, num_out=beams)
        cache.reorder(par)
        sc.copy_(s)
        tok.copy_(t.view(-1))

    cache, sc, tok = start()
    eager = []
    for _ in range(steps):
        step(cache, sc, tok)
        eager.append((sc.clone(), tok.clone()))
    cache.check_status()

    cache, sc, tok = start()
    keep = (sc.clone(), tok.clone(), [c.seq_lens.clone() for c in cache.layer_caches],
            cache.block_table.clone(), cache.pools.clone())
    host = [list(c.host_lengths) for c in cache.layer_caches]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(cache, sc, tok)                       # warm-up
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step(cache, sc, tok)
    torch.cuda.synchronize()
    sc.copy_(keep[0])
    tok.copy_(keep[1])
    for c, x, h in zip(cache.layer_caches, keep[2], host):
        c.seq_lens.copy_(x)
        c.host_lengths = h
    cache.block_table.copy_(keep[3])
    cache.pools.copy_(keep[4])
    for want in eager:
        graph.replay()
        for c in cache.layer_caches:
            c.advance_host_lengths(1)
        torch.cuda.synchronize()
        assert torch.equal(sc, want[0]) and torch.equal(tok, want[1])
    cache.check_status()


def test_refused_step_leaves_the_cache_as_it_was():
    m = tiny(torch.bfloat16, seed=8)
    ids = torch.randint(0, 512, (1, 21), generator=torch.Generator().manual_seed(4)).to(DEV)
    cache = m.make_beam_cache([21], 2, 40)
    tok = m.prefill(ids, cache.leaders()).topk(2).indices.view(-1)
    cache.fork()
    before = cache.pools.clone()
    with pytest.raises(ValueError, match="partition_tokens"):
        m.decode_step(tok, cache, partition_tokens=256)
    lc = cache.get_layer(0)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="out must"):
        lc.rope_append_decode(q, q[:, :2], q[:, :2], m.rope, out=q[..., :32])
    for lc in cache.layer_caches:
        assert lc.seq_lens.tolist() == [21, 21] and lc.host_lengths == [21, 21]
    assert torch.equal(cache.pools.nan_to_num(), before.nan_to_num())


def test_graphed_step_over_shared_prefixes():
    """A captured step of a beam layer: the results of eager steps, bit for bit (the kernel that
    reads the prompt once per prompt rounds otherwise than the one that reads it per beam)."""
    from llm_cuda_b200.models.llama3.kv_cache import GraphedDecodeStep

    def make():
        c = BeamKVCache(1, 2, 64, 400, 16, DEV, torch.bfloat16, [300, 130], 3,
                        generator=torch.Generator().manual_seed(5))
        c.pools.copy_(torch.randn(c.pools.shape, generator=torch.Generator().manual_seed(6)))
        c.fork()
        return c

    g = torch.Generator().manual_seed(7)
    rope = RopeTable(400, 64, 500000.0, DEV, torch.bfloat16)
    eager, graphed = make(), make()
    q, k, v = (torch.zeros(6, h, 1, 64, dtype=torch.bfloat16, device=DEV) for h in (8, 2, 2))
    with pytest.raises(ValueError, match="partition_tokens"):
        GraphedDecodeStep(graphed.get_layer(0), rope, q, k, v, partition_tokens=128)
    step = GraphedDecodeStep(graphed.get_layer(0), rope, q, k, v)
    for _ in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        want = eager.get_layer(0).rope_append_decode(q, k, v, rope)
        got = step.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want[:, :, 0])
    assert graphed.get_layer(0).host_lengths == eager.get_layer(0).host_lengths == [304] * 3 + [134] * 3
    assert torch.equal(graphed.pools, eager.pools)
    graphed.check_status()
