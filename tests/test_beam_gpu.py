"""Beam selection and cache reordering against plain 64-bit implementations."""

import math

import pytest
import torch

import llm_cuda_b200._native as N
from llm_cuda_b200.kernels.beam import beam_reorder, beam_select
from llm_cuda_b200.kernels.step_ops import argmax_rows

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
NEG = float("-inf")


def plain_select(logits, beam_scores, n, finished=None, eos=None):
    """Scores of every (beam, token) in 64 bits, sorted with ties to the lowest index."""
    G, K = beam_scores.shape
    x = logits.double().reshape(G, K, -1).cpu()
    V = x.shape[-1]
    b = beam_scores.double().cpu()[..., None]
    lse = torch.logsumexp(x, -1, keepdim=True)
    sc = torch.where(torch.isfinite(lse) & torch.isfinite(b), b + (x - lse), torch.tensor(NEG).double())
    if finished is not None:
        done = torch.full_like(x, NEG)
        done[..., eos] = torch.where(torch.isfinite(b[..., 0]), b[..., 0], torch.tensor(NEG).double())
        sc = torch.where(finished.cpu().bool()[..., None], done, sc)
    v, i = torch.sort(sc.reshape(G, K * V), dim=-1, descending=True, stable=True)
    return v[:, :n], (i // V)[:, :n].int(), (i % V)[:, :n]


def check_select(logits, beam_scores, n, finished=None, eos=None):
    s, b, t = beam_select(logits, beam_scores, num_out=n, finished=finished, eos_token_id=eos)
    torch.cuda.synchronize()
    rs, rb, rt = plain_select(logits, beam_scores, n, finished, eos)
    assert torch.equal(b.cpu(), rb) and torch.equal(t.cpu(), rt)
    # A score is rounded once to fp32; its log-sum-exp comes from exponentials good to 2^-21
    # (argument and function) and sums of them in fp32, at most 2^-20 off in all.
    fin = torch.isfinite(rs)
    assert torch.equal(torch.isfinite(s.cpu()), fin)
    tol = rs.abs() * 2.0 ** -24 + 2.0 ** -20
    assert ((s.cpu().double() - rs).abs()[fin] <= tol[fin]).all()
    assert (s.cpu()[~fin] == NEG).all()


def rand(G, K, V, dtype, seed, scale=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(G * K, V, generator=g, device=DEV) * scale).to(dtype)
    return x, torch.randn(G, K, generator=g, device=DEV) * 2 - 12


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("G,K,V,n", [
    (1, 1, 1, 1), (1, 4, 128256, 8), (3, 5, 50257, 10), (20, 4, 1003, 4), (2, 1, 7, 5),
    (1, 32, 4099, 64), (17, 8, 33, 16), (1, 3, 2, 6), (2, 16, 513, 33), (40, 2, 300, 64),
    (1, 17, 9000, 34), (5, 12, 64, 1)])
def test_select_matches_64_bit(G, K, V, n, dtype):
    x, s = rand(G, K, V, dtype, G * 1000 + K * 10 + n)
    check_select(x, s, n)


def test_select_ties_go_to_the_lowest_beam_and_token():
    """Equal logits everywhere, equal beams: the first tokens of the first beam."""
    x = torch.zeros(4, 2000, dtype=torch.bfloat16, device=DEV)
    s = torch.full((1, 4), -1.0, device=DEV)
    check_select(x, s, 64)
    x, s = rand(2, 4, 5000, torch.bfloat16, 1, scale=0.01)   # few distinct values, many ties
    x[4:] = x[:4]
    s[:] = -3.0
    check_select(x, s, 64)
    x[1] = x[0]                                              # two equal rows
    check_select(x, s, 33)


def test_select_zeros_of_both_signs_are_equal():
    x = torch.zeros(3, 1500, device=DEV)
    x[:, ::2] = -0.0
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        check_select(x.to(dtype), torch.tensor([[-2.0, -1.0, -2.0]], device=DEV), 20)


@pytest.mark.parametrize("n", [8, 64])
def test_select_logits_closer_than_scores(n):
    """Logits of 1e-22 and less: all scores round to -log(V), the order stays the logits'."""
    g = torch.Generator(device=DEV).manual_seed(n)
    row = torch.randperm(5000, generator=g, device=DEV).float() * 1e-26
    x = row.repeat(8, 1)
    s, b, t = beam_select(x, torch.zeros(1, 8, device=DEV), num_out=n)
    assert (b == 0).all()
    assert torch.equal(t[0], torch.argsort(row, descending=True)[:n])
    assert ((s + math.log(5000)).abs() <= 2.0 ** -19).all()   # 2^-20 and fp32 of 8.5


def test_select_sorted_rows():
    """Ascending logits make every tile better than all before it; descending ones none."""
    base = torch.arange(30000, device=DEV, dtype=torch.float32) / 1000
    x = torch.stack([base, base.flip(0), base, base.flip(0)])
    check_select(x, torch.tensor([[-1.0, -1.5, -2.0, -2.5]], device=DEV), 64)


def test_select_masked_and_infinite_logits():
    x, s = rand(3, 4, 4000, torch.float32, 2)
    x[torch.rand(12, 4000, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)) < 0.9] = NEG
    x[5] = NEG                            # a row with nothing left
    x[6, 17] = float("nan")               # a row with a NaN
    x[7, 100] = float("inf")
    x[8, 10:] = NEG                       # fewer tokens than candidates
    check_select(x, s, 16)
    check_select(x, s, 64)
    s[0, 1] = NEG                         # beams that are out
    s[0, 2] = float("nan")
    s[2, :] = NEG                         # a prompt with no beam at all
    check_select(x, s, 32)
    x[:] = NEG
    check_select(x, s, 8)


def test_select_lowest_values_as_mask():
    x, s = rand(2, 3, 3000, torch.float16, 4)
    x[:, 5:2990] = torch.finfo(torch.float16).min
    check_select(x, s, 24)


def log_softmax_select(logits, beam_scores, n):
    """As ``plain_select``, with the log-softmax formed from differences to the maximum, which
    64 bits hold even where the logits are too large for sums with them."""
    G, K = beam_scores.shape
    x = logits.double().reshape(G, K, -1).cpu()
    V = x.shape[-1]
    sc = beam_scores.double().cpu()[..., None] + torch.log_softmax(x, -1)
    v, i = torch.sort(sc.reshape(G, K * V), dim=-1, descending=True, stable=True)
    return v[:, :n], (i // V)[:, :n].int(), (i % V)[:, :n]


def check_large(x, s, n):
    got = beam_select(x, s, num_out=n)
    rs, rb, rt = log_softmax_select(x, s, n)
    assert torch.equal(got[1].cpu(), rb) and torch.equal(got[2].cpu(), rt)
    err = (got[0].cpu().double() - rs).abs()
    assert (err <= rs.abs() * 2.0 ** -24 + 2.0 ** -20).all()      # as in check_select


MASKS = [(dt, m) for dt in (torch.float32, torch.bfloat16, torch.float16)
         for m in ("min", -5e9, -1e10, -1e20, -1e30, -1e37) if m == "min" or dt != torch.float16]


@pytest.mark.parametrize("dtype,mask", MASKS)
def test_select_large_negative_masks(dtype, mask):
    """Finite masks of any size, over most of a row, over whole tiles, threads and splits of
    it and over all of it."""
    mask = torch.finfo(dtype).min if mask == "min" else mask
    x, s = rand(3, 4, 20011, dtype, 31)
    gone = torch.rand(4, 20011, device=DEV, generator=torch.Generator(device=DEV).manual_seed(32))
    x[:4].masked_fill_(gone < 0.99, mask)
    x[4, :15000] = mask                  # the first tiles of most threads
    x[5, 5000:] = mask
    x[6] = mask                          # all of a row: uniform
    x[7, :20010] = mask                  # one token left
    x[8:, 3:20000] = mask
    for n in (1, 8, 64):
        check_large(x, s, n)


@pytest.mark.parametrize("dtype,size", [(torch.float32, 1e38), (torch.bfloat16, 1e38),
                                        (torch.float32, 1e9), (torch.float16, 2e4)])
def test_select_logits_of_any_size(dtype, size):
    x, s = rand(2, 4, 5001, torch.float32, 33, scale=1.0)
    x = (x.clamp(-3.2, 3.2) * size).to(dtype)
    check_large(x, s, 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,pad", [(50257, 0), (4099, 0), (1001, 2), (20000, 3), (128255, 0)])
def test_select_equal_rows_tie_at_any_alignment(V, pad, dtype):
    """Rows of equal logits have equal scores wherever they begin: the lowest beam comes first."""
    for seed, K, n in ((1, 8, 64), (2, 5, 10), (3, 16, 33), (4, 32, 64)):
        x, s = rand(2, 1, V, dtype, 40 + seed)
        wide = torch.zeros(2 * K, V + pad, dtype=dtype, device=DEV)
        wide[:, :V] = x.repeat_interleave(K, 0)
        check_select(wide[:, :V], s.expand(2, K).contiguous(), n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_select_rows_at_every_offset(dtype):
    """Rows that begin anywhere between two 16-byte boundaries, of lengths around the vectors
    and tiles, with few distinct values (ties, cells and lists of many equal logits) and many;
    what lies around a row is NaN."""
    per = 16 // torch.empty(0, dtype=dtype).element_size()
    for V in (1, 2, per - 1, per, per + 1, 3 * per + 1, 1024, 1025, 8191, 8192 + per - 1, 40003):
        for off in range(per):
            few = (off + V) % 3 == 0
            x, s = rand(1, 3, V, dtype, V + off, scale=0.01 if few else 3.0)
            if few:
                x = (x * 400).round() / 4
            wide = torch.full((3, V + per + 1), float("nan"), dtype=dtype, device=DEV)
            wide[:, off:off + V] = x
            check_select(wide[:, off:off + V], s, min(64, 3 * V))


def test_select_finished_beams():
    x, s = rand(6, 4, 1000, torch.bfloat16, 5)
    fin = torch.zeros(6, 4, dtype=torch.bool, device=DEV)
    fin[0, 1] = fin[1, :] = fin[2, 0] = fin[3, 3] = True
    s[0, 1] = -0.5                        # a finished beam that leads
    x[5] = float("nan")                   # logits of a finished beam are not read
    fin[1, 1] = True
    check_select(x, s, 8, fin, 999)
    check_select(x, s, 64, fin, 0)
    check_select(x, s, 5, fin, 500)


def test_select_first_step_and_strided_rows():
    """Before the first token all beams but one are at -1e9; rows of a wider buffer, at an
    offset that no vector load divides."""
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.full((12, 2053), float("nan"), dtype=dtype, device=DEV)
        x, s = rand(3, 4, 2001, dtype, 6)
        wide[:, 5:2006] = x
        s[:, 1:] = -1e9
        check_select(wide[:, 5:2006], s, 8)
        check_select(wide[:, 5:2006].view(3, 4, 2001), s, 4)
        check_select(x.t().contiguous().t(), s, 4)          # columns contiguous: copied


def test_select_one_beam_is_argmax():
    x, _ = rand(9, 1, 128256, torch.bfloat16, 7)
    _, b, t = beam_select(x, torch.zeros(9, 1, device=DEV))
    assert torch.equal(t[:, 0], argmax_rows(x)) and not b.any()


def test_select_in_a_graph_and_on_a_stream():
    x, s = rand(4, 4, 32000, torch.bfloat16, 8)
    beam_select(x, s, num_out=8)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = beam_select(x, s, num_out=8)
    for seed in (9, 10):
        x2, s2 = rand(4, 4, 32000, torch.bfloat16, seed)
        x.copy_(x2)
        s.copy_(s2)
        graph.replay()
        torch.cuda.synchronize()
        rs, rb, rt = plain_select(x, s, 8)
        assert torch.equal(out[1].cpu(), rb) and torch.equal(out[2].cpu(), rt)


# -- reordering --------------------------------------------------------------------
def make_cache(G, K, layers, hkv, d, P, prompt_pages, own_pages, lens, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    per = prompt_pages + K * own_pages
    pages = G * per + 2
    order = torch.randperm(pages, generator=g)
    own = torch.empty(G, K, prompt_pages + own_pages, dtype=torch.int32)
    for gi in range(G):
        own[gi, :, :prompt_pages] = order[gi * per:gi * per + prompt_pages].int()
        own[gi, :, prompt_pages:] = order[gi * per + prompt_pages:(gi + 1) * per].int().view(K, -1)
    own = own.view(G * K, -1)
    pools = torch.randn(layers, 2, pages, hkv, P, d, generator=g).to(dtype)
    # a table as earlier steps leave it: full pages behind the prompt from any beam
    bt = own.clone()
    for gi in range(G):
        full = lens[gi] // P
        for c in range(prompt_pages, min(full, bt.shape[1])):
            pick = torch.randint(0, K, (K,), generator=g)
            bt[gi * K:(gi + 1) * K, c] = own[gi * K + pick, c]
    seq = torch.tensor([x for x in lens for _ in range(K)], dtype=torch.int32)
    return [t.to(DEV) for t in (pools, own, bt, seq)]


def plain_reorder(pools, own, bt, seq, parents):
    pools, bt0, out_bt = pools.clone(), bt.clone(), bt.clone()
    src = pools.clone()
    G, K = parents.shape
    P = pools.shape[4]
    for gi in range(G):
        for i in range(K):
            b, p = gi * K + i, gi * K + int(parents[gi, i])
            L = int(seq[b])
            full, fill = L // P, L % P
            out_bt[b, :full] = bt0[p, :full]
            out_bt[b, full:] = own[b, full:]
            if fill:
                pools[:, :, int(own[b, full]), :, :fill] = src[:, :, int(own[p, full]), :, :fill]
    return pools, out_bt


@pytest.mark.parametrize("G,K,layers,hkv,d,P,pp,op,lens,dtype", [
    (1, 4, 3, 8, 128, 16, 2, 2, [45], torch.bfloat16),
    (3, 8, 2, 2, 64, 16, 0, 3, [0, 16, 47], torch.float16),       # nothing held, no partial page
    (2, 1, 1, 1, 64, 8, 1, 1, [9, 15], torch.float32),
    (2, 32, 1, 4, 128, 16, 1, 1, [17, 31], torch.bfloat16),
    (5, 5, 4, 3, 40, 6, 2, 2, [13, 12, 23, 24, 18], torch.float32),   # 24: the cache is full
    (1, 12, 2, 2, 33, 64, 0, 1, [1], torch.float16),              # rows that 16 bytes do not divide
    (1, 3, 1, 2, 64, 1, 2, 5, [4], torch.bfloat16)])              # pages of one token
def test_reorder_matches_plain(G, K, layers, hkv, d, P, pp, op, lens, dtype):
    pools, own, bt, seq = make_cache(G, K, layers, hkv, d, P, pp, op, lens, dtype, K)
    g = torch.Generator().manual_seed(G)
    for step in range(4):
        parents = torch.randint(0, K, (G, K), generator=g, dtype=torch.int32)
        if step == 0:
            parents[:] = torch.arange(K)                   # nobody moves
        if step == 1:
            parents = parents * 0 + (K - 1)                # all from the last
        if step == 2:
            parents[:] = torch.arange(K).roll(1)           # a cycle
        rp, rb = plain_reorder(pools.cpu(), own.cpu(), bt.cpu(), seq.cpu(), parents)
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        beam_reorder(pools, own, bt, seq, parents.to(DEV), status=st)
        torch.cuda.synchronize()
        assert int(st.item()) == 0
        assert torch.equal(pools.cpu(), rp) and torch.equal(bt.cpu(), rb)


def test_reorder_leaves_a_bad_prompt_alone():
    pools, own, bt, seq = make_cache(3, 4, 2, 2, 64, 16, 1, 2, [20, 37, 18], torch.bfloat16, 1)
    parents = torch.tensor([[1, 0, 3, 2], [0, 4, 1, 1], [3, 3, 3, 3]], dtype=torch.int32)
    ref = parents.clone()
    ref[1] = torch.arange(4)                               # prompt 1 has a bad parent
    rp, rb = plain_reorder(pools.cpu(), own.cpu(), bt.cpu(), seq.cpu(), ref)
    rb[4:8] = bt[4:8].cpu()
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    beam_reorder(pools, own, bt, seq, parents.to(DEV), status=st)
    torch.cuda.synchronize()
    assert torch.equal(pools.cpu(), rp) and torch.equal(bt.cpu(), rb)
    with pytest.raises(N.DeviceStatusError, match="parent"):
        N.raise_on_status(st)
    parents[1] = 0
    for spoil, word in ((lambda: seq.__setitem__(5, 38), "parent"),
                        (lambda: (seq.__setitem__(5, 37), own.__setitem__((6, 2), -1)), "page"),
                        (lambda: (own.__setitem__((6, 2), 0), seq[4:8].fill_(49)), "length")):
        spoil()
        before = pools.clone(), bt.clone()
        only = torch.arange(4, dtype=torch.int32).repeat(3, 1)
        only[1] = 0
        beam_reorder(pools, own, bt, seq, only.to(DEV), status=st)
        torch.cuda.synchronize()
        assert torch.equal(pools, before[0]) and torch.equal(bt[4:8], before[1][4:8])
        with pytest.raises(N.DeviceStatusError, match=word):
            N.raise_on_status(st)


def test_no_prompts():
    s, b, t = beam_select(torch.zeros(0, 100, device=DEV), torch.zeros(0, 4, device=DEV), num_out=8)
    assert s.shape == b.shape == t.shape == (0, 8)
    s, b, t = beam_select(torch.zeros(0, 4, 100, device=DEV, dtype=torch.bfloat16),
                          torch.zeros(0, 4, device=DEV),
                          finished=torch.zeros(0, 4, dtype=torch.bool, device=DEV), eos_token_id=1)
    assert s.shape == b.shape == t.shape == (0, 4)
