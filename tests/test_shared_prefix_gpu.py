"""Shared-prefix decode attention against a 64-bit implementation.

The bound on an output element, with A = sum_t p_t |v_t| and u = eps / 2 of the tensor type:
  * the output is rounded once: u |o|;
  * 16-bit weights p_t may be rounded to the tensor type for the tensor cores: u A;
  * a score is a sum of d products in fp32 (d + 4 roundings of at most 2^-24 of the terms'
    magnitudes, the scaling and the exponent's argument among them): a relative error of
    each weight of e = (d + 4) 2^-24 max_t sum_i |q_i k_ti| scale, twice (numerator and
    normaliser): 2 e A; the exponential itself is good to 2^-21: 2 * 2^-21 A;
  * the weighted sums over n tokens add n 2^-24 A (numerator) and n 2^-24 A (normaliser), the
    join of the parts 16 * 2^-24 A.
"""

import math

import pytest
import torch

import llm_cuda_b200._native as N
from llm_cuda_b200.kernels.decode_attention import paged_decode
from llm_cuda_b200.kernels.shared_prefix import shared_prefix_decode

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


class Batch:
    """A paged batch with groups; every slot that no sequence holds is NaN, every table
    entry that no sequence uses is -1."""

    def __init__(self, sizes, shared, lens, hq, hkv, d, P, dtype, seed=0, extra_pages=3,
                 max_pages=None):
        g = torch.Generator().manual_seed(seed)
        self.sizes, self.shared, self.lens = sizes, shared, lens
        B = sum(sizes)
        starts = [0]
        for n in sizes:
            starts.append(starts[-1] + n)
        need = -(-max(max(lens), 1) // P)
        self.max_pages = max_pages or need + 1
        rows, nxt = [], 0
        group_of = [i for i, n in enumerate(sizes) for _ in range(n)]
        common = []
        for gi, n in enumerate(sizes):
            mine = [lens[b] for b in range(starts[gi], starts[gi + 1])]
            full = min(shared[gi], max(mine, default=0)) // P
            common.append(list(range(nxt, nxt + full)))
            nxt += full
        for b in range(B):
            n = -(-lens[b] // P)
            c = common[group_of[b]][:n]
            rows.append(c + list(range(nxt, nxt + n - len(c))))
            nxt += n - len(c)
        pages = nxt + extra_pages
        order = torch.randperm(pages, generator=g).tolist()
        bt = torch.full((B, self.max_pages), -1, dtype=torch.int32)
        for b, r in enumerate(rows):
            bt[b, :len(r)] = torch.tensor([order[x] for x in r], dtype=torch.int32)
        self.kp = torch.full((pages, hkv, P, d), float("nan"), dtype=dtype)
        self.vp = torch.full((pages, hkv, P, d), float("nan"), dtype=dtype)
        self.k, self.v = [], []
        for gi, n in enumerate(sizes):
            top = max([lens[b] for b in range(starts[gi], starts[gi + 1])], default=0)
            kc = torch.randn(hkv, min(shared[gi], top), d, generator=g).to(dtype)
            vc = torch.randn(hkv, min(shared[gi], top), d, generator=g).to(dtype)
            for b in range(starts[gi], starts[gi + 1]):
                L = lens[b]
                own = max(0, L - shared[gi])
                k = torch.cat([kc[:, :L], torch.randn(hkv, own, d, generator=g).to(dtype)], 1)
                v = torch.cat([vc[:, :L], torch.randn(hkv, own, d, generator=g).to(dtype)], 1)
                self.k.append(k)
                self.v.append(v)
                for i in range(0, L, P):
                    page = int(bt[b, i // P])
                    m = min(P, L - i)
                    self.kp[page, :, :m] = k[:, i:i + m]
                    self.vp[page, :, :m] = v[:, i:i + m]
        self.q = torch.randn(B, hq, d, generator=g).to(dtype)
        self.bt = bt.to(DEV)
        self.kp, self.vp, self.q = self.kp.to(DEV), self.vp.to(DEV), self.q.to(DEV)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.starts = torch.tensor(starts, dtype=torch.int32, device=DEV)
        self.shared_lens = torch.tensor(shared, dtype=torch.int32, device=DEV)
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def run(self, **kw):
        out = shared_prefix_decode(self.q, self.kp, self.vp, self.bt, self.seq_lens, self.starts,
                                   self.shared_lens, status=self.status, **kw)
        torch.cuda.synchronize()
        return out

    def check(self, out, scale=None):
        B, hq, d = self.q.shape
        hkv = self.kp.shape[1]
        r = hq // hkv
        u = torch.finfo(self.q.dtype).eps / 2
        scale = d ** -0.5 if scale is None else scale
        got = out.view(B, hq, d).double().cpu()
        assert torch.isfinite(got).all()
        for b in range(B):
            n = self.k[b].shape[1]
            if n == 0:
                assert not got[b].any()
                continue
            q = self.q[b].double().cpu()
            k = self.k[b].double().repeat_interleave(r, 0)
            v = self.v[b].double().repeat_interleave(r, 0)
            p = torch.softmax(torch.einsum("hd,htd->ht", q, k) * scale, -1)
            o = torch.einsum("ht,htd->hd", p, v)
            A = torch.einsum("ht,htd->hd", p, v.abs())
            mag = torch.einsum("hd,htd->ht", q.abs(), k.abs()).amax(-1, keepdim=True) * abs(scale)
            e = (d + 4) * 2.0 ** -24 * mag
            rel = (u if u > 2.0 ** -20 else 0.0) + 2 * e + 2 * 2.0 ** -21 \
                + (2 * n + 16) * 2.0 ** -24
            tol = u * o.abs() + rel * A + 1e-30
            bad = (got[b] - o).abs() > tol
            assert not bad.any(), (b, n, float(((got[b] - o).abs() / tol).max()))
        assert int(self.status.item()) == 0


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32

CASES = {
    # name: sizes, shared, lens, hq, hkv, d, P, dtype
    "beams": ([4, 4], [300, 40], [301, 310, 333, 305, 41, 44, 60, 57], 32, 8, 128, 16, BF),
    "one_token": ([2], [1], [1, 2], 8, 8, 64, 16, HF),
    "no_shared": ([3], [0], [5, 130, 16], 8, 2, 128, 16, BF),
    "all_shared": ([3], [257], [257, 257, 257], 32, 8, 128, 16, BF),
    "odd_everything": ([5, 1, 3], [129, 77, 0],
                       [129, 130, 200, 161, 400, 77, 1, 15, 64], 24, 2, 128, 128, BF),
    "empty_rows": ([4, 2], [100, 50], [120, 0, 101, 0, 0, 51], 16, 4, 64, 32, HF),
    "empty_group": ([2, 3], [90, 64], [0, 0, 65, 70, 64], 16, 4, 64, 16, BF),
    "shorter_than_shared": ([4], [500], [510, 40, 600, 501], 32, 8, 128, 16, BF),
    "many_rows": ([70], [520], [520 + (7 * i) % 150 for i in range(70)], 32, 8, 128, 16, BF),
    "three_row_tiles": ([150], [260], [260 + i % 9 for i in range(150)], 16, 4, 64, 16, BF),
    "wide_group_mha": ([33], [640], [641 + i for i in range(33)], 4, 4, 64, 64, HF),
    "big_ratio": ([9], [384], [400 + 3 * i for i in range(9)], 64, 1, 128, 16, BF),
    "fp32": ([3, 2], [200, 64], [210, 201, 280, 64, 99], 8, 2, 64, 64, FP),
    "fp32_d128": ([6], [1000], [1001, 1040, 1000, 1200, 1003, 0], 12, 4, 128, 16, FP),
    "d256": ([3], [150], [151, 160, 222], 8, 2, 256, 16, BF),
    "d80_p12": ([3], [150], [151, 160, 222], 6, 2, 80, 12, HF),
    "d33": ([2], [40], [44, 90], 3, 3, 33, 7, FP),
    "page_8": ([4], [400], [401, 402, 450, 480], 32, 8, 128, 8, BF),
    "page_256": ([4], [400], [401, 402, 450, 600], 32, 8, 64, 256, HF),
}


@pytest.mark.parametrize("force_generic", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_matches_64_bit(name, force_generic):
    b = Batch(*CASES[name], seed=len(name))
    b.check(b.run(force_generic=force_generic))


@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 63, 64, 127, 128, 129, 255, 256, 257, 1025])
def test_shared_lengths_around_tiles(L):
    b = Batch([3, 2], [L, L], [L, L + 1, L + 17, L + 128, L], 16, 4, 128, 16, BF, seed=L)
    b.check(b.run())


def test_long_prefix_over_many_blocks():
    """One prefix over all SMs, two row tiles, many partials per row."""
    b = Batch([40], [20000], [20000 + 5 * i for i in range(40)], 16, 2, 128, 64, BF, seed=5)
    b.check(b.run())


def test_more_groups_than_blocks():
    sizes = [1 + i % 3 for i in range(200)]
    shared = [(37 * i) % 300 for i in range(200)]
    lens = [shared[g] + (11 * g + j) % 40 for g, n in enumerate(sizes) for j in range(n)]
    b = Batch(sizes, shared, lens, 8, 2, 64, 16, BF, seed=9)
    b.check(b.run(max_group=3))


def test_sequences_outside_groups_and_beyond_max_group():
    b = Batch([6], [100], [101, 140, 100, 133, 180, 120], 16, 4, 128, 16, BF, seed=3)
    b.check(b.run(max_group=2))                    # four of the six read for themselves
    b.starts = torch.tensor([1, 4], dtype=torch.int32, device=DEV)
    b.check(b.run())                               # sequences 0, 4 and 5 are in no group
    b.starts = torch.zeros(1, dtype=torch.int32, device=DEV)
    b.shared_lens = torch.zeros(0, dtype=torch.int32, device=DEV)
    b.check(b.run())                               # no groups at all


def test_scale_strides_and_out():
    b = Batch([4], [200], [201, 220, 260, 300], 16, 4, 128, 16, BF, seed=4)
    wide = torch.full((4, 20, 128), float("nan"), dtype=BF, device=DEV)
    wide[:, 2:18] = b.q
    q = wide[:, 2:18]
    out = torch.empty(4, 16, 1, 128, dtype=BF, device=DEV)
    r = shared_prefix_decode(q.unsqueeze(2), b.kp, b.vp, b.bt, b.seq_lens, b.starts,
                             b.shared_lens, scale=0.3, out=out, status=b.status)
    torch.cuda.synchronize()
    assert r.data_ptr() == out.data_ptr() and r.shape == (4, 16, 1, 128)
    b.check(r, scale=0.3)


def test_equals_unshared_decode():
    b = Batch([8], [700], [700 + 9 * i for i in range(8)], 32, 8, 128, 16, BF, seed=6)
    bt = b.bt.clamp(min=0)
    kp, vp = torch.nan_to_num(b.kp), torch.nan_to_num(b.vp)
    ref = paged_decode(b.q, kp, vp, bt, b.seq_lens, status=b.status)
    torch.testing.assert_close(b.run().float(), ref.float(), rtol=0, atol=2e-2)


def test_infinite_and_large_scores():
    """Scores far apart (one key dominates) and of large magnitude stay finite."""
    b = Batch([4], [130], [131, 140, 150, 160], 8, 2, 128, 16, BF, seed=7)
    b.q *= 30
    b.check(b.run())


def test_nan_stays_in_its_sequence():
    """A NaN key in one sequence's own part reaches that sequence alone."""
    b = Batch([3], [64], [80, 80, 80], 8, 2, 128, 16, BF, seed=8)
    page = int(b.bt[1, 4])
    b.kp[page, :, 3] = float("nan")
    out = b.run()
    assert torch.isnan(out[1]).all()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()
    b.vp[int(b.bt[0, 1]), :, 0] = float("inf")     # shared: reaches all three
    out = b.run()
    assert not torch.isfinite(out).all(-1).any()


def test_captured_graph_follows_lengths_and_two_graphs_overlap():
    """Lengths are read on the device; two graphs with workspaces of their own may run on two
    streams at once."""
    def make(seed):
        b = Batch([5], [300], [310, 330, 300, 420, 301], 32, 8, 128, 16, BF, seed=seed)
        b.run()
        b.out = torch.empty_like(b.q)
        b.stream = torch.cuda.Stream()
        b.graph = torch.cuda.CUDAGraph()
        b.stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(b.graph, stream=b.stream):
            shared_prefix_decode(b.q, b.kp, b.vp, b.bt, b.seq_lens, b.starts, b.shared_lens,
                                 out=b.out, status=b.status)
        return b

    one, two = make(1), make(2)
    for _ in range(3):
        one.out.zero_()
        two.out.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(one.stream):
                one.graph.replay()
            with torch.cuda.stream(two.stream):
                two.graph.replay()
        torch.cuda.synchronize()
        one.check(one.out)
        two.check(two.out)
        for b in (one, two):               # the same launches with other lengths
            lens = [max(1, x - 7) for x in b.lens]
            b.lens = lens
            b.k = [k[:, :n] for k, n in zip(b.k, lens)]
            b.v = [v[:, :n] for v, n in zip(b.v, lens)]
            b.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            b.shared_lens.copy_(torch.tensor([min(290, min(lens))], dtype=torch.int32))


@pytest.mark.parametrize("force_generic", [False, True])
def test_pages_behind_2_31_elements(force_generic):
    """The same pages at the end of a pool of more than 2^31 elements: the same bits."""
    b = Batch([3], [200], [210, 300, 251], 8, 2, 128, 64, BF, seed=13)
    want = b.run(force_generic=force_generic)
    n = b.kp.shape[0]
    first = 2 ** 31 // b.kp[0].numel() + 1
    for name in ("kp", "vp"):
        small = getattr(b, name)
        pool = torch.empty(first + n, *small.shape[1:], dtype=BF, device=DEV)
        pool[first:] = small
        setattr(b, name, pool)
    b.bt = torch.where(b.bt >= 0, b.bt + first, b.bt)
    assert torch.equal(b.run(force_generic=force_generic), want)


def test_same_inputs_same_bits():
    b = Batch([20, 3], [900, 90], [901 + i for i in range(20)] + [90, 91, 99], 32, 8, 128, 16, BF,
              seed=11)
    first = b.run()
    for _ in range(3):
        assert torch.equal(b.run(), first)


@pytest.mark.parametrize("force_generic", [False, True])
@pytest.mark.parametrize("starts", [[0, 3, 1, 4], [0, 2, 3, 9], [-1, 2, 3, 4], [3, 0, 4, 2]])
def test_bad_groups_share_nothing(starts, force_generic):
    """One range that is none: the status word, and every sequence reads its own context."""
    b = Batch([2, 1, 1], [64, 64, 64], [70, 80, 90, 65], 8, 2, 128, 16, BF, seed=12)
    b.starts.copy_(torch.tensor(starts, dtype=torch.int32))
    out = b.run(force_generic=force_generic)
    with pytest.raises(N.DeviceStatusError, match="groups"):
        N.raise_on_status(b.status)
    b.status.zero_()
    b.check(out)


def test_bad_inputs_set_the_status_word():
    b = Batch([2, 2], [64, 64], [70, 80, 90, 65], 8, 2, 128, 16, BF, seed=12)
    b.bt[0, 1] = b.kp.shape[0]                    # one past the pool
    b.run()
    with pytest.raises(N.DeviceStatusError, match="page"):
        N.raise_on_status(b.status)
    b = Batch([2, 2], [64, 64], [70, 80, 90, 65], 8, 2, 128, 16, BF, seed=12)
    b.starts.copy_(torch.tensor([0, 3, 2], dtype=torch.int32))
    b.run()
    with pytest.raises(N.DeviceStatusError, match="groups"):
        N.raise_on_status(b.status)
    b.starts.copy_(torch.tensor([0, 2, 5], dtype=torch.int32))
    b.run()
    with pytest.raises(N.DeviceStatusError, match="groups"):
        N.raise_on_status(b.status)
    b = Batch([2, 2], [64, 64], [70, 80, 90, 65], 8, 2, 128, 16, BF, seed=12)
    b.seq_lens[3] = b.max_pages * 16 + 1
    b.kp, b.vp = torch.nan_to_num(b.kp), torch.nan_to_num(b.vp)
    b.run()
    with pytest.raises(N.DeviceStatusError, match="length"):
        N.raise_on_status(b.status)


@pytest.mark.parametrize("n,L,hq,hkv,d,P,dtype", [
    (40, 40007, 16, 2, 128, 64, BF), (9, 70001, 64, 2, 64, 16, HF), (37, 131072, 8, 1, 128, 256, BF)])
def test_long_prefix_with_wide_row_tiles(n, L, hq, hkv, d, P, dtype):
    """Enough work that a row tile has 256 rows; the 64-bit side runs on the GPU, the bound
    is the one above."""
    g = torch.Generator(device=DEV).manual_seed(L)
    own = [i % 5 for i in range(n)]
    full, f = L // P, L % P
    pages = full + n * 2
    kp = torch.randn(pages, hkv, P, d, device=DEV, generator=g).to(dtype)
    vp = torch.randn(pages, hkv, P, d, device=DEV, generator=g).to(dtype)
    bt = torch.full((n, full + 2), -1, dtype=torch.int32, device=DEV)
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    bt[:, :full] = order[:full]
    bt[:, full:] = order[full:].view(n, 2)
    ids = bt[:, full].long()
    for pool in (kp, vp):
        pool[ids, :, :f] = pool[ids[:1], :, :f].expand(n, -1, -1, -1)
    q = torch.randn(n, hq, d, device=DEV, generator=g).to(dtype)
    lens = torch.tensor([L + x for x in own], dtype=torch.int32, device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = shared_prefix_decode(q, kp, vp, bt, lens, torch.tensor([0, n], dtype=torch.int32, device=DEV),
                               torch.tensor([L], dtype=torch.int32, device=DEV), status=st).double()
    assert int(st.item()) == 0
    u = torch.finfo(dtype).eps / 2
    for b in range(0, n, 3):
        m = L + own[b]
        rows = bt[b, :-(-m // P)].long()
        for h in range(hkv):
            k = kp[rows, h].double().reshape(-1, d)[:m]
            v = vp[rows, h].double().reshape(-1, d)[:m]
            qs = q[b, h * (hq // hkv):(h + 1) * (hq // hkv)].double()
            p = torch.softmax(qs @ k.T * d ** -0.5, -1)
            o, A = p @ v, p @ v.abs()
            e = (d + 4) * 2.0 ** -24 * (qs.abs() @ k.abs().T).amax(-1, keepdim=True) * d ** -0.5
            tol = u * o.abs() + (u + 2 * e + 2 * 2.0 ** -21 + (2 * m + 16) * 2.0 ** -24) * A
            bad = (out[b, h * (hq // hkv):(h + 1) * (hq // hkv)] - o).abs() / tol
            assert float(bad.max()) <= 1.0


def test_many_units_per_block():
    """Every block works on several units in turn, each ending inside a chunk."""
    lens0 = [300 + (613 * i) % 1749 for i in range(16)]
    b = Batch([4] * 16, lens0, [x + 1 + (29 * i + j) % 128 for i, x in enumerate(lens0)
                                for j in range(4)], 32, 8, 128, 16, BF, seed=13)
    for _ in range(3):
        b.check(b.run(max_group=4))


def test_many_units_per_block_narrow_heads():
    lens0 = [200 + (413 * i) % 1333 for i in range(40)]
    b = Batch([3] * 40, lens0, [x + (29 * i + j) % 50 for i, x in enumerate(lens0)
                                for j in range(3)], 16, 4, 64, 32, HF, seed=14)
    for _ in range(3):
        b.check(b.run(max_group=3))


def test_batch_whose_tables_do_not_fit_shared_memory():
    sizes = [1 + i % 5 for i in range(1200)]
    shared = [(7 * i) % 40 for i in range(1200)]
    lens = [shared[g] + (3 * g + j) % 9 for g, n in enumerate(sizes) for j in range(n)]
    b = Batch(sizes, shared, lens, 2, 1, 128, 16, BF, seed=15)
    b.check(b.run(max_group=5))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("P", [8, 16, 32, 64, 128, 256, 384])
def test_every_page_size_of_the_tensor_cores(P, d, dtype):
    """Shared and own parts of several chunks with odd ends, narrow tiles and (the last group,
    of 70 x 2 rows per KV head) wide ones; pages of 8 tokens at head size 64 among them, whose V
    boxes lie closer together than those of two halves."""
    b = Batch([3, 2, 70], [300, 8, 133],
              [301, 463, 700, 9, 330] + [133 + (5 * i) % 37 for i in range(70)], 8, 4, d, P, dtype,
              seed=P + d)
    b.check(b.run())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("log2_weight", [-12.0, -20.5, -25.5, -28.0])
def test_small_weights_beside_a_large_one_fp16(log2_weight, own, d):
    """One token with (nearly) all of the weight and a value of 0, the others with so little that
    fp16 would drop them, and values of 1000.  Weights are 2^8 times their size against the
    greatest; where that is a subnormal of fp16 it is rounded by 2^-25, which is 2^-33 of the
    normaliser: n 2^-33 1000 beside the usual bound."""
    n = 250
    lens = [n + 1] * 3
    b = Batch([3], [0 if own else n], lens, 4, 2, d, 16, HF, seed=21)
    b.q.fill_(1.0)
    top = -log2_weight * math.log(2.0) * d ** 0.5 / d       # score 0 for the others
    for i in range(3):
        b.k[i].zero_()
        b.v[i].fill_(1000.0)
        b.k[i][:, 17] = top
        b.v[i][:, 17] = 0.0
        for t in range(n + 1):
            page = int(b.bt[i, t // 16])
            b.kp[page, :, t % 16] = b.k[i][:, t].to(DEV)
            b.vp[page, :, t % 16] = b.v[i][:, t].to(DEV)
    out = b.run()
    q = b.q[0, :2].double().cpu()
    p = torch.softmax(torch.einsum("hd,htd->ht", q, b.k[0].double()) * d ** -0.5, -1)
    o = torch.einsum("ht,htd->hd", p, b.v[0].double())
    # the usual bound (above), A = o here; fp16 results below 2^-14 are rounded by 2^-25
    e = (d + 4) * 2.0 ** -24 * float(b.k[0][0, 17].abs().sum()) * d ** -0.5
    rel = 2 * 2.0 ** -11 + 2 * e + 2 * 2.0 ** -21 + (2 * n + 18) * 2.0 ** -24
    tol = rel * o + n * 2.0 ** -33 * 1000 + 2.0 ** -25
    got = out.double().cpu().view(3, 2, 2, d)
    assert ((got - o[None, :, None]).abs() <= tol[None, :, None]).all(), \
        float(((got - o[None, :, None]).abs() / tol[None, :, None]).max())
    assert int(b.status.item()) == 0


@pytest.mark.parametrize("size", [30.0, 1000.0])
def test_large_scores_fp16(size):
    """Scores that differ by thousands: each row is (nearly) one value, and finite."""
    b = Batch([4], [700], [701, 740, 950, 1160], 8, 2, 128, 16, HF, seed=17)
    b.q *= size
    b.check(b.run())
