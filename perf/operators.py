"""Cases, plain forms and exact forms of the beam-search decode operators.

Three operators that one step of a beam search (or of a batch that shares a prompt) runs
between the projections of the decode model:

* ``prefix``: single-token decode attention over a paged cache whose sequences come in
  groups that share their first pages; the shared part of a group is read once.
* ``select``: log-softmax over the vocabulary, running beam scores added, the best ``n``
  continuations of every prompt over its beams and the whole vocabulary.
* ``reorder``: every beam continues from its parent: rows of the block table move, and the
  partly filled last page of each beam is copied, in every layer.

``own = False`` computes the plain form with elementary torch operations; ``own = True``
calls the framework.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------
def listed():
    return [
        # The first tokens of one user's beam search: 4 beams on a prompt of odd length.
        # All of it is latency.
        dict(name="prefix_beams_1x4", op="prefix", groups=1, group=4, ragged=False, prefix_lo=500,
             prefix_hi=500, suffix_lo=1, suffix_hi=24, empty=0, hq=32, hkv=8, d=128, page=16,
             dtype="bf16", lens=1),
        # A server's beam searches: 16 prompts of different lengths, 4 beams each.
        dict(name="prefix_beams_16x4", op="prefix", groups=16, group=4, ragged=False,
             prefix_lo=300, prefix_hi=2048, suffix_lo=1, suffix_hi=128, empty=0, hq=32, hkv=8,
             d=128, page=16, dtype="bf16", lens=2),
        # 64 requests behind one system prompt, each with its own dialogue behind it.
        dict(name="prefix_system_64", op="prefix", groups=1, group=64, ragged=False,
             prefix_lo=4096, prefix_hi=4096, suffix_lo=1, suffix_hi=1024, empty=0, hq=32, hkv=8,
             d=128, page=16, dtype="bf16", lens=3),
        # 8 questions about one long document: the key/value stream of the document.
        dict(name="prefix_document_8", op="prefix", groups=1, group=8, ragged=False,
             prefix_lo=131072, prefix_hi=131072, suffix_lo=1, suffix_hi=256, empty=0, hq=64,
             hkv=8, d=128, page=64, dtype="bf16", lens=4),
        # Many samples of one long prompt: enough rows to be bound by arithmetic.
        dict(name="prefix_samples_128", op="prefix", groups=1, group=128, ragged=False,
             prefix_lo=16384, prefix_hi=16384, suffix_lo=64, suffix_hi=512, empty=0, hq=64,
             hkv=8, d=128, page=16, dtype="bf16", lens=5),
        # A prefix cache's batch: groups of many sizes, prefixes of odd length, some absent,
        # some batch rows unused; half precision, narrow heads.
        dict(name="prefix_ragged_fp16", op="prefix", groups=7, group=37, ragged=True,
             prefix_lo=0, prefix_hi=1777, suffix_lo=0, suffix_hi=333, empty=5, hq=16, hkv=4,
             d=64, page=32, dtype="fp16", lens=6),
        # Single precision, as the smallest configuration runs it.
        dict(name="prefix_fp32", op="prefix", groups=3, group=5, ragged=False, prefix_lo=64,
             prefix_hi=1000, suffix_lo=1, suffix_hi=80, empty=0, hq=8, hkv=2, d=64, page=64,
             dtype="fp32", lens=7),
        # One user's step: 4 beams over the vocabulary, twice as many candidates kept.
        dict(name="select_1x4", op="select", groups=1, beams=4, n=8, vocab=128256, pad=0,
             finished=0.0, masked=0.0, first=False, dtype="bf16"),
        # A full batch: 64 prompts with 8 beams.
        dict(name="select_64x8", op="select", groups=64, beams=8, n=16, vocab=128256, pad=0,
             finished=0.0, masked=0.0, first=False, dtype="bf16"),
        # Odd sizes in single precision: some beams are done, some tokens forbidden, rows of a
        # wider buffer.
        dict(name="select_fp32_odd", op="select", groups=7, beams=5, n=10, vocab=50257, pad=47,
             finished=0.2, masked=0.05, first=False, dtype="fp32"),
        # The cache of one user's beams after a step, 32 layers.
        dict(name="reorder_1x4", op="reorder", groups=1, beams=4, layers=32, hkv=8, d=128, page=16,
             prompt_pages=32, own_pages=8, dtype="bf16", lens=11),
        # The cache of a full batch of beams.
        dict(name="reorder_64x8", op="reorder", groups=64, beams=8, layers=32, hkv=8, d=128,
             page=16, prompt_pages=2, own_pages=3, dtype="bf16", lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["prefix", "prefix", "select", "reorder"])
    if op == "prefix":
        hq, hkv, d, page = rng.choice([(32, 8, 128, 16), (64, 8, 128, 64), (64, 8, 128, 16),
                                       (16, 4, 64, 32), (8, 8, 64, 16), (24, 2, 128, 128)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 200_000_000 if dtype != "fp32" else 4_000_000   # rows x prefix tokens
        groups = _log(rng, 1, 24)
        group = _log(rng, 1, 128)
        while groups * group > 512:
            group = max(1, group // 2)
        hi = min(_log(rng, 64, 65536), max(64, most // (groups * group * hq)))
        suffix = _log(rng, 1, 700)
        while groups * group * suffix > 100_000:
            suffix = max(1, suffix // 2)
        return dict(op="prefix", groups=groups, group=group, ragged=rng.random() < 0.5,
                    prefix_lo=rng.randint(0, hi), prefix_hi=hi, suffix_lo=min(1, suffix),
                    suffix_hi=suffix, empty=rng.choice([0, 0, 1, 3]), hq=hq, hkv=hkv, d=d,
                    page=page, dtype=dtype, lens=rng.randrange(1 << 20))
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 10, 16, 24])
        vocab = _log(rng, 500, 128256)
        groups = _log(rng, 1, 64)
        while groups * beams * vocab > 64 * 8 * 128256:
            groups = max(1, groups // 2)
        return dict(op="select", groups=groups, beams=beams, n=rng.choice([beams, 2 * beams]),
                    vocab=vocab, pad=rng.choice([0, 0, 7, 64]),
                    finished=rng.choice([0.0, 0.0, 0.3]), masked=rng.choice([0.0, 0.0, 0.5]),
                    first=rng.random() < 0.2, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    beams = rng.choice([2, 3, 4, 5, 8, 12, 16])
    layers = rng.choice([1, 4, 16, 32])
    groups = _log(rng, 1, 64)
    while groups * beams * layers > 64 * 8 * 32:
        groups = max(1, groups // 2)
    hkv, d, page = rng.choice([(8, 128, 16), (2, 128, 16), (2, 64, 64), (4, 64, 32)])
    return dict(op="reorder", groups=groups, beams=beams, layers=layers, hkv=hkv, d=d, page=page,
                prompt_pages=rng.randint(0, 5), own_pages=rng.randint(1, 4),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), lens=rng.randrange(1 << 20))


# ---------------------------------------------------------------------------------
# What a case's numbers stand for
# ---------------------------------------------------------------------------------
def _prefix_shape(c):
    """(sequences of each group, shared tokens of each group, length of each sequence)."""
    r = random.Random(c["lens"])
    sizes = [r.randint(1, c["group"]) if c["ragged"] else c["group"] for _ in range(c["groups"])]
    if c["ragged"]:
        sizes[r.randrange(len(sizes))] = c["group"]
    shared = [r.randint(c["prefix_lo"], c["prefix_hi"]) for _ in sizes]
    if c["ragged"] and len(shared) > 1:
        shared[-1] = 0
    lens = [s + r.randint(c["suffix_lo"], c["suffix_hi"]) for s, n in zip(shared, sizes)
            for _ in range(n)]
    for _ in range(min(c["empty"], len(lens) - 1)):
        lens[r.randrange(len(lens))] = 0       # a row of the batch that no request uses
    return sizes, shared, lens


def _reorder_shape(c):
    """(tokens of each prompt's beams, parents within the prompt) of a reorder case."""
    r = random.Random(c["lens"])
    page, own_lo = c["page"], c["prompt_pages"] * c["page"]
    lens, parents = [], []
    for _ in range(c["groups"]):
        lens.append(own_lo + r.randint(1, c["own_pages"] * page - 1) if c["own_pages"] * page > 1
                    else own_lo)
        parents.append(sorted(r.choices(range(c["beams"]), weights=[2.0 / (1 + i) for i in
                                                                    range(c["beams"])],
                                        k=c["beams"])))
    return lens, parents


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["op"] == "prefix":
        sizes, shared, lens = _prefix_shape(case)
        P, d = case["page"], case["d"]
        starts = [0]
        for n in sizes:
            starts.append(starts[-1] + n)
        B = starts[-1]
        max_pages = max(1, max(-(-max(x, y) // P) for x, y in
                               zip(lens, [t for t, n in zip(shared, sizes) for _ in range(n)])))
        # logical tables first, then a random order of the pool
        rows, nxt = [], 0
        for gi, n in enumerate(sizes):
            common = list(range(nxt, nxt + shared[gi] // P))
            nxt += len(common)
            for b in range(starts[gi], starts[gi] + n):
                tail = -(-max(lens[b], shared[gi]) // P) - len(common)
                rows.append(common + list(range(nxt, nxt + tail)))
                nxt += tail
        pages = max(1, nxt)
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed)))
        bt = torch.zeros(B, max_pages, dtype=torch.int64)
        for b, r in enumerate(rows):
            bt[b, :len(r)] = torch.tensor(r, dtype=torch.int64)
        s["block_table"] = order[bt].to(torch.int32).to(dev)
        s["key_pages"] = torch.randn(pages, case["hkv"], P, d, device=dev, dtype=dt, generator=g)
        s["value_pages"] = torch.randn(pages, case["hkv"], P, d, device=dev, dtype=dt, generator=g)
        if any(t % P for t in shared):
            # A shared length inside a page: the rest of that page is each sequence's own, the
            # shared tokens in it are the same in all of them.
            for gi, n in enumerate(sizes):
                f = shared[gi] % P
                if f:
                    ids = s["block_table"][starts[gi]:starts[gi] + n, shared[gi] // P].long()
                    for pool in (s["key_pages"], s["value_pages"]):
                        pool[ids, :, :f] = pool[ids[:1], :, :f].expand(n, -1, -1, -1)
        s["q"] = torch.randn(B, case["hq"], d, device=dev, dtype=dt, generator=g)
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["group_starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        s["shared_lens"] = torch.tensor(shared, dtype=torch.int32, device=dev)
        s["max_group"] = max(sizes)
        s["max_shared"] = max(shared)
        s["max_own"] = max(0, max(x - t for x, t in
                                  zip(lens, [t for t, n in zip(shared, sizes) for _ in range(n)])))
    elif case["op"] == "select":
        G, K, V = case["groups"], case["beams"], case["vocab"]
        buf = torch.empty(G * K, V + case["pad"], device=dev, dtype=dt)
        buf.normal_(0.0, 3.0, generator=g)
        s["logits"] = buf[:, :V]
        if case["masked"]:
            s["logits"].masked_fill_(torch.rand(G * K, V, device=dev, generator=g)
                                     < case["masked"], float("-inf"))
        sc = torch.randn(G, K, device=dev, generator=g) * 2 - 12
        if case["first"]:
            sc[:, 1:] = -1e9               # before the first token all beams are the same
        s["beam_scores"] = sc
        s["finished"] = (torch.rand(G, K, device=dev, generator=g) < case["finished"]
                         if case["finished"] else None)
        s["eos"] = V // 3
    else:
        lens, parents = _reorder_shape(case)
        G, K, P = case["groups"], case["beams"], case["page"]
        mp = case["prompt_pages"] + case["own_pages"]
        per = case["prompt_pages"] + K * case["own_pages"]
        pages = G * per
        table = torch.empty(G, K, mp, dtype=torch.int64)
        for gi in range(G):
            table[gi, :, :case["prompt_pages"]] = gi * per + torch.arange(case["prompt_pages"])
            table[gi, :, case["prompt_pages"]:] = (
                gi * per + case["prompt_pages"]
                + torch.arange(K * case["own_pages"]).view(K, case["own_pages"]))
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed)))
        s["own_table"] = order[table.view(G * K, mp)].to(torch.int32).to(dev)
        s["block_table"] = s["own_table"].clone()
        s["pools"] = torch.empty(case["layers"], 2, pages, case["hkv"], P, case["d"], device=dev,
                                 dtype=dt).normal_(generator=g)
        s["seq_lens"] = torch.tensor([x for x in lens for _ in range(K)], dtype=torch.int32,
                                     device=dev)
        s["parents"] = torch.tensor(parents, dtype=torch.int32, device=dev)
    return s


# ---------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------
def _plain_prefix(s):
    """softmax(q k^T / sqrt(d)) v over each sequence's tokens; the keys and values of the
    shared tokens are gathered once for each group."""
    q, kp, vp, bt, lens = s["q"], s["key_pages"], s["value_pages"], s["block_table"], s["seq_lens"]
    B, hq, d = q.shape
    P, hkv = kp.shape[2], kp.shape[1]
    G, M, r = s["shared_lens"].shape[0], s["max_group"], hq // hkv
    dev = q.device
    starts = s["group_starts"].long()
    seq = torch.arange(B, device=dev)
    gid = torch.searchsorted(starts[1:].contiguous(), seq, right=True)
    at = seq - starts[gid]
    n = lens.long()
    own_from = torch.minimum(s["shared_lens"].long()[gid], n)
    qf = q.float().view(B, hkv, r, d) * (1.0 / math.sqrt(d))
    # tokens of the shared part, read through the table row of the group's first sequence
    tok = torch.arange(s["max_shared"], device=dev)
    ids = bt.long()[starts[:-1]][:, tok // P]                               # [G, Lp]
    kg = kp[ids, :, tok % P].float().permute(0, 2, 1, 3)                    # [G, hkv, Lp, d]
    qg = torch.zeros(G, M, hkv, r, d, device=dev)
    qg[gid, at] = qf
    qg = qg.permute(0, 2, 1, 3, 4).reshape(G, hkv, M * r, d)
    sg = (qg @ kg.transpose(2, 3)).view(G, hkv, M, r, -1)
    del kg
    sp = sg[gid, :, at]                                                     # [B, hkv, r, Lp]
    del sg
    sp.masked_fill_((tok >= own_from[:, None])[:, None, None], float("-inf"))
    # tokens of the sequence's own part
    pos = own_from[:, None] + torch.arange(s["max_own"], device=dev)        # [B, Ls]
    ok = pos < n[:, None]
    pid = bt.long().gather(1, (pos // P).clamp(max=bt.shape[1] - 1))
    ko = kp[pid, :, pos % P].float().permute(0, 2, 1, 3)
    so = qf @ ko.transpose(2, 3)
    so.masked_fill_(~ok[:, None, None], float("-inf"))
    sc = torch.cat([sp, so], -1)
    del sp, so
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    del sc
    l = p.sum(-1, keepdim=True)
    Lp = tok.numel()
    pg = torch.zeros(G, M, hkv, r, Lp, device=dev)
    pg[gid, at] = p[..., :Lp]
    vg = vp[ids, :, tok % P].float().permute(0, 2, 1, 3)
    og = (pg.permute(0, 2, 1, 3, 4).reshape(G, hkv, M * r, Lp) @ vg).view(G, hkv, M, r, d)
    o = og[gid, :, at] + p[..., Lp:] @ vp[pid, :, pos % P].float().permute(0, 2, 1, 3)
    o = torch.where(l > 0, o / l.clamp(min=1e-30), torch.zeros_like(o))
    return o.reshape(B, hq, d).to(q.dtype)


def _plain_select(s):
    """The n best of beam_score + log_softmax(logits) over beams and vocabulary, in 64 bits
    (candidates of different beams are often closer than 32 bits tell apart)."""
    sc, fin, c = s["beam_scores"], s["finished"], s["case"]
    G, K = sc.shape
    x = s["logits"].double().view(G, K, -1)
    V = x.shape[-1]
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    b = sc.double()[..., None]
    score = torch.where(torch.isfinite(lse) & torch.isfinite(b), b + (x - lse),
                        torch.full_like(x, float("-inf")))
    if fin is not None:
        done = torch.full_like(x, float("-inf"))
        done[..., s["eos"]] = sc.double()
        score = torch.where(fin[..., None], done, score)
    best, at = torch.sort(score.view(G, K * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :c["n"]], at[:, :c["n"]]
    return {"scores": best.float(), "beams": (at // V).to(torch.int32), "tokens": at % V}


def _plain_reorder(s):
    """Beam i of a prompt becomes a copy of beam parents[i]: it names the parent's full pages
    and gets the parent's tokens of the last page in its own."""
    pools, own_t, bt, lens = s["pools"], s["own_table"], s["block_table"], s["seq_lens"].long()
    G, K = s["parents"].shape
    P, mp = pools.shape[4], own_t.shape[1]
    dev = pools.device
    par = (s["parents"].long() + torch.arange(G, device=dev)[:, None] * K).view(-1)
    full, fill = lens // P, lens % P
    cols = torch.arange(mp, device=dev)
    bt.copy_(torch.where(cols < full[:, None], bt[par], own_t))
    tail = own_t.long().gather(1, full.clamp(max=mp - 1)[:, None])[:, 0]
    keep = (torch.arange(P, device=dev) < fill[:, None])[None, None, :, None, :, None]
    pools[:, :, tail] = torch.where(keep, pools[:, :, tail[par]], pools[:, :, tail])
    return {"pools": pools, "block_table": bt}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"prefix": _plain_prefix, "select": _plain_select,
                "reorder": _plain_reorder}[op](state)
    if op == "prefix":
        from llm_cuda_b200.kernels.shared_prefix import shared_prefix_decode

        return shared_prefix_decode(state["q"], state["key_pages"], state["value_pages"],
                                    state["block_table"], state["seq_lens"],
                                    state["group_starts"], state["shared_lens"],
                                    max_group=state["max_group"])
    from llm_cuda_b200.kernels.beam import beam_reorder, beam_select

    if op == "select":
        scores, beams, tokens = beam_select(state["logits"], state["beam_scores"],
                                            num_out=state["case"]["n"],
                                            finished=state["finished"],
                                            eos_token_id=state["eos"])
        return {"scores": scores, "beams": beams, "tokens": tokens}
    beam_reorder(state["pools"], state["own_table"], state["block_table"], state["seq_lens"],
                 state["parents"])
    return {"pools": state["pools"], "block_table": state["block_table"]}


# ---------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------
def work(case):
    e = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "prefix":
        sizes, shared, lens = _prefix_shape(case)
        tok, pages, b = 0, 0, 0
        for n, t in zip(sizes, shared):
            mine = lens[b:b + n]
            reach = min(t, max(mine))
            tok += reach + sum(max(0, x - t) for x in mine)
            pages += -(-reach // case["page"]) + sum(-(-max(0, x - t) // case["page"])
                                                     for x in mine)
            b += n
        return {"bytes": tok * case["hkv"] * case["d"] * 2 * e + pages * 4
                + 2 * len(lens) * case["hq"] * case["d"] * e,
                "flops": 4 * case["hq"] * case["d"] * sum(lens)}
    if case["op"] == "select":
        rows = case["groups"] * case["beams"]
        live = rows * (1.0 - case["finished"])
        return {"bytes": live * case["vocab"] * e + rows * 5 + case["groups"] * case["n"] * 16,
                "flops": 4 * live * case["vocab"]}
    lens, parents = _reorder_shape(case)
    one = case["hkv"] * case["d"] * e * 2 * case["layers"]          # a token of a beam
    moved = 0
    for t, par in zip(lens, parents):
        moves = [(i, p) for i, p in enumerate(par) if i != p]
        moved += t % case["page"] * (len(moves) + len({p for _, p in moves})) * one
        moved += len(moves) * 2 * 4 * (t // case["page"])
    return {"bytes": moved + 4 * case["groups"] * case["beams"] * 2, "flops": 0}


# ---------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prefix":
        # each sequence by itself, through its own row of the table
        lens = s["seq_lens"].tolist()
        B, hq, d = s["q"].shape
        hkv, P = s["key_pages"].shape[1], s["key_pages"].shape[2]
        out = torch.zeros(B, hq, d, device=s["q"].device, dtype=torch.float64)
        for b, n in enumerate(lens):
            if not n:
                continue
            ids = s["block_table"][b, :-(-n // P)].long()
            for h in range(hkv):
                k = s["key_pages"][ids, h].double().reshape(-1, d)[:n]
                v = s["value_pages"][ids, h].double().reshape(-1, d)[:n]
                hs = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
                w = torch.softmax(s["q"][b, hs].double() @ k.T / d ** 0.5, dim=-1)
                out[b, hs] = w @ v
        return out
    if case["op"] == "select":
        rows = []
        for gi in range(case["groups"]):
            cand = []
            for k in range(case["beams"]):
                base = float(s["beam_scores"][gi, k])
                if s["finished"] is not None and bool(s["finished"][gi, k]):
                    cand.append(torch.tensor([base], dtype=torch.float64, device="cuda"))
                    continue
                lp = torch.log_softmax(s["logits"][gi * case["beams"] + k].double(), -1)
                cand.append(base + torch.topk(lp, min(case["n"], case["vocab"])).values)
            cand.append(torch.full((case["n"],), float("-inf"), dtype=torch.float64,
                                   device="cuda"))
            rows.append(torch.topk(torch.cat(cand), case["n"]).values)
        return {"scores": torch.stack(rows), "beams": None, "tokens": None}
    lens, parents = _reorder_shape(case)
    old, K, P = s["pools"].clone(), case["beams"], case["page"]
    own_t = s["own_table"].tolist()
    for gi, (t, par) in enumerate(zip(lens, parents)):
        page, fill = t // P, t % P
        if not fill:
            continue
        for i, p in enumerate(par):
            dst, src = own_t[gi * K + i][page], own_t[gi * K + p][page]
            s["pools"][:, :, dst, :, :fill] = old[:, :, src, :, :fill]
    return {"pools": s["pools"], "block_table": None}
