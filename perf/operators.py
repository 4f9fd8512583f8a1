"""Cases for the operators of the paged KV cache: append, attention, attention weights, eviction.

A batch has `seqs` sequences.  Sequence s brings Q new rows, [q_start[s],
q_start[s + 1]) of the row arrays, and has L cached positions (its new rows'
included) on pages of `page` positions; row i sits at slot L - Q + i and sees
every slot up to its own whose page is mapped.  `own` False computes each
operator in plain torch operations, True through the C-ABI of
include/b2_kernels.h.

Fields of a case: op; seqs; long (how many sequences bring q_lo..q_hi new
rows; the others bring one, or none when idle is set); ctx_lo..ctx_hi
(positions cached before the new rows, spread over the logarithm); nq, nkv,
hd; page; layout ("head": pages of [head][position], "token": [position]
[head]); holes (leading pages given back and unmapped); sizes (the seed of
the lengths); tail (padding rows behind the last sequence); for eviction
budget, sink and recent.
"""
import ctypes
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BASE = dict(long=0, q_lo=1, q_hi=1, idle=False, nq=16, nkv=8, hd=128, page=64, layout="head", holes=False, sizes=1,
            tail=0, budget=0, sink=0, recent=0)


def case_of(name, op, **kw):
    c = dict(BASE, op=op, **kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step of 64 sequences of 128 to 4096 positions: latency
        case_of("append step x64", "append", seqs=64, ctx_lo=128, ctx_hi=4096),
        # a scheduler's step: three prompt chunks of about 2500 rows next to 29 single tokens
        case_of("append chunks", "append", seqs=32, long=3, q_lo=2000, q_hi=3000, ctx_lo=1, ctx_hi=8192, page=16, tail=5),
        # the first tokens of one short conversation: the smallest call
        case_of("attend one", "attend", seqs=1, ctx_lo=130, ctx_hi=130),
        # one decode step of 64 sequences of 128 to 4096 positions
        case_of("attend step x64", "attend", seqs=64, ctx_lo=128, ctx_hi=4096),
        # one decode step of a single very long context, 2 kv heads of 7 q heads
        case_of("attend long step", "attend", seqs=1, ctx_lo=200_001, ctx_hi=200_001, nq=14, nkv=2, page=128),
        # 60 embedding rows of an audio segment for each of 8 streams
        case_of("attend audio x8", "attend", seqs=8, long=8, q_lo=60, q_hi=60, ctx_lo=9, ctx_hi=700, page=16),
        # a 4096-row chunk of a prompt of 16 thousand tokens
        case_of("attend prompt", "attend", seqs=1, long=1, q_lo=4096, q_hi=4096, ctx_lo=12_288, ctx_hi=12_288),
        # decode steps of 40 sequences and prompt chunks of 4 others in one call, head_dim 64, token-major pages
        case_of("attend mixed", "attend", seqs=44, long=4, q_lo=300, q_hi=600, ctx_lo=64, ctx_hi=4096, nq=16, nkv=4,
                hd=64, page=32, layout="token", idle=True, tail=3),
        # the weights of one decode step of 64 sequences
        case_of("weights step x64", "weights", seqs=64, ctx_lo=128, ctx_hi=4096),
        # the weights of a 2048-row chunk at the end of a prompt of 8 thousand tokens
        case_of("weights prompt", "weights", seqs=1, long=1, q_lo=2048, q_hi=2048, ctx_lo=6144, ctx_hi=6144),
        # 16 sequences that reached 2048 to 4096 positions go back to 1024 of them
        case_of("evict x16", "evict", seqs=16, ctx_lo=2048, ctx_hi=4096, budget=1024, sink=4, recent=256),
        # one context of 100 thousand positions goes back to 20 thousand
        case_of("evict long", "evict", seqs=1, ctx_lo=100_003, ctx_hi=100_003, budget=20_000, sink=4, recent=2000,
                page=16, layout="token"),
    ]


def log_between(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "weights", "weights", "evict"])
    nq, nkv = rng.choice([(16, 8), (16, 8), (16, 4), (8, 8), (32, 4), (12, 4), (14, 2), (5, 1)])
    c = case_of(None, op, nq=nq, nkv=nkv, hd=rng.choice([128, 128, 64]), page=rng.choice([16, 32, 64, 128]),
                layout=rng.choice(["head", "head", "token"]), holes=rng.random() < 0.25, idle=rng.random() < 0.25,
                sizes=rng.randrange(1 << 30), tail=rng.choice([0, 0, 1, 7]))
    kind = "step" if op == "evict" else rng.choice(["step", "few", "chunk", "mixed"])
    if kind == "step":
        c["seqs"] = log_between(rng, 1, 100)
    elif kind == "few":  # a few drafted tokens for each sequence
        c["seqs"] = c["long"] = log_between(rng, 1, 40)
        c["q_lo"], c["q_hi"] = 2, 9
    elif kind == "chunk":
        c["seqs"] = c["long"] = rng.randint(1, 4)
        c["q_hi"] = log_between(rng, 17, 2400 // c["seqs"])
        c["q_lo"] = max(1, c["q_hi"] // 2)
    else:
        c["long"] = rng.randint(1, 3)
        c["seqs"] = c["long"] + log_between(rng, 1, 40)
        c["q_hi"] = log_between(rng, 17, 600)
        c["q_lo"] = max(2, c["q_hi"] // 3)
    # lengths: at most 16 thousand for chunks, and 200 thousand cached positions in all
    most = min(16_000 if kind in ("chunk", "mixed") else 100_000, 200_000 // c["seqs"])
    if kind == "mixed":
        most = min(most, 4096)
    c["ctx_hi"] = log_between(rng, 1, most)
    c["ctx_lo"] = max(1, c["ctx_hi"] // rng.choice([1, 2, 16, 64]))
    if op == "evict":
        c["budget"] = log_between(rng, 1, max(1, c["ctx_hi"]))
        c["sink"] = rng.randint(0, min(8, c["budget"]))
        c["recent"] = rng.randint(0, (c["budget"] - c["sink"]) // 2)
        c["idle"] = False
    return c


def lengths(case):
    """[(new rows, cached positions, leading unmapped pages)] of the sequences."""
    r = random.Random(case["sizes"])
    got = []
    for s in range(case["seqs"]):
        ctx = log_between(r, case["ctx_lo"], case["ctx_hi"])
        q = r.randint(case["q_lo"], case["q_hi"]) if s < case["long"] else 1
        if case["idle"] and s >= case["long"] and r.random() < 0.2:
            q = 0
        if case["op"] == "evict":
            q = 0
        lost = r.randint(0, ctx // case["page"] // 2) if case["holes"] else 0
        got.append((q, ctx + q, lost))
    r.shuffle(got)
    return got


def seen(case, q, length, lost):
    """Number of (row, slot) pairs of a sequence where the row sees the slot."""
    first = lost * case["page"]
    return sum(max(0, length - q + i + 1 - first) for i in range(q))


def work(case):
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    seqs = lengths(case)
    rows = sum(q for q, _, _ in seqs)
    cached = sum(n - lost * case["page"] for q, n, lost in seqs if q > 0)
    pairs = sum(seen(case, *s) for s in seqs)
    if case["op"] == "append":  # qkv in, q and the new K and V out, an angle row and a position for each row
        return {"bytes": rows * ((nq + 2 * nkv) * hd * 6 + hd * 4 + 4), "flops": rows * (nq + nkv) * hd * 7}
    if case["op"] == "attend":
        return {"bytes": cached * nkv * hd * 4 + rows * nq * (hd * 4 + 4), "flops": 4 * hd * pairs * nq}
    if case["op"] == "weights":
        total = sum(n for _, n, _ in seqs)
        return {"bytes": cached * nkv * hd * 2 + total * nkv * 8 + rows * nq * (hd * 2 + 4), "flops": 2 * hd * pairs * nq}
    kept = sum(min(case["budget"], n - lost * case["page"]) for _, n, lost in seqs)
    return {"bytes": nkv * (4 * sum(n for _, n, _ in seqs) + kept * (hd * 8 + 8)), "flops": nkv * kept}


def pool(g, n_pages, case):
    """A pool of pages as a [page][head][position][hd] tensor, in the case's layout."""
    nkv, hd, page = case["nkv"], case["hd"], case["page"]
    if case["layout"] == "head":
        return torch.randn(n_pages, nkv, page, hd, generator=g, device="cuda").half()
    return torch.randn(n_pages, page, nkv, hd, generator=g, device="cuda").half().transpose(1, 2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng(seed)
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    seqs = lengths(case)
    B, rows = len(seqs), sum(q for q, _, _ in seqs)
    M = rows + case["tail"]
    width = max(-(-n // page) for _, n, _ in seqs)
    used = sum(-(-n // page) for _, n, _ in seqs)
    kept_pages = -(-case["budget"] // page) if case["op"] == "evict" else 0
    order = r.permutation(used + B * kept_pages + 3).astype(np.int32)
    table = np.full((B, width), -1, np.int32)
    at = 0
    for s, (_, n, lost) in enumerate(seqs):
        k = -(-n // page)
        table[s, lost:k] = order[at + lost:at + k]
        at += k
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    qs = [q for q, _, _ in seqs]
    st = {"case": case, "M": M, "rows": rows, "max_q": max(1, max(qs)), "max_len": max(n for _, n, _ in seqs),
          "table": dev(table), "kv_len": dev(np.array([n for _, n, _ in seqs], np.int32)),
          "q_start": dev(np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)),
          # where each row belongs, as the program that built the batch knows it
          "row_seq": dev(np.repeat(np.arange(B), qs)), "row_idx": dev(np.concatenate([np.arange(q) for q in qs] + [[]]).astype(np.int64)),
          "k": pool(g, len(order), case), "v": pool(g, len(order), case)}
    if case["op"] == "append":
        slots = np.concatenate([np.arange(n - q, n) for q, n, _ in seqs] + [[]])
        ahead = int(r.integers(0, 1000))  # positions that earlier evictions took out of the cache
        st["pos"] = dev(np.concatenate([slots + ahead, np.zeros(case["tail"])]).astype(np.int32))
        angles = torch.arange(st["max_len"] + 1000, device="cuda", dtype=torch.float64)[:, None] * \
            1e6 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        st["cos"], st["sin"] = angles.cos().float(), angles.sin().float()
        st["qkv"] = torch.randn(M, (nq + 2 * nkv) * hd, generator=g, device="cuda") * 1.5
        st["qn"] = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
        st["kn"] = 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
        st["q16"] = torch.zeros(M, nq * hd, device="cuda", dtype=torch.float16)
    if case["op"] in ("attend", "weights"):
        st["q16"] = torch.randn(M, nq * hd, generator=g, device="cuda").half()
        st["out"] = torch.zeros(M, nq * hd, device="cuda", dtype=torch.float16)
        st["lse"] = torch.zeros(M, nq, device="cuda")
    if case["op"] == "weights":
        st["lse"][:rows] = plain_attention(st)[1]
    if case["op"] in ("weights", "evict"):
        st["prev"] = torch.empty(B, nkv, width * page, device="cuda").exponential_(1.0, generator=g)
        st["prev"] *= torch.randint(0, 2, st["prev"].shape, generator=g, device="cuda")  # many slots nobody looked at
        st["weights"] = torch.zeros_like(st["prev"])
    if case["op"] == "evict":
        mapped = [n - lost * page for _, n, lost in seqs]
        st["dst_table"] = dev(order[at:at + B * kept_pages].reshape(B, kept_pages))
        count = [min(case["budget"], n) for n in mapped]
        st["kept_seq"] = dev(np.repeat(np.arange(B), count))
        st["kept_idx"] = dev(np.concatenate([np.arange(n) for n in count]).astype(np.int64))
        st["kept"] = torch.full((B, nkv, case["budget"]), -1, device="cuda", dtype=torch.int32)
        st["dst_weights"] = torch.zeros(B, nkv, case["budget"], device="cuda")
        st["new_len"] = torch.zeros(B, device="cuda", dtype=torch.int32)
    return st


# ── plain forms ──


def gathered(st):
    """K and V in 32 bits as [seq][slot][head][hd], zero where nothing is mapped, and the mask of the mapped slots."""
    page = st["case"]["page"]
    slots = torch.arange(st["max_len"], device="cuda")
    pages = st["table"][:, slots // page]
    mapped = (pages >= 0) & (pages < st["k"].shape[0]) & (slots < st["kv_len"][:, None])
    at, off = pages.clamp(min=0).long(), (slots % page).expand(len(pages), -1)
    k, v = (torch.where(mapped[:, :, None, None], t[at, :, off], 0).float() for t in (st["k"], st["v"]))
    return k, v, mapped


def scores(st, k, mapped):
    """Scaled scores [seq][kv head][q head of the group][row][slot] with -inf where the row does not see the slot."""
    c = st["case"]
    nkv, group = c["nkv"], c["nq"] // c["nkv"]
    q_len = st["q_start"][1:] - st["q_start"][:-1]
    i = torch.arange(st["max_q"], device="cuda")
    rows = (st["q_start"][:-1, None] + i).clamp(max=max(0, st["M"] - 1)).long()
    q = st["q16"][rows].float().view(len(rows), st["max_q"], nkv, group, c["hd"])
    s = torch.einsum("bqgrd,blgd->bgrql", q, k).mul_(1.0 / math.sqrt(c["hd"]))
    slot = (st["kv_len"] - q_len)[:, None] + i
    sees = mapped[:, None, :] & (torch.arange(st["max_len"], device="cuda") <= slot[:, :, None])
    sees &= (i < q_len[:, None])[:, :, None]
    return s.masked_fill_(~sees[:, None, None], -math.inf)


def plain_attention(st):
    c = st["case"]
    k, v, mapped = gathered(st)
    s = scores(st, k, mapped)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bgrql,blgd->bqgrd", p, v)
    o = o / torch.where(total > 0, total, 1.0).permute(0, 3, 1, 2, 4)
    lse = (m + total.log()).squeeze(-1).permute(0, 3, 1, 2)
    at = (st["row_seq"], st["row_idx"])
    return o[at].reshape(-1, c["nq"] * c["hd"]).half(), lse[at].reshape(-1, c["nq"])


def plain_append(st):
    c, M = st["case"], st["rows"]
    nq, nkv, hd, page = c["nq"], c["nkv"], c["hd"], c["page"]
    x = st["qkv"][:M].view(M, nq + 2 * nkv, hd)
    qk, v = x[:, :nq + nkv], x[:, nq + nkv:]
    w = torch.cat([st["qn"].expand(nq, hd), st["kn"].expand(nkv, hd)])
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    pos = st["pos"][:M].long()
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    a, b = qk[..., :hd // 2], qk[..., hd // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    st["q16"][:M] = qk[:, :nq].reshape(M, nq * hd).half()
    q_len = st["q_start"][1:] - st["q_start"][:-1]
    slot = (st["kv_len"] - q_len)[st["row_seq"]] + st["row_idx"]
    at = st["table"][st["row_seq"], slot // page].long()
    st["k"][at, :, slot % page] = qk[:, nq:].half()
    st["v"][at, :, slot % page] = v.half()
    return {"q16": st["q16"], "k": st["k"], "v": st["v"]}


def plain_weights(st):
    c = st["case"]
    nkv, group = c["nkv"], c["nq"] // c["nkv"]
    k, _, mapped = gathered(st)
    s = scores(st, k, mapped)
    i = torch.arange(st["max_q"], device="cuda")
    rows = (st["q_start"][:-1, None] + i).clamp(max=max(0, st["M"] - 1)).long()
    lse = st["lse"][rows].view(len(rows), st["max_q"], nkv, group).permute(0, 2, 3, 1)[..., None]
    total = s.sub_(lse).exp_().sum((2, 3))
    n = st["max_len"]
    cached = (torch.arange(n, device="cuda") < st["kv_len"][:, None])[:, None]
    st["weights"][:, :, :n] = torch.where(cached, st["prev"][:, :, :n] + total, st["weights"][:, :, :n])
    return {"weights": st["weights"]}


def plain_evict(st):
    c = st["case"]
    page, budget, n = c["page"], c["budget"], st["max_len"]
    k, v, mapped = gathered(st)
    slots = torch.arange(n, device="cuda")
    w = st["prev"][:, :, :n]
    always = (slots < c["sink"]) | (slots >= st["kv_len"][:, None] - c["recent"])
    key = torch.where((mapped & always)[:, None], math.inf, torch.where(mapped[:, None], w, -math.inf))
    best = key.sort(stable=True, dim=-1, descending=True).indices[..., :budget]
    new_len = mapped.sum(-1).clamp(max=budget)
    full = torch.full((*key.shape[:2], budget), n, device="cuda")
    full[..., :best.shape[-1]] = best
    live = torch.arange(budget, device="cuda") < new_len[:, None, None]
    kept = torch.where(live, full, n).sort(-1).values
    st["kept"].copy_(torch.where(live, kept, st["kept"].long()))
    st["dst_weights"].copy_(torch.where(live, w.gather(-1, kept.clamp(max=n - 1)), st["dst_weights"]))
    st["new_len"].copy_(new_len)
    s, j = st["kept_seq"], st["kept_idx"]
    src, heads = kept[s, :, j], torch.arange(c["nkv"], device="cuda")
    to = st["dst_table"][s, j // page].long()
    st["k"][to, :, j % page] = k[s[:, None], src, heads].half()
    st["v"][to, :, j % page] = v[s[:, None], src, heads].half()
    return evicted(st)


def evicted(st):
    return {"kept": st["kept"], "weights": st["dst_weights"], "new_len": st["new_len"], "k": st["k"], "v": st["v"]}


# ── the framework's entry points ──


def library():
    path = os.path.join(ROOT, "rknn-matmul-parallel_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import b200_decoder
    return b200_decoder


def handle(st):
    """What a serving loop builds once and keeps: the cache's description, the workspace and the error flag."""
    bd, c, k = library(), st["case"], st["k"]
    kv = bd.B2PagedKV(k.data_ptr(), st["v"].data_ptr(), k.stride(0), k.stride(1), k.stride(2), k.shape[0], c["page"],
                      len(st["kv_len"]), st["table"].shape[1], st["table"].data_ptr(), st["kv_len"].data_ptr(),
                      st["q_start"].data_ptr())
    size = bd.capi().b2_attention_paged_workspace(len(st["kv_len"]), st["max_q"], c["nq"], c["nkv"], c["hd"])
    st["work"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
    st["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    st["kv"] = kv
    return kv


def called(st):
    bd, c = library(), st["case"]
    kv = ctypes.byref(st.get("kv") or handle(st))
    nq, nkv, hd, M = c["nq"], c["nkv"], c["hd"], st["M"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        bd.check(bd.capi().b2_qk_rope_kv_paged(
            st["q16"].data_ptr(), nq * hd, st["qkv"].data_ptr(), (nq + 2 * nkv) * hd, M, nq, nkv, hd, st["qn"].data_ptr(),
            st["kn"].data_ptr(), 1e-6, st["cos"].data_ptr(), st["sin"].data_ptr(), len(st["cos"]), 1, st["pos"].data_ptr(),
            kv, stream), "b2_qk_rope_kv_paged")
        return {"q16": st["q16"], "k": st["k"], "v": st["v"]}
    if c["op"] == "attend":
        bd.check(bd.capi().b2_attention_paged(
            st["out"].data_ptr(), st["lse"].data_ptr(), st["q16"].data_ptr(), nq * hd, M, st["max_q"], nq, nkv, hd, kv,
            st["work"].data_ptr(), st["err"].data_ptr(), stream), "b2_attention_paged")
        return {"out": st["out"], "lse": st["lse"]}
    if c["op"] == "weights":
        bd.check(bd.capi().b2_attention_paged_weights(
            st["weights"].data_ptr(), st["prev"].data_ptr(), st["prev"].stride(1), st["q16"].data_ptr(), nq * hd,
            st["lse"].data_ptr(), M, st["max_q"], nq, nkv, hd, kv, st["err"].data_ptr(), stream),
            "b2_attention_paged_weights")
        return {"weights": st["weights"]}
    bd.check(bd.capi().b2_kv_evict_paged(
        kv, nkv, hd, st["prev"].data_ptr(), st["prev"].stride(1), c["budget"], c["sink"], c["recent"],
        st["dst_table"].data_ptr(), st["dst_table"].shape[1], st["kept"].data_ptr(), st["dst_weights"].data_ptr(),
        st["new_len"].data_ptr(), stream), "b2_kv_evict_paged")
    return evicted(st)


def run(st):
    if own:
        return called(st)
    if st["case"]["op"] == "attend":
        out, lse = plain_attention(st)
        st["out"][:st["rows"]] = out
        st["lse"][:st["rows"]] = lse
        return {"out": st["out"], "lse": st["lse"]}
    return {"append": plain_append, "weights": plain_weights, "evict": plain_evict}[st["case"]["op"]](st)


# ── in 64 bits, a sequence and a head at a time ──


def exact(case, seed):
    st = prepare(case, seed)
    nq, nkv, hd, page, op = case["nq"], case["nkv"], case["hd"], case["page"], case["op"]
    group, seqs, f64 = nq // nkv, lengths(case), torch.float64
    k, v = st["k"].to(f64), st["v"].to(f64)
    table = st["table"].tolist()
    if op == "append":
        q16 = st["q16"].to(f64)
        x = st["qkv"].to(f64).view(st["M"], -1, hd)
        row = 0
        for s, (q, n, _) in enumerate(seqs):
            y, pos = x[row:row + q].clone(), st["pos"][row:row + q].long()
            for lo, hi, w in ((0, nq, st["qn"]), (nq, nq + nkv, st["kn"])):
                y[:, lo:hi] *= ((y[:, lo:hi] ** 2).mean(-1, keepdim=True) + 1e-6) ** -0.5 * w.to(f64)
            turn = torch.complex(st["cos"][pos].to(f64), st["sin"][pos].to(f64))[:, None]
            z = torch.complex(y[:, :nq + nkv, :hd // 2], y[:, :nq + nkv, hd // 2:]) * turn
            y[:, :nq + nkv] = torch.cat([z.real, z.imag], -1)
            q16[row:row + q] = y[:, :nq].flatten(1)
            for p in range((n - q) // page, -(-n // page)):  # the pages that the new rows reach
                lo, hi = max(n - q, p * page), min(n, (p + 1) * page)
                new = y[lo - (n - q):hi - (n - q)].transpose(0, 1)
                k[table[s][p], :, lo - p * page:hi - p * page] = new[nq:nq + nkv]
                v[table[s][p], :, lo - p * page:hi - p * page] = new[nq + nkv:]
            row += q
        return {"q16": q16, "k": k, "v": v}
    if op == "evict":
        w64 = st["prev"].cpu().numpy()
        kept, dst_w = st["kept"].cpu().numpy().copy(), np.zeros(st["dst_weights"].shape)
        new_len, dst = [], st["dst_table"].tolist()
        for s, (_, n, lost) in enumerate(seqs):
            new_len.append(min(case["budget"], n - lost * page))
            for g in range(nkv):
                must = [j for j in range(lost * page, n) if j < case["sink"] or j >= n - case["recent"]]
                held = set(must)
                rest = sorted((j for j in range(lost * page, n) if j not in held), key=lambda j: (-w64[s, g, j], j))
                for a, j in enumerate(sorted(must + rest[:new_len[s] - len(must)])):
                    kept[s, g, a], dst_w[s, g, a] = j, w64[s, g, j]
            src, to = torch.from_numpy(kept[s, :, :new_len[s]].astype(np.int64)).cuda(), torch.arange(new_len[s], device="cuda")
            at, here = torch.tensor(table[s], device="cuda"), torch.tensor(dst[s], device="cuda")
            for g in range(nkv):
                for t in (k, v):
                    t[here[to // page], g, to % page] = t[at[src[g] // page], g, src[g] % page]
        return {"kept": torch.from_numpy(kept), "weights": torch.from_numpy(dst_w), "new_len": torch.tensor(new_len, dtype=torch.int32),
                "k": k, "v": v}
    out, lse = st["out"].to(f64), st["lse"].to(f64)
    weights = st["weights"].to(f64) if op == "weights" else None
    row = 0
    for s, (q, n, lost) in enumerate(seqs):
        at = torch.tensor(table[s][lost:-(-n // page)], device="cuda")
        first = lost * page
        sees = torch.arange(first, n, device="cuda") <= torch.arange(n - q, n, device="cuda")[:, None]
        for g in range(nkv):
            keys, values = (t[at, g].reshape(-1, hd)[:n - first] for t in (k, v))
            total = torch.zeros(n - first, dtype=f64, device="cuda")
            for h in range(g * group, (g + 1) * group):
                x = st["q16"][row:row + q, h * hd:(h + 1) * hd].to(f64) @ keys.T / hd ** 0.5
                x[~sees] = -math.inf
                if op == "weights":
                    total += (x - lse[row:row + q, h, None]).exp().sum(0)
                elif q:
                    out[row:row + q, h * hd:(h + 1) * hd] = torch.softmax(x, -1) @ values
                    lse[row:row + q, h] = torch.logsumexp(x, -1)
            if op == "weights":
                weights[s, g, :first] = st["prev"][s, g, :first]
                weights[s, g, first:n] = st["prev"][s, g, first:n] + total
        row += q
    return {"weights": weights} if op == "weights" else {"out": out, "lse": lse}
