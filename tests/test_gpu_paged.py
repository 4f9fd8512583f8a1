"""The paged KV cache operators (b2_qk_rope_kv_paged, b2_attention_paged,
b2_attention_paged_weights, b2_kv_evict_paged) against a plain 64-bit form.

Everything a sequence does not own holds NaN: slots past kv_len, unmapped
pages, spare pages, padding columns of the row arrays.  What a call must leave
alone holds a marker and is compared bit by bit.

Tolerances.  u = 2^-11 is half a step of FP16.  The score of a row and a slot is
a sum of hd exact products added in FP32, in any order and with truncation:
off by at most e = (hd + 2) 2^-23 sum|q k| / sqrt(hd), and its exponential by a
factor 1 +- (e + 2^-20).  The softmax weights are rounded to FP16 (u each), the
output too, so an output may be off by u |o| + (u + 2 (e + 2^-20)) sum p |v|, plus
half of FP16's smallest subnormal step.  The second-order terms are covered by the factor 1.01."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import b200_decoder as bd  # noqa: E402

if not torch.cuda.is_available():  # pragma: no cover - CPU containers
    pytest.skip("needs a CUDA device", allow_module_level=True)

DEV = torch.device("cuda:0")
U = 2.0 ** -11
F64 = torch.float64


def stream():
    return torch.cuda.current_stream().cuda_stream


class Paged:
    """A batch over a paged cache.  seqs: (new rows, kv_len, unmapped page indexes)."""

    def __init__(self, seqs, nq=16, nkv=8, hd=128, page=64, layout="head", seed=0, tail=0, scale=1.0, bad=-1,
                 extra_pages=3, extra_cols=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = np.random.default_rng(seed)
        self.seqs, self.nq, self.nkv, self.hd, self.page, self.G = seqs, nq, nkv, hd, page, nq // nkv
        B = len(seqs)
        self.width = max([1] + [-(-n // page) for _, n, _ in seqs]) + extra_cols
        count = sum(-(-n // page) for _, n, _ in seqs)
        self.n_pages = count + extra_pages
        order = r.permutation(self.n_pages)
        table = np.full((B, self.width), bad, np.int64)
        at = 0
        for s, (_, n, holes) in enumerate(seqs):
            for p in range(-(-n // page)):
                if p not in holes:
                    table[s, p] = order[at]
                at += 1
        self.spare = [int(x) for x in order[at:]]
        self.table = torch.from_numpy(table.astype(np.int32)).to(DEV)
        self.kv_len = torch.tensor([n for _, n, _ in seqs], dtype=torch.int32, device=DEV)
        starts = np.concatenate([[0], np.cumsum([q for q, _, _ in seqs])])
        self.rows = int(starts[-1])
        self.M = self.rows + tail
        self.starts = starts
        self.q_start = torch.from_numpy(starts.astype(np.int32)).to(DEV)
        self.k, self.v = self._pools(layout)
        self.q16 = (torch.randn(max(1, self.M), nq * hd + 8, generator=g, device=DEV) * scale).half()
        self.q16[:, nq * hd:] = math.nan  # padding columns
        for s, (_, n, holes) in enumerate(seqs):
            for p in range(-(-n // page)):
                if p in holes:
                    continue
                m = min(page, n - p * page)
                for t in (self.k, self.v):
                    t[table[s, p], :, :m] = (torch.randn(nkv, m, hd, generator=g, device=DEV) * scale).half()
        size = bd.capi().b2_attention_paged_workspace(B, max(1, self.M), nq, nkv, hd)
        self.work = torch.zeros(size, dtype=torch.uint8, device=DEV)
        self.err = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.max_q = max([1] + [q for q, _, _ in seqs])

    def _pools(self, layout):
        n, h, p, d = self.n_pages, self.nkv, self.page, self.hd
        nan = lambda *shape: torch.full(shape, math.nan, dtype=torch.float16, device=DEV)  # noqa: E731
        if layout == "head":
            return nan(n, h, p, d), nan(n, h, p, d)
        if layout == "token":
            return nan(n, p, h, d).transpose(1, 2), nan(n, p, h, d).transpose(1, 2)
        both = nan(n, 3, h, p, d + 8)  # K and V of one layer among others, padded rows
        return both[:, 0, :, :, :d], both[:, 2, :, :, :d]

    def kv(self, q_start=None):
        k, qs = self.k, self.q_start if q_start is None else q_start
        assert k.stride() == self.v.stride() and k.stride(3) == 1
        return bd.B2PagedKV(k.data_ptr(), self.v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), self.n_pages,
                            self.page, len(self.seqs), self.table.shape[1], self.table.data_ptr(),
                            self.kv_len.data_ptr(), qs.data_ptr())

    def attend(self, max_q=None, want_lse=True, st=None):
        out = torch.full((max(1, self.M), self.nq * self.hd), 7.0, dtype=torch.float16, device=DEV)
        lse = torch.full((max(1, self.M), self.nq), 7.0, device=DEV)
        bd.check(bd.capi().b2_attention_paged(
            out.data_ptr(), lse.data_ptr() if want_lse else None, self.q16.data_ptr(), self.q16.stride(0), self.M,
            self.max_q if max_q is None else max_q, self.nq, self.nkv, self.hd, ctypes.byref(self.kv()),
            self.work.data_ptr(), self.err.data_ptr(), stream() if st is None else st), "b2_attention_paged")
        return out, lse

    def weigh(self, lse, prev, out, max_q=None):
        bd.check(bd.capi().b2_attention_paged_weights(
            out.data_ptr(), None if prev is None else prev.data_ptr(), out.stride(1), self.q16.data_ptr(),
            self.q16.stride(0), lse.data_ptr(), self.M, self.max_q if max_q is None else max_q, self.nq, self.nkv,
            self.hd, ctypes.byref(self.kv()), self.err.data_ptr(), stream()), "b2_attention_paged_weights")
        return out

    def slots(self, s):
        """Mapped slots below kv_len of sequence s (host list) and their K, V [slot][head][hd] in 64 bits."""
        n = self.seqs[s][1]
        row = self.table[s].tolist()
        js = [j for j in range(min(n, len(row) * self.page)) if 0 <= row[j // self.page] < self.n_pages]
        pg = torch.tensor([row[j // self.page] for j in js], dtype=torch.long, device=DEV)
        off = torch.tensor([j % self.page for j in js], dtype=torch.long, device=DEV)
        j = torch.tensor(js, dtype=torch.long, device=DEV)
        return j, self.k[pg, :, off].to(F64), self.v[pg, :, off].to(F64)

    def reference(self):
        """out, lse, the tolerance of out, and that of lse, for the rows of the sequences."""
        nq, hd, G = self.nq, self.hd, self.G
        out = torch.zeros(self.rows, nq, hd, dtype=F64, device=DEV)
        lse = torch.full((self.rows, nq), -math.inf, dtype=F64, device=DEV)
        tol, tl = torch.zeros_like(out), torch.zeros_like(lse)
        for s, (q, n, _) in enumerate(self.seqs):
            j, K, V = self.slots(s)
            if q == 0 or len(j) == 0:
                continue
            r = slice(int(self.starts[s]), int(self.starts[s]) + q)
            Q = self.q16[r, :nq * hd].to(F64).view(q, nq, hd)
            K, V = (t.repeat_interleave(G, 1) for t in (K, V))
            x = torch.einsum("rhd,jhd->hrj", Q, K) / math.sqrt(hd)
            mag = torch.einsum("rhd,jhd->hrj", Q.abs(), K.abs()) / math.sqrt(hd)
            sees = j[None] <= (n - q + torch.arange(q, device=DEV))[:, None]
            x = x.masked_fill(~sees, -math.inf)
            m = x.amax(-1, keepdim=True)
            p = (x - torch.where(m == -math.inf, 0.0, m)).exp()
            l = p.sum(-1, keepdim=True)
            p = p / torch.where(l > 0, l, 1.0)
            e = (hd + 2) * 2.0 ** -23 * mag.masked_fill(~sees, 0).amax(-1) + 2.0 ** -20
            o = torch.einsum("hrj,jhd->rhd", p, V)
            a = torch.einsum("hrj,jhd->rhd", p, V.abs())
            out[r] = o
            tol[r] = U * o.abs() + (U + 2 * e.T[..., None]) * a
            lse[r] = (m + l.log())[..., 0].T
            tl[r] = e.T + 2.0 ** -21 * (1 + lse[r].abs().nan_to_num(posinf=0))
        return out.reshape(self.rows, -1), lse, 1.01 * tol.reshape(self.rows, -1) + 2.0 ** -25, tl


def check_attention(b, out, lse, max_q=None):
    """out and lse of a call on b, with rows past max_q of a sequence and the tail untouched."""
    assert b.err.item() == 0
    assert not b.work[:4096].any(), "counters stay zero"
    ro, rl, tol, tl = b.reference()
    done = torch.zeros(out.shape[0], dtype=torch.bool, device=DEV)
    for s, (q, _, _) in enumerate(b.seqs):
        a = int(b.starts[s])
        done[a:a + min(q, q if max_q is None else max_q)] = True
    assert bool((out[~done] == 7).all()) and bool((lse[~done] == 7).all())
    n = b.rows
    d = (out[:n].to(F64) - ro).abs()
    ok = (d <= tol) | ~done[:n, None]
    assert bool(ok.all()), (int((~ok).sum()), float((d / tol)[done[:n]].max()), torch.nonzero(~ok)[:4].tolist())
    dl = lse[:n].to(F64)
    empty = rl == -math.inf
    assert bool(((dl == -math.inf) == empty)[done[:n]].all())
    okl = ((dl - rl).abs() <= tl) | empty | ~done[:n, None]
    assert bool(okl.all()), float(((dl - rl).abs() / tl)[~empty & done[:n, None]].max())


HEADS = [(16, 8, 128), (16, 4, 64), (3, 1, 128), (14, 2, 128), (32, 4, 64), (5, 1, 64), (8, 8, 128), (16, 1, 128)]


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_attention_lengths(nq, nkv, hd, page):
    """Cached lengths from nothing to several blocks, one to a few new rows, idle sequences."""
    seqs = [(1, n, ()) for n in (1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 257, 1000)]
    seqs += [(0, 40, ()), (0, 0, ()), (2, 2, ()), (3, 66, ()), (2, 300, ())]
    b = Paged(seqs, nq, nkv, hd, page, layout=["head", "token", "mixed"][page % 3], seed=page + nq, tail=3)
    check_attention(b, *b.attend())


@pytest.mark.parametrize("q", [2, 4, 5, 8, 9, 16, 17, 33, 64, 65, 100, 128, 130, 257, 400])
@pytest.mark.parametrize("nq,nkv,hd,page", [(16, 8, 128, 64), (16, 4, 64, 16), (3, 1, 128, 32), (16, 1, 64, 128),
                                            (7, 1, 128, 16)])
def test_attention_chunks(nq, nkv, hd, page, q):
    """Chunks of new rows behind caches of several lengths, next to single tokens."""
    seqs = [(q, q, ()), (1, 70, ()), (q, q + 1, ()), (q - 1, q + 63, ()), (0, 9, ()), (q, q + 517, ()), (1, 1, ())]
    b = Paged(seqs, nq, nkv, hd, page, layout="token" if q % 2 else "head", seed=q, tail=1)
    check_attention(b, *b.attend())


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("q", [1, 3, 70, 200])
@pytest.mark.parametrize("bad", [-1, 1 << 30, -(1 << 31), None])
def test_attention_unmapped_pages(page, q, bad):
    """Unmapped pages in front, in the middle, at the end and everywhere; rows that see nothing at all."""
    n = 5 * page + 3 + q
    k = -(-n // page)
    seqs = [(q, n, (0,)), (q, n, (0, 1, 2)), (q, n, (2,)), (q, n, (1, 3)), (q, n, (k - 1,)), (q, n, tuple(range(k))),
            (q, n, (0, k - 1)), (q, n, ()), (q, q, tuple(range(-(-q // page))))]
    if bad is None:  # the first id past the pool
        bad = sum(-(-m // page) for _, m, _ in seqs) + 3
    b = Paged(seqs, 8, 4, 128, page, seed=page + q, bad=bad)
    check_attention(b, *b.attend())


@pytest.mark.parametrize("q", [2, 40, 150])
def test_attention_fewer_cached_than_new(q):
    """kv_len below the number of new rows: the first rows have no slot and see nothing."""
    b = Paged([(q, q - 1, ()), (q, 1, ()), (q, 0, ()), (1, 0, ()), (q, q // 2, ())], 4, 2, 64, 16, seed=q)
    check_attention(b, *b.attend())


@pytest.mark.parametrize("q", [1, 6, 90])
def test_attention_kv_len_beyond_table(q):
    """kv_len past what the table can hold: the slots behind it are not there."""
    b = Paged([(q, 128, ()), (q, 100, ())], 4, 2, 128, 64, seed=q)
    b.table = b.table[:, :1].contiguous()
    b.width = 1
    check_attention(b, *b.attend())


@pytest.mark.parametrize("nq,nkv,hd,page,q,n", [(2, 1, 128, 128, 1, 30_011), (14, 2, 128, 16, 1, 20_000),
                                                (16, 8, 64, 64, 4, 9_000), (4, 4, 128, 32, 1, 12_345),
                                                (2, 1, 128, 64, 100, 20_100), (8, 1, 64, 32, 70, 33_333)])
def test_attention_long(nq, nkv, hd, page, q, n):
    """Contexts that many CTAs share; the pieces are merged in a fixed order, so calls repeat bit by bit."""
    b = Paged([(q, n, ())], nq, nkv, hd, page, seed=n)
    out, lse = b.attend()
    check_attention(b, out, lse)
    for _ in range(3):
        o2, l2 = b.attend()
        assert torch.equal(out, o2) and torch.equal(lse, l2)


@pytest.mark.parametrize("seqs_n", [1, 31, 32, 33, 64, 500, 1024])
def test_attention_many_sequences(seqs_n):
    r = np.random.default_rng(seqs_n)
    seqs = [(int(r.integers(0, 3)), int(r.integers(3, 90)), ()) for _ in range(seqs_n)]
    b = Paged(seqs, 4, 2, 64, 16, seed=seqs_n, tail=2)
    check_attention(b, *b.attend())


@pytest.mark.parametrize("seqs,max_q", [([(9, 30, ()), (1, 5, ())], 4), ([(300, 300, ()), (2, 70, ())], 130),
                                        ([(70, 200, ())], 1)])
def test_attention_max_q_cuts(seqs, max_q):
    """Rows past the first max_q of a sequence are left as they were."""
    b = Paged(seqs, 4, 2, 128, 32, seed=max_q)
    out, lse = b.attend(max_q=max_q)
    check_attention(b, out, lse, max_q=max_q)


def test_attention_without_lse():
    b = Paged([(1, 700, ()), (90, 300, ())], seed=3)
    out, _ = b.attend()
    again, untouched = b.attend(want_lse=False)
    assert torch.equal(out, again) and bool((untouched == 7).all())


@pytest.mark.parametrize("q", [1, 5, 130])
def test_attention_extreme_scores(q):
    """Scores of +-2000 (one slot takes everything), equal scores, and the type's lowest values in K."""
    b = Paged([(q, 200 + q, ()), (q, 300 + q, ()), (q, 150 + q, ())], 4, 2, 128, 64, seed=q, scale=12.0)
    pages = b.table.tolist()
    for p in pages[1][:5]:
        b.k[p][~b.k[p].isnan()] = 0.25  # every slot weighs the same
    b.k[pages[2][0], :, 3] = -65504.0
    b.k[pages[2][1], :, 5] = 65504.0
    # scores near 1e6 x 2^-17 relative error say nothing about a softmax, so q is small there
    r = slice(int(b.starts[2]), int(b.starts[2]) + q)
    b.q16[r, :512] *= 2.0 ** -12
    check_attention(b, *b.attend())


@pytest.mark.parametrize("q", [1, 4, 140])
def test_attention_non_finite_values(q):
    """Infinities in slots nobody sees change nothing; a NaN in a seen slot reaches the rows that see it."""
    b = Paged([(q, 160 + q, (1,)), (q, 90 + q, ())], 4, 2, 128, 64, seed=q)
    for p in b.spare:
        b.k[p], b.v[p] = math.inf, -math.inf
    out, lse = b.attend()
    check_attention(b, out, lse)
    page = int(b.table[1, 0])
    b.k[page, 1, 7] = math.nan  # kv head 1 of sequence 1
    out2, lse2 = b.attend()
    r = slice(int(b.starts[1]), int(b.starts[1]) + q)
    assert bool(out2[r, 256:].isnan().all()) and bool(lse2[r, 2:].isnan().all())
    out2[r, 256:], lse2[r, 2:] = out[r, 256:], lse[r, 2:]
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("q", [1, 90])
def test_attention_graph_streams_and_shared_workspace(q):
    """Captured and replayed with other lengths, on another stream, with one workspace for calls of other shapes."""
    small = Paged([(1, 33, ())], 8, 1, 64, 16, seed=9)
    b = Paged([(q, 500 + q, ()), (q, 1200 + q, ()), (1, 64, ())], seed=q)
    small.work = b.work
    side = torch.cuda.Stream()
    b.attend()  # the first call sets the kernels up outside the capture
    torch.cuda.synchronize()
    out = torch.full((b.M, b.nq * b.hd), 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full((b.M, b.nq), 7.0, device=DEV)
    kv = b.kv()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        bd.check(bd.capi().b2_attention_paged(
            out.data_ptr(), lse.data_ptr(), b.q16.data_ptr(), b.q16.stride(0), b.M, b.max_q, b.nq, b.nkv, b.hd,
            ctypes.byref(kv), b.work.data_ptr(), b.err.data_ptr(), torch.cuda.current_stream().cuda_stream))
    graph.replay()
    torch.cuda.synchronize()
    check_attention(b, out, lse)
    check_attention(small, *small.attend())
    # shorter contexts for the same graph: the first two sequences lose their newest slots
    b.seqs = [(q, 100 + q, ()), (q, 700 + q, ()), (1, 64, ())]
    b.kv_len.copy_(torch.tensor([n for _, n, _ in b.seqs], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    check_attention(b, out, lse)


# ── append ──


def rope_reference(b, qkv, qn, kn, cos, sin, pos, style):
    """q and k rows [M][head][hd] in 64 bits, and their rounding tolerances' magnitudes."""
    nq, nkv, hd = b.nq, b.nkv, b.hd
    x = qkv[:, :(nq + 2 * nkv) * hd].to(F64).view(len(qkv), nq + 2 * nkv, hd)
    y = x[:, :nq + nkv].clone()
    for lo, hi, w in ((0, nq, qn), (nq, nq + nkv, kn)):
        if w is not None:
            y[:, lo:hi] = y[:, lo:hi] / (y[:, lo:hi].square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.to(F64)
    c, s = cos[pos.clamp(0, len(cos) - 1).long()].to(F64)[:, None], sin[pos.clamp(0, len(cos) - 1).long()].to(F64)[:, None]
    z, mag = torch.empty_like(y), torch.empty_like(y)
    a, d = (y[..., 0::2], y[..., 1::2]) if style == 0 else (y[..., :hd // 2], y[..., hd // 2:])
    for t, u, v, m in ((z, a * c - d * s, d * c + a * s, 0), (mag, (a * c).abs() + (d * s).abs(), (d * c).abs() + (a * s).abs(), 1)):
        if style == 0:
            t[..., 0::2], t[..., 1::2] = u, v
        else:
            t[..., :hd // 2], t[..., hd // 2:] = u, v
    return z, x[:, nq + nkv:], mag


@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("nq,nkv,hd,page,layout", [(16, 8, 128, 64, "head"), (3, 1, 128, 16, "token"),
                                                   (14, 2, 64, 32, "mixed"), (5, 5, 64, 128, "head"),
                                                   (1, 1, 128, 64, "token")])
def test_append(nq, nkv, hd, page, layout, norm, style):
    """Rows of sequences of every kind: idle, one, a chunk over pages, slots that are unmapped, negative or past the
    table, positions outside the angle tables, padding rows."""
    seqs = [(1, 1, ()), (0, 30, ()), (40, 170, ()), (1, 129, ()), (9, 9, ()), (5, 3, ()), (3, 200, (-(-200 // page) - 1,)),
            (1, 64, ()), (0, 0, ()), (2, 65, ())]
    b = Paged(seqs, nq, nkv, hd, page, layout, seed=nq + style, tail=2)
    g = torch.Generator(device=DEV).manual_seed(nq)
    width = (nq + 2 * nkv) * hd
    qkv = torch.randn(b.M, width + 4, generator=g, device=DEV) * 2
    qkv[:, width:] = math.nan
    qn, kn = ((1 + 0.2 * torch.randn(hd, generator=g, device=DEV)) if norm else None for _ in range(2))
    angle = torch.rand(400, hd // 2, generator=g, device=DEV, dtype=F64) * 6.3
    cos, sin = angle.cos().float(), angle.sin().float()
    slot = torch.cat([torch.arange(n - q, n) for q, n, _ in seqs] + [torch.zeros(2)]).int().to(DEV)
    pos = (slot + 37).clamp(min=0)
    pos[2], pos[50] = 400, -1  # outside the tables: these rows are left out
    q16 = torch.full((b.M, nq * hd + 4), 7.0, dtype=torch.float16, device=DEV)
    before = [t.clone() for t in (b.k, b.v)]
    for p in (pos, None):
        b.k.copy_(before[0]), b.v.copy_(before[1]), q16.fill_(7.0)
        bd.check(bd.capi().b2_qk_rope_kv_paged(
            q16.data_ptr(), q16.stride(0), qkv.data_ptr(), qkv.stride(0), b.M, nq, nkv, hd,
            qn.data_ptr() if norm else None, kn.data_ptr() if norm else None, 1e-6, cos.data_ptr(), sin.data_ptr(), 400,
            style, None if p is None else p.data_ptr(), ctypes.byref(b.kv()), stream()), "b2_qk_rope_kv_paged")
        at = slot if p is None else p
        z, v, mag = rope_reference(b, qkv, qn, kn, cos, sin, at, style)
        # FP32: the norm's three roundings and the sum of squares, two products and a sum: 16 half steps of the terms
        tol = U * z.abs() + 16 * 2.0 ** -24 * mag + 2.0 ** -25
        k_exp, v_exp = (t.to(F64) for t in before)
        k_tol = torch.zeros_like(k_exp)
        row = 0
        for s, (q, n, holes) in enumerate(seqs):
            for i in range(q):
                m, j = row, n - q + i
                row += 1
                if not 0 <= int(at[m]) < 400:
                    assert bool((q16[m] == 7).all())
                    continue
                d = (q16[m, :nq * hd].to(F64).view(nq, hd) - z[m, :nq]).abs()
                assert bool((d <= tol[m, :nq]).all()), (m, float((d / tol[m, :nq]).max()))
                if j < 0 or j // page in holes:
                    continue
                pg = int(b.table[s, j // page])
                k_exp[pg, :, j % page], k_tol[pg, :, j % page] = z[m, nq:], tol[m, nq:]
                v_exp[pg, :, j % page] = v[m].half().to(F64)
        assert bool((q16[b.rows:] == 7).all()) and bool((q16[:, nq * hd:] == 7).all())
        same = (b.k.to(F64) - k_exp).abs() <= k_tol
        assert bool((same | (b.k.isnan() & k_exp.isnan())).all())
        got = b.v.to(F64)
        assert bool(((got == v_exp) | (got.isnan() & v_exp.isnan())).all())


# ── attention weights ──


def check_weights(b, lse, prev, out, ldw, mark):
    for s, (q, n, _) in enumerate(b.seqs):
        j, K, _ = b.slots(s)
        r = slice(int(b.starts[s]), int(b.starts[s]) + q)
        total = torch.zeros(b.nkv, max(1, n), dtype=F64, device=DEV)
        tol = torch.zeros_like(total)
        if q and len(j):
            Q = b.q16[r, :b.nq * b.hd].to(F64).view(q, b.nkv, b.G, b.hd)
            x = torch.einsum("rghd,jgd->ghrj", Q, K) / math.sqrt(b.hd)
            mag = torch.einsum("rghd,jgd->ghrj", Q.abs(), K.abs()) / math.sqrt(b.hd)
            le = lse[r].to(F64).view(q, b.nkv, b.G).permute(1, 2, 0)[..., None]
            sees = (j[None] <= (n - q + torch.arange(q, device=DEV))[:, None]) & (le > -math.inf)
            p = torch.where(sees, (x - le.nan_to_num(neginf=0)).exp(), 0.0)
            e = (b.hd + 2) * 2.0 ** -23 * mag + 2.0 ** -22 * (x.abs() + le.nan_to_num(neginf=0).abs()) + 2.0 ** -20
            total[:, j] = p.sum((1, 2))
            tol[:, j] = (p * e).sum((1, 2)) + (q * b.G + 8) * 2.0 ** -24 * total[:, j]
        m = min(n, ldw)
        was = torch.zeros_like(total[:, :m]) if prev is None else prev[s, :, :m].to(F64)
        d = (out[s, :, :m].to(F64) - (was + total[:, :m])).abs()
        t = 1.01 * tol[:, :m] + 2.0 ** -23 * (was + total[:, :m]).abs()
        assert bool((d <= t).all()), (s, float((d / t.clamp(min=1e-30)).max()))
        assert bool((out[s, :, m:] == mark).all())
    assert b.err.item() == 0


@pytest.mark.parametrize("with_prev", [True, False])
@pytest.mark.parametrize("nq,nkv,hd,page", [(16, 8, 128, 64), (14, 2, 64, 16), (3, 1, 128, 32), (16, 1, 64, 128)])
@pytest.mark.parametrize("q", [1, 2, 7, 33, 130, 300])
def test_weights(nq, nkv, hd, page, q, with_prev):
    seqs = [(q, q, ()), (q, q + 1, ()), (1, 70, ()), (0, 40, ()), (q, q + 300, (1,)), (q, q - 1, ()), (1, 1, ()), (0, 0, ()),
            (q, q + 129, (0, 1))]
    b = Paged(seqs, nq, nkv, hd, page, layout="token" if q % 2 else "head", seed=q, tail=2)
    _, lse = b.attend()
    ldw = q + 310
    prev = torch.rand(len(seqs), nkv, ldw, device=DEV) if with_prev else None
    out = torch.full((len(seqs), nkv, ldw), 7.0, device=DEV)
    b.weigh(lse, prev, out)
    check_weights(b, lse, prev, out, ldw, 7.0)
    again = torch.full_like(out, 7.0)
    b.weigh(lse, prev, again)
    assert torch.equal(out, again)
    if with_prev:  # in place
        here = torch.where(out == 7.0, 7.0, prev)
        b.weigh(lse, here, here)
        assert torch.equal(here, out)


@pytest.mark.parametrize("q", [1, 200])
def test_weights_of_one_row_sum_to_the_group(q):
    """Every row gives each of its q heads a total of one."""
    b = Paged([(q, 900 + q, ())], seed=q)
    _, lse = b.attend()
    out = b.weigh(lse, None, torch.zeros(1, b.nkv, 900 + q, device=DEV))
    # 1100 slots of e ~ 2^-13 relative error at most
    assert bool(((out.to(F64).sum(-1) / (q * b.G) - 1).abs() < 2.0 ** -12).all())


def test_weights_narrow_rows_and_max_q():
    """Weight rows shorter than the cache, and rows past max_q that give nothing."""
    b = Paged([(5, 200, ()), (80, 100, ())], 4, 2, 64, 32, seed=4)
    _, lse = b.attend()
    out = torch.full((2, 2, 90), 7.0, device=DEV)
    b.weigh(lse, None, out)
    check_weights(b, lse, None, out, 90, 7.0)
    few = lse.clone()
    few[3:5], few[5 + 3:] = -math.inf, -math.inf
    out2 = torch.full((2, 2, 90), 7.0, device=DEV)
    b.weigh(lse, None, out2, max_q=3)
    check_weights(b, few, None, out2, 90, 7.0)


# ── eviction ──


def evict(b, w, budget, sink, recent, dst, dst_weights=True):
    B = len(b.seqs)
    kept = torch.full((B, b.nkv, max(1, budget)), -7, dtype=torch.int32, device=DEV)
    dw = torch.full((B, b.nkv, max(1, budget)), -7.0, device=DEV)
    n = torch.full((B,), -7, dtype=torch.int32, device=DEV)
    bd.check(bd.capi().b2_kv_evict_paged(
        ctypes.byref(b.kv()), b.nkv, b.hd, w.data_ptr(), w.stride(1), budget, sink, recent, dst.data_ptr(), dst.shape[1],
        kept.data_ptr(), dw.data_ptr() if dst_weights else None, n.data_ptr(), stream()), "b2_kv_evict_paged")
    return kept, dw, n


def evict_reference(b, w, budget, sink, recent):
    """[(kept slots per kv head)] per sequence."""
    got = []
    for s, (_, n, _) in enumerate(b.seqs):
        js = b.slots(s)[0].tolist()
        heads = []
        for g in range(b.nkv):
            row = w[s, g].tolist()
            val = lambda j: (row[j] if j < len(row) else 0.0) + 0.0  # noqa: E731
            must = {j for j in js if j < sink or j >= n - recent}
            rest = sorted((j for j in js if j not in must), key=lambda j: (math.isnan(val(j)), 0 if math.isnan(val(j)) else -val(j), j))
            heads.append(sorted(list(must) + rest[:max(0, min(budget, len(js)) - len(must))]))
        got.append(heads)
    return got


@pytest.mark.parametrize("budget,sink,recent", [(64, 4, 16), (100, 0, 0), (1, 0, 0), (1, 1, 0), (1, 0, 1), (37, 37, 0),
                                                (200, 0, 200), (5000, 4, 100), (0, 0, 0)])
@pytest.mark.parametrize("hd,page,layout", [(128, 64, "head"), (64, 16, "token"), (128, 32, "mixed")])
def test_evict(budget, sink, recent, hd, page, layout):
    seqs = [(0, 500, ()), (0, 1, ()), (0, 0, ()), (0, 64, ()), (0, 301, (0, 2)), (0, 150, tuple(range(-(-150 // page)))),
            (0, 1500, (1,)), (0, 99, ())]
    per = max(1, -(-budget // page))
    b = Paged(seqs, 4, 2, hd, page, layout, seed=budget, extra_pages=per * len(seqs) + 2)
    dst = torch.tensor(b.spare[:per * len(seqs)], dtype=torch.int32, device=DEV).view(len(seqs), per)
    if per > 1:
        dst[3, 1] = -1  # an unmapped destination
    g = torch.Generator(device=DEV).manual_seed(budget)
    w = torch.rand(len(seqs), 2, 1400, generator=g, device=DEV)  # narrower than the longest sequence
    w[0, 0, :400] = 0.5        # equal weights: the lowest slots
    w[0, 1, 100:300] = 0.0
    w[0, 1, 150:160] = -0.0    # equal to 0
    w[3, 0, 10:20] = math.nan  # last
    w[3, 1, 5], w[3, 1, 7] = math.inf, -1.0
    before = [t.clone() for t in (b.k, b.v)]
    kept, dw, n = evict(b, w, budget, sink, recent, dst)
    ref = evict_reference(b, w, budget, sink, recent)
    k_exp, v_exp = (t.clone() for t in before)
    for s, heads in enumerate(ref):
        assert int(n[s]) == len(heads[0])
        for h, js in enumerate(heads):
            assert kept[s, h, :len(js)].tolist() == js, (s, h)
            assert bool((kept[s, h, len(js):] == -7).all()) and bool((dw[s, h, len(js):] == -7).all())
            if not js:
                continue
            j = torch.tensor(js, device=DEV)
            exp = torch.where(j < 1400, w[s, h, j.clamp(max=1399)], 0.0)
            assert bool(((dw[s, h, :len(js)] == exp) | exp.isnan()).all())
            to = torch.arange(len(js), device=DEV)
            on = dst[s, to // page] >= 0
            src, at = b.table[s, j // page].long()[on], dst[s, to // page].long()[on]
            for t, e in ((before[0], k_exp), (before[1], v_exp)):
                e[at, h, (to % page)[on]] = t[src, h, (j % page)[on]]
    for t, e in ((b.k, k_exp), (b.v, v_exp)):
        assert bool(((t == e) | (t.isnan() & e.isnan())).all())
    k2, _, n2 = evict(b, w, budget, sink, recent, dst, dst_weights=False)
    assert torch.equal(k2, kept) and torch.equal(n2, n)


@pytest.mark.parametrize("n,budget", [(40_000, 10_000), (40_000, 39_999), (70_001, 1), (20_000, 20_000)])
def test_evict_long(n, budget):
    page = 128
    per = -(-budget // page)
    b = Paged([(0, n, ()), (0, n // 3, ())], 2, 1, 64, page, seed=n, extra_pages=2 * per + 1)
    dst = torch.tensor(b.spare[:2 * per], dtype=torch.int32, device=DEV).view(2, per)
    w = (torch.rand(2, 1, n, device=DEV) * 50).floor() / 50  # many equal weights
    kept, dw, got = evict(b, w, budget, min(2, budget), min(100, budget // 4), dst)
    for s, heads in enumerate(evict_reference(b, w, budget, min(2, budget), min(100, budget // 4))):
        assert kept[s, 0, :int(got[s])].tolist() == heads[0]
        j = torch.tensor(heads[0], device=DEV)
        to = torch.arange(len(j), device=DEV)
        assert torch.equal(dw[s, 0, :len(j)], w[s, 0, j])
        assert torch.equal(b.v[dst[s, to // page].long(), 0, to % page], b.v[b.table[s, j // page].long(), 0, j % page])


# ── all of them, as a serving loop uses them ──


def test_serving_loop():
    """Two sequences: prompts in chunks, decode steps, then eviction to a budget, then more steps at positions that
    the cache no longer counts.  Every step's attention is checked against the cache as it stands, the cache against
    the rows it was given."""
    nq, nkv, hd, page, budget = 8, 4, 128, 16, 48
    L, G = bd.capi(), nq // nkv
    n_pages = 64
    k, v = (torch.full((n_pages, nkv, page, hd), math.nan, dtype=torch.float16, device=DEV) for _ in range(2))
    free = list(np.random.default_rng(1).permutation(n_pages))
    own = [[], []]
    length, pos = [0, 0], [0, 0]
    angle = torch.arange(512, device=DEV, dtype=F64)[:, None] * 1e4 ** (-torch.arange(hd // 2, device=DEV, dtype=F64) / 64)
    cos, sin = angle.cos().float(), angle.sin().float()
    g = torch.Generator(device=DEV).manual_seed(5)
    weights = torch.zeros(2, nkv, 256, device=DEV)
    work = torch.zeros(L.b2_attention_paged_workspace(2, 64, nq, nkv, hd), dtype=torch.uint8, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    kept_rows = [[torch.zeros(0, hd, dtype=F64, device=DEV)] * nkv for _ in range(2)]  # K the cache should hold

    def ints(a):
        return torch.tensor(a, dtype=torch.int32, device=DEV)

    for step, news in enumerate([(30, 1), (40, 25), (1, 1), (1, 0), "evict", (1, 1), (5, 1), (1, 60), "evict", (1, 1)]):
        if news == "evict":
            table = ints([o + [-1] * (16 - len(o)) for o in own])
            per = -(-budget // page)
            fresh = [[free.pop() for _ in range(per)] for _ in range(2)]
            kv = bd.B2PagedKV(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), n_pages, page, 2, 16,
                              table.data_ptr(), (kl := ints(length)).data_ptr(), None)
            kept = torch.zeros(2, nkv, budget, dtype=torch.int32, device=DEV)
            new_len, to = ints([0, 0]), ints(fresh)
            moved = torch.zeros(2, nkv, budget, device=DEV)
            bd.check(L.b2_kv_evict_paged(ctypes.byref(kv), nkv, hd, weights.data_ptr(), 256, budget, 4, 16, to.data_ptr(),
                                         per, kept.data_ptr(), moved.data_ptr(), new_len.data_ptr(), stream()))
            length = new_len.tolist()
            assert length == [min(budget, n) for n in kl.tolist()]
            weights.zero_()
            for s in range(2):
                free.extend(own[s])
                own[s] = fresh[s][:-(-length[s] // page)]
                free.extend(fresh[s][len(own[s]):])
                weights[s, :, :length[s]] = moved[s, :, :length[s]]
                for h in range(nkv):
                    kept_rows[s][h] = kept_rows[s][h][kept[s, h, :length[s]].long()]
            continue
        for s in range(2):
            length[s] += news[s]
            while len(own[s]) * page < length[s]:
                own[s].append(free.pop())
        M = sum(news)
        qkv = torch.randn(M, (nq + 2 * nkv) * hd, generator=g, device=DEV)
        at = ints(list(range(pos[0], pos[0] + news[0])) + list(range(pos[1], pos[1] + news[1])))
        table, kl, qs = ints([o + [-1] * (16 - len(o)) for o in own]), ints(length), ints([0, news[0], M])
        kv = bd.B2PagedKV(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), n_pages, page, 2, 16,
                          table.data_ptr(), kl.data_ptr(), qs.data_ptr())
        b = Paged([(news[s], length[s], ()) for s in range(2)], nq, nkv, hd, page, extra_pages=0)
        b.k, b.v, b.n_pages, b.table, b.work, b.err = k, v, n_pages, table, work, err
        b.q16 = torch.zeros(M, nq * hd, dtype=torch.float16, device=DEV)
        bd.check(L.b2_qk_rope_kv_paged(b.q16.data_ptr(), nq * hd, qkv.data_ptr(), qkv.stride(0), M, nq, nkv, hd, None, None,
                                       1e-6, cos.data_ptr(), sin.data_ptr(), 512, 1, at.data_ptr(), ctypes.byref(kv),
                                       stream()))
        z, _, _ = rope_reference(b, qkv, None, None, cos, sin, at, 1)
        out, lse = b.attend()
        check_attention(b, out, lse)
        before = weights.clone()
        b.weigh(lse, weights, weights)
        check_weights(b, lse, before, weights, 256, 0.0)
        for s in range(2):
            r = slice(int(b.starts[s]), int(b.starts[s]) + news[s])
            _, K, _ = b.slots(s)
            for h in range(nkv):
                kept_rows[s][h] = torch.cat([kept_rows[s][h], z[r, nq + h]])
                assert bool(((K[:, h] - kept_rows[s][h]).abs() <= U * kept_rows[s][h].abs() + 2.0 ** -18).all())
            pos[s] += news[s]
    assert err.item() == 0


# ── what one row may see and another may not, and sizes past the usual ──


@pytest.mark.parametrize("nq,nkv,hd,page", [(4, 2, 128, 64), (2, 2, 64, 16), (16, 1, 128, 32), (3, 1, 64, 128)])
@pytest.mark.parametrize("q", [2, 5, 16, 40, 140, 300])
def test_attention_non_finite_values_of_later_rows(nq, nkv, hd, page, q):
    """An infinite or NaN V (an overflow in the cache) reaches the rows that see it, in its column of its kv head,
    and no row before it."""
    G = nq // nkv
    seqs = [(q, 200 + q, ()), (q, q, ()), (q, q + 31, (0,)), (1, 80, ())]
    b = Paged(seqs, nq, nkv, hd, page, seed=q)
    hit = torch.zeros(b.M, nq, hd, dtype=torch.bool, device=DEV)
    clean, _ = b.attend()
    kept = b.v.clone()
    for s, row, d, bad in [(0, 1, 3, math.inf), (0, q - 1, 3, -math.inf), (0, q // 2, hd - 1, math.nan),
                           (1, 0, 9, math.inf), (1, q - 1, 10, math.nan), (2, q // 3, 0, -math.inf), (3, 0, 1, math.nan)]:
        j, h = seqs[s][1] - seqs[s][0] + row, (row + d) % nkv
        if j // page in seqs[s][2]:
            continue
        b.v[b.table[s, j // page], h, j % page, d] = bad
        a = int(b.starts[s])
        hit[a + row:a + seqs[s][0], h * G:(h + 1) * G, d] = True
    out, lse = b.attend()
    b.v.copy_(kept)
    hit = hit.view(b.M, -1)
    assert not bool(out[hit].isfinite().any()) and bool(out[~hit].isfinite().all())
    check_attention(b, torch.where(hit, clean, out), lse)


@pytest.mark.parametrize("q", [1, 6, 40, 140, 300])
def test_weights_non_finite_keys(q):
    """K that is not finite at one slot gives that slot's weight, and no other's, whoever sees it."""
    b = Paged([(q, 180 + q, ()), (q, q + 5, ())], 4, 2, 128, 64, seed=q)
    _, lse = b.attend()
    ldw = 200 + q
    out = b.weigh(lse, None, torch.zeros(2, 2, ldw, device=DEV))
    check_weights(b, lse, None, out, ldw, 0.0)
    where = [(0, 0, 180 + q // 2), (1, 1, q + 4), (0, 1, 17)]
    for s, h, j in where:
        b.k[b.table[s, j // 64], h, j % 64, 5] = math.nan
    got = b.weigh(lse, None, torch.zeros(2, 2, ldw, device=DEV))
    for s, h, j in where:
        assert math.isnan(got[s, h, j].item())
        got[s, h, j] = out[s, h, j]
    assert torch.equal(got, out)


def test_weights_of_rows_without_weight():
    """Rows whose lse is -infinity give exactly nothing, whatever their scores."""
    b = Paged([(150, 400, ()), (3, 200, ())], 4, 2, 64, 32, seed=2)
    none = torch.full((b.M, b.nq), -math.inf, device=DEV)
    out = b.weigh(none, None, torch.full((2, 2, 400), 7.0, device=DEV))
    assert not bool(out[0].any()) and not bool(out[1, :, :200].any())


@pytest.mark.parametrize("G,seqs_n,q", [(16, 100, 400), (8, 900, 33), (1, 1, 2500)])
def test_attention_many_chunks(G, seqs_n, q):
    """More tiles than the chunk kernel keeps places for, many sequences of chunks, one head of its own."""
    b = Paged([(q, q + (s * 7) % 50, ()) for s in range(seqs_n)], G, 1, 64, 64, seed=G)
    out, lse = b.attend()
    check_attention(b, out, lse)
    prev = torch.rand(seqs_n, 1, q + 50, device=DEV)
    w = b.weigh(lse, prev, prev.clone())
    for s in range(0, seqs_n, 37):  # every row gives each of its heads one
        n = b.seqs[s][1]
        given = (w - prev)[s, 0, :n].to(F64).sum() / (q * G)
        assert abs(float(given) - 1) < 2.0 ** -10


@pytest.mark.parametrize("seqs_n,n", [(150, 60_000), (1, 400_000)])
def test_evict_more_slots_than_fit(seqs_n, n):
    """More slots than the CTAs of one kv head hold keys for."""
    page, budget = 128, 5000
    per = -(-budget // page)
    b = Paged([(0, n, ())] + [(0, 40 + s, ()) for s in range(seqs_n - 1)], 1, 1, 64, page, seed=1,
              extra_pages=per * seqs_n + 1)
    dst = torch.tensor(b.spare[:per * seqs_n], dtype=torch.int32, device=DEV).view(seqs_n, per)
    w = (torch.rand(seqs_n, 1, n, device=DEV) * 1000).floor()
    kept, dw, got = evict(b, w, budget, 3, 500, dst)
    for s, heads in enumerate(evict_reference(b, w, budget, 3, 500)):
        assert kept[s, 0, :int(got[s])].tolist() == heads[0]
        j = torch.tensor(heads[0], device=DEV)
        to = torch.arange(len(j), device=DEV)
        assert torch.equal(dw[s, 0, :len(j)], w[s, 0, j])
        assert torch.equal(b.k[dst[s, to // page].long(), 0, to % page], b.k[b.table[s, j // page].long(), 0, j % page])


@pytest.mark.parametrize("q", [1, 90])
def test_pages_far_apart(q):
    """Pages of one layer in a pool whose offsets pass 32 bits."""
    b = Paged([(q, 300 + q, ()), (q, q + 20, ())], 4, 2, 128, 64, seed=q, extra_pages=20)
    stride, n = 1 << 28, b.n_pages
    big = torch.empty(n * stride, dtype=torch.float16, device=DEV)
    k, v = (big.as_strided((n, 2, 64, 128), (stride, 64 * 128, 128, 1), at) for at in (0, stride // 2))
    k.copy_(b.k)
    v.copy_(b.v)
    assert int(b.table.max()) * stride > 1 << 32  # elements
    b.k, b.v = k, v
    out, lse = b.attend()
    check_attention(b, out, lse)
    w = b.weigh(lse, None, torch.zeros(2, 2, 400, device=DEV))
    check_weights(b, lse, None, w, 400, 0.0)
    qkv = torch.randn(b.M, (4 + 2 * 2) * 128, device=DEV)
    pos = torch.arange(b.M, dtype=torch.int32, device=DEV)
    cos, sin = torch.ones(b.M, 64, device=DEV), torch.zeros(b.M, 64, device=DEV)
    bd.check(bd.capi().b2_qk_rope_kv_paged(b.q16.data_ptr(), b.q16.stride(0), qkv.data_ptr(), qkv.stride(0), b.M, 4, 2,
                                           128, None, None, 1e-6, cos.data_ptr(), sin.data_ptr(), b.M, 0, pos.data_ptr(),
                                           ctypes.byref(b.kv()), stream()))
    for s in range(2):
        for i in (0, q - 1):
            j, m = b.seqs[s][1] - q + i, int(b.starts[s]) + i
            at = int(b.table[s, j // 64])
            assert torch.equal(b.k[at, :, j % 64], qkv[m, 512:768].half().view(2, 128))
            assert torch.equal(b.v[at, :, j % 64], qkv[m, 768:].half().view(2, 128))
    dst = torch.tensor(b.spare[:8], dtype=torch.int32, device=DEV).view(2, 4)
    kept, _, got = evict(b, w, 200, 4, 16, dst)
    for s in range(2):
        m = int(got[s])
        assert m == min(200, b.seqs[s][1])
        to = torch.arange(m, device=DEV)
        for h in range(2):
            j = kept[s, h, :m].long()
            assert torch.equal(b.v[dst[s, to // 64].long(), h, to % 64], b.v[b.table[s, j // 64].long(), h, j % 64])


def test_captured_step():
    """Append, attention and weights captured as one step and replayed on other rows and lengths, and the eviction
    after it: what the calls give one by one."""
    nq, nkv, hd, page = 8, 2, 128, 32
    b = Paged([(1, 100, ()), (70, 200, ()), (1, 333, ())], nq, nkv, hd, page, seed=3, extra_pages=16)
    M = b.M
    qkv = torch.randn(M, (nq + 2 * nkv) * hd, device=DEV)
    pos = torch.arange(M, dtype=torch.int32, device=DEV)
    angle = torch.rand(M, hd // 2, device=DEV) * 6
    cos, sin = angle.cos(), angle.sin()
    out = torch.zeros(M, nq * hd, dtype=torch.float16, device=DEV)
    lse = torch.zeros(M, nq, device=DEV)
    w = torch.zeros(3, nkv, 340, device=DEV)
    dst = torch.tensor(b.spare[:12], dtype=torch.int32, device=DEV).view(3, 4)
    kept, moved = torch.zeros(3, nkv, 120, dtype=torch.int32, device=DEV), torch.zeros(3, nkv, 120, device=DEV)
    new = torch.zeros(3, dtype=torch.int32, device=DEV)
    kv, L = b.kv(), bd.capi()

    def step():
        st = torch.cuda.current_stream().cuda_stream
        bd.check(L.b2_qk_rope_kv_paged(b.q16.data_ptr(), b.q16.stride(0), qkv.data_ptr(), qkv.stride(0), M, nq, nkv, hd,
                                       None, None, 1e-6, cos.data_ptr(), sin.data_ptr(), M, 1, pos.data_ptr(),
                                       ctypes.byref(kv), st))
        bd.check(L.b2_attention_paged(out.data_ptr(), lse.data_ptr(), b.q16.data_ptr(), b.q16.stride(0), M, M, nq, nkv,
                                      hd, ctypes.byref(kv), b.work.data_ptr(), b.err.data_ptr(), st))
        bd.check(L.b2_attention_paged_weights(w.data_ptr(), w.data_ptr(), 340, b.q16.data_ptr(), b.q16.stride(0),
                                              lse.data_ptr(), M, M, nq, nkv, hd, ctypes.byref(kv), b.err.data_ptr(), st))
        bd.check(L.b2_kv_evict_paged(ctypes.byref(kv), nkv, hd, w.data_ptr(), 340, 120, 4, 16, dst.data_ptr(), 4,
                                     kept.data_ptr(), moved.data_ptr(), new.data_ptr(), st))

    results = (out, lse, w, kept, moved, new, b.k, b.v)
    start = [t.clone() for t in results]
    step()
    torch.cuda.synchronize()
    assert b.err.item() == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        step()
    for news in ([1, 70, 1], [70, 1, 1], [0, 30, 42], [2, 2, 2]):
        lens = [n + q for n, q in zip((60, 40, 200), news)]
        b.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        b.q_start.copy_(torch.tensor([0, *np.cumsum(news)], dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, device=DEV))
        got = []
        for run in (step, graph.replay):
            for t, s in zip(results, start):
                t.copy_(s)
            run()
            torch.cuda.synchronize()
            got.append([t.clone() for t in results])
        for a, c in zip(*got):
            assert torch.equal(a.nan_to_num(9.0), c.nan_to_num(9.0))
    assert b.err.item() == 0


def test_calls_at_once():
    """Calls with workspaces of their own on two streams, over the same pages."""
    b = Paged([(1, 900, ()), (200, 700, ()), (1, 50, ()), (9, 300, ())], seed=6)
    out, lse = b.attend()
    check_attention(b, out, lse)
    w = b.weigh(lse, None, torch.zeros(4, b.nkv, 900, device=DEV))
    sides = [torch.cuda.Stream() for _ in range(2)]
    works = [b.work, torch.zeros_like(b.work)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for st, work in zip(sides, works):
            with torch.cuda.stream(st):
                b.work = work
                o, l = b.attend(st=st.cuda_stream)
                x = torch.zeros_like(w)
                bd.check(bd.capi().b2_attention_paged_weights(
                    x.data_ptr(), None, 900, b.q16.data_ptr(), b.q16.stride(0), l.data_ptr(), b.M, b.max_q, b.nq, b.nkv,
                    b.hd, ctypes.byref(b.kv()), b.err.data_ptr(), st.cuda_stream))
                got.append((o, l, x))
    torch.cuda.synchronize()
    for o, l, x in got:
        assert torch.equal(o, out) and torch.equal(l, lse) and torch.equal(x, w)


@pytest.mark.parametrize("q", [2, 6, 40, 140, 300])
def test_weights_of_a_row_that_is_not_a_number(q):
    """A row whose sum is NaN or infinite reaches the slots that it sees and no others."""
    b = Paged([(q, 180 + q, ()), (q, q + 5, ())], 4, 2, 64, 64, seed=q)
    _, lse = b.attend()
    ldw = 200 + q
    out = b.weigh(lse, None, torch.zeros(2, 2, ldw, device=DEV))
    row = q // 2
    lse[row, 0] = math.nan                 # sequence 0, kv head 0: slots 0 .. 180 + row
    lse[int(b.starts[1]) + row, 3] = math.nan  # sequence 1, kv head 1: slots 0 .. 5 + row
    got = b.weigh(lse, None, torch.zeros(2, 2, ldw, device=DEV))
    assert bool(got[0, 0, :181 + row].isnan().all()) and bool(got[1, 1, :6 + row].isnan().all())
    got[0, 0, :181 + row], got[1, 1, :6 + row] = out[0, 0, :181 + row], out[1, 1, :6 + row]
    assert torch.equal(got, out)


@pytest.mark.parametrize("G,q,seqs_n", [(16, 200, 1024), (2, 4, 1024), (2, 9, 64)])
def test_sequences_that_share_rows(G, q, seqs_n):
    """Row ranges that are no partition: the first sequence's rows and the caller's memory stay right, and the
    workspace serves the next call."""
    one = Paged([(q, 300 + q, ())], G, 1, 64, 64, seed=5)
    b = Paged([(0, 300 + q, ())] * seqs_n, G, 1, 64, 64, seed=6)
    b.M, b.rows, b.max_q, b.q16 = one.M, one.rows, q, one.q16
    b.k, b.v, b.n_pages = one.k, one.v, one.n_pages
    b.table = one.table.repeat(seqs_n, 1)
    b.work = torch.zeros_like(b.work)
    b.q_start = torch.tensor([0, q] * (seqs_n // 2) + [0], dtype=torch.int32, device=DEV)
    out, lse = b.attend()
    assert b.err.item() == 0 and not bool(b.work[:4096].any())
    check_attention(one, out, lse)
    w = torch.full((seqs_n, 1, 300 + q), 7.0, device=DEV)
    b.weigh(lse, None, w)
    # (not bit by bit: how many CTAs share a slot's rows, and so the order of its sum, depends on the batch)
    check_weights(one, lse, None, w[:1], 300 + q, 7.0)
    assert not bool(w[1].any())
    one.work = b.work
    check_attention(one, *one.attend())


def test_no_rows():
    """A batch whose sequences are all idle: nothing to append or attend, the weights are what they were."""
    b = Paged([(0, 100, ()), (0, 7, ())], 4, 2, 64, 16)
    L, kv = bd.capi(), b.kv()
    before = [t.clone() for t in (b.k, b.v)]
    cos = torch.ones(128, 32, device=DEV)
    bd.check(L.b2_qk_rope_kv_paged(None, 256, None, 512, 0, 4, 2, 64, None, None, 1e-6, cos.data_ptr(), cos.data_ptr(), 128,
                                   0, None, ctypes.byref(kv), stream()))
    bd.check(L.b2_attention_paged(None, None, None, 256, 0, 0, 4, 2, 64, ctypes.byref(kv), b.work.data_ptr(),
                                  b.err.data_ptr(), stream()))
    prev = torch.rand(2, 2, 100, device=DEV)
    for p, max_q in ((prev, 0), (None, 0), (prev, 64)):
        out = torch.full((2, 2, 100), 7.0, device=DEV)
        bd.check(L.b2_attention_paged_weights(out.data_ptr(), None if p is None else p.data_ptr(), 100, None, 256, None, 0,
                                              max_q, 4, 2, 64, ctypes.byref(kv), b.err.data_ptr(), stream()))
        exp = torch.zeros_like(out) if p is None else p.clone()
        exp[1, :, 7:] = 7.0
        assert torch.equal(out, exp)
    for t, e in zip((b.k, b.v), before):
        assert torch.equal(t.nan_to_num(9.0), e.nan_to_num(9.0))


def test_evict_to_nothing():
    """A budget of 0 keeps nothing and needs no place for it."""
    b = Paged([(0, 100, ()), (0, 0, ())], 4, 2, 64, 16)
    before = b.k.clone()
    w, n = torch.rand(2, 2, 100, device=DEV), torch.full((2,), 7, dtype=torch.int32, device=DEV)
    bd.check(bd.capi().b2_kv_evict_paged(ctypes.byref(b.kv()), 2, 64, w.data_ptr(), 100, 0, 0, 0, None, 0, None, None,
                                         n.data_ptr(), stream()))
    assert n.tolist() == [0, 0] and torch.equal(b.k.nan_to_num(9.0), before.nan_to_num(9.0))


@pytest.mark.parametrize("seqs", [[(90, 90, ())], [(60, 700, ())] * 3, [(300, 4000, ()), (200, 9000, ())],
                                  [(40, 2500, ()), (1, 30, ())]])
def test_attention_chunks_alone_repeat(seqs):
    """Chunks only, or next to one token: most CTAs of the kernel behind the chunks have no tile of their own and go
    straight to the merge of the chunks' pieces.  Calls one right behind the other give the same bits."""
    b = Paged(seqs, seed=len(seqs))
    out, lse = b.attend()
    check_attention(b, out, lse)
    o2, l2 = torch.empty_like(out), torch.empty_like(lse)
    kv, L = b.kv(), bd.capi()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        for _ in range(50):
            bd.check(L.b2_attention_paged(o2.data_ptr(), l2.data_ptr(), b.q16.data_ptr(), b.q16.stride(0), b.M, b.max_q, b.nq,
                                          b.nkv, b.hd, ctypes.byref(kv), b.work.data_ptr(), b.err.data_ptr(),
                                          torch.cuda.current_stream().cuda_stream))
    for _ in range(4):
        o2.fill_(7.0), l2.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o2, out) and torch.equal(l2, lse)
    assert b.err.item() == 0 and not b.work[:4096].any()


def test_mixed_steps_back_to_back():
    """Append and attention of chunks next to single tokens, 24 steps without a host in between: the kernel of the
    single tokens, which begins beside that of the chunks, finds what the append just wrote.  Same bits as the same
    steps with the GPU idle between any two calls."""
    nq, nkv, hd = 8, 4, 128
    b = Paged([(50, 130, ()), (1, 700, ()), (1, 64, ()), (3, 900, ()), (120, 1000, ())], nq, nkv, hd, 32, seed=8)
    M, L, kv = b.M, bd.capi(), b.kv()
    angle = torch.rand(M, hd // 2, device=DEV) * 6
    cos, sin = angle.cos(), angle.sin()
    pos = torch.arange(M, dtype=torch.int32, device=DEV)
    qkv = torch.randn(24, M, (nq + 2 * nkv) * hd, device=DEV)
    b.q16 = torch.zeros(M, nq * hd, dtype=torch.float16, device=DEV)
    start = [t.clone() for t in (b.k, b.v)]

    def steps(idle):
        b.k.copy_(start[0]), b.v.copy_(start[1])
        out, lse = torch.zeros(24, M, nq * hd, dtype=torch.float16, device=DEV), torch.zeros(24, M, nq, device=DEV)
        torch.cuda.synchronize()
        for i in range(24):
            bd.check(L.b2_qk_rope_kv_paged(b.q16.data_ptr(), nq * hd, qkv[i].data_ptr(), qkv.stride(1), M, nq, nkv, hd, None,
                                           None, 1e-6, cos.data_ptr(), sin.data_ptr(), M, 1, pos.data_ptr(),
                                           ctypes.byref(kv), stream()))
            if idle:
                torch.cuda.synchronize()
            bd.check(L.b2_attention_paged(out[i].data_ptr(), lse[i].data_ptr(), b.q16.data_ptr(), nq * hd, M, b.max_q, nq, nkv,
                                          hd, ctypes.byref(kv), b.work.data_ptr(), b.err.data_ptr(), stream()))
            if idle:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert b.err.item() == 0 and not b.work[:4096].any()
        return out, lse

    out, lse = steps(True)
    check_attention(b, out[-1], lse[-1])
    for _ in range(3):
        o2, l2 = steps(False)
        assert torch.equal(o2, out) and torch.equal(l2, lse)


def test_weights_back_to_back():
    """Append and weights of chunks next to single tokens, 24 steps without a host in between: the same bits as with
    the GPU idle between any two calls."""
    nq, nkv, hd = 8, 4, 128
    b = Paged([(50, 130, ()), (1, 700, ()), (1, 64, ()), (3, 900, ()), (120, 1000, ())], nq, nkv, hd, 32, seed=9)
    M, L, kv = b.M, bd.capi(), b.kv()
    angle = torch.rand(M, hd // 2, device=DEV) * 6
    cos, sin = angle.cos(), angle.sin()
    pos = torch.arange(M, dtype=torch.int32, device=DEV)
    qkv = torch.randn(24, M, (nq + 2 * nkv) * hd, device=DEV)
    b.q16 = torch.zeros(M, nq * hd, dtype=torch.float16, device=DEV)
    lse = torch.rand(M, nq, device=DEV) + 8
    start = [t.clone() for t in (b.k, b.v)]

    def steps(idle):
        b.k.copy_(start[0]), b.v.copy_(start[1])
        out = torch.zeros(24, 5, nkv, 1000, device=DEV)
        torch.cuda.synchronize()
        for i in range(24):
            bd.check(L.b2_qk_rope_kv_paged(b.q16.data_ptr(), nq * hd, qkv[i].data_ptr(), qkv.stride(1), M, nq, nkv, hd, None,
                                           None, 1e-6, cos.data_ptr(), sin.data_ptr(), M, 1, pos.data_ptr(),
                                           ctypes.byref(kv), stream()))
            if idle:
                torch.cuda.synchronize()
            b.weigh(lse, out[i - 1] if i else None, out[i])
            if idle:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return out

    out = steps(True)
    check_weights(b, lse, out[-2], out[-1], 1000, 0.0)
    for _ in range(3):
        assert torch.equal(steps(False), out)


@pytest.mark.parametrize("q", [3, 20, 60])
@pytest.mark.parametrize("G,n", [(16, (1 << 27) + 700), (16, (1 << 28) + 80), (16, 2**31 - 1), (8, (1 << 28) + 700),
                                 (2, (1 << 30) + 900), (16, (1 << 27) - 50)])
def test_weights_far_below_the_new_rows(G, n, q):
    """Slots so far before the new rows that the distance times the group passes 32 bits: every row sees them."""
    b = Paged([(q, 128 + q, ()), (1, 40, ())], G, 1, 64, 64, seed=G + q)
    b.seqs[0] = (q, n, ())  # a table of 128 slots and a bit, all of them before the first new row
    b.kv_len[0] = n
    b.table = b.table[:, :2].contiguous()
    r = slice(0, q)
    K = b.slots(0)[1][:, 0]
    x = torch.einsum("rgd,jd->rgj", b.q16[r, :G * 64].to(F64).view(q, G, 64), K) / 8
    lse = torch.full((b.M, G), 3.0, device=DEV)
    lse[:q] = x.logsumexp(-1).float()
    out = b.weigh(lse, None, torch.full((2, 1, 200), 7.0, device=DEV))
    exp = (x - lse[:q].to(F64)[..., None]).exp().sum((0, 1))
    # scores are off by (hd + 2) 2^-23 sum|q k| / 8 at most, here below 2^-13; the other roundings below 2^-15
    assert bool(((out[0, 0, :128].to(F64) - exp).abs() <= 2.0 ** -12 * exp).all())
    assert bool((out[0, 0, 128:] == 7).all()) and b.err.item() == 0


@pytest.mark.parametrize("q", [2, 20])
def test_first_page_and_a_window_far_behind(q):
    """One context of 150 million slots of which the first page and the newest are mapped: attention and weights."""
    nq, hd, page = 16, 64, 128
    n, pages = 150_000_000, -(-150_000_000 // 128)
    b = Paged([(q, 2 * page + q, ())], nq, 1, hd, page, seed=q)
    first, late = int(b.table[0, 0]), [int(x) for x in b.table[0, 1:]]
    window = (n - q) // page  # the page of the first new row
    b.k[late[0]], b.v[late[0]] = (torch.randn(1, page, hd, device=DEV).half() for _ in range(2))
    b.table = torch.full((1, pages), -1, dtype=torch.int32, device=DEV)
    b.table[0, 0], b.table[0, window - 1] = first, late[0]
    for p in range(window, pages):
        b.table[0, p] = late[1] if p == window else b.spare[p - window - 1]
    m = n - window * page  # slots cached on the pages from `window` on
    for i in range(0, m, page):
        at = int(b.table[0, window + i // page])
        for t in (b.k, b.v):
            t[at, :, :min(page, m - i)] = torch.randn(1, min(page, m - i), hd, device=DEV).half()
    b.seqs, b.kv_len[0] = [(q, n, ())], n
    near = torch.arange((window - 1) * page, n, device=DEV)
    j = torch.cat([torch.arange(page, device=DEV), near])
    at, off = b.table[0, j // page].long(), j % page
    b.slots = lambda s: (j, b.k[at, :, off].to(F64), b.v[at, :, off].to(F64))
    out, lse = b.attend()
    check_attention(b, out, lse)
    K, Q = b.slots(0)[1][:, 0], b.q16[:q, :nq * hd].to(F64).view(q, nq, hd)
    x = torch.einsum("rgd,jd->rgj", Q, K) / 8
    x = x.masked_fill((j[None] > n - q + torch.arange(q, device=DEV)[:, None])[:, None], -math.inf)
    exp = (x - lse[:q].to(F64)[..., None]).exp().sum((0, 1))
    got = b.weigh(lse, None, torch.full((1, 1, n), 7.0, device=DEV))[0, 0]
    assert bool(((got[j].to(F64) - exp).abs() <= 2.0 ** -12 * exp).all())
    assert not bool(got[page:(window - 1) * page].any()) and b.err.item() == 0


@pytest.mark.parametrize("q", [6, 60, 150, 300])
def test_weights_without_excluded_rows(q):
    """Rows that the caller excludes (lse -infinity) give nothing whatever q holds there, and slots whose K is not
    finite get nothing from them; the other rows' weights stay what they were."""
    b = Paged([(q, 180 + q, ()), (q, q + 5, ())], 4, 2, 64, 64, seed=q)
    _, lse = b.attend()
    out = torch.arange(b.M, device=DEV) % 3 == 1  # excluded rows
    out[:min(q, 140)] |= q >= 150                 # a whole tile of them
    lse[out] = -math.inf
    ldw = 200 + q
    exp = b.weigh(lse, None, torch.zeros(2, 2, ldw, device=DEV))
    check_weights(b, lse, None, exp, ldw, 0.0)
    b.q16[out, :256] = math.nan
    assert torch.equal(b.weigh(lse, None, torch.zeros(2, 2, ldw, device=DEV)), exp)
    b.q16[out, :256] = math.inf
    assert torch.equal(b.weigh(lse, None, torch.zeros(2, 2, ldw, device=DEV)), exp)
    b.q16[out, :256] = 1.0
    lse[:q] = -math.inf  # all of sequence 0
    b.k[b.table[0, 1], :, 3], b.k[b.table[0, 0], 1, 7, 5] = math.inf, math.nan
    assert not bool(b.weigh(lse, None, torch.full((2, 2, ldw), 7.0, device=DEV))[0, :, :180 + q].any())


def test_evict_arrays_side_by_side():
    """The arrays that an eviction reads and writes one right behind the other: no overlap, no refusal."""
    b = Paged([(0, 100, ()), (0, 60, ())], 2, 1, 64, 16, extra_pages=8)
    sizes = [2 * 100, 2 * 32, 2 * 32, 2, 2 * 7, 2, 2 * 2]  # weights, kept, moved weights, new_len, table, kv_len, dst
    at = [sum(sizes[:i]) for i in range(len(sizes))]
    pool = torch.zeros(sum(sizes), dtype=torch.int32, device=DEV)
    w, kept, dw, new, table, kl, dst = (pool[a:a + n] for a, n in zip(at, sizes))
    w.view(torch.float32).copy_(torch.rand(200, device=DEV))
    table.copy_(b.table.flatten()), kl.copy_(b.kv_len), dst.copy_(torch.tensor(b.spare[:4]))
    ref = evict_reference(b, w.view(torch.float32).view(2, 1, 100), 32, 2, 5)
    kv = b.kv()
    kv.page_table, kv.kv_len = table.data_ptr(), kl.data_ptr()
    bd.check(bd.capi().b2_kv_evict_paged(ctypes.byref(kv), 1, 64, w.data_ptr(), 100, 32, 2, 5, dst.data_ptr(), 2,
                                         kept.data_ptr(), dw.data_ptr(), new.data_ptr(), stream()))
    assert new.tolist() == [32, 32] and kept.view(2, 32).tolist() == [ref[0][0], ref[1][0]]
    assert torch.equal(dw.view(torch.float32).view(2, 32),
                       torch.stack([w.view(torch.float32)[s * 100:][kept.view(2, 32)[s].long()] for s in range(2)]))


def test_evict_budget_of_any_size():
    """A budget far beyond the slots there are (rows of kept as long as an int counts) keeps them all."""
    budget = 2**31 - 1
    b = Paged([(0, 500, (1,))], 2, 1, 64, 16, extra_pages=40)
    kept = torch.empty(budget, dtype=torch.int32, device=DEV)
    kept[:600] = -7
    dst = torch.tensor([b.spare[:32]], dtype=torch.int32, device=DEV)
    w, n = torch.rand(1, 1, 500, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    bd.check(bd.capi().b2_kv_evict_paged(ctypes.byref(b.kv()), 1, 64, w.data_ptr(), 500, budget, 4, 2**31 - 100, dst.data_ptr(),
                                         32, kept.data_ptr(), None, n.data_ptr(), stream()), "b2_kv_evict_paged")
    j = b.slots(0)[0]
    assert int(n) == 484 and torch.equal(kept[:484], j.int()) and bool((kept[484:600] == -7).all())
    to = torch.arange(484, device=DEV)
    for t in (b.k, b.v):
        assert torch.equal(t[dst[0, to // 16].long(), 0, to % 16], t[b.table[0, j // 16].long(), 0, j % 16])


def test_evict_sink_and_recent_count_unmapped_slots():
    """The first and last slots are kept by their place, not as the first and last that are mapped."""
    b = Paged([(0, 320, (0, 4))], 2, 1, 64, 64, extra_pages=4)  # slots 64 .. 255 are mapped
    w = torch.arange(320, 0, -1, device=DEV, dtype=torch.float32).view(1, 1, 320)
    w[0, 0, 64:70], w[0, 0, 250:256] = -1.0, -2.0
    dst = torch.tensor([b.spare[:3]], dtype=torch.int32, device=DEV)
    for sink, recent, first, last in ((4, 64, (), ()), (66, 64, (64, 65), ()), (4, 66, (), (254, 255)), (67, 67, (64, 65, 66), (253, 254, 255))):
        kept, _, n = evict(b, w, 150, sink, recent, dst)
        rest = [j for j in range(70, 250)][:150 - len(first) - len(last)]
        assert int(n) == 150 and kept[0, 0].tolist() == [*first, *rest, *last]


@pytest.mark.parametrize("nq,nkv,qs", [(4, 2, (15, 16, 17, 20, 21, 31, 32, 33)), (16, 1, (1, 2, 3, 4, 5)), (5, 1, (6, 7, 8, 9, 13))])
def test_weights_around_the_kernels_border(nq, nkv, qs):
    """Sequences on both sides of where the two kernels divide them, in one call and one by one."""
    seqs = [(q, 200 + 7 * q, (1,)) for q in qs]
    b = Paged(seqs, nq, nkv, 128, 32, seed=nq)
    _, lse = b.attend()
    ldw = 450
    check_weights(b, lse, None, b.weigh(lse, None, torch.full((len(seqs), nkv, ldw), 0.0, device=DEV)), ldw, 0.0)
    for q in qs:
        one = Paged([(q, 200 + 7 * q, ())], nq, nkv, 128, 32, seed=q)
        _, lse = one.attend()
        check_weights(one, lse, None, one.weigh(lse, None, torch.full((1, nkv, ldw), 0.0, device=DEV)), ldw, 0.0)


# ── waits that run out ──


@pytest.mark.parametrize("limit", [-1, 0, 2, 8])
@pytest.mark.parametrize("hd,seqs", [(128, [(1, 3000, ())] * 40), (64, [(2, 900 + 50 * i, (1,)) for i in range(30)]),
                                     (128, [(300, 2300, ()), (70, 900, ()), (300, 300, ())]),
                                     (64, [(500, 1500, ()), (1, 2000, ()), (90, 90, ()), (3, 700, ())])])
def test_waits_that_run_out(hd, seqs, limit, monkeypatch):
    """With a limit of a few polls ordinary waits run out: the kernels return by themselves, err tells it, what is not
    theirs stays, and with work and err zeroed the next call is right.  A call whose waits were all short enough is
    right too."""
    b = Paged(seqs, 8, 4, hd, 32, seed=hd, tail=2)
    out, lse = b.attend()
    check_attention(b, out, lse)
    ldw = max(n for _, n, _ in seqs)
    w = b.weigh(lse, None, torch.full((len(seqs), 4, ldw), 7.0, device=DEV))
    pools = [t.clone() for t in (b.k, b.v)]
    gave_up = [0, 0]
    for _ in range(3):
        torch.full((256 << 20,), 1, dtype=torch.uint8, device=DEV)  # K and V out of L2
        monkeypatch.setenv("B2_PAGED_POLL_LIMIT", str(limit))
        o2, l2 = b.attend()
        torch.cuda.synchronize()
        if b.err.item():
            gave_up[0] += 1
            assert bool((o2[b.rows:] == 7).all()) and bool((l2[b.rows:] == 7).all())
        else:
            assert torch.equal(o2, out) and torch.equal(l2, lse)
        b.work.zero_(), b.err.zero_()
        torch.full((256 << 20,), 1, dtype=torch.uint8, device=DEV)
        w2 = b.weigh(lse, None, torch.full_like(w, 7.0))
        torch.cuda.synchronize()
        if b.err.item():
            gave_up[1] += 1
            for s, (_, n, _) in enumerate(seqs):
                assert bool((w2[s, :, n:] == 7).all())
        else:
            assert torch.equal(w2, w)
        b.err.zero_()
        monkeypatch.delenv("B2_PAGED_POLL_LIMIT")
        o2, l2 = b.attend()
        assert torch.equal(o2, out) and torch.equal(l2, lse)
        assert torch.equal(b.weigh(lse, None, torch.full_like(w, 7.0)), w)
        assert b.err.item() == 0 and not b.work[:4096].any()
    for t, e in zip((b.k, b.v), pools):
        assert torch.equal(t.nan_to_num(9.0), e.nan_to_num(9.0))
    if limit < 0:  # a poll takes 1.5 us, and the attention's first copies from HBM take longer
        assert gave_up[0]


@pytest.mark.parametrize("q", [1, 5, 80])
def test_pages_that_sequences_share(q):
    """A common prefix: four sequences whose tables begin with the same pages, each with rows of its own behind."""
    b = Paged([(q, 160 + q + 9 * i, ()) for i in range(4)], 4, 2, 64, 32, seed=q, extra_pages=20)
    b.table[1:, :5] = b.table[0, :5]
    out, lse = b.attend()
    check_attention(b, out, lse)
    ldw = 200 + q
    w = b.weigh(lse, None, torch.zeros(4, 2, ldw, device=DEV))
    check_weights(b, lse, None, w, ldw, 0.0)
    dst = torch.tensor(b.spare[:16], dtype=torch.int32, device=DEV).view(4, 4)
    before = [t.clone() for t in (b.k, b.v)]
    kept, _, n = evict(b, w, 100, 4, 20, dst)
    for s, heads in enumerate(evict_reference(b, w, 100, 4, 20)):
        for h, js in enumerate(heads):
            assert int(n[s]) == 100 and kept[s, h].tolist() == js
            j, to = torch.tensor(js, device=DEV), torch.arange(100, device=DEV)
            for t, e in zip((b.k, b.v), before):
                assert torch.equal(t[dst[s, to // 32].long(), h, to % 32], e[b.table[s, j // 32].long(), h, j % 32])


@pytest.mark.parametrize("norms", ["q", "k", "both"])
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("nq,nkv,hd,rows", [(16, 8, 128, 1300), (5, 5, 64, 2700), (3, 1, 128, 5000), (7, 1, 64, 30)])
def test_append_many_rows(nq, nkv, hd, rows, style, norms):
    """More rows than warps (each takes a whole row then), norm weights of q or of k alone, angle tables at an odd
    address; K, V and q of every row against the 64-bit form."""
    b = Paged([(rows // 2, rows // 2 + 40, ()), (1, 900, ()), (rows - rows // 2 - 1, rows + 3, ())], nq, nkv, hd, 32, seed=rows)
    g = torch.Generator(device=DEV).manual_seed(rows)
    qkv = torch.randn(b.M, (nq + 2 * nkv) * hd, generator=g, device=DEV) * 2
    qn, kn = (1 + 0.2 * torch.randn(hd, generator=g, device=DEV) if norms in (n, "both") else None for n in "qk")
    angle = torch.rand(700, hd // 2, generator=g, device=DEV, dtype=F64) * 6.3
    tables = []
    for t in (angle.cos(), angle.sin()):
        pool = torch.zeros(t.numel() + 1, device=DEV)
        tables.append(pool[1:].view(700, hd // 2).copy_(t))
    pos = torch.randint(0, 700, (b.M,), generator=g, device=DEV, dtype=torch.int32)
    q16 = torch.full((b.M, nq * hd), 7.0, dtype=torch.float16, device=DEV)
    bd.check(bd.capi().b2_qk_rope_kv_paged(
        q16.data_ptr(), nq * hd, qkv.data_ptr(), qkv.stride(0), b.M, nq, nkv, hd, None if qn is None else qn.data_ptr(),
        None if kn is None else kn.data_ptr(), 1e-6, tables[0].data_ptr(), tables[1].data_ptr(), 700, style, pos.data_ptr(),
        ctypes.byref(b.kv()), stream()), "b2_qk_rope_kv_paged")
    z, v, mag = rope_reference(b, qkv, qn, kn, *tables, pos, style)
    tol = U * z.abs() + 16 * 2.0 ** -24 * mag + 2.0 ** -25  # as in test_append
    assert bool(((q16.to(F64).view(b.M, nq, hd) - z[:, :nq]).abs() <= tol[:, :nq]).all())
    for s, (q, n, _) in enumerate(b.seqs):
        j = torch.arange(n - q, n, device=DEV)
        r = slice(int(b.starts[s]), int(b.starts[s]) + q)
        at = b.table[s, j // 32].long()
        assert bool(((b.k[at, :, j % 32].to(F64) - z[r, nq:]).abs() <= tol[r, nq:]).all())
        assert torch.equal(b.v[at, :, j % 32], v[r].half())
