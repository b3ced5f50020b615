"""sjh_attn_scored against float64, at the edges of its tiles, lists and masks.

The bound.  A score is off by ds: (Dh + 3) 2^-24 scale sum |q k| of its product,
8 2^-24 of its own size for the scalings and roundings after it, cap 2e-6 for
the cap (a polynomial within 6e-7, or exponential, reciprocal and one
cancellation of an ulp of the cap each), 4 2^-24 of the bias.  A weight is then
off by a factor 1 + d, |d| <= 2 ds (its score and the softmax offset's) + 16
2^-24 (exponential, offset, rescales), and bf16's P rounds by 2^-8 more; the sum
of the weights adds the same rounded ones, so o is off by |d| sum_j w_j |v_j -
o|, to first order (1.05 covers the rest), plus 2 (n + 8) 2^-24 sum_j w_j |v_j|
for the sums and their joining, plus the output's rounding."""
import ctypes as C

import numpy as np
import pytest

import snapjudge_amd as sj

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def ints(x):
    return torch.from_numpy(np.asarray(x, np.int32)).cuda()


class Case:
    """Tensors of a batch: sequences back to back with a gap row between, all
    rows of o preset to 7."""

    def __init__(self, ql, kl, H=2, Hkv=0, Dh=64, dtype="bf16", cap=0.0, slopes=None, window=0, causal=False, prefix=None, docs=None,
                 q_pos=None, scale=0.0, seed=0, amp=1.0):
        self.__dict__.update({k: v for k, v in locals().items() if k != "self"})
        self.Hkv = Hkv or H
        g = torch.Generator(device="cuda").manual_seed(seed + 7 * len(kl) + sum(kl))
        td = torch.bfloat16 if dtype == "bf16" else torch.float32
        self.ql, self.kl = list(ql), list(kl)
        self.qs = np.cumsum([0] + [n + 1 for n in ql])[:-1]
        self.ks = np.cumsum([0] + [n + 2 for n in kl])[:-1]
        self.nq, self.nk = int(sum(ql) + len(ql)), int(sum(kl) + 2 * len(kl))
        R = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.q = (amp * R(self.nq, H, Dh)).to(td)
        self.k, self.v = R(self.nk, self.Hkv, Dh).to(td), R(self.nk, self.Hkv, Dh).to(td)
        self.o = torch.full((self.nq, H, Dh), 7.0, dtype=td, device="cuda")
        self.q_pos = [k - q for q, k in zip(ql, kl)] if q_pos is None else q_pos
        self.sl = None if slopes is None else torch.tensor(slopes, dtype=torch.float32, device="cuda")
        self.kd = self.qd = None
        if docs is not None:  # docs(b, j): document of key j
            kd, qd = np.full(self.nk, -9, np.int32), np.full(self.nq, -8, np.int32)
            for b, (q, k) in enumerate(zip(ql, kl)):
                kd[self.ks[b]:self.ks[b] + k] = [docs(b, j) for j in range(k)]
                qd[self.qs[b]:self.qs[b] + q] = [docs(b, self.q_pos[b] + i) for i in range(q)]
            self.kd, self.qd = kd, qd

    def args(self, **over):
        P = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.keep = [ints(self.qs), ints(self.ql), ints(self.ks), ints(self.kl), ints(self.q_pos)]
        self.keep += [None if self.prefix is None else ints(self.prefix), None if self.qd is None else ints(self.qd), None if self.kd is None else ints(self.kd)]
        qs, ql, ks, kl, qp, pre, qd, kd = (P(t) for t in self.keep)
        a = sj.AttnScoredArgs(q=P(self.q), k=P(self.k), v=P(self.v), o=P(self.o), q_start=qs, q_len=ql, k_start=ks, k_len=kl, q_pos=qp, prefix=pre,
                              q_doc=qd, k_doc=kd, slopes=P(self.sl), scale=self.scale, softcap=self.cap, window=self.window, causal=int(self.causal),
                              B=len(self.ql), H=self.H, Hkv=self.Hkv, Dh=self.Dh, q_rows=self.nq, k_rows=self.nk, max_q=max(self.ql),
                              max_k=max(self.kl), dtype=sj.SJH_BF16 if self.dtype == "bf16" else sj.SJH_F32)
        for k, v in over.items():
            setattr(a, k, v)
        n = sj.lib().sjh_attn_scored_workspace(C.byref(a))
        assert n >= 0, sj.lib().sjh_last_error()
        if n:
            # (nothing in it is read that the call has not written)
            self.ws = torch.full((n // 4,), float("nan"), device="cuda")
            a.workspace, a.workspace_bytes = self.ws.data_ptr(), n
        return a

    def run(self, stream=None, **over):
        a = self.args(**over)
        sj.check(sj.lib().sjh_attn_scored(C.byref(a), stream))
        torch.cuda.synchronize()
        return self.o

    def see(self, b, i0, i1):
        p = np.arange(self.q_pos[b] + i0, self.q_pos[b] + i1)[:, None]
        j = np.arange(self.kl[b])[None]
        see = np.ones((i1 - i0, self.kl[b]), bool)
        if self.causal:
            see &= j <= p
        if self.window:
            see &= np.abs(p - j) <= self.window
        if self.kd is not None:
            see &= self.qd[self.qs[b] + i0:self.qs[b] + i1, None] == self.kd[None, self.ks[b]:self.ks[b] + self.kl[b]]
        if self.prefix is not None:
            see |= j < self.prefix[b]
        return see, np.abs(p - j)

    def check(self, seqs=None, rows=None):
        got = self.o.double().cpu().numpy()
        q, k, v = (t.double().cpu().numpy() for t in (self.q, self.k, self.v))
        G = self.H // self.Hkv
        scale = self.scale or self.Dh ** -0.5
        scale = float(np.float32(scale))
        written = np.zeros(self.nq, bool)
        for b in range(len(self.ql)):
            written[self.qs[b]:self.qs[b] + self.ql[b]] = True
        assert np.all(got[~written] == 7)  # rows of no sequence
        for b in seqs if seqs is not None else range(len(self.ql)):
            i0, i1 = rows or (0, self.ql[b])
            i1 = min(i1, self.ql[b])
            if i1 <= i0:
                continue
            see, dist = self.see(b, i0, i1)
            for h in range(self.H):
                qq = q[self.qs[b] + i0:self.qs[b] + i1, h]
                kk, vv = (x[self.ks[b]:self.ks[b] + self.kl[b], h // G] for x in (k, v))
                o = got[self.qs[b] + i0:self.qs[b] + i1, h]
                dead = ~see.any(1)
                assert np.all(o[dead] == 0), (b, h)
                if dead.all():
                    continue
                with np.errstate(invalid="ignore", over="ignore"):
                    s = np.where(see, qq @ kk.T * scale, 0.0)
                    ds = (self.Dh + 3) * U * scale * np.where(see, np.abs(qq) @ np.abs(kk).T, 0.0) + 8 * U * np.abs(s)
                if self.cap:
                    s = self.cap * np.tanh(s / self.cap)
                    ds = ds + 2e-6 * self.cap
                if self.sl is not None:
                    bias = float(self.sl[h]) * dist
                    s, ds = s - bias, ds + 4 * U * np.where(see, bias, 0)
                s = np.where(see, s, -np.inf)
                w = np.exp(s - np.where(dead, 0, s.max(1))[:, None])
                w = w / np.maximum(w.sum(1, keepdims=True), 1e-300)
                d = 2 * np.where(see, ds, 0).max(1) + 16 * U + (2.0 ** -8 if self.dtype == "bf16" else 0)
                for i in np.flatnonzero(~dead):
                    vis = see[i]
                    x, wi = vv[vis], w[i][vis][:, None]
                    if not np.isfinite(x).all():
                        # sums with infinities and NaN as they come
                        with np.errstate(invalid="ignore"):
                            want = (wi * x).sum(0)
                        fin = np.isfinite(x).all(0)
                        assert np.array_equal(np.isnan(o[i]), np.isnan(want)) and np.array_equal(o[i][np.isinf(want)], want[np.isinf(want)])
                    else:
                        fin = slice(None)
                    x = x[:, fin]
                    want = (wi * x).sum(0)
                    lim = 1.05 * d[i] * (wi * np.abs(x - want)).sum(0) + 2 * (vis.sum() + 8) * U * (wi * np.abs(x)).sum(0)
                    lim = lim + (2.0 ** -8 if self.dtype == "bf16" else U) * (np.abs(want) + lim) + 1e-38
                    err = np.abs(o[i][fin] - want)
                    assert np.all(err <= lim), (b, h, i0 + i, float((err / lim).max()))


def halves(b, j):
    return 3 * (j // 37) - 5


# lengths at the edges of a wave's 32 queries, a block's 128, a tile's 64 keys; no
# queries, no keys; each modification alone and all together; head groups
MODS = {
    "plain": dict(),
    "cap": dict(cap=5.0, amp=4.0),
    "cap_small": dict(cap=50.0),
    "bias": dict(slopes=[0.5, 0.03]),
    "causal": dict(causal=True),
    "window": dict(window=20),
    "docs": dict(docs=halves),
    "all": dict(cap=9.0, amp=4.0, slopes=[0.25, 0.01], causal=True, window=90, docs=halves, prefix="some"),
}
LENS = [(1, 1), (31, 64), (33, 65), (0, 5), (7, 0), (128, 128), (130, 200), (64, 63)]


@pytest.mark.parametrize("dtype,Dh", [("bf16", 64), ("bf16", 128), ("bf16", 32), ("f32", 64), ("f32", 8), ("f32", 128)])
@pytest.mark.parametrize("mod", sorted(MODS))
def test_attn_scored(mod, dtype, Dh):
    print(f"attn_scored {mod} {dtype} Dh={Dh}", flush=True)
    kw = dict(MODS[mod])
    if kw.get("prefix") == "some":
        kw["prefix"] = [0, 3, 65, 1, 0, 70, 10, 64]
    # (positions of queries whose keys are fewer: some before the first, all after the last)
    c = Case([q for q, _ in LENS], [k for _, k in LENS], Dh=Dh, dtype=dtype, q_pos=[max(k - q, 0) for q, k in LENS], **kw)
    c.run()
    c.check()


# enough blocks for the shape that shares tiles between waves (B x H x blocks >= 256)
@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("mod", sorted(MODS))
def test_attn_scored_many_blocks(mod, Dh):
    print(f"attn_scored many {mod} Dh={Dh}", flush=True)
    kw = dict(MODS[mod])
    lens = [(5 * i) % 141 + (i == 0) for i in range(64)]
    if kw.get("prefix") == "some":
        kw["prefix"] = [(3 * i) % 80 for i in range(64)]
    if "slopes" in kw:
        kw["slopes"] = kw["slopes"] * 2
    c = Case(lens, lens, H=4, Hkv=2, Dh=Dh, **kw)
    c.run()
    c.check(seqs=range(0, 64, 5))


@pytest.mark.parametrize("Dh,dtype", [(64, "bf16"), (128, "bf16"), (64, "f32")])
@pytest.mark.parametrize("H,Hkv,q", [(8, 2, 1), (8, 2, 8), (8, 1, 5), (6, 6, 3), (4, 2, 33)])
def test_attn_scored_few_queries_of_long_sequences(H, Hkv, q, Dh, dtype):
    # splits, head groups in one block, more than 4096 keys (a second word of tiles)
    print(f"attn_scored tail H={H}/{Hkv} q={q} Dh={Dh} {dtype}", flush=True)
    for kw in (dict(cap=8.0, amp=3.0, causal=True), dict(slopes=[0.5 ** (i + 1) for i in range(H)], prefix=[100, 0, 64]),
               dict(docs=lambda b, j: j * 7 % 3, window=2500), dict(docs=lambda b, j: j // 2000)):
        c = Case([q, 1, q], [4500, 1, 4161], H=H, Hkv=Hkv, Dh=Dh, dtype=dtype, **kw)
        c.run()
        c.check()


def test_attn_scored_long_rows_and_sparse_masks():
    # whole sequences past a word of tiles, whose masks leave most tiles unread
    print("attn_scored long", flush=True)
    for kw in (dict(docs=lambda b, j: (j * 2654435761 >> 7) % 5 if j % 700 < 40 else j // 700, causal=True), dict(window=3, prefix=[70]),
               dict(docs=lambda b, j: -(j // 90), slopes=[0.1] * 4, cap=20.0)):
        c = Case([8300], [8300], H=4, seed=3, **kw)
        c.run()
        for r in (0, 60, 4090, 8290):
            c.check(rows=(r, r + 12))


@pytest.mark.parametrize("dtype,Dh,q", [("bf16", 64, 40), ("bf16", 64, 3), ("bf16", 128, 40), ("bf16", 64, 300), ("f32", 64, 40), ("f32", 32, 3)])
def test_attn_scored_masked_values_take_no_part(dtype, Dh, q):
    # infinities and NaN in keys and values that some queries see and others do
    # not, in one tile: the first are as the sum has it, the others untouched
    print(f"attn_scored infinities {dtype} Dh={Dh} q={q}", flush=True)
    B = 48 if q == 300 else 2  # (300: the shape of shared tiles)
    c = Case([q] * B, [max(q, 200)] * B, H=2, Dh=Dh, dtype=dtype, docs=lambda b, j: j // 25, q_pos=[0] * B, cap=10.0, amp=2.0)
    inf, nan = float("inf"), float("nan")
    for b in (0, 1):
        s = int(c.ks[b])
        c.v[s + 30, :, :5] = inf
        c.v[s + 31, :, 3:8] = -inf
        c.v[s + 60, :, 1] = nan
        c.k[s + 110] = nan
        c.v[s + 110] = nan
        c.v[s + 199] = -inf
        c.k[s + 150] = inf
    c.run()
    # a NaN key's score makes its document's queries NaN: left to the next loop
    got = c.o.double().cpu().numpy()
    for b in (0, 1):
        for i in range(q):
            d = i // 25
            row = got[c.qs[b] + i]
            if d in (4, 6):  # a NaN score, an infinite key (0 * inf or inf in its product, capped or NaN)
                continue
            c.check(seqs=[b], rows=(i, i + 1))
            if d not in (1, 2, 7):
                assert np.isfinite(row).all()
    if q > 100:
        assert np.isnan(got[c.qs[0] + 100:c.qs[0] + 125]).all()


def test_attn_scored_all_scores_alike_large_and_offset():
    # scores far outside the exponential's range, equal ones, and a cap that saturates
    for kw in (dict(amp=200.0), dict(amp=200.0, cap=50.0), dict(amp=0.0), dict(amp=30.0, cap=1e-3), dict(amp=3.0, cap=1e4), dict(amp=3.0, slopes=[40.0, 500.0])):
        print("attn_scored", kw, flush=True)
        c = Case([100], [170], q_pos=[35], **kw)
        c.run()
        c.check()
    # far keys alone: every bias beyond the range of a difference of exponents from 0
    c = Case([40], [3000], q_pos=[2900], slopes=[3.0, 0.5], prefix=[50], docs=lambda b, j: 1 if j < 2000 else j)
    c.run()
    c.check()


def test_attn_scored_strides_and_alignment():
    # packed q|k|v rows, as the projection writes them; rows no vector load takes
    print("attn_scored strides", flush=True)
    for off in (0, 1):
        for dtype in ("bf16", "f32"):
            c = Case([70, 50], [70, 50], H=3, Dh=64, dtype=dtype, causal=True)
            D = 3 * 64
            rows = c.nk
            buf = torch.randn(off + rows * 3 * D + 8, device="cuda").to(c.q.dtype)
            qkv = buf[off:off + rows * 3 * D].view(rows, 3, 3, 64)
            c.qs, c.nq = c.ks, c.nk
            ob = torch.full((off + rows * (D + 3 * off + 4),), 7.0, device="cuda", dtype=c.q.dtype)
            ld_o = D + 3 * off + 4
            o = ob[off:].view(rows, ld_o)[:, :D]
            c.q, c.k, c.v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
            c.o = o
            a = c.args(ld_q=3 * D, ld_k=3 * D, ld_v=3 * D, ld_o=ld_o)
            sj.check(sj.lib().sjh_attn_scored(C.byref(a), None))
            torch.cuda.synchronize()
            m = torch.ones_like(ob, dtype=torch.bool)
            m[off:].view(rows, ld_o)[:, :D] = False
            assert torch.all(ob[m] == 7)
            c.o = o.reshape(rows, 3, 64)
            c.check()


def test_attn_scored_offsets_past_32_bits():
    # one query at the end of a cache whose rows span more than 4 GiB
    n, ld = 300_000, 8192
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of free device memory")
    print("attn_scored 5 GB of keys", flush=True)
    for dtype, td, ldd in (("bf16", torch.bfloat16, ld), ("f32", torch.float32, ld // 2)):
        c = Case([1], [300], H=1, Dh=64, dtype=dtype, window=200, prefix=[10])
        kb, vb = (torch.empty(n, ldd, dtype=td, device="cuda") for _ in range(2))
        # the last 300 keys are the case's; the prefix its first ones
        for big, small in ((kb, c.k), (vb, c.v)):
            big[n - 300:, :64] = small[:300, 0]
            big[:10, :64] = small[:10, 0]
        small_k, small_v = c.k, c.v
        c.k, c.v = kb, vb
        c.kl, c.ks, c.q_pos, c.nk = [n], [0], [n - 1], n
        c.run(ld_k=ldd, ld_v=ldd)
        c.k, c.v = small_k, small_v
        c.kl, c.q_pos, c.nk = [300], [299], 302
        c.check()


def test_attn_scored_device_tables_are_clamped():
    # starts and lengths that leave the buffers or the bounds read and write
    # nothing outside: the rows there are take part, no more
    print("attn_scored clamped", flush=True)
    c = Case([40, 30], [60, 30])
    a = c.args()
    bad = [ints([0, 1 << 30]), ints([1 << 30, -5]), ints([-7, 40]), ints([60, 1 << 30])]
    a.q_start, a.q_len, a.k_start, a.k_len = (t.data_ptr() for t in bad)
    pos, pre = ints([-(1 << 31), (1 << 31) - 1]), ints([(1 << 31) - 1, -4])
    a.q_pos, a.prefix = pos.data_ptr(), pre.data_ptr()
    guard = c.o.clone()
    sj.check(sj.lib().sjh_attn_scored(C.byref(a), None))
    torch.cuda.synchronize()
    assert torch.equal(c.o[40:], guard[40:])  # max_q rows of sequence 0, none of 1
    c.ql, c.qs, c.kl, c.ks, c.q_pos = [40], [0], [60], [0], [0]
    c.check()


def test_attn_scored_in_graphs_on_streams_and_twice_at_once():
    # a replayed graph and calls on two streams, a workspace each, give the eager bits
    print("attn_scored graphs", flush=True)
    cs = [Case([3, 2], [4000, 2500], H=4, Hkv=2, seed=i, causal=True, docs=lambda b, j: j // 900) for i in range(2)]
    want = [c.run().clone() for c in cs]
    calls = [c.args() for c in cs]
    assert all(a.workspace_bytes > 0 for a in calls)
    keep = [c.ws for c in cs]  # noqa: F841
    streams = [torch.cuda.Stream() for _ in cs]
    graphs = []
    for a, s in zip(calls, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            sj.check(sj.lib().sjh_attn_scored(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        graphs.append(g)
    for _ in range(3):
        for c in cs:
            c.o.fill_(7.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(c.o, w) for c, w in zip(cs, want))
        for c in cs:
            c.o.fill_(7.0)
        torch.cuda.synchronize()
        for a, s in zip(calls, streams):
            sj.check(sj.lib().sjh_attn_scored(C.byref(a), C.c_void_p(s.cuda_stream)))
        torch.cuda.synchronize()
        assert all(torch.equal(c.o, w) for c, w in zip(cs, want))


@pytest.mark.parametrize("Dh,q,B", [(64, 100, 4), (128, 100, 4), (64, 3, 1)])
def test_attn_scored_small_values_under_low_scores(Dh, q, B):
    """Every score at the cap's lower end (weights 2^-95 of 1), values of 1e-12: their
    products are below fp32's range without a maximum."""
    print(f"attn_scored small values {Dh} {q}", flush=True)
    c = Case([q] * B, [q] * B, H=64, Dh=Dh, cap=66.0)
    c.q.fill_(9.0)
    c.k.fill_(-9.0)
    c.v *= 1e-12
    c.run()
    c.check(seqs=[B - 1])
    assert float(c.o[:q].abs().max()) > 0


@pytest.mark.parametrize("H,q", [(2, 3), (64, 130)])
@pytest.mark.parametrize("cap", [1e9, 1e10, 1e37])
def test_attn_scored_caps_far_above_the_scores(cap, H, q):
    """cap tanh(s / cap) = s to 2^-40 here.  A score is off by 1e-5 of its size (the
    polynomial's factor of it, 9e-6, and fp32's roundings), a weight by twice the
    largest score's and bf16's 2^-8, as in the bound above."""
    print(f"attn_scored cap {cap} {H} {q}", flush=True)
    c = Case([q] * 4, [300] * 4, H=H, cap=cap, amp=60.0)
    c.run()
    got = c.o.double().cpu().numpy()
    q_, k, v = (t.double().cpu().numpy() for t in (c.q, c.k, c.v))
    for b in (0, 3):
        for h in (0, H - 1):
            s = q_[c.qs[b]:c.qs[b] + q, h] @ k[c.ks[b]:c.ks[b] + 300, h].T / 8
            assert np.abs(s).max() > 100  # (144 in log2: past fp32 without a maximum)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            vv = v[c.ks[b]:c.ks[b] + 300, h]
            want = w @ vv
            d = 2 * 1e-5 * np.abs(s).max(1, keepdims=True) + 16 * U + 2.0 ** -8
            lim = 1.05 * d * np.einsum("ij,ijd->id", w, np.abs(vv[None] - want[:, None])) + 2 * 308 * U * (w @ np.abs(vv))
            lim = lim + 2.0 ** -8 * (np.abs(want) + lim)
            err = np.abs(got[c.qs[b]:c.qs[b] + q, h] - want)
            assert np.all(err <= lim), (b, h, float((err / lim).max()))


@pytest.mark.parametrize("Dh,H,Hkv", [(64, 8, 2), (128, 8, 2), (64, 32, 1)])
def test_attn_scored_many_sequences_of_few_tokens(Dh, H, Hkv):
    """More sequences than CUs, the queries of a key head's heads in one block of 32."""
    print(f"attn_scored many few {Dh} {H} {Hkv}", flush=True)
    ql, kl = ([1, 2, 0, 4], [1, 64, 3, 130]) if H == 8 else ([1, 1, 0, 1], [700, 64, 3, 65])
    c = Case(ql * 80, kl * 80, H=H, Hkv=Hkv, Dh=Dh, cap=20.0, causal=True, prefix=[0, 5, 1, 40] * 80, docs=lambda b, j: j // 33)
    c.run()
    c.check(seqs=[0, 1, 2, 3, 158, 159, 318, 319])


@pytest.mark.parametrize("B,H,Hkv", [(3, 9, 9), (3, 9, 3), (1, 30, 30), (5, 12, 3)])
@pytest.mark.parametrize("causal", [False, True])
def test_attn_scored_orders_of_blocks(B, H, Hkv, causal):
    """Pairs of sequence and key head that fill the XCDs' turns and that do not; every
    block of every head is written (the rows of one are told apart by their values)."""
    print(f"attn_scored orders {B} {H} {Hkv} {causal}", flush=True)
    L = [1300 - 7 * b for b in range(B)]
    c = Case(L, L, H=H, Hkv=Hkv, causal=causal, cap=30.0, window=200)
    c.run()
    for b in range(B):
        assert not bool((c.o[c.qs[b]:c.qs[b] + L[b]] == 7).all(-1).any()), b
    for rows in ((0, 40), (630, 650), (1260, 1300)):
        c.check(seqs=[0, B - 1], rows=rows)
