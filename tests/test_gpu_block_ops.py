"""A sandwich-normed encoder block with adapters, packed documents and capped
scores, run from the three operators as a program would: one stream, one
workspace that the calls take in turn, no wait between them, QKV read in place
by its strides.  Every step is then held to float64 of the buffers that it read
(with the bounds of the operators' own tests), and the block, captured, gives
the same bits on every replay."""
import ctypes as C

import numpy as np
import pytest

import snapjudge_amd as sj

torch = pytest.importorskip("torch")
import test_gpu_add_norm as tn  # noqa: E402
import test_gpu_attn_scored as ta  # noqa: E402
import test_gpu_lora as tl  # noqa: E402

pytestmark = pytest.mark.gpu


class Block:
    def __init__(self, lens, L, H, Dh, F, R, n, dtype, docs, causal, prefix, slopes=None, cap=30.0, window=0):
        B, D = len(lens), H * Dh
        M = B * L
        g = torch.Generator(device="cuda").manual_seed(M + D)
        td, self.code, self.u = tn.DT[dtype]
        self.__dict__.update({k: v for k, v in locals().items() if k != "self"})
        R_ = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.x = R_(M, D)
        self.norms = [1 + 0.1 * R_(D) for _ in range(5)]
        ad = np.repeat(np.arange(B) % (n + 1) - 1, L)  # one request's rows each; some with none
        mk = lambda N, K, **kw: tl.Case(M, N, K, R, n, ad, dtype=dtype, scale=True, **kw)  # noqa: E731
        self.qkv, self.wo, self.up, self.down = mk(3 * D, D), mk(D, D, seed=1), mk(F, D, act=1, seed=2), mk(D, F, seed=3)
        for c in (self.qkv, self.wo, self.up, self.down):
            c.w.mul_(c.K ** -0.5)
            c.a.mul_(c.K ** -0.5)
        at = ta.Case(lens, lens, H=H, Dh=Dh, dtype=dtype, cap=cap, slopes=slopes, window=window, causal=causal, prefix=prefix, docs=docs, q_pos=[0] * B)
        at.qs = at.ks = np.arange(B) * L
        at.nq = at.nk = M
        if docs is not None:
            at.qd = at.kd = np.concatenate([[docs(b, j) if j < lens[b] else -1 for j in range(L)] for b in range(B)]).astype(np.int32)
        at.q, at.k, at.v = (self.qkv.out[:M].view(M, 3, H, Dh)[:, i] for i in range(3))
        at.o = torch.full((M, H, Dh), 7.0, dtype=td, device="cuda")
        self.at = at
        self.y1, self.y2 = (torch.empty(M, D, dtype=td, device="cuda") for _ in range(2))
        self.y3 = torch.empty(M, D, dtype=td, device="cuda")
        self.x1, self.x2 = torch.empty_like(self.x), torch.empty_like(self.x)
        self.qkv.x, self.wo.x, self.up.x, self.down.x = self.y1, at.o.view(M, D), self.y2, self.up.out[:M]
        ang = torch.arange(L, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, Dh, 2, device="cuda") / Dh)
        self.cos, self.sin = ang.cos().contiguous(), ang.sin().contiguous()
        # the calls' arguments, kept as a program keeps them; one workspace for all
        self.calls = [c.args() for c in (self.qkv, self.wo, self.up, self.down)]
        self.aa = at.args(ld_q=3 * D, ld_k=3 * D, ld_v=3 * D)
        n_ws = max([self.aa.workspace_bytes] + [c.workspace_bytes for c in self.calls])
        self.ws = torch.full((n_ws // 4 + 4,), float("nan"), device="cuda")
        for c in self.calls + [self.aa]:
            c.workspace, c.workspace_bytes = self.ws.data_ptr(), n_ws

    def norm(self, x, r, xo, y, post, w, **kw):
        d = dict(x=x, y=y, pre_w=w, x_scale=1.0, r_scale=1.0, eps=1e-6, pre_norm=sj.SJH_NORM_RMS, M=self.M, D=self.D, dtype=self.code)
        if r is not None:
            d.update(r=r, x_out=xo, post_w=post, post_norm=sj.SJH_NORM_RMS)
        a = sj.AddNormArgs(**{k: (v.data_ptr() if torch.is_tensor(v) else v) for k, v in d.items()})
        sj.check(sj.lib().sjh_add_norm(C.byref(a), self.st))

    def run(self, stream):
        self.st = stream
        lib = sj.lib()
        gemm = lambda i: sj.check(lib.sjh_gemm_lora(C.byref(self.calls[i]), stream))  # noqa: E731
        w = self.norms
        self.norm(self.x, None, None, self.y1, None, w[0])
        gemm(0)
        # (the rotated rows are the projection's output; kept apart for its check)
        self.raw.copy_(self.qkv.out)
        sj.check(lib.sjh_rope(self.qkv.out.data_ptr(), self.cos.data_ptr(), self.sin.data_ptr(), self.M, self.L, self.H, self.Dh, self.code, stream))
        sj.check(lib.sjh_attn_scored(C.byref(self.aa), stream))
        gemm(1)
        self.norm(self.x, self.wo.out, self.x1, self.y2, w[1], w[2])
        gemm(2)
        gemm(3)
        self.norm(self.x1, self.down.out, self.x2, self.y3, w[3], w[4])

    raw = property(lambda self: self.__dict__.setdefault("_raw", torch.empty_like(self.qkv.out)))

    def outputs(self):
        return [self.qkv.out, self.at.o, self.wo.out, self.x1, self.y2, self.up.out, self.down.out, self.x2, self.y3]

    def check_norm(self, x, r, post, w, xo, y):
        N = tn.npd
        zero = np.zeros((self.M, self.D))
        want, ex, wy, ey = tn.oracle(N(x), zero if r is None else N(r[:self.M]), "none" if r is None else "rms", "rms", N(post), None, N(w), None,
                                     None, None, 1.0, 0.0 if r is None else 1.0, 1e-6)
        if xo is not None:
            assert np.all(np.abs(N(xo) - want) <= 1.05 * ex)
        assert np.all(np.abs(N(y) - wy) <= 1.05 * (ey + self.u * (np.abs(wy) + ey)) + 1e-30)

    def check(self):
        w = self.norms
        self.check_norm(self.x, None, None, w[0], None, self.y1)
        rot, self.qkv.out = self.qkv.out, self.raw
        self.qkv.check()
        self.qkv.out = rot
        # the rotation, from the rows before it: two products, a sum, one rounding
        M, H, Dh = self.M, self.H, self.Dh
        v = self.raw[:M].double().view(M, 3, H, Dh)
        c, s = (t.double().repeat(self.B, 1)[:, None, None] for t in (self.cos, self.sin))
        lo, hi = v[:, :2, :, :Dh // 2], v[:, :2, :, Dh // 2:]
        want = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
        mag = torch.cat([(lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()], -1)
        got = rot[:M].double().view(M, 3, H, Dh)
        assert torch.equal(got[:, 2], v[:, 2])
        assert torch.all((got[:, :2] - want).abs() <= self.u * want.abs() + 4 * 2.0 ** -24 * mag)
        self.at.check()
        self.wo.check()
        self.check_norm(self.x, self.wo.out, w[1], w[2], self.x1, self.y2)
        self.up.check()
        self.down.check()
        self.check_norm(self.x1, self.down.out, w[3], w[4], self.x2, self.y3)


DOC = lambda b, j: j // 37  # noqa: E731
CASES = {
    "bf16 documents": dict(lens=[130, 0, 77, 1], L=130, H=2, Dh=64, F=520, R=8, n=2, dtype="bf16", docs=DOC, causal=False, prefix=[0, 0, 3, 0]),
    "bf16 causal": dict(lens=[300, 299], L=300, H=4, Dh=128, F=640, R=33, n=1, dtype="bf16", docs=None, causal=True, prefix=None, slopes=[0.5, 0.1, 0.0, 0.02]),
    "bf16 tokens": dict(lens=[2] * 9, L=2, H=6, Dh=64, F=100, R=4, n=3, dtype="bf16", docs=None, causal=True, prefix=None, cap=0.0, window=1),
    "f32": dict(lens=[40, 61], L=64, H=3, Dh=32, F=90, R=5, n=2, dtype="f32", docs=DOC, causal=False, prefix=[2, 0]),
}


@pytest.mark.parametrize("name", sorted(CASES))
def test_block(name):
    print(f"block {name}", flush=True)
    t = Block(**CASES[name])
    t.raw
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        t.run(st.cuda_stream)
    torch.cuda.synchronize()
    t.check()
    want = [o.clone() for o in t.outputs()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        t.run(st.cuda_stream)
    for i in range(3):
        for o in t.outputs():
            if o is not t.at.o:
                o[:t.M].fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for j, (o, w) in enumerate(zip(t.outputs(), want)):
            assert torch.equal(o, w), (i, j)
