"""sjh_gemm_lora against float64, at the edges of its tiles and row blocks.

The bound.  The base's sum is off by (K + 2) 2^-24 sum |x w|, t by (K + 3) 2^-24
scale sum |x a| and, for the bf16 pipes, one rounding of 2^-8 |t|; both enter the
output through |b|, whose own products add (R + 4) 2^-24 sum |t b|, and the joint
sum 2^-24 of its size.  GELU's slope is at most 1.13, its bf16 form within
4.3e-7 of the exact one and four roundings; a bf16 output rounds by 2^-8."""
import ctypes as C

import numpy as np
import pytest

import snapjudge_amd as sj

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def P(t):
    return None if t is None else t.data_ptr()


class Case:
    def __init__(self, M, N, K, R, n, adapter, dtype="bf16", act=0, bias=True, scale=True, off=0, pad=0, seed=0):
        g = torch.Generator(device="cuda").manual_seed(M + 3 * N + 7 * K + 11 * R + seed)
        td = torch.float32 if dtype == "f32" else torch.bfloat16
        self.__dict__.update({k: v for k, v in locals().items() if k not in ("self", "g", "td")})

        def R_(*s):
            n_ = int(np.prod(s))
            return torch.randn(n_ + off, generator=g, device="cuda").to(td)[off:].view(*s)

        self.ld = K + pad
        self.x = R_(M, self.ld)
        self.a, self.b = R_(n, R, K), R_(n, N, R)
        self.bv = torch.randn(N, generator=g, device="cuda") if bias else None
        self.sv = torch.rand(n, generator=g, device="cuda") - 0.5 if scale else None
        self.ad = None if adapter is None else torch.from_numpy(np.asarray(adapter, np.int32)).cuda()
        if dtype == "fp8":
            w = torch.randn(N, K, generator=g, device="cuda")
            self.ws = (w.abs().amax(1) / 448).contiguous()
            self.w = (w / self.ws[:, None]).to(torch.float8_e4m3fn)
        else:
            self.w, self.ws = R_(N, K), None
        self.ld_out = N + pad
        self.out = torch.full((M + 1, self.ld_out), 7.0, device="cuda", dtype=td)

    def args(self, **over):
        n = sj.lib().sjh_gemm_lora_workspace(self.M, self.R)
        self.work = torch.full((n // 4 + 4,), float("nan"), device="cuda")
        a = sj.LoraArgs(x=P(self.x), w=P(self.w), w_scale=P(self.ws), bias=P(self.bv), a=P(self.a), b=P(self.b), scale=P(self.sv),
                        adapter=P(self.ad), out=P(self.out), workspace=P(self.work), workspace_bytes=n, ld_x=self.ld, ld_out=self.ld_out, M=self.M,
                        N=self.N, K=self.K, R=self.R, n_adapters=self.n, act=self.act, dtype=sj.SJH_F32 if self.dtype == "f32" else sj.SJH_BF16)
        for k, v in over.items():
            setattr(a, k, v)
        return a

    def run(self, stream=None, **over):
        sj.check(sj.lib().sjh_gemm_lora(C.byref(self.args(**over)), stream))
        torch.cuda.synchronize()
        return self.out

    def check(self, rows=None):
        rows = np.arange(self.M) if rows is None else np.asarray(rows)
        d = lambda t: t.double().cpu().numpy()  # noqa: E731
        x, a, b = d(self.x)[rows, :self.K], d(self.a), d(self.b)
        w = d(self.w.float()) * (d(self.ws)[:, None] if self.ws is not None else 1)
        bias = d(self.bv) if self.bv is not None else np.zeros(self.N)
        ad = np.zeros(self.M, int) if self.ad is None else self.ad.cpu().numpy()
        y = x @ w.T + bias
        e = (self.K + 4) * U * (np.abs(x) @ np.abs(w).T + np.abs(bias))
        half = 2.0 ** -8 if self.dtype != "f32" else 0.0
        for k in range(self.n):
            r = np.flatnonzero(ad[rows] == k)
            if len(r) == 0:
                continue
            s = float(self.sv[k]) if self.sv is not None else 1.0
            t = s * (x[r] @ a[k].T)
            et = (self.K + 3) * U * abs(s) * (np.abs(x[r]) @ np.abs(a[k]).T)
            et = et + half * (np.abs(t) + et)
            y[r] += t @ b[k].T
            e[r] += (et + (self.R + 4) * U * (np.abs(t) + et)) @ np.abs(b[k]).T
        e = e + U * np.abs(y)
        if self.act == 1:
            z = 0.5 * y * (1 + torch.erf(torch.from_numpy(y / np.sqrt(2))).numpy())
            y, e = z, 1.13 * e + 5e-7 + 6 * U * np.abs(y)
        elif self.act == 2:
            y = np.maximum(y, 0)
        got = d(self.out)
        assert np.all(got[self.M] == 7) and np.all(got[:, self.N:] == 7)
        err, lim = np.abs(got[rows, :self.N] - y), e + half * (np.abs(y) + e)
        assert np.all(err <= lim), (float((err / lim).max()), np.argwhere(err > lim)[:5])


def mixed(M, n, seed=0):
    return np.random.default_rng(seed).integers(-1, n + 1, size=M)


def runs(M, n, rows):
    """Requests of `rows` rows each, one in three without an adapter."""
    return [(-1 if (i // rows) % 3 == 2 else (i // rows) % n) for i in range(M)]


# one row; rows of a partial block; every tile shape of the bf16 kernels (32- and
# 64-column tiles, 128x64, 128x128, the persistent one with its half units); ranks
# of a part of a step, one, several, past one sweep of the first product, odd ones
SHAPES = [(1, 64, 64, 16, 1), (9, 300, 128, 8, 16), (33, 96, 768, 16, 5), (300, 520, 192, 24, 3), (257, 2304, 64, 64, 4),
          (1100, 770, 256, 40, 6), (3000, 1152, 128, 16, 7), (6200, 1156, 128, 80, 5), (12000, 1540, 64, 32, 9), (70, 36, 320, 13, 4), (40, 64, 64, 1, 2),
          (515, 1024, 128, 130, 3), (20, 32, 64, 256, 2)]


@pytest.mark.parametrize("dtype", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("M,N,K,R,n", SHAPES)
def test_lora(M, N, K, R, n, dtype):
    if dtype == "f32" and M > 3000:
        pytest.skip("the fp32 kernel's tiles do not change past this")
    for i, ad in enumerate((mixed(M, n), runs(M, n, 45), runs(M, n, 700))):
        print(f"lora M={M} N={N} K={K} R={R} n={n} {dtype} {i}", flush=True)
        c = Case(M, N, K, R, n, ad, dtype=dtype, act=i)
        if dtype == "fp8" and N % 4:  # (as sjh_gemm_fp8w)
            with pytest.raises(sj.SjhError, match="N % 4"):
                c.run()
            continue
        c.run()
        c.check(rows=None if M * N < 2e6 else np.unique(np.r_[np.arange(0, M, 53), np.arange(min(M, 70)), np.arange(max(0, M - 70), M)]))


# shapes of the fp32-product kernel: K no multiple of 64, rows no vector load takes, bf16 among them
# the first product's blocks of 64 rows: one piece of K, fewer and more than its
# ring holds; a rank block, two and four, a second sweep; blocks of one adapter, of
# none, of many, and where requests meet
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("M,N,K,R,n,rows", [(8192, 64, 64, 16, 70, 1), (8200, 40, 192, 24, 5, 100), (8255, 96, 320, 65, 3, 64), (9001, 36, 768, 130, 2, 5000)])
def test_lora_many_rows(M, N, K, R, n, rows, dtype):
    print(f"lora many {M}x{N}x{K} R={R} n={n} {rows} {dtype}", flush=True)
    c = Case(M, N, K, R, n, mixed(M, n) if rows == 1 else runs(M, n, rows), dtype=dtype)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K,R,n,off,pad", [(5, 3, 1, 1, 1, 0, 0), (33, 70, 51, 7, 3, 0, 0), (200, 130, 128, 16, 4, 1, 1), (700, 600, 100, 33, 5, 0, 3), (1, 9, 64, 4, 2, 1, 0)])
def test_lora_any_shape(M, N, K, R, n, off, pad, dtype):
    print(f"lora any M={M} N={N} K={K} R={R} off={off} pad={pad} {dtype}", flush=True)
    for act, ad in ((0, mixed(M, n)), (1, None)):
        c = Case(M, N, K, R, n, ad, dtype=dtype, act=act, off=off, pad=pad, bias=act == 0, scale=act == 0)
        c.run()
        c.check()


def test_lora_strides_and_no_adapters():
    print("lora strides", flush=True)
    c = Case(130, 128, 192, 16, 3, mixed(130, 3), pad=8)
    c.run()
    c.check()
    # no adapters: sjh_gemm's bits; a row without one among others: the same
    for M, N in ((40, 256), (300, 768), (6200, 1156)):
        c = Case(M, N, 128, 16, 4, mixed(M, 4), act=1)
        ref = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
        sj.check(sj.lib().sjh_gemm(P(c.x), P(c.w), C.cast(P(c.bv), C.POINTER(C.c_float)), P(ref), M, N, 128, 1, sj.SJH_BF16, None))
        none = ((c.ad < 0) | (c.ad >= 4))
        assert torch.equal(c.run()[:M][none], ref[none])
        c.out[:M] = 3.0
        assert torch.equal(c.run(n_adapters=0, a=None, b=None, workspace=None, R=0)[:M], ref)


@pytest.mark.parametrize("dtype", ["bf16", "fp8", "f32"])
@pytest.mark.parametrize("M,N", [(50, 96), (300, 520), (6200, 1156)])
def test_lora_adapters_keep_to_their_rows(M, N, dtype):
    # an adapter of infinities and NaN, and a row of them: no other row changes
    if dtype == "f32" and M > 3000:
        pytest.skip("the fp32 kernel's tiles do not change past this")
    print(f"lora infinities M={M} N={N} {dtype}", flush=True)
    c = Case(M, N, 128, 16, 4, mixed(M, 4), dtype=dtype)
    want = c.run().clone()
    c.a[2, 3], c.b[2, ::3] = float("nan"), float("inf")
    row = int(torch.nonzero(c.ad == 1)[0])
    c.x[row, 5] = float("inf")
    got = c.run()
    hit = (c.ad == 2)
    hit[row] = True
    keep = ~hit
    assert torch.equal(got[:M][keep], want[:M][keep]) and torch.all(got[M] == 7)
    assert not torch.isfinite(got[:M][c.ad == 2]).any()
    assert not torch.isfinite(got[row]).any()


def test_lora_in_a_graph_and_on_streams():
    print("lora graph", flush=True)
    cs = [Case(m, 768, 256, 16, 5, mixed(m, 5, m)) for m in (20, 700)]
    want = [c.run().clone() for c in cs]
    calls, streams, graphs = [c.args() for c in cs], [torch.cuda.Stream() for _ in cs], []
    for a, s in zip(calls, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            sj.check(sj.lib().sjh_gemm_lora(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        graphs.append(g)
    for _ in range(3):
        for how in ("replay", "call"):
            for c in cs:
                c.out.fill_(7.0)
            torch.cuda.synchronize()
            for a, g, s in zip(calls, graphs, streams):
                if how == "replay":
                    with torch.cuda.stream(s):
                        g.replay()
                else:
                    sj.check(sj.lib().sjh_gemm_lora(C.byref(a), C.c_void_p(s.cuda_stream)))
            torch.cuda.synchronize()
            assert all(torch.equal(c.out, w) for c, w in zip(cs, want)), how
