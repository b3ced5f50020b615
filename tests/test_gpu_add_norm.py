"""sjh_add_norm against float64, at the edges of its kernels' row shapes.

The bounds.  A norm's value is off by the rounding of v - shift, of its mean
(taken in double, rounded once), of the difference, the inverse deviation and
two products and a sum: (|d| + |mean d| + |y| 8) 2^-24 with |d| and |mean d| in
deviations; d lies within the row's spread, at most sqrt(2 D) deviations of one
another.  x' adds four roundings of its terms.  What r's norm is off by reaches
x', and x' relative to its own deviation reaches y."""
import ctypes as C

import numpy as np
import pytest

import snapjudge_amd as sj

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
U = 2.0 ** -24
KIND = {"none": sj.SJH_NORM_NONE, "ln": sj.SJH_NORM_LAYER, "rms": sj.SJH_NORM_RMS}
DT = {"bf16": (torch.bfloat16, sj.SJH_BF16, 2.0 ** -8), "f32": (torch.float32, sj.SJH_F32, U)}


def call(stream=None, **kw):
    a = sj.AddNormArgs(**{k: (v.data_ptr() if torch.is_tensor(v) else v) for k, v in kw.items()})
    sj.check(sj.lib().sjh_add_norm(C.byref(a), stream))


def norm64(v, kind, w, b, eps):
    """The norm in float64, and the deviation it divides by."""
    if kind == "none":
        return v, np.ones((len(v), 1))
    m = v.mean(1, keepdims=True) if kind == "ln" else 0.0
    sd = np.sqrt(((v - m) ** 2).mean(1, keepdims=True) + eps)
    return (v - m) / sd * (1.0 if w is None else w) + (0.0 if b is None else b), sd


def norm_err(v, sd, kind, w):
    """What a norm's rounding leaves, for values v."""
    if kind == "none":
        return 0.0
    spread = (v.max(1, keepdims=True) - v.min(1, keepdims=True)) if kind == "ln" else np.abs(v)
    return (3 * spread / sd + 8 * np.abs(v - (v.mean(1, keepdims=True) if kind == "ln" else 0)) / sd) * U * (1.0 if w is None else np.abs(w))


def oracle(x, r, post, pre, pw, pb, w, b, gate, rows, xs, rs, eps):
    u, sd = norm64(r, post, pw, pb, eps)
    eu = norm_err(r, sd, post, pw) + 2 * U * np.abs(u)
    g = 1.0 if gate is None else gate[np.zeros(len(x), int) if rows is None else np.clip(rows, 0, len(gate) - 1)]
    xo = xs * x + rs * g * u
    ex = 4 * U * (np.abs(xs * x) + np.abs(rs * g * u)) + np.abs(rs * g) * eu
    y, sdx = norm64(xo, pre, w, b, eps)
    aw = 1.0 if w is None else np.abs(w)
    z = np.abs(norm64(xo, pre, None, None, eps)[0]).max(1, keepdims=True)
    ey = ex if pre == "none" else norm_err(xo, sdx, pre, w) + 2 * U * np.abs(y) + aw * ex.max(1, keepdims=True) / sdx * (2 + z)
    return xo, ex, y, ey


def npd(t):
    return None if t is None else t.double().cpu().numpy()


# rows of a part of a wave's piece, one piece, several, the last wave-owned row,
# the first and last that a workgroup owns; widths no vector load divides
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("post,pre", [("none", "ln"), ("rms", "rms"), ("ln", "none"), ("ln", "ln"), ("none", "none"), ("rms", "ln")])
@pytest.mark.parametrize("M,D", [(1, 1), (3, 4), (5, 63), (2, 256), (9, 260), (600, 768), (3, 771), (1300, 1023), (4, 1024), (3, 1028), (2, 2049), (3, 4096), (2, 8190), (2, 8192)])
def test_add_norm(M, D, post, pre, dtype):
    print(f"add_norm M={M} D={D} {post} {pre} {dtype}", flush=True)
    td, code, u = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(M * 31 + D)
    R = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    n_gates = 1 + M % 3
    x, r = R(M, D) * 2 + 1, (R(M, D) + 0.5).to(td)
    pw, pb, w, b = R(D) + 1, R(D), R(D) + 1, R(D)
    gate, rows = R(n_gates, D), torch.randint(-1, n_gates + 1, (M,), generator=g, device="cuda", dtype=torch.int32)
    xo, y = torch.full((M + 1, D), 7.0, device="cuda"), torch.full((M + 1, D), 7.0, device="cuda", dtype=td)
    eps = 1e-5
    call(x=x, r=r, x_out=xo, y=y, post_w=pw, post_b=pb, pre_w=w, pre_b=b, gate=gate, gate_row=rows, n_gates=n_gates, x_scale=1.25,
         r_scale=0.5, eps=eps, post_norm=KIND[post], pre_norm=KIND[pre], M=M, D=D, dtype=code)
    xw, ex, yw, ey = oracle(npd(x), npd(r), post, pre, npd(pw), npd(pb), npd(w), npd(b), npd(gate), rows.cpu().numpy(), 1.25, 0.5, eps)
    assert np.all(np.abs(npd(xo)[:M] - xw) <= ex)
    assert np.all(np.abs(npd(y)[:M] - yw) <= ey * 1.01 + u * np.abs(yw) + 1e-37)
    assert torch.all(xo[M] == 7) and torch.all(y[M] == 7)  # nothing behind the last row


def test_add_norm_optional_parts_strides_and_places():
    # no block output, no weights, no y or no x_out; x_out in x's place and y in
    # r's; rows further apart than their width, and addresses no vector load takes
    g = torch.Generator(device="cuda").manual_seed(5)
    R = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    M, D = 37, 516
    for off, pad in ((0, 4), (1, 3), (0, 0)):
        print(f"add_norm offset {off} pad {pad}", flush=True)
        ld = D + pad
        xb, rb = R(off + M * ld), R(off + M * ld).bfloat16()
        x, r = (t[off:].view(M, ld)[:, :D] for t in (xb, rb))
        xw, ex, yw, ey = oracle(npd(x), npd(r), "rms", "ln", None, None, None, None, None, None, 0.5, 2.0, 1e-6)
        rest = (xb.clone(), rb.clone())
        kw = dict(x=x, r=r, x_scale=0.5, r_scale=2.0, eps=1e-6, post_norm=2, pre_norm=1, M=M, D=D, dtype=sj.SJH_BF16, ld_x=ld, ld_r=ld)
        xo = torch.empty(M, D, device="cuda")
        call(x_out=xo, **kw)
        y = torch.empty(M, D, device="cuda", dtype=torch.bfloat16)
        call(y=y, **kw)
        call(x_out=x, y=r, ld_xo=ld, ld_y=ld, **kw)
        assert torch.equal(x, xo) and torch.equal(r, y)
        assert np.all(np.abs(npd(xo) - xw) <= ex) and np.all(np.abs(npd(y) - yw) <= ey * 1.01 + 2.0 ** -8 * np.abs(yw))
        # only the rows themselves were written
        for buf, was in zip((xb, rb), rest):
            m = torch.ones_like(buf, dtype=torch.bool)
            m[off:].view(M, ld)[:, :D] = False
            assert torch.equal(buf[m], was[m])
    call(x=x, x_out=xo, x_scale=3.0, eps=0.0, M=M, D=D, dtype=sj.SJH_BF16, ld_x=ld)
    assert torch.equal(xo, x * 3.0)
    call(x=0, x_out=0, M=0, D=4, dtype=0)  # no rows


def test_add_norm_keeps_to_its_rows_and_holds_offsets():
    # NaN and infinite rows reach no other; a large offset costs no accuracy; magnitudes
    # whose squares leave fp32 are normed as any
    g = torch.Generator(device="cuda").manual_seed(6)
    M, D = 12, 768
    x = torch.randn(M, D, generator=g, device="cuda")
    y, y2 = (torch.empty(M, D, device="cuda") for _ in range(2))
    kw = dict(eps=1e-5, x_scale=1.0, pre_norm=1, M=M, D=D, dtype=sj.SJH_F32)
    call(x=x, y=y, **kw)
    z = x.clone()
    z[3, 100], z[7, 0] = float("nan"), float("inf")
    call(x=z, y=y2, **kw)
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[[3, 7]] = False
    assert torch.equal(y[keep], y2[keep]) and torch.isnan(y2[[3, 7]]).all()
    for D2 in (D, 2048):
        off = (torch.randint(-500, 500, (M, D2), generator=g, device="cuda") * 2.0 ** -6 + 4096).contiguous()  # exact in fp32
        y = torch.empty(M, D2, device="cuda")
        call(x=off, y=y, eps=1e-5, x_scale=1.0, pre_norm=1, M=M, D=D2, dtype=sj.SJH_F32)
        want, sd = norm64(npd(off), "ln", None, None, 1e-5)
        assert np.all(np.abs(npd(y) - want) <= norm_err(npd(off), sd, "ln", None))
        for kind in (1, 2):
            big = torch.randn(M, D2, generator=g, device="cuda") * 1e25
            call(x=big, y=y, eps=1e-5, x_scale=1.0, pre_norm=kind, M=M, D=D2, dtype=sj.SJH_F32)
            want, sd = norm64(npd(big), ("", "ln", "rms")[kind], None, None, 1e-5)
            assert np.all(np.abs(npd(y) - want) <= norm_err(npd(big), sd, ("", "ln", "rms")[kind], None) + 4 * U * np.abs(want))


def test_add_norm_in_a_graph_and_on_a_stream():
    g = torch.Generator(device="cuda").manual_seed(7)
    M, D = 300, 1024
    x, r = torch.randn(M, D, generator=g, device="cuda"), torch.randn(M, D, generator=g, device="cuda").bfloat16()
    xo, y = torch.empty_like(x), torch.empty_like(r)
    kw = dict(x=x, r=r, x_out=xo, y=y, x_scale=1.0, r_scale=1.0, eps=1e-5, post_norm=2, pre_norm=1, M=M, D=D, dtype=sj.SJH_BF16)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        call(stream=C.c_void_p(torch.cuda.current_stream().cuda_stream), **kw)
    for i in range(3):
        x.copy_(torch.randn(M, D, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = xo.clone(), y.clone()
        call(**kw)
        torch.cuda.synchronize()
        assert torch.equal(got[0], xo) and torch.equal(got[1], y), i


@pytest.mark.parametrize("post,pre", [("none", "ln"), ("rms", "ln"), ("ln", "rms")])
@pytest.mark.parametrize("M,D", [(700, 260), (900, 1023), (2000, 1028), (1500, 2049), (800, 8190)])
def test_add_norm_in_place(M, D, post, pre):
    """x_out = x and y = r give the bits of outputs of their own."""
    print(f"add_norm in place {M}x{D} {post} {pre}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(D)
    x, r = (torch.randn(M, D, generator=g, device="cuda") + 3 for _ in range(2))
    kw = dict(x_scale=1.5, r_scale=2.0, eps=1e-5, post_norm=KIND[post], pre_norm=KIND[pre], M=M, D=D, dtype=sj.SJH_F32)
    xo, y = torch.empty_like(x), torch.empty_like(r)
    call(x=x, r=r, x_out=xo, y=y, **kw)
    torch.cuda.synchronize()
    for _ in range(3):
        x1, r1 = x.clone(), r.clone()
        call(x=x1, r=r1, x_out=x1, y=r1, **kw)
        torch.cuda.synchronize()
        assert torch.equal(x1, xo) and torch.equal(r1, y)
