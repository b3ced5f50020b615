"""The kernel-level operators of an encoder block beyond the plain one.

A block of an encoder whose checkpoint has norms on both sides of it, gates per
request, capped or distance-biased attention over packed documents, and low-rank
adapters chosen per request, calls three operators:

  norm  sjh_add_norm     x' = x_scale x + r_scale gate * post(r);  y = pre(x')
  lora  sjh_gemm_lora    out = act(x W^T + bias + scale_a (x A_a^T) B_a^T), a the row's adapter
  attn  sjh_attn_scored  softmax over the visible keys of cap tanh(q.k scale / cap) - slope |p - j|, times v

Key j is visible to the query at position p where j lies in the sequence's
prefix, or where it is not after p (causal), at most ``window`` away and of p's
document, as far as each of these is asked for.

Widths are those of the encoders the benchmark runs (768 and 1024 hidden, 12 and
16 heads of 64, gated layers of 2624), row counts those of its batches: one
request of a few words up to 64 rows of up to 512 tokens, documents of 8192.
``own`` False computes each operator in its plain form in 32 bits; True calls
the framework's kernels.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

EPS = 1e-5
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one short request, all of its tokens: launches and latency
        dict(name="norm_request", op="norm", M=17, D=768, post="rms", pre="rms", gates=1, x_scale=1.0, dtype="bf16"),
        # the throughput batch of the wide encoder, a gate row per request, LayerNorm after the block
        dict(name="norm_bulk", op="norm", M=18432, D=1024, post="ln", pre="rms", gates=64, x_scale=1.0, dtype="bf16"),
        # an encoder that scales its residual stream, fp32 checks, an odd width no vector load divides
        dict(name="norm_odd", op="norm", M=1501, D=771, post="none", pre="ln", gates=0, x_scale=1.4, dtype="fp32"),
        # single tokens of different requests, each with an adapter of its own
        dict(name="lora_tokens", op="lora", M=9, N=2304, K=768, R=16, adapters=16, requests=9, act=0, dtype="bf16"),
        # a batch of requests over a dozen adapters, some rows without one, GELU product
        dict(name="lora_requests", op="lora", M=1501, N=1152, K=768, R=16, adapters=12, requests=24, act=1, dtype="bf16"),
        # the QKV product of the throughput batch, adapters of rank 64
        dict(name="lora_bulk", op="lora", M=18432, N=2304, K=768, R=64, adapters=24, requests=64, act=0, dtype="bf16"),
        # a base held in fp8 under bf16 adapters, down projection of the wide encoder
        dict(name="lora_fp8", op="lora", M=4033, N=1024, K=2624, R=32, adapters=8, requests=16, act=0, dtype="fp8"),
        # one short request
        dict(name="attn_request", op="attn", B=1, lo=73, hi=73, H=12, Hkv=12, Dh=64, cap=30.0, slopes=True, window=0, causal=False,
             prefix=0, docs_lo=0, docs_hi=0, tail=0, dtype="bf16"),
        # typed questions behind a shared state: every question sees the state and itself
        dict(name="attn_questions", op="attn", B=12, lo=500, hi=1000, H=16, Hkv=16, Dh=64, cap=50.0, slopes=False, window=0, causal=False,
             prefix=400, docs_lo=15, docs_hi=60, tail=0, dtype="bf16"),
        # rows packed with documents of any length
        dict(name="attn_packed", op="attn", B=16, lo=1800, hi=2048, H=12, Hkv=12, Dh=64, cap=50.0, slopes=False, window=0, causal=False,
             prefix=0, docs_lo=30, docs_hi=700, tail=0, dtype="bf16"),
        # long documents read from left to right behind a two-way prefix, distance-biased
        dict(name="attn_long", op="attn", B=2, lo=5000, hi=8192, H=12, Hkv=12, Dh=64, cap=0.0, slopes=True, window=0, causal=True,
             prefix=300, docs_lo=0, docs_hi=0, tail=0, dtype="bf16"),
        # the last few tokens of long texts against the keys held of them, shared key heads of 128
        dict(name="attn_tail", op="attn", B=3, lo=6000, hi=8191, H=16, Hkv=4, Dh=128, cap=50.0, slopes=False, window=0, causal=True,
             prefix=0, docs_lo=0, docs_hi=0, tail=5, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["norm", "lora", "attn", "attn"])
        if op == "norm":
            c = dict(op=op, M=_log(rng, 1, 30000), D=rng.choice([768, 1024, 768, 1024, 256, 512, _log(rng, 8, 4096)]), post=rng.choice(["none", "ln", "rms"]),
                     pre=rng.choice(["none", "ln", "rms"]), gates=rng.choice([0, 1, rng.randint(2, 64)]), x_scale=rng.choice([1.0, 1.4]),
                     dtype=rng.choice(["bf16", "bf16", "bf16", "fp32"]))
        elif op == "lora":
            dtype = rng.choice(["bf16", "bf16", "bf16", "fp8", "fp32"])
            M = _log(rng, 1, 2000 if dtype == "fp32" else 20000)
            c = dict(op=op, M=M, N=rng.choice([768, 1024, 1152, 2304, 2624, 4 * rng.randint(40, 700)]), K=64 * rng.choice([12, 16, 18, 41, rng.randint(4, 47)]),
                     R=rng.choice([8, 16, 16, 32, 64, rng.randint(1, 64)]), adapters=rng.randint(1, 24), requests=min(M, rng.randint(1, 64)),
                     act=rng.choice([0, 0, 1, 2]), dtype=dtype)
        else:
            hi = _log(rng, 1, 8192)
            tail = rng.choice([0, 0, 0, rng.randint(1, 16)])
            docs = rng.choice([(0, 0), (0, 0), (1, max(1, hi // 3)), (20, 600)])
            H = rng.choice([12, 16])
            c = dict(op=op, B=_log(rng, 1, 24), lo=rng.randint(max(1, hi // 8), hi), hi=hi, H=H, Hkv=rng.choice([H, H, 4]), Dh=rng.choice([64, 64, 64, 128, 32]),
                     cap=rng.choice([0.0, 30.0, 50.0]), slopes=rng.choice([False, True]), window=rng.choice([0, 0, 64, rng.randint(1, 1500)]),
                     causal=rng.choice([False, False, True]), prefix=rng.choice([0, 0, rng.randint(1, 500)]), docs_lo=docs[0], docs_hi=docs[1], tail=tail,
                     dtype=rng.choice(["bf16", "bf16", "bf16", "fp32"]))
        w = work(c)
        # no more than the largest listed case; fp32, and heads of other sizes, are for small batches
        slow = c["op"] == "attn" and (c["dtype"] == "fp32" or c["Dh"] == 32) or c["dtype"] == "fp32" and c["op"] == "lora"
        if w["flops"] <= (1e10 if slow else 1.6e11) and _cells(c) <= 1.4e9 and w["bytes"] <= 3e8:
            return c


# ------------------------------------------------------------------ sizes --
def _spread(B, lo, hi):
    """B lengths evenly over [lo, hi]."""
    return [lo + round((hi - lo) * (i + 0.5) / B) for i in range(B)] if B > 1 else [hi]


def _klens(c):
    return _spread(c["B"], c["lo"], c["hi"])


def _qlens(c):
    """Queries of each sequence: all of its tokens, or its last one to ``tail``."""
    if not c["tail"]:
        return _klens(c)
    return [min(n, 1 + (i + c["tail"] - 1) % c["tail"]) for i, n in enumerate(_klens(c))]


def _doc_ids(c, n):
    """Document of each of a sequence's n tokens; those of the prefix are one of their own."""
    r = random.Random(7 * n + 1)
    ids = [0] * min(c["prefix"], n)
    d = 0
    while len(ids) < n:
        d += 1
        ids += [(d * 37) % 1009 + 1] * r.randint(c["docs_lo"], c["docs_hi"])
    return np.array(ids[:n], np.int32)


def _visible(c, n, nq):
    """[nq] numbers of visible keys of a sequence's last nq queries of n keys."""
    p = np.arange(n - nq, n)
    lo, hi = np.zeros(nq, np.int64), np.full(nq, n, np.int64)
    if c["window"]:
        lo, hi = np.maximum(p - c["window"], 0), np.minimum(p + c["window"] + 1, n)
    if c["causal"]:
        hi = np.minimum(hi, p + 1)
    if c["docs_hi"]:
        ids = _doc_ids(c, n)
        edge = np.flatnonzero(np.diff(ids)) + 1
        starts = np.concatenate([[0], edge])
        ends = np.concatenate([edge, [n]])
        d = np.searchsorted(starts, p, side="right") - 1
        lo, hi = np.maximum(lo, starts[d]), np.minimum(hi, ends[d])
    pre = min(c["prefix"], n)
    return pre + np.maximum(hi - np.maximum(lo, pre), 0)


def _cells(c):
    """Scores a plain form holds, a bound on its time."""
    return c["H"] * sum(n * q for n, q in zip(_klens(c), _qlens(c))) if c["op"] == "attn" else 0


def _segments(c):
    """(first row, rows, adapter) of each request; one request in eight has no adapter."""
    G, M = c["requests"], c["M"]
    cut = [M * i // G for i in range(G + 1)]
    return [(cut[i], cut[i + 1] - cut[i], -1 if i % 8 == 5 else (5 * i + 3) % c["adapters"]) for i in range(G)]


def work(c):
    es = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "norm":
        M, D = c["M"], c["D"]
        vec = (c["post"] != "none") + (c["pre"] != "none") + (c["pre"] == "ln") + c["gates"]
        return {"bytes": M * D * (8 + 2 * es) + 4 * D * vec + (4 * M if c["gates"] > 1 else 0), "flops": 16 * M * D}
    if c["op"] == "lora":
        M, N, K, R = c["M"], c["N"], c["K"], c["R"]
        seg = [(n, a) for _, n, a in _segments(c) if a >= 0 and n > 0]
        used, rows = len({a for _, a in seg}), sum(n for n, _ in seg)
        ws = N * K + 4 * N if c["dtype"] == "fp8" else es * N * K
        return {"bytes": es * (M * K + M * N + used * R * (K + N)) + ws + 4 * N + 4 * M, "flops": 2 * M * N * K + 2 * rows * R * (K + N)}
    kl, ql = _klens(c), _qlens(c)
    pairs = c["H"] * sum(int(_visible(c, n, q).sum()) for n, q in zip(kl, ql))
    nb = es * c["Dh"] * (2 * c["H"] * sum(ql) + 2 * c["Hkv"] * sum(kl)) + (4 * (sum(kl) + sum(ql)) if c["docs_hi"] else 0)
    return {"bytes": nb, "flops": 4 * c["Dh"] * pairs}


# ----------------------------------------------------------------- inputs --
def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT.get(c["dtype"], torch.bfloat16)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")

    def ints(x):
        return torch.from_numpy(np.asarray(x, np.int32)).cuda()

    if c["op"] == "norm":
        M, D, G = c["M"], c["D"], c["gates"]
        t = {"x": r(M, D) * 3 + r(1, D), "r": (r(M, D) + 0.3 * r(1, D)).to(dt)}
        for side in ("post", "pre"):
            t[side + "_w"] = 1 + 0.1 * r(D) if c[side] != "none" else None
        t["pre_b"] = 0.1 * r(D) if c["pre"] == "ln" else None
        t["gate"] = torch.sigmoid(r(G, D)) if G else None
        # requests one after another, a gate row each
        t["gate_row"] = ints(np.random.default_rng(seed).permutation(G)[np.arange(M) * G // M]) if G > 1 else None
        return t
    if c["op"] == "lora":
        M, N, K, R, n = (c[k] for k in ("M", "N", "K", "R", "adapters"))
        w = r(N, K) * 0.03
        t = {"x": r(M, K).to(dt), "bias": 0.02 * r(N), "a": (r(n, R, K) / math.sqrt(K)).to(dt), "b": (r(n, N, R) * 0.1).to(dt),
             "scale": 0.5 + torch.rand(n, generator=g, device="cuda")}
        if c["dtype"] == "fp8":  # e4m3 codes, one scale per output row
            t["w_scale"] = w.abs().amax(1) / 448.0
            t["w"] = (w / t["w_scale"][:, None]).to(torch.float8_e4m3fn)
        else:
            t["w"], t["w_scale"] = w.to(dt), None
        ad = np.empty(M, np.int32)
        for first, rows, a in _segments(c):
            ad[first:first + rows] = a
        t["adapter"] = ints(ad)
        return t
    perm = np.random.default_rng(seed).permutation(c["B"])
    kl, ql = [np.array(v)[perm] for v in (_klens(c), _qlens(c))]
    H, Hkv, Dh = c["H"], c["Hkv"], c["Dh"]
    t = {"kl": kl.tolist(), "ql": ql.tolist()}
    t["q"] = (2.0 * r(int(ql.sum()), H, Dh)).to(dt)
    t["k"], t["v"] = (r(int(kl.sum()), Hkv, Dh).to(dt) for _ in range(2))
    t["q_start"], t["k_start"] = ints(np.cumsum(ql) - ql), ints(np.cumsum(kl) - kl)
    t["q_len"], t["k_len"], t["q_pos"] = ints(ql), ints(kl), ints(kl - ql)
    t["prefix"] = ints(np.minimum(c["prefix"], kl)) if c["prefix"] else None
    t["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H) if c["slopes"] else None
    t["k_doc"] = t["q_doc"] = None
    if c["docs_hi"]:
        ids = [_doc_ids(c, n) for n in kl]
        t["k_doc"] = ints(np.concatenate(ids))
        t["q_doc"] = ints(np.concatenate([d[len(d) - q:] for d, q in zip(ids, ql)]))
    return t


def prepare(case, seed):
    c = case
    st = {"case": c, "in": _inputs(c, seed)}
    if own:
        st["call"], st["out"], st["keep"] = _call(c, st["in"])
    return st


# ---------------------------------------------------------------- own calls --
def _call(c, t):
    """The entry point, its arguments, the buffers that a program keeps for it."""
    import ctypes

    import snapjudge_amd as sj

    lib = sj.lib()
    dt = sj.SJH_F32 if c["dtype"] == "fp32" else sj.SJH_BF16
    keep = [t]

    def p(x):
        return None if x is None else x.data_ptr()

    def workspace(n):
        w = torch.empty(max(int(n), 1), dtype=torch.uint8, device="cuda")
        keep.append(w)
        return w.data_ptr(), int(n)

    if c["op"] == "norm":
        kinds = {"none": sj.SJH_NORM_NONE, "ln": sj.SJH_NORM_LAYER, "rms": sj.SJH_NORM_RMS}
        out = (torch.empty_like(t["x"]), torch.empty_like(t["r"]))
        a = sj.AddNormArgs(x=p(t["x"]), r=p(t["r"]), x_out=p(out[0]), y=p(out[1]), post_norm=kinds[c["post"]], post_w=p(t["post_w"]),
                           pre_norm=kinds[c["pre"]], pre_w=p(t["pre_w"]), pre_b=p(t["pre_b"]), gate=p(t["gate"]), n_gates=c["gates"],
                           gate_row=p(t["gate_row"]), x_scale=c["x_scale"], r_scale=1.0, eps=EPS, M=c["M"], D=c["D"], dtype=dt)
        fn = lib.sjh_add_norm
    elif c["op"] == "lora":
        out = torch.empty(c["M"], c["N"], dtype=t["x"].dtype, device="cuda")
        ws, n = workspace(lib.sjh_gemm_lora_workspace(c["M"], c["R"]))
        a = sj.LoraArgs(x=p(t["x"]), w=p(t["w"]), w_scale=p(t["w_scale"]), bias=p(t["bias"]), a=p(t["a"]), b=p(t["b"]), scale=p(t["scale"]),
                        adapter=p(t["adapter"]), out=p(out), workspace=ws, workspace_bytes=n, M=c["M"], N=c["N"], K=c["K"], R=c["R"],
                        n_adapters=c["adapters"], act=c["act"], dtype=dt)
        fn = lib.sjh_gemm_lora
    else:
        out = torch.empty_like(t["q"])
        a = sj.AttnScoredArgs(q=p(t["q"]), k=p(t["k"]), v=p(t["v"]), o=p(out), q_start=p(t["q_start"]), q_len=p(t["q_len"]), k_start=p(t["k_start"]),
                              k_len=p(t["k_len"]), q_pos=p(t["q_pos"]), B=c["B"], H=c["H"], Hkv=c["Hkv"], Dh=c["Dh"], q_rows=len(t["q"]),
                              k_rows=len(t["k"]), max_q=max(t["ql"]), max_k=max(t["kl"]), softcap=c["cap"], slopes=p(t["slopes"]),
                              window=c["window"], causal=int(c["causal"]), prefix=p(t["prefix"]), q_doc=p(t["q_doc"]), k_doc=p(t["k_doc"]), dtype=dt)
        a.workspace, a.workspace_bytes = workspace(lib.sjh_attn_scored_workspace(ctypes.byref(a)))
        fn = lib.sjh_attn_scored
    ref = ctypes.byref(a)
    return (lambda: sj.check(fn(ref, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))), out, keep


# -------------------------------------------------------------- plain forms --
def _norm(x, kind, w, b):
    if kind == "none":
        return x
    if kind == "ln":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    return y if b is None else y + b


def _plain_norm(c, t):
    u = _norm(t["r"].float(), c["post"], t["post_w"], None)
    if t["gate"] is not None:
        u = u * (t["gate"][t["gate_row"].long()] if t["gate_row"] is not None else t["gate"])
    x = c["x_scale"] * t["x"] + u
    return x, _norm(x, c["pre"], t["pre_w"], t["pre_b"]).to(t["r"].dtype)


def _plain_lora(c, t):
    x = t["x"].float()
    w = t["w"].float()
    if t["w_scale"] is not None:
        w = w * t["w_scale"][:, None]
    y = x @ w.t() + t["bias"]
    for first, rows, a in _segments(c):
        if a >= 0 and rows > 0:
            s = slice(first, first + rows)
            y[s] += t["scale"][a] * ((x[s] @ t["a"][a].float().t()) @ t["b"][a].float().t())
    if c["act"] == 1:
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif c["act"] == 2:
        y = y.clamp(min=0)
    return y.to(t["x"].dtype)


def _mask(c, t, n, nq, q0, k0):
    """[nq, n] truth of what a sequence's queries see, and their distances."""
    p = torch.arange(n - nq, n, device="cuda")[:, None]
    j = torch.arange(n, device="cuda")[None]
    see = torch.ones(nq, n, dtype=torch.bool, device="cuda")
    if c["causal"]:
        see &= j <= p
    if c["window"]:
        see &= (p - j).abs() <= c["window"]
    if c["docs_hi"]:
        see &= t["q_doc"][q0:q0 + nq, None] == t["k_doc"][None, k0:k0 + n]
    if c["prefix"]:
        see |= j < c["prefix"]
    return see, (p - j).abs()


def _plain_attn(c, t):
    H, G, Dh = c["H"], c["H"] // c["Hkv"], c["Dh"]
    out = torch.empty_like(t["q"])
    q0 = k0 = 0
    for n, nq in zip(t["kl"], t["ql"]):
        see, dist = _mask(c, t, n, nq, q0, k0)
        # heads at once as far as their scores take a gigabyte
        hs = G * max(1, min(c["Hkv"], int(2.5e8 / (n * nq * G))))
        for h in range(0, H, hs):
            he = min(h + hs, H)
            q = t["q"][q0:q0 + nq, h:he].transpose(0, 1).float()
            k, v = (t[x][k0:k0 + n, h // G:he // G].transpose(0, 1).float().repeat_interleave(G, 0) for x in ("k", "v"))
            s = torch.bmm(q, k.transpose(1, 2).contiguous()) * Dh ** -0.5
            if c["cap"]:
                s = c["cap"] * torch.tanh(s / c["cap"])
            if t["slopes"] is not None:
                s = s - t["slopes"][h:he, None, None] * dist
            s = s.masked_fill(~see, -math.inf)
            e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
            o = torch.bmm(e, v.contiguous()) / e.sum(-1, keepdim=True).clamp(min=1e-30)
            out[q0:q0 + nq, h:he] = o.transpose(0, 1).to(out.dtype)
        q0, k0 = q0 + nq, k0 + n
    return out


def run(state):
    if own:
        state["call"]()
        return state["out"]
    return {"norm": _plain_norm, "lora": _plain_lora, "attn": _plain_attn}[state["case"]["op"]](state["case"], state["in"])


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    c, t = case, _inputs(case, seed)

    def d(x):
        return x.to(torch.float64)

    if c["op"] == "norm":
        def norm(z, kind, w, b):
            if kind == "none":
                return z
            m = z.mean(1) if kind == "ln" else torch.zeros(len(z), dtype=z.dtype, device=z.device)
            dev = z - m[:, None]
            z = dev / ((dev ** 2).sum(1) / z.shape[1] + EPS).sqrt()[:, None] * d(w)
            return z if b is None else z + d(b)

        u = norm(d(t["r"]), c["post"], t["post_w"], None)
        if c["gates"]:
            rows = t["gate_row"] if t["gate_row"] is not None else torch.zeros(c["M"], dtype=torch.int32, device="cuda")
            u = u * d(t["gate"]).index_select(0, rows)
        x = d(t["x"]) * c["x_scale"] + u
        return x, norm(x, c["pre"], t["pre_w"], t["pre_b"])
    if c["op"] == "lora":
        w = d(t["w"].float())
        if t["w_scale"] is not None:
            w = w * d(t["w_scale"]).unsqueeze(1)
        y = torch.nn.functional.linear(d(t["x"]), w, d(t["bias"]))
        for a in range(c["adapters"]):
            rows = torch.nonzero(t["adapter"] == a).flatten()
            if len(rows):
                full = d(t["b"][a]) @ d(t["a"][a]) * d(t["scale"][a])  # the adapter's whole matrix [N, K]
                y[rows] += torch.nn.functional.linear(d(t["x"][rows]), full)
        if c["act"] == 1:
            return y * torch.special.ndtr(y)
        return torch.where(y > 0, y, torch.zeros_like(y)) if c["act"] == 2 else y
    G = c["H"] // c["Hkv"]
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for n, nq in zip(t["kl"], t["ql"]):
        for r0 in range(0, nq, 2048):  # rows at once
            r1 = min(r0 + 2048, nq)
            pos = torch.arange(n - nq + r0, n - nq + r1, device="cuda")
            gap = pos.unsqueeze(1) - torch.arange(n, device="cuda")
            hide = torch.zeros(gap.shape, dtype=torch.bool, device="cuda")
            if c["causal"]:
                hide |= gap < 0
            if c["window"]:
                hide |= gap.abs() > c["window"]
            if c["docs_hi"]:
                hide |= t["q_doc"][q0 + r0:q0 + r1].unsqueeze(1) != t["k_doc"][k0:k0 + n]
            hide[:, :c["prefix"]] = hide[:, :c["prefix"]] & (c["prefix"] == 0)
            for h in range(c["H"]):
                kk, vv = d(t["k"][k0:k0 + n, h // G]), d(t["v"][k0:k0 + n, h // G])
                z = d(t["q"][q0 + r0:q0 + r1, h]) @ kk.t().contiguous() / math.sqrt(c["Dh"])
                if c["cap"]:
                    z = torch.tanh(z / c["cap"]) * c["cap"]
                if t["slopes"] is not None:
                    z = z - d(t["slopes"][h]) * gap.abs()
                z[hide] = -math.inf
                none = hide.all(1)
                z[none] = 0.0
                w = torch.softmax(z, 1)
                w[none] = 0.0
                out[q0 + r0:q0 + r1, h] = w @ vv
        q0, k0 = q0 + nq, k0 + n
    return out
