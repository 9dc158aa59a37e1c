"""Timed cases of the windowed / paged attention operators and of the query-key norm with position rotation.

`run` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, with `own` set, through
patchaugnet_amd.attention.  `exact` states the same operators in 64 bits, one head at a time, without this repository's code.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
_EPS = 1e-6


def listed():
    return [
        # one step of a served stream: a single new token for each of eight sequences; launch latency is all there is
        dict(name="norm-step", op="norm", dtype="bfloat16", B=8, N=1, H=8, Hk=2, D=64, rot=64, axes=0, far=200000, train=False),
        # training pass over the points of a level, rotated by their three coordinates: 18 clouds of 1024 points (the quadruplet tuple)
        dict(name="norm-coords-train", op="norm", dtype="float32", B=18, N=1024, H=8, Hk=8, D=64, rot=48, axes=3, far=0, train=True),
        # training pass over long token sequences with shared key heads
        dict(name="norm-long-train", op="norm", dtype="bfloat16", B=8, N=4096, H=16, Hk=4, D=128, rot=128, axes=0, far=4096, train=True),
        # one small cloud level, exact type, every point sees its neighbours in the serial order on both sides
        dict(name="window-small", op="window", dtype="float32", B=1, N=64, M=64, H=8, Hk=8, D=32, left=16, right=16, sinks=1, ragged=0, chunk=False, train=False),
        # a padded batch of 32 clouds with different point counts, windows on both sides
        dict(name="window-ragged", op="window", dtype="float16", B=32, N=1001, M=1001, H=8, Hk=8, D=64, left=64, right=64, sinks=4, ragged=7, chunk=False, train=False),
        # a long prompt, causal, shared key heads
        dict(name="window-long", op="window", dtype="bfloat16", B=4, N=16384, M=16384, H=16, Hk=4, D=128, left=1023, right=0, sinks=4, ragged=0, chunk=False, train=False),
        # training pass in the framework's own type over the quadruplet tuple's 1024-point level
        dict(name="window-train-f32", op="window", dtype="float32", B=18, N=1024, M=1024, H=8, Hk=8, D=32, left=128, right=128, sinks=4, ragged=0, chunk=False, train=True),
        # training pass over 4096-point serial orders, causal, shared key heads
        dict(name="window-train-bf16", op="window", dtype="bfloat16", B=4, N=4096, M=4096, H=16, Hk=4, D=64, left=511, right=0, sinks=4, ragged=0, chunk=False, train=True),
        # one stream with a short cache: latency
        dict(name="paged-short", op="paged", dtype="bfloat16", B=1, top=100, page=16, H=8, Hk=2, D=64, left=-1, sinks=0, ragged=3),
        # many streams with long caches of different lengths, everything visible
        dict(name="paged-long", op="paged", dtype="bfloat16", B=48, top=16384, page=64, H=32, Hk=8, D=128, left=-1, sinks=0, ragged=5),
        # one new token of each of 32 streams into the cache
        dict(name="append-step", op="append", dtype="bfloat16", B=32, T=1, top=4000, page=16, Hk=8, D=128, ragged=11),
        # prompts of different lengths into the cache
        dict(name="append-prompt", op="append", dtype="float16", B=16, T=2048, top=2048, page=64, Hk=8, D=128, ragged=13),
    ]


# --------------------------------------------------------------------------------------------------------------------- drawn cases
def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    hk = rng.choice([1, 2, 3, 4, 8])
    return hk * rng.choice([1, 1, 2, 3, 4, 8]), hk


def _draw_once(rng):
    op = rng.choice(["norm", "norm", "window", "window", "window", "paged", "paged", "append"])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    h, hk = _heads(rng)
    if op == "norm":
        axes = rng.choice([0, 0, 1, 3])
        d = rng.choice([32, 40, 64, 66, 80, 96, 128, 192, 256])
        step = 2 * max(axes, 1)
        rot = d // step * step if rng.random() < 0.5 else rng.randrange(1, d // step + 1) * step
        return dict(op=op, dtype=dtype, B=_logint(rng, 1, 32), N=_logint(rng, 1, 8192), H=h, Hk=hk, D=d, rot=rot, axes=axes,
                    far=_logint(rng, 16, 1000000) if axes == 0 else 0, train=rng.random() < 0.6)
    if op == "window":
        n = _logint(rng, 1, 16384)
        chunk = rng.random() < 0.25
        m = n + _logint(rng, 1, 16384) if chunk else n
        left = _logint(rng, 1, 2048) if rng.random() < 0.85 else -1
        right = rng.choice([0, 0, 0, left if left >= 0 else -1, _logint(rng, 1, 256)])
        return dict(op=op, dtype=dtype, B=_logint(rng, 1, 32), N=n, M=m, H=h, Hk=hk, D=rng.choice([16, 32, 40, 64, 72, 96, 128]),
                    left=left, right=right, sinks=rng.choice([0, 1, 4, 16, 70]), ragged=rng.randrange(1, 1000) if rng.random() < 0.5 else 0,
                    chunk=chunk, train=rng.random() < 0.5)
    if op == "paged":
        return dict(op=op, dtype=dtype, B=_logint(rng, 1, 128), top=_logint(rng, 1, 32768), page=rng.choice([8, 16, 24, 32, 64, 100, 128]), H=h, Hk=hk,
                    D=rng.choice([16, 32, 64, 80, 96, 128]), left=rng.choice([-1, -1, _logint(rng, 1, 4096)]), sinks=rng.choice([0, 1, 4, 33]),
                    ragged=rng.randrange(1, 1000))
    t = _logint(rng, 1, 2048)
    return dict(op=op, dtype=dtype, B=_logint(rng, 1, 64), T=t, top=t + _logint(rng, 1, 2048), page=rng.choice([8, 16, 24, 32, 64, 128]), Hk=hk,
                D=rng.choice([16, 32, 64, 80, 96, 128]), ragged=rng.randrange(1, 1000))


def draw(rng):
    """A case of the same ranges that costs no more than the largest listed one (32-bit cases: a quarter of it, their plain and own rates are lower)."""
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        case = _draw_once(rng)
        if case["op"] in ("window", "paged") and case["B"] * max(case.get("M", 0), case.get("top", 0)) * case["Hk"] * case["D"] > 48 * 16384 * 8 * 128:
            continue
        if case["op"] == "window" and case["B"] * case["H"] * case["N"] * case["M"] > 4 * 16 * 16384 * 16384:
            continue
        w = work(case)
        cut = 4 if case["dtype"] == "float32" else 1
        if w["bytes"] <= most["bytes"] and w["flops"] * cut <= most["flops"]:
            return case


# ------------------------------------------------------------------------------------------------------------------------- the cases' data
def _lengths(case):
    """Lengths of the sequences of a batch, from the case alone (its mix number), the first one the longest allowed."""
    rs = np.random.RandomState(case["ragged"])
    if case["op"] == "append":
        top, low = case["T"], 1
    elif case["op"] == "paged":
        top, low = case["top"], max(1, case["top"] // 4)
    else:
        top, low = case["N"], max(1, case["N"] // 4)
    if not case["ragged"]:
        return np.full(case["B"], top, dtype=np.int64)
    out = rs.randint(low, top + 1, size=case["B"]).astype(np.int64)
    out[0] = top
    return out


def _starts(case):
    """Position of the first query (window, with a cached prefix) or of the first new token (append)."""
    rs = np.random.RandomState(1000 + case["ragged"])
    if case["op"] == "append":
        room = case["top"] - case["T"]
        return rs.randint(0, room + 1, size=case["B"]).astype(np.int64)
    if not case["chunk"]:
        return np.zeros(case["B"], dtype=np.int64)
    room = case["M"] - case["N"]
    out = rs.randint(0, room + 1, size=case["B"]).astype(np.int64)
    out[0] = room
    return out


def _counts(case):
    """Keys in view of every query of the batch, summed: a range count, no mask is built."""
    if case["op"] == "paged":
        p = _lengths(case) - 1
        left, right, sinks, length = case["left"], 0, case["sinks"], p + 1
    else:
        starts, rows = _starts(case), _lengths(case)
        p = np.concatenate([s + np.arange(r) for s, r in zip(starts, rows)])
        length = np.repeat(starts + rows, rows)
        left, right, sinks = case["left"], case["right"], case["sinks"]
    hi = length if right < 0 else np.minimum(length, p + right + 1)          # one past the last key in view
    lo = np.zeros_like(p) if left < 0 else np.maximum(p - left, 0)
    return int(np.sum(np.maximum(hi - lo, 0) + np.minimum(np.minimum(lo, sinks), hi)))


def work(case):
    s = _SIZE[case["dtype"]]
    op = case["op"]
    if op == "norm":
        rows = case["B"] * case["N"]
        x = rows * (case["H"] + case["Hk"]) * case["D"]
        moved = x * s * (4 if case["train"] else 2) + rows * 4 * max(case["axes"], 1)
        return {"bytes": moved, "flops": x * (18 if case["train"] else 7)}
    if op == "window":
        rows = int(_lengths(case).sum())
        keys = int((_lengths(case) + _starts(case)).sum())
        q, kv = rows * case["H"] * case["D"], keys * case["Hk"] * case["D"]
        moved = (2 * q + 2 * kv) * s
        flops = 4 * case["D"] * case["H"] * _counts(case)
        if case["train"]:                                    # read q, k, v, dout, write out, dq, dk, dv: each once
            moved, flops = (4 * q + 4 * kv) * s, flops * 7 // 2
        return {"bytes": moved, "flops": flops}
    if op == "paged":
        seen = _counts(case)
        return {"bytes": 2 * seen * case["Hk"] * case["D"] * s + 2 * case["B"] * case["H"] * case["D"] * s, "flops": 4 * case["D"] * case["H"] * seen}
    new = int(_lengths(case).sum())
    return {"bytes": 4 * new * case["Hk"] * case["D"] * s, "flops": 0}


def _table(case, gen, lengths):
    """Pages of a pool dealt out in a random order: (table (B, pages per sequence), pages in the pool)."""
    per = [-(-int(n) // case["page"]) for n in lengths]
    width, total = max(per), sum(per) + 3
    order = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.zeros((case["B"], width), dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    """Inputs on the GPU.  Queries and keys are the unit-variance rows that the norm hands on, values and gradients are normal."""
    host = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=dev, device="cuda") * scale).to(dt)

    st = {"case": case}
    op = case["op"]
    if op == "norm":
        B, N, H, Hk, D = (case[k] for k in ("B", "N", "H", "Hk", "D"))
        qkv = normal(B, N, H + 2 * Hk, D, scale=1.7)                         # one projection's output: queries, keys and values side by side
        st["q"], st["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hk]
        st["qw"] = 1.0 + 0.2 * torch.randn(D, generator=dev, device="cuda")
        st["kw"] = 1.0 + 0.2 * torch.randn(D, generator=dev, device="cuda")
        if case["axes"]:
            st["positions"] = torch.rand(B, N, case["axes"], generator=dev, device="cuda") * 2 - 1
            f = case["rot"] // (2 * case["axes"])
            st["inv_freq"] = (math.pi * 64.0 ** (torch.arange(f, dtype=torch.float64) / max(f, 1))).expand(case["axes"], f).contiguous().float().cuda()
        else:
            first = torch.randint(0, max(case["far"] - N, 1), (B, 1), generator=host)
            st["positions"] = (first + torch.arange(N)).to(torch.int32).cuda()
            f = case["rot"] // 2
            st["inv_freq"] = (10000.0 ** -(torch.arange(f, dtype=torch.float64) / f)).view(1, f).float().cuda()
        if case["train"]:
            for k in ("q", "k", "qw", "kw"):
                st[k].requires_grad_()
            st["dq"], st["dk"] = normal(B, N, H, D), normal(B, N, Hk, D)
        return st
    if op == "window":
        B, N, M, H, Hk, D = (case[k] for k in ("B", "N", "M", "H", "Hk", "D"))
        st["q"], st["k"], st["v"] = normal(B, N, H, D), normal(B, M, Hk, D), normal(B, M, Hk, D)
        starts, rows = _starts(case), _lengths(case)
        st["lengths"] = torch.from_numpy(starts + rows).to(torch.int32).cuda() if case["ragged"] or case["chunk"] else None
        st["q_start"] = torch.from_numpy(starts).to(torch.int32).cuda() if case["chunk"] else None
        if case["train"]:
            for k in ("q", "k", "v"):
                st[k].requires_grad_()
            st["dout"] = normal(B, N, H, D)
        return st
    lengths = _lengths(case)
    ends = lengths + _starts(case) if op == "append" else lengths
    table, pages = _table(case, host, ends)
    st["table"] = table.cuda()
    st["k_pages"] = normal(pages, case["page"], case["Hk"], case["D"])
    st["v_pages"] = normal(pages, case["page"], case["Hk"], case["D"])
    if op == "paged":
        st["q"] = normal(case["B"], case["H"], case["D"])
        st["lengths"] = torch.from_numpy(lengths).to(torch.int32).cuda()
    else:
        st["k"], st["v"] = normal(case["B"], case["T"], case["Hk"], case["D"]), normal(case["B"], case["T"], case["Hk"], case["D"])
        st["starts"] = torch.from_numpy(_starts(case)).to(torch.int32).cuda()
        st["counts"] = torch.from_numpy(lengths).to(torch.int32).cuda()
    return st


def _opt(n):
    return None if n < 0 else n


def run(st):
    return _run_own(st) if own else _PLAIN[st["case"]["op"]](st)


def _run_own(st):
    from patchaugnet_amd import attention
    c = st["case"]
    if c["op"] == "norm":
        q, k = attention.qk_norm_rotary(st["q"], st["k"], st["qw"], st["kw"], positions=st["positions"], inv_freq=st["inv_freq"], eps=_EPS)
        if not c["train"]:
            return q, k
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (st["q"], st["k"], st["qw"], st["kw"]), (st["dq"], st["dk"]))
    if c["op"] == "window":
        out = attention.window_attention(st["q"], st["k"], st["v"], left=_opt(c["left"]), right=_opt(c["right"]), sinks=c["sinks"],
                                         lengths=st["lengths"], q_start=st["q_start"])
        if not c["train"]:
            return out
        return (out.detach(),) + torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["dout"])
    if c["op"] == "paged":
        return attention.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], left=_opt(c["left"]), sinks=c["sinks"])
    attention.paged_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["starts"], counts=st["counts"])
    return st["k_pages"], st["v_pages"]


# --------------------------------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(st):
    c = st["case"]
    half = c["rot"] // 2
    with torch.no_grad():
        pos = st["positions"].double()
        pos = pos if c["axes"] else pos.unsqueeze(-1)
        ang = (pos.unsqueeze(-1) * st["inv_freq"].double()).flatten(-2)       # far positions lose their angle in 32 bits
        cos, sin = ang.cos().float().unsqueeze(2), ang.sin().float().unsqueeze(2)

        def rotate(x, s):
            u, v = x[..., :half], x[..., half:2 * half]
            return torch.cat([u * cos - v * s, u * s + v * cos, x[..., 2 * half:]], dim=-1)

        outs, grads, wgrads = [], [], []
        for x, w, g in ((st["q"], st["qw"], st.get("dq")), (st["k"], st["kw"], st.get("dk"))):
            xf = x.float()
            r = (xf.square().mean(-1, keepdim=True) + _EPS).rsqrt()
            n = xf * r
            outs.append(rotate(n * w, sin).to(x.dtype))
            if g is not None:
                t = rotate(g.float(), -sin)
                wgrads.append((t * n).sum((0, 1, 2)))
                t = t * w
                grads.append((r * (t - n * (t * n).mean(-1, keepdim=True))).to(x.dtype))
    return tuple(outs) if st.get("dq") is None else tuple(outs + grads + wgrads)


def _view(c, p, j, length):
    """Which keys j (row vector) a query at p (column vector) sees."""
    vis = (j < length) & (p < length)
    if c["right"] >= 0:
        vis = vis & (j <= p + c["right"])
    if c["left"] >= 0:
        vis = vis & ((j >= p - c["left"]) | (j < c["sinks"]))
    return vis


def _plain_window(st, block=512):
    """Blocks of queries against the keys that any of them can see: the first tokens and one contiguous range."""
    c = st["case"]
    B, N, M, H, Hk, D = (c[k] for k in ("B", "N", "M", "H", "Hk", "D"))
    G, scale = H // Hk, 1.0 / math.sqrt(D)
    dt = st["q"].dtype
    with torch.no_grad():
        length = st["lengths"].long().view(B, 1, 1) if st["lengths"] is not None else torch.full((B, 1, 1), M, device="cuda")
        start = st["q_start"].long().view(B, 1, 1) if st["q_start"] is not None else torch.zeros((B, 1, 1), dtype=torch.long, device="cuda")
        kf, vf = (st[n].float().permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))                     # (B, Hk, M, D)
        qf = st["q"].float().view(B, N, Hk, G, D).permute(0, 2, 3, 1, 4).contiguous()                    # (B, Hk, G, N, D)
        out = torch.empty_like(qf)
        train = c["train"]
        if train:
            do = st["dout"].float().view(B, N, Hk, G, D).permute(0, 2, 3, 1, 4).contiguous()
            dq, dk, dv = torch.empty_like(qf), torch.zeros_like(kf), torch.zeros_like(vf)
        low, high = (0, M - N) if c["chunk"] else (0, 0)
        for i0 in range(0, N, block):
            i1 = min(i0 + block, N)
            lo = 0 if c["left"] < 0 else max(0, i0 + low - c["left"])
            hi = M if c["right"] < 0 else min(M, i1 + high + c["right"])
            first = min(lo, c["sinks"])
            js = torch.cat([torch.arange(first, device="cuda"), torch.arange(lo, max(hi, lo), device="cuda")])
            p = start + torch.arange(i0, i1, device="cuda").view(1, -1, 1)
            vis = _view(c, p, js.view(1, 1, -1), length)                                                  # (B, rows, keys)
            vis = vis.view(B, 1, 1, i1 - i0, -1).expand(B, Hk, G, -1, -1).reshape(B, Hk, G * (i1 - i0), -1)
            ks, vs = kf[:, :, js], vf[:, :, js]
            qs = qf[:, :, :, i0:i1].reshape(B, Hk, G * (i1 - i0), D)
            s = torch.matmul(qs, ks.transpose(2, 3).contiguous()) * scale
            s = s.masked_fill(~vis, float("-inf"))
            top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full(s.shape[:-1] + (1,), float("-inf"))
            e = (s - top.clamp_min(-1e30)).exp()
            tot = e.sum(-1, keepdim=True)
            prob = e / tot.clamp_min(1e-30)
            o = torch.matmul(prob, vs)
            out[:, :, :, i0:i1] = o.view(B, Hk, G, i1 - i0, D)
            if train:
                g = do[:, :, :, i0:i1].reshape(B, Hk, G * (i1 - i0), D)
                dv.index_add_(2, js, torch.matmul(prob.transpose(2, 3).contiguous(), g))
                dp = torch.matmul(g, vs.transpose(2, 3).contiguous())
                ds = prob * (dp - (g * o).sum(-1, keepdim=True)) * scale
                dq[:, :, :, i0:i1] = torch.matmul(ds, ks).view(B, Hk, G, i1 - i0, D)
                dk.index_add_(2, js, torch.matmul(ds.transpose(2, 3).contiguous(), qs))

        def back_q(t):
            return t.permute(0, 3, 1, 2, 4).reshape(B, N, H, D).to(dt)

        def back_kv(t):
            return t.permute(0, 2, 1, 3).contiguous().to(dt)

        if not train:
            return back_q(out)
        return back_q(out), back_q(dq), back_kv(dk), back_kv(dv)


def _plain_paged(st):
    c = st["case"]
    B, H, Hk, D = (c[k] for k in ("B", "H", "Hk", "D"))
    G = H // Hk
    with torch.no_grad():
        lengths = st["lengths"].long()
        j = torch.arange(st["table"].shape[1] * c["page"], device="cuda").view(1, -1)
        vis = j < lengths.view(B, 1)
        if c["left"] >= 0:
            vis = vis & ((j >= lengths.view(B, 1) - 1 - c["left"]) | (j < c["sinks"]))
        out = torch.empty_like(st["q"])
        for b in range(B):
            js = vis[b].nonzero().flatten()
            page, at = st["table"][b].long()[js // c["page"]], js % c["page"]
            k, v = (st[n][page, at].float().permute(1, 0, 2) for n in ("k_pages", "v_pages"))             # (Hk, keys, D)
            q = st["q"][b].float().view(Hk, G, D)
            s = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(D)
            e = (s - s.amax(-1, keepdim=True)).exp()
            out[b] = torch.matmul(e / e.sum(-1, keepdim=True), v.contiguous()).view(H, D).to(out.dtype)
    return out


def _plain_append(st):
    c = st["case"]
    with torch.no_grad():
        t = torch.arange(c["T"], device="cuda").view(1, -1)
        b, i = (t < st["counts"].long().view(-1, 1)).nonzero(as_tuple=True)
        j = st["starts"].long()[b] + i
        page, at = st["table"].long()[b, j // c["page"]], j % c["page"]
        st["k_pages"][page, at] = st["k"][b, i]
        st["v_pages"][page, at] = st["v"][b, i]
    return st["k_pages"], st["v_pages"]


_PLAIN = {"norm": _plain_norm, "window": _plain_window, "paged": _plain_paged, "append": _plain_append}


# ------------------------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "window": _exact_window, "paged": _exact_paged, "append": _exact_append}[case["op"]](case, st)


def _exact_norm(c, st):
    half, axes = c["rot"] // 2, max(c["axes"], 1)
    f = half // axes
    pos = st["positions"].double().reshape(c["B"], c["N"], axes)
    z = torch.empty(c["B"], c["N"], 1, half, dtype=torch.complex128, device="cuda")
    for a in range(axes):
        for i in range(f):
            ang = pos[:, :, a] * float(st["inv_freq"][a, i])
            z[:, :, 0, a * f + i] = torch.complex(torch.cos(ang), torch.sin(ang))

    def turn(x, by):
        w = torch.complex(x[..., :half], x[..., half:c["rot"]]) * by
        return torch.cat([w.real, w.imag, x[..., c["rot"]:]], dim=-1)

    outs, dxs, dws = [], [], []
    for x, w, g in ((st["q"], st["qw"], st.get("dq")), (st["k"], st["kw"], st.get("dk"))):
        x, w = x.double(), w.double()
        rms = torch.sqrt((x * x).sum(-1, keepdim=True) / c["D"] + _EPS)
        outs.append(turn(x / rms * w, z))
        if g is not None:
            u = turn(g.double(), z.conj())
            dws.append((u * x / rms).sum((0, 1, 2)))
            u = u * w
            dxs.append(u / rms - x * (u * x).sum(-1, keepdim=True) / (c["D"] * rms ** 3))
    return tuple(outs + dxs + dws)


def _exact_window(c, st):
    """Head by head on dense score matrices; the mask from the definition."""
    B, N, M, H, Hk, D = (c[k] for k in ("B", "N", "M", "H", "Hk", "D"))
    if B * H * N * M * D * (7 if c["train"] else 2) > 3e13:
        return None
    lens, starts = _starts(c) + _lengths(c), _starts(c)
    if not (c["ragged"] or c["chunk"]):
        lens = np.full(B, M)
    out = torch.zeros(B, N, H, D, dtype=torch.float64, device="cuda")
    if c["train"]:
        dq, dk, dv = torch.zeros_like(out), torch.zeros(B, M, Hk, D, dtype=torch.float64, device="cuda"), torch.zeros(B, M, Hk, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, m = int(min(N, max(lens[b] - starts[b], 0))), int(min(lens[b], M))           # rows and keys of this sequence
        pos = int(starts[b]) + torch.arange(n, device="cuda")
        gap = torch.arange(m, device="cuda")[None, :] - pos[:, None]                     # key minus query
        hide = torch.zeros(n, m, dtype=torch.bool, device="cuda")
        if c["left"] >= 0:
            hide |= gap < -c["left"]
        hide[:, :c["sinks"]] = False
        if c["right"] >= 0:
            hide |= gap > c["right"]
        for h in range(H):
            g = h * Hk // H
            q, k, v = st["q"][b, :n, h].double(), st["k"][b, :m, g].double(), st["v"][b, :m, g].double()
            s = (q @ k.t().contiguous()).div_(math.sqrt(D)).masked_fill_(hide, float("-inf"))
            pr = torch.softmax(s, dim=1).nan_to_num_(nan=0.0)
            o = pr @ v
            out[b, :n, h] = o
            if c["train"]:
                do = st["dout"][b, :n, h].double()
                dv[b, :m, g] += pr.t().contiguous() @ do
                ds = (do @ v.t().contiguous()).sub_((do * o).sum(1, keepdim=True)).mul_(pr).div_(math.sqrt(D))
                dq[b, :n, h] = ds @ k
                dk[b, :m, g] += ds.t().contiguous() @ q
    return (out, dq, dk, dv) if c["train"] else out


def _exact_paged(c, st):
    B, H, Hk, D, page = (c[k] for k in ("B", "H", "Hk", "D", "page"))
    out = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    lens, table = _lengths(c), st["table"].cpu()
    for b in range(B):
        n = int(lens[b])
        ids = table[b, :-(-n // page)].long().cuda()
        lo = 0 if c["left"] < 0 else max(0, n - 1 - c["left"])
        keep = torch.tensor(sorted(set(range(lo, n)) | set(range(min(c["sinks"], n)))), device="cuda")
        for g in range(Hk):
            k = st["k_pages"][ids, :, g].reshape(-1, D)[keep].double()
            v = st["v_pages"][ids, :, g].reshape(-1, D)[keep].double()
            heads = slice(g * H // Hk, (g + 1) * H // Hk)
            pr = torch.softmax((st["q"][b, heads].double() / math.sqrt(D)) @ k.t().contiguous(), dim=1)
            out[b, heads] = pr @ v
    return out


def _exact_append(c, st):
    k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
    lens, starts, table = _lengths(c), _starts(c), st["table"].cpu().numpy()
    slot = torch.full((k_pages.shape[0] * c["page"],), -1, dtype=torch.long)
    for b in range(c["B"]):
        j = starts[b] + np.arange(lens[b])
        where = table[b, j // c["page"]].astype(np.int64) * c["page"] + j % c["page"]
        slot[torch.from_numpy(where)] = torch.from_numpy(b * c["T"] + np.arange(lens[b]))
    slot = slot.cuda()
    hit = (slot >= 0).nonzero().flatten()
    for pool, new in ((k_pages, st["k"]), (v_pages, st["v"])):
        pool.view(-1, c["Hk"], c["D"])[hit] = new.double().reshape(-1, c["Hk"], c["D"])[slot[hit]]
    return k_pages, v_pages
