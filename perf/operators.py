"""The operators of an attention block over packed structures, in plain torch and as the library's calls.

`norm_rotate`: queries and keys normalised per head and rotated by angles that are linear in an atom's (token's) position, forward and
backward.  `structure_attention`: attention inside every structure of a packed batch (grouped heads, causal or not, any lengths), forward,
backward, and with single queries over long keys.  The plain forms compute in 32 bits (angles in 64) and round once at the end.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# ------------------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # a serving step: one new token of each of 8 sequences, far positions, norm and rotation
        dict(name="rotate_step_8", op="rotate", n=8, hq=16, hk=4, d=128, dtype="bf16", axes=1, norm=True, pairing="halves", span=100000.0,
             train=False),
        # the batch of 512 molecules (10 to 40 atoms) that the benchmark poses: 4 heads x 32, axes x, y, z; gradients down to the positions
        dict(name="rotate_molecules", op="rotate", n=12803, hq=4, hk=4, d=32, dtype="f32", axes=3, norm=True, pairing="halves", span=20.0,
             train=True),
        # a prompt batch of a model with grouped heads
        dict(name="rotate_prompt", op="rotate", n=32771, hq=32, hk=8, d=128, dtype="bf16", axes=3, norm=True, pairing="halves", span=4096.0,
             train=False),
        # training with rotation alone, neighbouring pairs
        dict(name="rotate_train", op="rotate", n=16411, hq=16, hk=16, d=64, dtype="f16", axes=2, norm=False, pairing="neighbors", span=512.0,
             train=True),
        # every atom of a molecule attends to all of it: the 512-molecule batch
        dict(name="attend_molecules", op="attend", layout="ragged", structures=512, lo=10, hi=40, layout_seed=7, hq=4, hk=4, d=32,
             dtype="f32", causal=False, train=False),
        dict(name="attend_molecules_train", op="attend", layout="ragged", structures=512, lo=10, hi=40, layout_seed=7, hq=4, hk=4, d=32,
             dtype="f32", causal=False, train=True),
        # one solvated-polymer sized structure of 5,000 atoms
        dict(name="attend_polymer_train", op="attend", layout="ragged", structures=1, lo=5000, hi=5000, layout_seed=1, hq=4, hk=4, d=32,
             dtype="f32", causal=False, train=True),
        # whole prompts / trajectories, causal, from one token to thousands, an empty one among them
        dict(name="attend_prompts", op="attend", layout="list", lengths="8192,37,4099,0,513,2048,1,1111", hq=32, hk=8, d=128, dtype="bf16",
             causal=True, train=False),
        dict(name="attend_prompts_train", op="attend", layout="list", lengths="8192,37,4099,0,513,2048,1,1111", hq=32, hk=8, d=128,
             dtype="bf16", causal=True, train=True),
        # structures of a few hundred atoms, wide features
        dict(name="attend_structures_train", op="attend", layout="ragged", structures=24, lo=150, hi=900, layout_seed=3, hq=16, hk=16, d=64,
             dtype="f16", causal=False, train=True),
        # single queries over long keys: one new frame (token) of each trajectory
        dict(name="attend_single", op="attend", layout="single", structures=48, lo=17, hi=16000, layout_seed=5, hq=32, hk=8, d=128,
             dtype="bf16", causal=True, train=False),
        # the block as a readout of per-atom features uses it: norm and rotation by the coordinates, then attention, forward and backward
        # down to the positions
        dict(name="block_train", op="block", layout="ragged", structures=64, lo=20, hi=700, layout_seed=9, hq=4, hk=4, d=32, dtype="f32",
             causal=False, axes=3, pairing="halves", span=20.0, train=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["rotate", "rotate", "attend", "attend", "attend", "single", "block"])
    d = rng.choice([32, 64, 80, 96, 128])
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 2, 4])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    seed = rng.randrange(1 << 20)
    if kind == "rotate":
        n = log(1, 16000)
        return dict(op="rotate", n=n, hq=hq, hk=hk, d=d, dtype=dtype, axes=rng.choice([1, 2, 3]), norm=rng.random() < 0.7,
                    pairing=rng.choice(["halves", "neighbors"]), span=float(log(10, 100000)), train=rng.random() < 0.5)
    if kind == "single":
        return dict(op="attend", layout="single", structures=log(1, 64), lo=1, hi=log(100, 12000), layout_seed=seed, hq=hq, hk=hk, d=d,
                    dtype=dtype, causal=rng.random() < 0.5, train=False)
    hi = log(16, 4000 if dtype != "f32" else 1500)
    case = dict(op="attend", layout="ragged", structures=max(1, min(600, int(log(4000, 14000) / hi))), lo=rng.choice([0, 1, hi // 2]), hi=hi,
                layout_seed=seed, hq=hq, hk=hk, d=d, dtype=dtype, causal=rng.random() < 0.5, train=rng.random() < 0.6)
    if kind == "block":
        case.update(op="block", dtype="f32", hi=min(hi, 1500), axes=rng.choice([1, 3]), pairing=rng.choice(["halves", "neighbors"]), span=20.0,
                    train=True)
        case["lo"] = min(max(1, case["lo"]), case["hi"])
    return case


def _lengths(case):
    """Lengths of queries and of keys, from the case alone."""
    if case["layout"] == "list":
        L = [int(x) for x in case["lengths"].split(",")]
        return L, L
    r = random.Random(case["layout_seed"])
    L = [r.randint(case["lo"], case["hi"]) for _ in range(case["structures"])]
    return ([1] * len(L), L) if case["layout"] == "single" else (L, L)


def _pairs(lq, lk, causal):
    """Allowed (query, key) pairs of one head: query i sees the keys up to i + lk - lq where causal."""
    total = 0
    for a, b in zip(lq, lk):
        if not causal:
            total += a * b
        else:
            rows = min(a, b)                       # rows that see anything: the last min(a, b), from b - rows + 1 keys to b
            total += rows * (b - rows + 1 + b) // 2
    return total


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["op"] == "rotate":
        n = case["n"]
        values = n * (hq + hk) * d
        byt = values * size * (4 if case["train"] else 2) + n * case["axes"] * 4 * (2 if case["train"] else 1) + case["axes"] * d // 2 * 4
        return dict(bytes=byt, flops=values * (20 if case["train"] else 8))
    lq, lk = _lengths(case)
    nq, nk = sum(lq), sum(lk)
    byt = (2 * nq * hq + 2 * nk * hk) * d * size * (2 if case["train"] else 1)
    flops = _pairs(lq, lk, case["causal"]) * hq * d * (14 if case["train"] else 4)
    if case["op"] == "block":
        byt += nq * case["axes"] * 4
        flops += nq * (hq + hk) * d * 20
    return dict(bytes=byt, flops=flops)


# ------------------------------------------------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hk, d = case["hq"], case["hk"], case["d"]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    st = dict(case=case, scale=1.0 / math.sqrt(d))
    if case["op"] == "rotate":
        nq = nk = case["n"]
    else:
        st["lq"], st["lk"] = _lengths(case)
        nq, nk = sum(st["lq"]), sum(st["lk"])
        st["starts_q"], st["starts_k"] = (np.concatenate([[0], np.cumsum(x)]).astype(np.int32) for x in (st["lq"], st["lk"]))
        if own:
            from so3lr_b200.attention import PackedStructures
            st["packed"] = PackedStructures(st["starts_q"], None if case["layout"] != "single" else st["starts_k"], causal=case["causal"])
        else:
            # the same knowledge for the plain form: rows of a padded batch, where that is the smaller thing
            st["pad"] = _padding(st) if _use_padding(st) else None
    st["q"], st["k"] = normal(nq, hq, d), normal(nk, hk, d)
    if case["op"] != "rotate":
        st["v"] = normal(nk, hk, d)
        if case["train"]:
            st["g"] = normal(nq, hq, d)
    if case["op"] in ("rotate", "block"):
        axes = case["axes"]
        if axes == 3:                     # coordinates, or time / height / width
            pos = torch.rand(nq, 3, generator=g, device="cuda") * (case["span"] or 20.0)
        elif case["op"] == "block":       # the index inside the sequence
            pos = torch.cat([torch.arange(n, dtype=torch.float32) for n in st["lq"]]).cuda()[:, None]
        else:
            pos = torch.floor(torch.rand(nq, axes, generator=g, device="cuda") * case["span"])
        st["positions"] = pos.contiguous()
        # pair p turns with axis p mod axes, the frequencies falling from 1
        p = torch.arange(d // 2)
        f = torch.zeros(axes, d // 2)
        f[p % axes, p] = (1000.0 ** (-(p // axes).double() / max(1, (d // 2) // axes))).float()
        st["frequencies"] = f.cuda()
        if case["op"] == "block" or case["norm"]:
            st["wq"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).float()
            st["wk"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).float()
        if case["op"] == "rotate" and case["train"]:
            st["gq"], st["gk"] = normal(nq, hq, d), normal(nk, hk, d)
    return st


def _use_padding(st):
    """A padded batch where its logits take at most 1 GB and its keys 4, else sequence by sequence."""
    b, mq, mk, c = len(st["lq"]), max(st["lq"]), max(st["lk"]), st["case"]
    return b * c["hq"] * mq * mk * 4 <= 1 << 30 and b * c["hq"] * mk * c["d"] * 4 <= 1 << 32


def _padding(st):
    """Row numbers (B, L) of a padded batch (the row behind the last one where there is none) and the allowed pairs (B, 1, Lq, Lk)."""
    def rows(lengths, starts):
        n = torch.as_tensor(np.asarray(lengths)).cuda()
        at = torch.arange(max(lengths), device="cuda")[None, :]
        there = at < n[:, None]
        return torch.where(there, torch.as_tensor(starts[:-1].astype(np.int64)).cuda()[:, None] + at, int(starts[-1])), there, n, at

    rq, tq, nq, aq = rows(st["lq"], st["starts_q"])
    rk, tk, nk, ak = rows(st["lk"], st["starts_k"])
    allowed = tq[:, :, None] & tk[:, None, :]
    if st["case"]["causal"]:
        allowed &= ak[:, None, :] <= aq[:, :, None] + (nk - nq)[:, None, None]
    return rq, rk, allowed[:, None]


# ------------------------------------------------------------------------------------------------------------ plain forms


def _cos_sin(positions, frequencies):
    theta = positions.double() @ frequencies.double()
    return torch.cos(theta).float()[:, None, :], torch.sin(theta).float()[:, None, :]


def _split(x, pairing):
    return (x[..., 0::2], x[..., 1::2]) if pairing == "neighbors" else x.chunk(2, dim=-1)


def _join(a, b, pairing):
    return torch.stack([a, b], dim=-1).flatten(-2) if pairing == "neighbors" else torch.cat([a, b], dim=-1)


def _rotate(x, w, cs, pairing, eps=1e-6):
    """Norm and rotation in 32 bits: the rotated rows and what the reverse pass needs."""
    x = x.float()
    r = None if w is None else torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    a, b = _split(x if w is None else x * r * w, pairing)
    c, s = cs
    return _join(a * c - b * s, a * s + b * c, pairing), (x, r)


def _rotate_back(g, out, saved, w, cs, pairing):
    """(dx, dw, dtheta) of `_rotate`; dw None without a norm."""
    (x, r), (c, s) = saved, cs
    g1, g2 = _split(g.float(), pairing)
    o1, o2 = _split(out, pairing)
    dtheta = (g2 * o1 - g1 * o2).sum(1)
    gy = _join(g1 * c + g2 * s, g2 * c - g1 * s, pairing)
    if w is None:
        return gy, None, dtheta
    xh = x * r
    gw = gy * w
    return r * (gw - xh * (gw * xh).mean(-1, keepdim=True)), (gy * xh).sum((0, 1)), dtheta


def _attend(q, k, v, allowed, scale):
    """softmax(scale q k^T) v over the allowed pairs, head axis ahead of the rows; rows without keys give zero."""
    s = (q @ k.transpose(-1, -2)) * scale
    s = s.masked_fill(~allowed, float("-inf")) if allowed is not None else s
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    return p @ v, p


def _attend_back(q, k, v, p, o, g, scale):
    dp = g @ v.transpose(-1, -2)
    ds = p * (dp - (g * o).sum(-1, keepdim=True)) * scale
    return ds @ k, ds.transpose(-1, -2) @ q, p.transpose(-1, -2) @ g


def _heads_first(x, times=1):
    """(..., n, h, d) -> (..., h times, n, d)"""
    x = x.transpose(-2, -3)
    return x.repeat_interleave(times, dim=-3) if times > 1 else x


def _one(q, k, v, g, allowed, scale):
    """Output and gradients (rows first) of one structure, or of a padded batch of them."""
    times, hk = q.shape[-2] // k.shape[-2], k.shape[-2]
    Q, K, V = _heads_first(q), _heads_first(k, times), _heads_first(v, times)
    o, p = _attend(Q, K, V, allowed, scale)
    if g is None:
        return (o.transpose(-2, -3),)
    dq, dk, dv = _attend_back(Q, K, V, p, o, _heads_first(g), scale)
    dk, dv = (x.unflatten(-3, (hk, times)).sum(-3) for x in (dk, dv))
    return tuple(x.transpose(-2, -3) for x in (o, dq, dk, dv))


def _attention(st, q, k, v, g):
    """In 32 bits: output (and gradients of q, k, v), packed as the inputs are."""
    q, k, v = q.float(), k.float(), v.float()
    g = None if g is None else g.float()
    if st["pad"] is not None:
        rq, rk, allowed = st["pad"]

        def pick(x, rows):
            return torch.cat([x, x.new_zeros(1, *x.shape[1:])])[rows]

        res = _one(pick(q, rq), pick(k, rk), pick(v, rk), None if g is None else pick(g, rq), allowed, st["scale"])

        def back(x, rows, n):
            return x.new_zeros(n + 1, *x.shape[2:]).index_copy_(0, rows.flatten(), x.flatten(0, 1).contiguous())[:n]

        at = ((rq, len(q)), (rq, len(q)), (rk, len(k)), (rk, len(k)))
        return tuple(back(x, *a) for x, a in zip(res, at))
    out = tuple(torch.zeros_like(x) for x in ((q,) if g is None else (q, q, k, v)))
    for a, b, c, d in zip(st["starts_q"][:-1], st["starts_q"][1:], st["starts_k"][:-1], st["starts_k"][1:]):
        if a == b or c == d:
            continue
        allowed = None
        if st["case"]["causal"]:
            allowed = torch.ones(b - a, d - c, dtype=torch.bool, device="cuda").tril(int((d - c) - (b - a)))
        res = _one(q[a:b], k[c:d], v[c:d], None if g is None else g[a:b], allowed, st["scale"])
        out[0][a:b] = res[0]
        if g is not None:
            out[1][a:b], out[2][c:d], out[3][c:d] = res[1:]
    return out


def _plain(st):
    case, dt = st["case"], st["q"].dtype
    if case["op"] == "attend":
        res = _attention(st, st["q"], st["k"], st["v"], st.get("g"))
        return dict(zip(("out", "dq", "dk", "dv"), (x.to(dt) for x in res)))
    wq, wk, pairing = st.get("wq"), st.get("wk"), case["pairing"]
    cs = _cos_sin(st["positions"], st["frequencies"])
    (oq, sq), (ok, sk) = _rotate(st["q"], wq, cs, pairing), _rotate(st["k"], wk, cs, pairing)
    res = {}
    if case["op"] == "rotate":
        res.update(q=oq.to(dt), k=ok.to(dt))
        if not case["train"]:
            return res
        gq, gk = st["gq"], st["gk"]
    else:
        out, gq, gk, dv = _attention(st, oq, ok, st["v"], st["g"])
        res.update(out=out.to(dt), dv=dv.to(dt))
    dq, dwq, tq = _rotate_back(gq, oq, sq, wq, cs, pairing)
    dk, dwk, tk = _rotate_back(gk, ok, sk, wk, cs, pairing)
    res.update(dq=dq.to(dt), dk=dk.to(dt), dpositions=(tq + tk) @ st["frequencies"].T)
    if wq is not None:
        res.update(dwq=dwq, dwk=dwk)
    return res


# ------------------------------------------------------------------------------------------------------------ the library's calls


def _calls(st):
    from so3lr_b200.attention import norm_rotate, structure_attention
    case = st["case"]
    if case["op"] == "attend" and not case["train"]:
        return dict(out=structure_attention(st["q"], st["k"], st["v"], st["packed"], scale=st["scale"]))
    if case["op"] == "rotate" and not case["train"]:
        q, k = norm_rotate(st["q"], st["k"], st["positions"], st["frequencies"], q_weight=st.get("wq"), k_weight=st.get("wk"),
                           pairing=case["pairing"])
        return dict(q=q, k=k)
    leaf = {n: st[n].detach().requires_grad_() for n in ("q", "k", "v", "positions", "wq", "wk") if n in st}
    if case["op"] == "attend":
        out = structure_attention(leaf["q"], leaf["k"], leaf["v"], st["packed"], scale=st["scale"])
        got = torch.autograd.grad(out, [leaf["q"], leaf["k"], leaf["v"]], st["g"])
        return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *got)))
    q, k = norm_rotate(leaf["q"], leaf["k"], leaf["positions"], st["frequencies"], q_weight=leaf.get("wq"), k_weight=leaf.get("wk"),
                       pairing=case["pairing"])
    names = [n for n in ("v", "q", "k", "positions", "wq", "wk") if n in leaf]
    if case["op"] == "rotate":
        got = torch.autograd.grad([q, k], [leaf[n] for n in names], [st["gq"], st["gk"]])
        res = dict(q=q.detach(), k=k.detach())
    else:
        out = structure_attention(q, k, leaf["v"], st["packed"], scale=st["scale"])
        got = torch.autograd.grad(out, [leaf[n] for n in names], st["g"])
        res = dict(out=out.detach())
    res.update({"d" + n: g for n, g in zip(names, got)})
    return res


def run(state):
    return _calls(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------ 64 bits


def _exact_rotate(x, w, positions, frequencies, pairing, eps=1e-6):
    """Pairs as complex numbers times exp(i theta)."""
    if w is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + eps) * w
    half = x.shape[-1] // 2
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], half, 2)) if pairing == "neighbors" else torch.complex(x[..., :half], x[..., half:])
    theta = (positions[:, :, None] * frequencies[None]).sum(1)
    z = z * torch.polar(torch.ones_like(theta), theta)[:, None, :]
    return torch.view_as_real(z).reshape(x.shape) if pairing == "neighbors" else torch.cat([z.real, z.imag], -1)


def _exact_attention(st, q, k, v, g):
    """Structure by structure and head by head; the gradients by automatic differentiation."""
    case = st["case"]
    times = case["hq"] // case["hk"]
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for n, (lq, lk) in enumerate(zip(st["lq"], st["lk"])):
        a, c = int(st["starts_q"][n]), int(st["starts_k"][n])
        if not lq or not lk:
            continue
        bias = None
        if case["causal"]:
            i, j = torch.arange(lq, device="cuda")[:, None], torch.arange(lk, device="cuda")[None, :]
            bias = torch.where(j > i + (lk - lq), float("-inf"), 0.0).double()
        per = max(1, min(case["hk"], (1 << 27) // (lq * lk * times)))
        for h in range(0, case["hk"], per):
            hk, hq = slice(h, min(h + per, case["hk"])), slice(h * times, min(h + per, case["hk"]) * times)
            with torch.enable_grad():
                Q, K, V = (x.detach().requires_grad_(g is not None) for x in (q[a:a + lq, hq], k[c:c + lk, hk], v[c:c + lk, hk]))
                KK, VV = (x[:, :, None].expand(-1, -1, times, -1).flatten(1, 2) for x in (K, V))
                s = torch.einsum("ihd,jhd->hij", Q, KK) * st["scale"]
                if bias is not None:
                    s = s + bias
                o = torch.einsum("hij,jhd->ihd", torch.nan_to_num(torch.exp(s - torch.logsumexp(s, -1, keepdim=True)), nan=0.0), VV)
                out[a:a + lq, hq] = o.detach()
                if g is not None:
                    dq[a:a + lq, hq], dk[c:c + lk, hk], dv[c:c + lk, hk] = torch.autograd.grad(o, (Q, K, V), g[a:a + lq, hq])
    return out, dq, dk, dv


def exact(case, seed):
    st = prepare(case, seed)
    x = {n: st[n].double() for n in ("q", "k", "v", "g", "gq", "gk", "positions", "frequencies", "wq", "wk") if n in st}
    if case["op"] == "attend":
        res = _exact_attention(st, x["q"], x["k"], x["v"], x.get("g"))
        return dict(zip(("out", "dq", "dk", "dv"), res if case["train"] else res[:1]))
    names = [n for n in ("q", "k", "positions", "wq", "wk") if n in x]
    with torch.enable_grad():
        leaf = {n: x[n].requires_grad_() for n in names}
        q, k = (_exact_rotate(leaf[n], leaf.get("w" + n), leaf["positions"], x["frequencies"], case["pairing"]) for n in ("q", "k"))
        if case["op"] == "rotate":
            res = dict(q=q.detach(), k=k.detach())
            gq, gk = x.get("gq"), x.get("gk")
        else:
            out, gq, gk, dv = _exact_attention(st, q.detach(), k.detach(), x["v"], x["g"])
            res = dict(out=out, dv=dv)
        if case["train"]:
            got = torch.autograd.grad([q, k], [leaf[n] for n in names], [gq, gk])
            res.update({"d" + n: t for n, t in zip(names, got)})
    return res
