"""structure_attention and norm_rotate on the GPU against their formulas in 64 bits.

Tolerances are bounds, derived ahead of the first run.  u = eps / 2 of the type is the error of one rounding relative to the value.
 * logits: a float32 dot product of d terms is off by at most (d + 4) 2^-24 of sum |q||k| (float32 inputs: each product of two split operands
   by 2^-21 more); times scale this is `e`, and a probability by the factor exp(2 max e) - 1 <= 3 max e, plus 2^-20 for the
   exponential, the running rescaling and the normalisation.
 * a probability (dS likewise) is rounded to the inputs' type ahead of the second product: u sum |P||v|, and the result once: u |o|.
 * sums of L terms in float32: L 2^-24 of the sum of their magnitudes.
 * float16 has steps of 2^-24 below 2^-14: a probability relative to its row's largest (forward) and dS are off by up to 2^-25 each on the way
   into their products besides u, the former over a sum of at least one.  (2^15 P goes into dv: nothing to add there.)
 * delta = g . o uses the rounded o: (u + (d + 4) 2^-24) sum |g||o|; float32 inputs: the error of o itself in place of u |o|.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from so3lr_b200.attention import PackedStructures, norm_rotate, structure_attention  # noqa: E402

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def starts(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def reference(q, k, v, g, lq, lk, causal, scale, dtype):
    """(values, bounds) of out, dq, dk, dv in float64."""
    u = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    up = 2.0 ** -21 if dtype == torch.float32 else u          # rounding of P and dS on the way into a product
    w = u if u else 2.0 ** -24
    step = 2.0 ** -25 if dtype == torch.float16 else 0.0
    q, k, v, g = (x.double() for x in (q, k, v, g))
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    val = [torch.zeros_like(x) for x in (q, q, k, v)]
    err = [torch.zeros_like(x) for x in (q, q, k, v)]
    a = c = 0
    for n, m in zip(lq, lk):
        if n and m:
            for h in range(hq):
                j = h // (hq // hk)
                Q, K, V, G = q[a:a + n, h], k[c:c + m, j], v[c:c + m, j], g[a:a + n, h]
                s = scale * Q @ K.T
                ok = torch.ones(n, m, dtype=torch.bool, device=q.device)
                if causal:
                    ok = torch.arange(m, device=q.device)[None] <= torch.arange(n, device=q.device)[:, None] + (m - n)
                P = torch.softmax(s.masked_fill(~ok, -float("inf")), -1).nan_to_num(0.0)
                O, dP = P @ V, G @ V.T
                delta = (G * O).sum(-1, keepdim=True)
                dS = P * (dP - delta)
                e = scale * (Q.abs() @ K.abs().T) * ((d + 4) * 2.0 ** -24 + (2.0 ** -21 if not u else 0))
                rel = (3 * torch.where(ok, e, 0.0).amax(-1, keepdim=True) + 2.0 ** -20 + m * 2.0 ** -24).expand(n, m)
                eO = ((rel + up + m * 2.0 ** -24) * P + step * ok) @ V.abs() + w * O.abs()
                edelta = (G.abs() * (eO + O.abs() * ((d + 4) * 2.0 ** -24))).sum(-1, keepdim=True)
                edP = (G.abs() @ V.abs().T) * ((d + 4) * 2.0 ** -24 + (2.0 ** -21 if not u else 0))
                edS = P * (edP + edelta) + rel * dS.abs() * 1.01 + rel * P * (edP + edelta)
                eS2 = edS + (up + max(m, n) * 2.0 ** -24) * (dS.abs() + edS) + step * ok
                val[0][a:a + n, h] += O
                err[0][a:a + n, h] += eO
                val[1][a:a + n, h] += scale * dS @ K
                err[1][a:a + n, h] += scale * eS2 @ K.abs()
                val[2][c:c + m, j] += scale * dS.T @ Q
                err[2][c:c + m, j] += scale * eS2.T @ Q.abs()
                val[3][c:c + m, j] += P.T @ G
                err[3][c:c + m, j] += ((rel + up + n * hq * 2.0 ** -24) * P).T @ G.abs()
        a, c = a + n, c + m
    # the final rounding; 16-bit types also underflow to their smallest steps
    tiny = 0.0 if dtype == torch.float32 else torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return val, [x * 1.01 + w * (y.abs() + x) + tiny for x, y in zip(err, val)]


def inputs(lq, lk, hq, hk, d, dtype, seed=0, extra=0, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shapes = ((sum(lq) + extra, hq, d), (sum(lk) + extra, hk, d), (sum(lk) + extra, hk, d), (sum(lq) + extra, hq, d))
    return [(torch.randn(*s, generator=gen, device="cuda") * size).to(dtype) for s in shapes]


def within(got, val, err, names=("out", "dq", "dk", "dv")):
    for n, x, y, e in zip(names, got, val, err):
        assert torch.isfinite(x).all(), n
        off = (x.double() - y).abs()
        assert (off <= e).all(), f"{n}: off by {float((off - e).max()):.3g} more than the bound, {float((off / (e + 1e-300)).max()):.3g} times it"


def train(q, k, v, g, packed, scale=None):
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out = structure_attention(q, k, v, packed, scale=scale)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), g))


ODD = [0, 1, 2, 63, 64, 65, 15, 0, 16, 17, 127, 128, 129, 200]
CASES = [
    # lq, lk (None: the same rows), heads, key heads, d, causal
    (ODD, None, 2, 2, 32, False), (ODD, None, 4, 2, 64, True), (ODD, None, 3, 1, 128, True), (ODD, None, 2, 1, 96, False),
    # the same short ones beside a long one, which decides on the kernels
    (ODD + [650], None, 2, 2, 32, False), (ODD + [650], None, 4, 2, 64, True), ([601, 7, 0, 640], None, 2, 1, 16, True),
    (ODD + [301], None, 3, 1, 112, False), ([650, 40, 1], [5, 700, 130], 2, 1, 48, True), ([1300], None, 2, 2, 64, False),
    ([20, 31, 5, 1, 0, 16], None, 2, 2, 64, False), ([33, 40, 10], None, 4, 2, 32, True), ([9, 2, 16], None, 2, 1, 128, True),
    ([17, 24, 1, 0, 16], None, 4, 2, 96, False), ([48, 31, 16, 2], None, 2, 2, 16, True), ([3, 30, 8], [40, 2, 0], 8, 2, 64, False),
    ([300, 1, 77], None, 4, 4, 80, True), ([257], None, 2, 1, 16, True), ([511, 513], None, 1, 1, 128, False), ([1000], None, 2, 2, 48, True),
    # more keys than queries, fewer (rows that see nothing), none at all
    ([5, 70, 100, 3, 0, 90], [64, 200, 40, 0, 10, 1], 4, 2, 64, True), ([5, 70, 100, 3, 0, 90], [64, 200, 40, 0, 10, 1], 4, 2, 64, False),
    # one query per structure: the keys' axis is split and joined
    ([1] * 7, [1, 64, 65, 1000, 0, 5000, 130], 8, 2, 128, True), ([1, 0, 1, 2], [3000, 50, 0, 700], 4, 4, 32, False),
    ([3, 16, 1], [777, 20, 4097], 4, 1, 112, True),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lq,lk,hq,hk,d,causal", CASES)
def test_against_the_formula(lq, lk, hq, hk, d, causal, dtype):
    lk = lq if lk is None else lk
    q, k, v, g = inputs(lq, lk, hq, hk, d, TYPES[dtype], seed=len(lq) + d)
    packed = PackedStructures(starts(lq), starts(lk), causal=causal)
    val, err = reference(q, k, v, g, lq, lk, causal, d ** -0.5, q.dtype)
    got = train(q, k, v, g, packed)
    within(got, val, err)
    # without gradients, and again: the same bits
    assert torch.equal(structure_attention(q, k, v, packed), got[0])
    for x, y in zip(got, train(q, k, v, g, packed)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_large_logits_and_given_scale(dtype):
    lq = [90, 200]
    q, k, v, g = inputs(lq, lq, 2, 1, 64, TYPES[dtype], seed=5, size=3.0)
    packed = PackedStructures(starts(lq), causal=True)
    val, err = reference(q, k, v, g, lq, lq, True, 0.4, q.dtype)
    within(train(q, k, v, g, packed, 0.4), val, err)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths", [[70, 130], [20, 9]])
def test_strides_rows_behind_and_neighbours(dtype, lengths):
    """Operands cut out of one projection, rows behind the last structure (NaN there), and a structure whose values are not finite."""
    hq, hk, d, extra = 4, 2, 64, 5
    n = sum(lengths)
    gen = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(n + extra, (hq + 2 * hk) * d, generator=gen, device="cuda").to(TYPES[dtype])
    qkv[n:] = float("nan")
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hk * d, hk * d], dim=1))
    g = torch.randn(n + extra, hq, d, generator=gen, device="cuda").to(q.dtype)
    packed = PackedStructures(starts(lengths))
    val, err = reference(q[:n], k[:n], v[:n], g[:n], lengths, lengths, False, d ** -0.5, q.dtype)
    got = train(q, k, v, g, packed)
    within([x[:n] for x in got], val, err)
    assert all((x[n:] == 0).all() for x in got)
    # head-major storage, and a cotangent broadcast over the heads
    q2, k2 = q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1)
    assert not q2.is_contiguous()
    for x, y in zip(train(q2, k2, v, g, packed), got):
        assert torch.equal(x, y)
    gb = g[:, :1].expand(-1, hq, -1)
    for x, y in zip(train(q, k, v, gb, packed), train(q, k, v, gb.contiguous(), packed)):
        assert torch.equal(x, y)
    # an odd storage offset: not 16-byte aligned
    off = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape).copy_(q)
    assert off.data_ptr() % 16 and torch.equal(structure_attention(off, k, v, packed), got[0])
    # the second structure's values stay its own
    k3, v3 = k.clone(), v.clone()
    k3[lengths[0] + 1], v3[lengths[0] + 2] = float("inf"), float("nan")
    for x, y in zip(train(q, k3, v3, g, packed), got):
        assert torch.equal(x[:lengths[0]], y[:lengths[0]])


def test_gradients_against_differences():
    lq, lk, d = [9, 70], [30, 66], 32
    q, k, v, g = inputs(lq, lk, 4, 2, d, torch.float32, seed=11)
    packed = PackedStructures(starts(lq), starts(lk), causal=True)
    _, *grads = train(q, k, v, g, packed)
    val, _ = reference(q, k, v, g, lq, lk, True, d ** -0.5, torch.float32)
    # central differences of the float64 formula along a direction: step^2 / 6 of the third derivative, 1e-4^2 -> 1e-7 of the value's size
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i, (x, dx) in enumerate(zip((q, k, v), grads)):
        t = torch.randn(x.shape, generator=gen, device="cuda").double()
        f = []
        for sign in (1, -1):
            y = [z.double() for z in (q, k, v)]
            y[i] = y[i] + sign * 1e-4 * t
            f.append((reference(*y, g, lq, lk, True, d ** -0.5, torch.float32)[0][0] * g.double()).sum())
        want = float((f[0] - f[1]) / 2e-4)
        assert abs(float((dx.double() * t).sum()) - want) <= 1e-5 * float((dx.double() * t).abs().sum()) + 1e-5


@pytest.mark.parametrize("lq,lk,hq,hk", [([200, 30], [200, 30], 4, 2), ([1, 1], [3000, 900], 8, 2)])
def test_streams_capture_and_concurrent_graphs(lq, lk, hq, hk):
    """Another stream; two captured graphs of the same layout replayed side by side with fresh inputs."""
    d = 64
    packed = PackedStructures(starts(lq), starts(lk), causal=True)
    sets = [inputs(lq, lk, hq, hk, d, torch.bfloat16, seed=s) for s in range(4)]
    want = [train(*s, packed) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train(*sets[0], packed)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(got, want[0]):
        assert torch.equal(x, y)
    graphs, held, outs = [], [], []
    for s in sets[:2]:
        hold = [x.clone() for x in s]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = train(*hold, packed)
        graphs.append(graph), held.append(hold), outs.append(out)
    streams = [torch.cuda.Stream() for _ in graphs]
    for rnd in range(3):
        for i, (graph, st) in enumerate(zip(graphs, streams)):
            for x, y in zip(held[i], sets[(i + rnd) % 4]):
                x.copy_(y)
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for i, out in enumerate(outs):
            for x, y in zip(out, want[(i + rnd) % 4]):
                assert torch.equal(x, y)


def test_no_rows_at_all():
    for lq, lk in (([], []), ([0, 0], [0, 0]), ([3, 2], [0, 0]), ([0, 0], [4, 1])):
        q, k, v, g = inputs(lq, lk, 2, 1, 32, torch.float32)
        for x in train(q, k, v, g, PackedStructures(starts(lq), starts(lk))):
            assert (x == 0).all()


def test_refusals():
    q, k, v, _ = inputs([5], [5], 4, 2, 32, torch.float32)
    packed = PackedStructures([0, 5])
    for a in ((q.double(), k, v), (q, k.half(), v), (q, k, v[:4]), (q[:4], k, v), (q, k[:4], v[:4]), (q[:, :3], k, v), (q[..., :24], k[..., :24], v[..., :24]),
              (q, k[:, :0], v[:, :0]), (q.cpu(), k, v), (q, k.cpu(), v), (q, k[..., :16], v[..., :16])):
        with pytest.raises(ValueError):
            structure_attention(*a, packed)
    for s in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            structure_attention(q, k, v, packed, scale=s)
    with pytest.raises(ValueError):
        structure_attention(q, k, v, [0, 5])
    out = structure_attention(q.requires_grad_(), k, v, packed)
    (dq,) = torch.autograd.grad(out.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):        # differentiable once
        dq.sum().backward()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError):
            PackedStructures([0, 5])


# ------------------------------------------------------------------------------------------------------------ norm and rotation


def rotate_reference(x, w, theta, pairing, eps=1e-6):
    """In float64, differentiable."""
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    c, s = torch.cos(theta)[:, None], torch.sin(theta)[:, None]
    a, b = (x[..., ::2], x[..., 1::2]) if pairing == "neighbors" else x.chunk(2, -1)
    y = (a * c - b * s, a * s + b * c)
    return torch.stack(y, -1).flatten(-2) if pairing == "neighbors" else torch.cat(y, -1)


ROTATIONS = [
    # n, heads, key heads, d, axes, norm, pairing
    (1, 1, 1, 16, 1, True, "halves"), (7, 4, 2, 32, 3, True, "neighbors"), (130, 3, 0, 64, 2, True, "halves"), (1000, 8, 2, 128, 1, True, "halves"),
    (33, 5, 5, 80, 3, False, "neighbors"), (257, 2, 1, 96, 4, False, "halves"), (64, 2, 2, 256, 1, True, "neighbors"), (5000, 4, 4, 32, 3, True, "halves"),
    (19, 40, 8, 128, 0, True, "halves"), (3, 6, 3, 48, 2, True, "neighbors"), (40000, 1, 1, 32, 2, True, "halves"),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,hq,hk,d,axes,norm,pairing", ROTATIONS)
def test_norm_rotate_against_the_formula(n, hq, hk, d, axes, norm, pairing, dtype):
    t = TYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(n + d)

    def normal(*s):
        return torch.randn(*s, generator=gen, device="cuda")

    q, k, gq, gk = normal(n, hq, d).to(t), normal(n, hk, d).to(t) if hk else None, normal(n, hq, d).to(t), normal(n, hk, d).to(t) if hk else None
    pos = (normal(n, axes) * 3000).float() if axes else None           # far positions: the angle needs its fraction
    freq = torch.rand(axes, d // 2, generator=gen, device="cuda") if axes else None
    wt = torch.float32 if d != 64 else t                               # weights of the rows' own type once
    wq = (1 + 0.1 * normal(d)).to(wt) if norm else None
    wk = (1 + 0.1 * normal(d)).to(wt) if norm and hk else None
    given = {"q": q, "k": k, "positions": pos, "wq": wq, "wk": wk}

    leaf = {m: x.double().requires_grad_() for m, x in given.items() if x is not None}
    theta = leaf["positions"] @ freq.double() if axes else torch.zeros(n, d // 2, dtype=torch.float64, device="cuda")
    want = [rotate_reference(leaf[m], leaf.get("w" + m), theta, pairing) for m in ("q", "k") if m in leaf]
    wgrad = dict(zip(leaf, torch.autograd.grad(want, list(leaf.values()), [x.double() for x in (gq, gk) if x is not None])))

    mine = {m: x.detach().requires_grad_() for m, x in given.items() if x is not None}
    got = norm_rotate(mine["q"], mine.get("k"), mine.get("positions"), freq, q_weight=mine.get("wq"), k_weight=mine.get("wk"), pairing=pairing)
    assert (got[1] is None) == (k is None)
    got = [x for x in got if x is not None]
    ggrad = dict(zip(mine, torch.autograd.grad(got, list(mine.values()), [x for x in (gq, gk) if x is not None])))

    # float32 arithmetic: the mean's d terms (d 2^-24), a root, a quotient, five products and sums, the cosine (2^-23): less than
    # (d + 16) 2^-23 of the pair's length; one rounding to the type
    u = torch.finfo(t).eps / 2
    small = (d + 16) * 2.0 ** -23
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps

    def pair_length(x):
        return (x.detach().square() + _partner(x.detach(), pairing).square()).sqrt()

    for x, y in zip(got, want):
        assert ((x.detach().double() - y.detach()).abs() <= u * y.detach().abs() + small * pair_length(y) + tiny).all()
    for m in ("q", "k"):
        if m not in leaf:
            continue
        x, g, w = leaf[m].detach(), (gq if m == "q" else gk).double(), leaf.get("w" + m)
        r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) if norm else torch.ones_like(x[..., :1])
        gw = pair_length(g) * (w.detach().abs().amax() if norm else 1)
        # dx = r (gy w - xhat mean(..)): magnitudes of both terms
        bound = r * (gw + (x.abs() * r * (gw * x.abs() * r).mean(-1, keepdim=True) if norm else 0))
        y = wgrad[m]
        assert ((ggrad[m].double() - y).abs() <= u * y.abs() + 2 * small * bound + tiny).all(), m
    # sums over n rows and heads: (terms + d + 16) 2^-23 of the sum of magnitudes at the very worst, here with the depth of the sums
    # (at most 2,048 terms are added one after the other)
    deep = (min(n * max(hq, hk, 1), 2048) + d + 64) * 2.0 ** -23
    for m in ("wq", "wk"):
        if m in leaf:
            x, g = leaf[m[1]].detach(), (gq if m == "wq" else gk).double()
            xh = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
            mag = (pair_length(g) * xh.abs()).sum((0, 1))
            uw = 2.0 ** -24 if wt == torch.float32 else u
            assert ((ggrad[m].double() - wgrad[m]).abs() <= uw * wgrad[m].abs() + deep * mag).all(), m
    if axes:
        mag = sum((pair_length(g.double()) * pair_length(y)).sum((1, 2)) for g, y in zip((gq, gk), want))
        off = (ggrad["positions"].double() - wgrad["positions"]).abs()
        assert (off <= (small + 128 * 2.0 ** -23) * mag[:, None] * float(freq.max())).all()
    # the same bits again, without gradients too
    again = norm_rotate(q, k, pos, freq, q_weight=wq, k_weight=wk, pairing=pairing)
    for x, y in zip(got, [z for z in again if z is not None]):
        assert torch.equal(x, y)


def _partner(x, pairing):
    if pairing == "neighbors":
        return x.unflatten(-1, (-1, 2)).flip(-1).flatten(-2)
    return x.roll(x.shape[-1] // 2, -1)


def test_norm_rotate_only_differences_matter():
    """The product of two rotated rows does not change when all positions move: float64 angles, one rounding of the shift."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.randn(50, 2, 64, generator=gen, device="cuda") for _ in range(2))
    pos = torch.rand(50, 3, generator=gen, device="cuda", dtype=torch.float64) * 20
    f = torch.rand(3, 32, generator=gen, device="cuda")
    s = []
    for shift in (0.0, 1.0e6):
        a, b = norm_rotate(q, k, pos + shift, f)
        s.append(torch.einsum("ihd,jhd->hij", a, b))
    # each rotated value is off by some 2^-22 of its pair, 64 of them are summed
    assert (s[0] - s[1]).abs().max() <= 64 * 2.0 ** -20


def test_norm_rotate_strides_streams_and_capture():
    gen = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn(100, 8 * 64, generator=gen, device="cuda").to(torch.bfloat16)
    q, k = qkv[:, :256].unflatten(1, (4, 64)), qkv[:, 256:384].unflatten(1, (2, 64))
    pos = torch.arange(100, device="cuda").double()[:, None].expand(-1, 2)          # not contiguous
    f = torch.rand(2, 32, generator=gen, device="cuda")
    w = torch.ones(64, device="cuda")
    want = norm_rotate(q.contiguous(), k.contiguous(), pos.contiguous(), f, q_weight=w, k_weight=w)
    for x, y in zip(norm_rotate(q, k, pos, f, q_weight=w, k_weight=w), want):
        assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm_rotate(q, k, pos, f, q_weight=w, k_weight=w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    torch.cuda.synchronize()
    graph, buf = torch.cuda.CUDAGraph(), torch.zeros_like(q.contiguous())
    with torch.cuda.graph(graph):
        got = norm_rotate(buf, None, pos, f, q_weight=w)
    buf.copy_(q)
    graph.replay()
    assert torch.equal(got[0], want[0])
    # no rows, no heads
    assert norm_rotate(q[:0], k[:0], pos[:0], f)[0].shape == (0, 4, 64)
    leaf = w.clone().requires_grad_()
    a, _ = norm_rotate(q[:0], None, pos[:0], f, q_weight=leaf)
    assert (torch.autograd.grad(a.sum(), leaf)[0] == 0).all()


def test_norm_rotate_one_side_of_the_gradient():
    """Only one output used: the other's cotangent is zero."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k = (torch.randn(20, 2, 32, generator=gen, device="cuda").requires_grad_() for _ in range(2))
    pos = torch.rand(20, 3, generator=gen, device="cuda").requires_grad_()
    f = torch.rand(3, 16, generator=gen, device="cuda")
    a, b = norm_rotate(q, k, pos, f)
    dq, dk, dp = torch.autograd.grad(b.square().sum() + b.sum(), (q, k, pos))
    assert (dq == 0).all()
    a2, _ = norm_rotate(k, None, pos, f)
    dk2, dp2 = torch.autograd.grad(a2.square().sum() + a2.sum(), (k, pos))
    assert torch.equal(dk, dk2) and torch.allclose(dp, dp2, rtol=1e-5, atol=1e-5)


def test_norm_rotate_refusals():
    q, k = torch.zeros(5, 4, 32, device="cuda"), torch.zeros(5, 2, 32, device="cuda")
    pos, f, w = torch.zeros(5, 3, device="cuda"), torch.zeros(3, 16, device="cuda"), torch.ones(32, device="cuda")
    for args, kw in (((q, k), {}), ((q, k, pos), {}), ((q, k, None, f), {}), ((q, k[:4], pos, f), {}), ((q, k.half(), pos, f), {}),
                     ((q, k, pos[:4], f), {}), ((q, k, pos.half(), f), {}), ((q, k, pos.cpu(), f), {}), ((q, k, pos, f.double()), {}),
                     ((q, k, pos, f[:2]), {}), ((q, k, pos, f[:, :8]), {}), ((q, k, pos, f.clone().requires_grad_()), {}),
                     ((q, k, pos, f), dict(pairing="rows")), ((q, k, pos, f), dict(q_weight=w)), ((q, k, pos, f), dict(k_weight=w)),
                     ((q, None, pos, f), dict(q_weight=w, k_weight=w)), ((q, k, pos, f), dict(q_weight=w[:16], k_weight=w)),
                     ((q, k, pos, f), dict(q_weight=w, k_weight=w.double())), ((q, k), dict(q_weight=w, k_weight=w, eps=-1.0)),
                     ((q[..., :24], k[..., :24], pos, f[:, :12]), {}), ((q, k, pos[:, :0], f[:0]), {})):
        with pytest.raises(ValueError):
            norm_rotate(*args, **kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lk,d", [(300, 32), (300, 64), (300, 128), (40, 64), (1000, 128)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_one_value_that_is_not_finite_shows(lk, d, dtype, value):
    # one key of the first structure: every one of its rows attends to it, wherever it stands in its tile; the second structure is spared
    q, k, v, _ = inputs([lk, 280], [lk, 280], 1, 1, d, TYPES[dtype], seed=2)
    q[:, :, 0] = 1.0
    packed = PackedStructures(starts([lk, 280]))
    clean = structure_attention(q, k, v, packed)
    for j in list(range(8)) + [lk - 1, lk - 2, lk - 3, lk - 4]:
        bad = k.clone()
        bad[j, 0, 0] = value
        out = structure_attention(q, bad, v, packed)
        assert not torch.isfinite(out[:lk]).any(), j
        assert torch.equal(out[lk:], clean[lk:])


def test_rows_with_free_strides_and_scales_that_change():
    # one row, one head: the strides of these axes mean nothing, whatever they are
    gen = torch.Generator(device="cuda").manual_seed(6)
    q = torch.randn(40, generator=gen, device="cuda").as_strided((1, 2, 16), (33, 16, 1))
    k = torch.randn(40, 20, generator=gen, device="cuda")[:, None, :16].as_strided((40, 1, 16), (20, 3, 1))
    packed = PackedStructures([0, 1], [0, 40])
    assert q.stride(0) % 4 and k.stride(1) % 4
    want = torch.softmax(0.25 * torch.einsum("qhd,kd->hqk", q.double(), k[:, 0].double()), -1)
    want = torch.einsum("hqk,kd->qhd", want, k[:, 0].double())
    got = structure_attention(q, k, k, packed)
    # 16 terms a logit of size 4 and 40 a value: below 100 roundings of 2^-24
    assert (got.double() - want).abs().max() <= 100 * 2.0 ** -24 * k.abs().max()
    turned = norm_rotate(q, None, torch.ones(1, 1, device="cuda"), torch.zeros(1, 8, device="cuda"))[0]
    assert torch.equal(turned, q)
    scale = torch.tensor(0.5)
    first = structure_attention(q, k, k, packed, scale=scale)
    scale.fill_(2.0)
    assert torch.equal(structure_attention(q, k, k, packed, scale=scale), structure_attention(q, k, k, packed, scale=2.0))
    assert not torch.equal(structure_attention(q, k, k, packed, scale=scale), first)


@pytest.mark.parametrize("heads", [1, 3, 5])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_rotate_without_eps_and_keys(heads, dtype):
    # counts of heads that are no power of two leave lanes without a head
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(9, heads, 32, generator=gen, device="cuda").to(TYPES[dtype])
    pos, f, w = torch.rand(9, 3, generator=gen, device="cuda"), torch.rand(3, 16, generator=gen, device="cuda"), torch.rand(32, generator=gen, device="cuda") + 0.5
    leaves = [t.clone().requires_grad_() for t in (x, pos, w)]
    g = torch.randn(9, heads, 32, generator=gen, device="cuda").to(TYPES[dtype])
    out = norm_rotate(leaves[0], None, leaves[1], f, q_weight=leaves[2], eps=0.0)[0]
    got = torch.autograd.grad(out, leaves, g)
    ref = [t.detach().double().requires_grad_() for t in leaves]
    y = rotate_reference(ref[0], ref[2], ref[1] @ f.double(), "halves", eps=0.0)
    want = torch.autograd.grad(y, ref, g.double())
    for name, a, b in zip(("x", "positions", "weight"), got, want):
        # sums of up to 9 heads rows of a hundred float32 operations, and a rounding of 16-bit results
        step = 2.0 ** -8 if a.dtype == torch.bfloat16 else 2.0 ** -15
        assert (a.double() - b).abs().max() <= step * b.abs().max(), name


def test_more_rows_than_an_index_holds_are_refused():
    many = torch.zeros(1, 1, 16, dtype=torch.bfloat16, device="cuda").expand(2 ** 31, 1, 16)
    one = torch.zeros(1, 1, 16, dtype=torch.bfloat16, device="cuda")
    packed = PackedStructures([0, 1])
    for q, k in ((many, one), (one, many)):
        with pytest.raises(ValueError, match="rows"):
            structure_attention(q, k, k, packed)
    with pytest.raises(ValueError, match="rows"):
        norm_rotate(many, None, torch.zeros(1, 1, device="cuda").expand(2 ** 31, 1), torch.zeros(1, 8, device="cuda"))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hq,hk,d,causal,seed", [(16, 16, 32, False, 0), (12, 4, 64, True, 1), (14, 7, 128, True, 2), (16, 1, 48, False, 3)])
def test_more_items_than_the_chip_takes_at_once(hq, hk, d, causal, seed, dtype):
    # lengths of both sides from none to 500, in any order: every CTA works on many items, some of them without any row of the other side
    rng = np.random.default_rng(seed)
    lq, lk = (np.where(rng.random(30) < 0.15, 0, rng.integers(1, 500, 30)).tolist() for _ in range(2))
    q, k, v, g = inputs(lq, lk, hq, hk, d, TYPES[dtype], seed=seed, extra=3)
    packed = PackedStructures(starts(lq), starts(lk), causal=causal)
    val, err = reference(q, k, v, g, lq, lk, causal, d ** -0.5, q.dtype)
    got = train(q, k, v, g, packed)
    within(got, val, err)
    # beside another call of the same kind, and replayed: the same bits
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        beside = train(q, k, v, g, packed)
    again = train(q, k, v, g, packed)
    torch.cuda.synchronize()
    for x, y, z in zip(got, again, beside):
        assert torch.equal(x, y) and torch.equal(x, z)
    no_wait_ran_out()


def no_wait_ran_out():
    import ctypes

    from so3lr_b200._lib import check, lib
    word = ctypes.c_int(-1)
    check(lib.so3lr_b200_structure_attention_error(ctypes.byref(word)), "structure_attention_error")
    assert word.value == 0


@pytest.mark.parametrize("dtype,d", [("f32", 32), ("f32", 64), ("bf16", 64), ("f16", 128)])
@pytest.mark.parametrize("side", ["queries", "keys"])
def test_long_runs_of_items_that_meet_nothing(side, dtype, d):
    # hundreds of structures without any key (any query) beside two that have both
    full, none = [131] * 401, [0] * 200 + [250] + [0] * 199 + [140]
    lq, lk = (full, none) if side == "queries" else (none, full)
    q, k, v, g = inputs(lq, lk, 8, 4, d, TYPES[dtype], seed=11)
    packed = PackedStructures(starts(lq), starts(lk))
    val, err = reference(q, k, v, g, lq, lk, False, d ** -0.5, q.dtype)
    within(train(q, k, v, g, packed), val, err)
    no_wait_ran_out()
