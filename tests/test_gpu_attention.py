"""Kernel attention against the formula in float64, element by element.

Error bounds, with u the half step of a 16-bit type (fp32 inputs: pairs of
fp16 halves, 2^-21 for a product of two pairs without its smallest term),
E = 2^-23 for each fp32 addition, n terms in a sum:
  score  a ((D + 4) E + pair) sum |q k|, and a few steps of the score, the
         cap and the distance term
  P      relative 2 max err(score) + 2^-19
  out    sum P |v| (u + rel P + (n + 4) E) + half a step of out
  D_i    sum |do| (out's bound with P as a pair, 2^-16, in u's place)
  dS     P (rel P (|dP| + |D|) + err dP + err D); times q or k also u |dS|
  dq dk  the same with dS (1 - tanh^2); dv as out
An fp16 number below its normal range has an absolute half step of 2^-25, and a
pair's low half reaches there too: P is held up to 2^7 or more; dS at 2^13 or
more for 2 D max |do| max |v| (elements' maxima), so dS is off by 2^-37 of
D max |do| max |v|; and each fp32 tensor's pairs at 2^13 or more for its largest
element, so their elements are off by 2^-38 of it.
Positions and sigma get dS as it is, in fp32.
"""
import math
import threading

import pytest
import torch

import rapidalign_b200 as ra

pytestmark = pytest.mark.gpu

E = 2.0 ** -23
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(nq, nk, heads, kv, dim, dtype, pos, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=g, device="cuda")

    d = dict(q=(rn(sum(nq), heads, dim) * spread).to(dtype), k=rn(sum(nk), kv, dim).to(dtype),
             v=rn(sum(nk), kv, dim).to(dtype), g=rn(sum(nq), heads, dim).to(dtype))
    if pos:
        d["q_pos"], d["k_pos"] = rn(sum(nq), pos), rn(sum(nk), pos)
        d["sigma"] = torch.tensor([0.3 * 1.7 ** (i % 4) for i in range(heads)], device="cuda")
    return d


def ptr(n):
    return torch.tensor([0] + list(n), device="cuda").cumsum(0)


def exact(d, nq, nk, scale, cap, q_mask=None, k_mask=None):
    """Float64 results and bounds, as dicts of flat tensors."""
    dtype = d["q"].dtype
    u = torch.finfo(dtype).eps / 2
    pair = 2.0 ** -21 if dtype == torch.float32 else 0.0
    up = pair if pair else u  # of an operand held in 16 bits
    fine = 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -20
    tiny = torch.finfo(dtype).tiny
    w = {n: t.double() for n, t in d.items()}
    names = [n for n in ("q", "k", "v", "q_pos", "k_pos", "sigma") if n in d]
    heads, kv = w["q"].shape[1], w["k"].shape[1]
    D = w["q"].shape[2]
    head = torch.arange(heads, device="cuda") // (heads // kv)
    out, b_out = torch.zeros_like(w["q"]), torch.zeros_like(w["q"])
    gr = {n: torch.zeros_like(w[n]) for n in names}
    b = {n: torch.zeros_like(w[n]) for n in names}
    keep_q = torch.ones(sum(nq), dtype=torch.bool, device="cuda") if q_mask is None else q_mask
    keep_k = torch.ones(sum(nk), dtype=torch.bool, device="cuda") if k_mask is None else k_mask
    small_ds = 0.0
    # of an element of q, k, v, do held as a pair
    s_el = {x: (2.0 ** -38 * float(w[x][keep].abs().max()) if pair and keep.any() else 0.0)
            for x, keep in (("q", keep_q), ("k", keep_k), ("v", keep_k), ("g", keep_q))}
    if dtype != torch.bfloat16 and keep_q.any() and keep_k.any():
        small_ds = D * float(w["g"][keep_q].abs().max() * w["v"][keep_k].abs().max()) * 2.0 ** -37
    a0 = c0 = 0
    for n, m in zip(nq, nk):
        I = torch.nonzero(keep_q[a0:a0 + n])[:, 0] + a0
        J = torch.nonzero(keep_k[c0:c0 + m])[:, 0] + c0
        a0, c0 = a0 + n, c0 + m
        if not I.numel() or not J.numel():
            continue
        q = w["q"][I].transpose(0, 1)
        k, v = (w[x][J].transpose(0, 1)[head] for x in ("k", "v"))
        go = w["g"][I].transpose(0, 1)
        U = scale * q @ k.transpose(1, 2)
        ez = abs(scale) * ((D + 4) * E + pair) * (q.abs() @ k.abs().transpose(1, 2))
        ez = ez + abs(scale) * (s_el["q"] * k.abs().sum(-1)[:, None]
                                + s_el["k"] * q.abs().sum(-1)[:, :, None])
        S = cap * torch.tanh(U / cap) if cap else U
        ez = ez + 8 * E * (S.abs() + cap)
        slope = 1 - (S / cap) ** 2 if cap else torch.ones_like(S)
        eslope = (16 * E + 2 * ez / cap) if cap else torch.zeros_like(S)
        if "sigma" in w:
            diff = w["q_pos"][I][:, None] - w["k_pos"][J][None]
            r2 = diff.square().sum(-1)
            bias = r2 / (2 * w["sigma"][:, None, None] ** 2)
            S = S - bias
            ez = ez + 16 * E * bias
        P = torch.softmax(S, -1)
        # an error where P vanishes moves nothing: weigh by what P can become
        rp = (2 * torch.where(P > 1e-30, ez, torch.zeros_like(ez)).amax(-1, keepdim=True)
              + 2.0 ** -19)
        peak = P.amax(-1, keepdim=True)
        smallp = 0.0 if dtype == torch.bfloat16 else 2.0 ** -31 * (2.0 ** -8 if pair else 1)
        nj, ni = J.numel(), I.numel()
        o = P @ v
        bo = lambda r: (P * (r + rp + (nj + 4) * E) + smallp * peak) @ v.abs() \
            + s_el["v"]  # noqa: E731
        out[I] = o.transpose(0, 1)
        b_out[I] = (bo(up) + u * o.abs()).transpose(0, 1)
        dP = go @ v.transpose(1, 2)
        Di = (go * o).sum(-1, keepdim=True)
        edp = ((D + 4) * E + pair) * (go.abs() @ v.abs().transpose(1, 2))
        edp = edp + s_el["g"] * v.abs().sum(-1)[:, None] + s_el["v"] * go.abs().sum(-1)[:, :, None]
        eD = (go.abs() * (bo(fine) + (D + 4) * E * o.abs())).sum(-1, keepdim=True)
        dS = P * (dP - Di)
        # exponentials below 2^-126 are flushed to zero
        eS = 2.0 ** -126 * (dP.abs() + Di.abs())
        eS = eS + P * (rp * (dP.abs() + Di.abs()) + edp + eD + 4 * E * (dP - Di).abs())
        if "sigma" in w:
            s2 = w["sigma"][:, None, None] ** 2
            for name, idx, dim, sgn in (("q_pos", I, 1, -1), ("k_pos", J, 0, 1)):
                per = (dS / s2)[..., None] * diff
                # each head's sum over the other side, then over the heads
                gr[name][idx] = sgn * per.sum((0, dim + 1))
                e = ((eS + 6 * E * dS.abs() + (nj + ni + heads + 8) * E * dS.abs()) / s2)[..., None] \
                    * diff.abs()
                b[name][idx] = e.sum((0, dim + 1)) + E * gr[name][idx].abs()
            gr["sigma"] += (dS * r2).sum((1, 2)) / w["sigma"] ** 3
            b["sigma"] += ((eS + (nj + 16) * E * dS.abs()) * r2).sum((1, 2)) / w["sigma"] ** 3
        dU = dS * slope
        eU = eS * slope + dS.abs() * eslope + up * dU.abs() + small_ds + 4 * E * dU.abs()
        gr["q"][I] = (scale * dU @ k).transpose(0, 1)
        b["q"][I] = (abs(scale) * (eU + ((nj + 4) * E + pair) * dU.abs()) @ k.abs()).transpose(0, 1)
        b["q"][I] += abs(scale) * s_el["k"] * dU.abs().sum(-1).T[..., None]
        dk = scale * dU.transpose(1, 2) @ q
        n_all = ni * (heads // kv)
        bk = abs(scale) * (eU + ((n_all + 4) * E + pair) * dU.abs()).transpose(1, 2) @ q.abs()
        dv = P.transpose(1, 2) @ go
        bv = (P * (up + rp + (n_all + 4) * E + pair) + 2.0 ** -36).transpose(1, 2) @ go.abs()
        bk = bk + abs(scale) * s_el["q"] * dU.abs().sum(1)[..., None]
        bv = bv + s_el["g"] * P.sum(1)[..., None]
        for name, t, e in (("k", dk, bk), ("v", dv, bv)):
            fold = lambda x: x.reshape(kv, heads // kv, *x.shape[1:]).sum(1).transpose(0, 1)  # noqa: E731
            gr[name][J] = fold(t)
            b[name][J] = fold(e)
    for n in ("q", "k", "v"):
        b[n] = b[n] + u * gr[n].abs() + tiny
    for n in names[3:]:
        b[n] = b[n] + 4 * E * gr[n].abs() + 1e-30
    return (out, b_out + tiny), {n: (gr[n], b[n]) for n in names}


def close(got, want, bound, what):
    got = got.detach()
    assert torch.isfinite(got).all(), what
    off = (got.double() - want).abs() - bound
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, (what, worst, float(bound.max()), float((off + bound).max()))


def check(d, nq, nk, scale=None, cap=0.0, dense=False, masks=(None, None), call=None):
    names = [n for n in ("q", "k", "v", "q_pos", "k_pos", "sigma") if n in d]
    leaves = {n: d[n].detach().requires_grad_(True) for n in names}
    kw = dict(scale=scale, softcap=cap, **{n: leaves[n] for n in names[3:]})
    if dense:
        B = len(nq)

        def pad(t):
            return t.reshape(B, -1, *t.shape[1:])
        kw.update({n: pad(kw[n]) for n in ("q_pos", "k_pos") if n in kw})

        def fn(no_grad=False):
            m = [None if t is None else t.reshape(B, -1) for t in masks]
            return ra.kernel_attention_dense(pad(leaves["q"]), pad(leaves["k"]), pad(leaves["v"]),
                                             *m, **kw).reshape(d["q"].shape)
    else:
        seg = ra.attention_segments(ptr(nq), ptr(nk))

        def fn():
            return ra.pyg_kernel_attention(leaves["q"], leaves["k"], leaves["v"], segments=seg,
                                           q_mask=masks[0], k_mask=masks[1], **kw)
    o = fn()
    grads = torch.autograd.grad(o, [leaves[n] for n in names], d["g"])
    with torch.no_grad():
        o2 = fn()
    (o64, bo), g64 = exact(d, nq, nk, d["q"].shape[2] ** -0.5 if scale is None else scale, cap,
                           *masks)
    close(o, o64, bo, "out")
    close(o2, o64, bo, "out without gradients")
    for n, g in zip(names, grads):
        assert g.dtype == d[n].dtype and g.shape == d[n].shape
        close(g, *g64[n], "d" + n)
    return o, grads


RAGGED = [([1], [1]), ([3], [2]), ([64], [64]), ([65], [127]), ([128], [129]), ([130], [300]),
          ([0, 5, 0, 200, 1], [4, 0, 0, 77, 130]), ([33, 2, 512], [33, 2, 512]),
          ([1, 1, 1], [70, 1, 1000])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nk", RAGGED)
def test_lengths(nq, nk, dtype, cuda_device):
    check(make(nq, nk, 4, 2, 32, dtype, 3, seed=len(nq)), nq, nk)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 5, 8, 16, 24, 40, 64, 72, 96, 128, 136, 256])
def test_head_widths(dim, dtype, cuda_device):
    n = [40, 150]
    check(make(n, n, 2, 2, dim, dtype, 2, seed=dim), n, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pos", [0, 1, 2, 3])
@pytest.mark.parametrize("cap", [0.0, 2.0, 30.0])
def test_positions_and_cap(cap, pos, dtype, cuda_device):
    nq, nk = [70, 129], [140, 90]
    check(make(nq, nk, 3, 1, 48, dtype, pos, seed=pos), nq, nk, cap=cap, scale=-0.3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_dense_masks(dtype, cuda_device):
    """Any pattern of masks, a cloud with none valid, NaN and infinities in
    masked rows."""
    B, N, M = 5, 90, 140
    nq, nk = [N] * B, [M] * B
    d = make(nq, nk, 4, 4, 64, dtype, 3, seed=5)
    g = torch.Generator(device="cuda").manual_seed(6)
    mq = torch.rand(B * N, generator=g, device="cuda") > 0.3
    mk = torch.rand(B * M, generator=g, device="cuda") > 0.4
    mk[2 * M:3 * M] = False
    mk[M:M + 130] = False
    mq[3 * N:4 * N] = False
    clean = check(d, nq, nk, dense=True, masks=(mq, mk))
    dirty = {n: t.clone() for n, t in d.items()}
    for i, n in enumerate(("q", "g", "k", "v")):
        bad = ~mq if i < 2 else ~mk
        dirty[n][bad] = math.nan
        if n == "k":
            dirty[n][bad.nonzero()[::2, 0]] = math.inf
    dirty["q_pos"][~mq] = math.nan
    dirty["k_pos"][~mk] = -math.inf
    o, grads = check(dirty, nq, nk, dense=True, masks=(mq, mk))
    assert torch.equal(o, clean[0])
    assert all(torch.equal(a, b) for a, b in zip(grads, clean[1]))
    assert not o[~mq].any() and not o[2 * N:3 * N].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_neighbours_do_not_leak(dtype, cuda_device):
    """NaN in one graph reaches no other, tiles and alignment aside."""
    n = [50, 3, 200, 77]
    d = make(n, n, 2, 1, 32, dtype, 2, seed=8)
    names = ("q", "k", "v", "q_pos", "k_pos", "sigma")
    p = ptr(n)

    def run(x):
        leaves = [x[k].detach().requires_grad_(True) for k in names]
        o = ra.pyg_kernel_attention(*leaves[:3], q_ptr=p, q_pos=leaves[3], k_pos=leaves[4],
                                    sigma=leaves[5])
        return (o, *torch.autograd.grad(o, leaves[:5], x["g"]))

    bad = {k: t.clone() for k, t in d.items()}
    rows = slice(53, 253)
    for x in (d, bad):  # fp16 operands are scaled by their tensor's maximum: in a clean row
        for k in ("q", "k", "v", "g"):
            x[k][0, 0, 0] = 8.0
    want = run(d)
    for k in ("q", "k", "v", "g"):
        bad[k][rows] = math.nan
    got = run(bad)
    for a, b in zip(got, want):
        assert torch.equal(a[:53], b[:53]) and torch.equal(a[253:], b[253:])
        assert torch.isnan(a[rows]).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_keys_few_queries(dtype, cuda_device):
    nq, nk = [1, 3], [40000, 5000]
    check(make(nq, nk, 8, 2, 64, dtype, 3, seed=9), nq, nk)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [8, 24, 64, 104])
@pytest.mark.parametrize("nq,heads,kv", [([1, 1, 1, 1], 1, 1), ([1, 0, 1, 1], 4, 2),
                                         ([2, 1, 0, 2], 2, 1), ([1, 1, 1, 1], 8, 1),
                                         ([8, 3, 1, 0], 3, 3)])
def test_few_rows(nq, heads, kv, dim, dtype, cuda_device):
    """Up to eight rows a graph and key head, short and long key ranges,
    masks, the cap."""
    nk = [3000, 5, 600, 0]
    d = make(nq, nk, heads, kv, dim, dtype, 3, seed=dim + heads)
    check(d, nq, nk)
    g = torch.Generator(device="cuda").manual_seed(4)
    mq = torch.rand(sum(nq), generator=g, device="cuda") > 0.2
    mk = torch.rand(sum(nk), generator=g, device="cuda") > 0.3
    mk[3000:3005] = False
    for n in ("k", "v"):
        d[n][~mk] = math.nan
    d["k_pos"][~mk] = math.inf
    check(d, nq, nk, masks=(mq, mk), cap=4.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_queries_few_keys(dtype, cuda_device):
    nq, nk = [20000, 1], [1, 2]
    check(make(nq, nk, 2, 2, 32, dtype, 0, seed=10), nq, nk)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype, cuda_device):
    """Maxima that grow along the keys, weights of 0 and 1."""
    n = [300]
    d = make(n, n, 2, 2, 64, dtype, 3, seed=11)
    ramp = torch.linspace(0.01, 6, 300, device="cuda")[:, None, None]
    d["k"] = (d["k"].float() * ramp).to(dtype)
    check(d, n, n, scale=0.5)
    d["k"] = d["k"].flip(0)
    check(d, n, n, scale=0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype, cuda_device):
    """A fused projection's slices, heads first, broadcast heads and rows."""
    n = [31, 140]
    rows, H, D = sum(n), 4, 32
    d = make(n, n, H, H, D, dtype, 2, seed=12)
    fused = torch.zeros(rows, 3 * H * D + 5, dtype=dtype, device="cuda")
    views = [fused[:, 2 + i * H * D:2 + (i + 1) * H * D].view(rows, H, D) for i in range(3)]
    for t, name in zip(views, "qkv"):
        t.copy_(d[name])
    seg = ra.attention_segments(ptr(n))
    kw = dict(segments=seg, q_pos=d["q_pos"], k_pos=d["k_pos"], sigma=d["sigma"])
    want = ra.pyg_kernel_attention(d["q"], d["k"], d["v"], **kw)
    assert torch.equal(ra.pyg_kernel_attention(*views, **kw), want) or \
        (ra.pyg_kernel_attention(*views, **kw).float() - want.float()).abs().max() < 0.02
    heads_first = [d[x].transpose(0, 1).contiguous().transpose(0, 1) for x in "qkv"]
    assert torch.equal(ra.pyg_kernel_attention(*heads_first, **kw), want)
    one = d["k"][:, :1]
    a = ra.pyg_kernel_attention(d["q"], one.expand(rows, H, D), d["v"], **kw)
    b = ra.pyg_kernel_attention(d["q"], one.expand(rows, H, D).contiguous(), d["v"], **kw)
    assert torch.equal(a, b)
    # gradients of a broadcast input add up
    src = d["k"][:1, :1].detach().requires_grad_(True)
    full = src.detach().expand(rows, H, D).contiguous().requires_grad_(True)
    g1, = torch.autograd.grad(ra.pyg_kernel_attention(d["q"], src.expand(rows, H, D), d["v"], **kw),
                              src, d["g"])
    g2, = torch.autograd.grad(ra.pyg_kernel_attention(d["q"], full, d["v"], **kw), full, d["g"])
    assert torch.equal(g1, g2.sum((0, 1), keepdim=True))


def test_kernel_weights_without_scores(cuda_device):
    """q = k = 0: the normalised Gaussian kernel of the framework's sums."""
    n, m = 60, 45
    x, y = torch.randn(n, 3, device="cuda"), torch.randn(m, 3, device="cuda")
    z = torch.zeros(n, 1, 8, device="cuda")
    v = torch.ones(m, 1, 8, device="cuda") * torch.arange(m, device="cuda")[:, None, None]
    o = ra.pyg_kernel_attention(z, torch.zeros(m, 1, 8, device="cuda"), v,
                                q_ptr=ptr([n]), k_ptr=ptr([m]), q_pos=x, k_pos=y, sigma=0.7)
    k = torch.exp(-(x.double()[:, None] - y.double()[None]).square().sum(-1) / (2 * 0.7 ** 2))
    want = (k @ torch.arange(m, device="cuda").double()) / k.sum(1)
    assert (o[:, 0, 0].double() - want).abs().max() < 44 * 2.0 ** -17


def test_self_attention_positions(cuda_device):
    """One position tensor for both sides, a scalar sigma, batch vectors."""
    n = [20, 41]
    d = make(n, n, 2, 2, 16, torch.float32, 3, seed=14)
    batch = torch.repeat_interleave(torch.arange(2, device="cuda"), torch.tensor(n, device="cuda"))
    p = d["q_pos"].detach().requires_grad_(True)
    s = torch.tensor(0.8, device="cuda", requires_grad=True)
    o = ra.pyg_kernel_attention(d["q"], d["k"], d["v"], q_batch=batch, q_pos=p, sigma=s)
    gp, gs = torch.autograd.grad(o, [p, s], d["g"])
    pq, pk = (d["q_pos"].detach().clone().requires_grad_(True) for _ in range(2))
    sg = torch.full((2,), 0.8, device="cuda", requires_grad=True)
    o2 = ra.pyg_kernel_attention(d["q"], d["k"], d["v"], q_ptr=ptr(n), k_ptr=ptr(n), q_pos=pq,
                                 k_pos=pk, sigma=sg)
    a, b, c = torch.autograd.grad(o2, [pq, pk, sg], d["g"])
    assert torch.equal(o, o2) and torch.equal(gp, a + b) and torch.equal(gs, c.sum())


@pytest.mark.parametrize("dtype", DTYPES)
def test_some_gradients(dtype, cuda_device):
    """Each gradient alone is what it is among all."""
    n = [90, 200]
    d = make(n, n, 4, 2, 64, dtype, 3, seed=15)
    names = ("q", "k", "v", "q_pos", "k_pos", "sigma")
    seg = ra.attention_segments(ptr(n))

    def grads(wanted):
        x = {k: d[k].detach().requires_grad_(k in wanted) for k in names}
        o = ra.pyg_kernel_attention(x["q"], x["k"], x["v"], segments=seg, q_pos=x["q_pos"],
                                    k_pos=x["k_pos"], sigma=x["sigma"])
        return torch.autograd.grad(o, [x[k] for k in wanted], d["g"])

    every = dict(zip(names, grads(names)))
    for k in names:
        assert torch.equal(grads((k,))[0], every[k])


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeatable(dtype, cuda_device):
    n = [700, 33, 128, 400]
    d = make(n, n, 4, 2, 64, dtype, 3, seed=16)
    runs = [check(d, n, n) for _ in range(2)]
    assert torch.equal(runs[0][0], runs[1][0])
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))


def test_differences(cuda_device):
    """Directional derivatives against central differences of <out, g>: off by
    about h^2 of the third derivative (< 1e-3 of the gradient's norm at this
    h) and by the outputs' rounding, 2^-21 |out| |g| / h."""
    n = [60, 100]
    d = make(n, n, 2, 1, 32, torch.float32, 3, seed=17)
    d["sigma"] = torch.tensor([0.8, 1.5], device="cuda")
    names = ("q", "k", "v", "q_pos", "k_pos", "sigma")
    x = {k: d[k].detach().requires_grad_(True) for k in names}
    seg = ra.attention_segments(ptr(n))

    def f(x):
        return ra.pyg_kernel_attention(x["q"], x["k"], x["v"], segments=seg, q_pos=x["q_pos"],
                                       k_pos=x["k_pos"], sigma=x["sigma"], softcap=3.0)

    o = f(x)
    grads = torch.autograd.grad(o, [x[k] for k in names], d["g"])
    gen = torch.Generator(device="cuda").manual_seed(3)
    h = 2.0 ** -6
    noise = 2.0 ** -21 * float(o.detach().norm() * d["g"].norm()) / h
    for k, g in zip(names, grads):
        step = torch.randn(g.shape, generator=gen, device="cuda")
        step = step / step.norm()
        with torch.no_grad():
            up = f({**x, k: x[k] + h * step}).double()
            down = f({**x, k: x[k] - h * step}).double()
        got = float(((up - down) * d["g"].double()).sum() / (2 * h))
        want = float((g.double() * step.double()).sum())
        assert abs(got - want) <= 2e-3 * float(g.norm()) + noise, k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_other_stream_and_capture(dtype, cuda_device):
    n = [100, 260]
    names = ("q", "k", "v", "q_pos", "k_pos", "sigma")
    d = make(n, n, 4, 2, 64, dtype, 3, seed=18)
    x = {k: d[k].detach().requires_grad_(True) for k in names}
    seg = ra.attention_segments(ptr(n))

    def step():
        o = ra.pyg_kernel_attention(x["q"], x["k"], x["v"], segments=seg, q_pos=x["q_pos"],
                                    k_pos=x["k_pos"], sigma=x["sigma"])
        return (o.detach(), *torch.autograd.grad(o, [x[k] for k in names], d["g"]))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    other = make(n, n, 4, 2, 64, dtype, 3, seed=19)
    with torch.no_grad():
        for k in names:
            x[k].copy_(other[k])
        d["g"].copy_(other["g"])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 40, 128])
def test_few_rows_of_slices_replayed(dim, dtype, cuda_device):
    """One query a graph against slices of a fused projection whose other
    columns hold NaN, and a replayed graph of it on new values."""
    nq, nk = [1, 1, 1], [9000, 1, 33]
    d = make(nq, nk, 6, 2, dim, dtype, 2, seed=dim)
    fused = torch.full((sum(nk), 2, 2 * dim + 24), math.nan, dtype=dtype, device="cuda")
    k, v = fused[..., 8:8 + dim], fused[..., 16 + dim:16 + 2 * dim]
    k.copy_(d["k"]), v.copy_(d["v"])
    d["k"], d["v"] = k, v
    seg = ra.attention_segments(ptr(nq), ptr(nk))

    def step():
        return ra.pyg_kernel_attention(d["q"], k, v, segments=seg, q_pos=d["q_pos"],
                                       k_pos=d["k_pos"], sigma=d["sigma"])

    (o64, bo), _ = exact(d, nq, nk, dim ** -0.5, 0.0)
    close(step(), o64, bo, "out")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n, t in make(nq, nk, 6, 2, dim, dtype, 2, seed=dim + 1).items():
        d[n].copy_(t)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, step())
    (o64, bo), _ = exact(d, nq, nk, dim ** -0.5, 0.0)
    close(held, o64, bo, "replayed out")


def test_calls_from_two_threads(cuda_device):
    """Calls at the same time, each on its own stream: what each is alone."""
    sizes = [([1] * 5, [700, 3, 64, 65, 2000]), ([90, 200], [90, 200])]
    data = [make(*n, 4, 2, 64, torch.bfloat16, 3, seed=i) for i, n in enumerate(sizes)]
    segs = [ra.attention_segments(ptr(a), ptr(b)) for a, b in sizes]

    def step(i):
        x = {n: t.detach().requires_grad_(n != "g") for n, t in data[i].items()}
        o = ra.pyg_kernel_attention(x["q"], x["k"], x["v"], segments=segs[i], q_pos=x["q_pos"],
                                    k_pos=x["k_pos"], sigma=x["sigma"])
        return (o.detach(), *torch.autograd.grad(o, [x["q"], x["k"], x["v"]], x["g"]))

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[i].extend(step(i) for _ in range(20))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20
        assert all(torch.equal(a, b) for g in got[i] for a, b in zip(g, want[i]))


def test_refusals_on_the_device(cuda_device):
    q = torch.zeros(6, 2, 8, device="cuda")
    with pytest.raises(ValueError, match="start at 0"):
        ra.attention_segments(torch.tensor([1, 6], device="cuda"))
    with pytest.raises(ValueError, match="match node stacks"):
        ra.attention_segments(torch.tensor([0, 4, 3, 6], device="cuda"))
    with pytest.raises(ValueError, match="same length"):
        ra.attention_segments(torch.tensor([0, 6], device="cuda"),
                              torch.tensor([0, 3, 6], device="cuda"))
    with pytest.raises(ValueError, match="equal number of nodes"):
        ra.pyg_kernel_attention(q, q, q, q_ptr=torch.tensor([0, 5], device="cuda"))
    seg = ra.attention_segments(torch.tensor([0, 6], device="cuda"))
    with pytest.raises(ValueError, match="either segments or"):
        ra.pyg_kernel_attention(q, q, q, segments=seg, q_ptr=torch.tensor([0, 6], device="cuda"))
    with pytest.raises(ValueError, match="masks must have shape"):
        ra.pyg_kernel_attention(q, q, q, segments=seg, q_mask=torch.ones(5, device="cuda"))
    with pytest.raises(ValueError, match="sorted"):
        ra.pyg_kernel_attention(q, q, q, q_batch=torch.tensor([0, 0, 2, 1, 1, 1], device="cuda"))


def test_the_plan_is_its_own(cuda_device):
    """Writing to the offsets afterwards changes nothing."""
    p = torch.tensor([0, 2, 6], device="cuda")
    q = torch.randn(6, 2, 8, device="cuda")
    seg = ra.attention_segments(p)
    want = ra.pyg_kernel_attention(q, q, q, segments=seg)
    p.fill_(1 << 40)
    assert torch.equal(ra.pyg_kernel_attention(q, q, q, segments=seg), want)


def test_nothing_to_do(cuda_device):
    z = torch.zeros(0, 2, 8, device="cuda", requires_grad=True)
    one = torch.randn(3, 2, 8, device="cuda", requires_grad=True)
    p0, p3 = (torch.tensor([0, n], device="cuda") for n in (0, 3))
    o = ra.pyg_kernel_attention(z, one, one, q_ptr=p0, k_ptr=p3)
    assert o.shape == (0, 2, 8)
    g = torch.autograd.grad(o.sum(), [z, one])
    assert g[0].shape == (0, 2, 8) and not g[1].any()
    o = ra.pyg_kernel_attention(one, z, z, q_ptr=p3, k_ptr=p0)
    assert not o.any()
    g = torch.autograd.grad(o.sum(), [one, z])
    assert not g[0].any()
    none = torch.tensor([0], device="cuda")
    assert ra.pyg_kernel_attention(z, z, z, q_ptr=none).shape == (0, 2, 8)
    e = torch.zeros(0, 4, 2, 8, device="cuda")
    assert ra.kernel_attention_dense(e, e, e).shape == (0, 4, 2, 8)


def test_attention_trains_a_classifier_head(cuda_device):
    """The two operators as they are used together: embeddings made by
    attention inside each graph, scored against a table; gradients of the
    whole against float64 autograd of the plain formulas.  The embeddings
    and logits carry fp32 steps only: 1e-5 of each gradient's norm."""
    n = [40, 100, 7]
    H, D, V = 2, 16, 50
    d = make(n, n, H, H, D, torch.float32, 3, seed=20)
    table = torch.randn(V, H * D, device="cuda")
    target = torch.randint(0, V, (sum(n),), device="cuda")
    names = ("q", "k", "v", "q_pos", "sigma")
    x = {k: d[k].detach().requires_grad_(True) for k in names}
    t = table.detach().requires_grad_(True)
    o = ra.pyg_kernel_attention(x["q"], x["k"], x["v"], q_ptr=ptr(n), q_pos=x["q_pos"],
                                sigma=x["sigma"])
    loss, lse = ra.linear_cross_entropy(o.reshape(sum(n), H * D), t, target)
    got = torch.autograd.grad(loss, [x[k] for k in names] + [t])
    y = {k: d[k].double().requires_grad_(True) for k in names}
    t64 = table.double().requires_grad_(True)
    outs, a = [], 0
    for m in n:
        r = slice(a, a + m)
        a += m
        s = torch.einsum("ihd,jhd->hij", y["q"][r], y["k"][r]) / D ** 0.5
        r2 = (y["q_pos"][r][:, None] - y["q_pos"][r][None]).square().sum(-1)
        s = s - r2 / (2 * y["sigma"][:, None, None] ** 2)
        outs.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), y["v"][r]))
    z = torch.cat(outs).reshape(sum(n), H * D) @ t64.T
    want_loss = (torch.logsumexp(z, 1) - z.gather(1, target[:, None])[:, 0]).mean()
    want = torch.autograd.grad(want_loss, [y[k] for k in names] + [t64])
    assert abs(float(loss.detach()) - float(want_loss.detach())) < 1e-5
    for g, w in zip(got, want):
        assert (g.double() - w).norm() <= 1e-5 * w.norm()
