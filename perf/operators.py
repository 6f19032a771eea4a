"""Cases of the softmax operators: attention over ragged batches of graphs and
the cross entropy over a large table, forward and backward.

``run`` computes a case in its plain form (elementary torch operations in 32
bits, rounded once at the end), or through ``rapidalign_b200`` when ``own``
is set.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_IGNORE = -100


def _attn(name, **kw):
    case = dict(name=name, op="attention", layout="ragged", graphs=1, nmin=1, nmax=1, kmin=0,
                kmax=0, heads=4, kv_heads=4, dim=32, dtype="fp32", pos=3, cap=0.0, train=True)
    case.update(kw)
    return case


def _ce(name, **kw):
    case = dict(name=name, op="cross_entropy", rows=1, vocab=1, dim=128, dtype="fp32", cap=0.0,
                train=True)
    case.update(kw)
    return case


def listed():
    return [
        # one small cloud of the single-pair configuration: latency
        _attn("attn_one_cloud", graphs=1, nmin=128, nmax=128),
        # node embeddings (D = 128) of a ragged batch of 64-512 nodes, as the
        # embedding workload has them, trained in fp32 with learned sigmas
        _attn("attn_embed_fp32", graphs=256, nmin=64, nmax=512),
        # the same batch in mixed precision, wider heads, two heads a key
        _attn("attn_embed_bf16", graphs=512, nmin=64, nmax=512, heads=4, kv_heads=2, dim=64,
              dtype="bf16"),
        # big graphs up to the ragged workload's largest cloud, no positions,
        # capped scores
        _attn("attn_big_bf16", graphs=32, nmin=33, nmax=2048, heads=8, kv_heads=8, dim=128,
              dtype="bf16", pos=0, cap=30.0),
        # padded clouds with masks (64 x 1024, 512-1024 valid), evaluation
        _attn("attn_dense_fp16", layout="dense", graphs=64, nmin=512, nmax=1024, heads=4,
              kv_heads=4, dim=64, dtype="fp16", train=False),
        # one query a graph: attention pooling of a served batch
        _attn("attn_pool", graphs=1024, nmin=1, nmax=1, kmin=64, kmax=512, heads=8, kv_heads=2,
              dim=64, dtype="bf16", train=False),
        # one query against one huge cloud
        _attn("attn_one_query", graphs=1, nmin=1, nmax=1, kmin=262144, kmax=262144, heads=8,
              kv_heads=2, dim=64, dtype="bf16", train=False),
        # a small classification step: latency
        _ce("ce_small", rows=128, vocab=1000),
        # every node of an embedding batch against a table of classes, fp32
        _ce("ce_embed_fp32", rows=65537, vocab=4099, dim=128),
        # a large vocabulary, mixed-precision training
        _ce("ce_train_bf16", rows=8192, vocab=131072, dim=1024, dtype="bf16"),
        # evaluation over an odd vocabulary with capped logits
        _ce("ce_eval_fp16", rows=4096, vocab=50001, dim=512, dtype="fp16", cap=30.0, train=False),
        # scoring a few tokens: the table is read once
        _ce("ce_few_rows", rows=5, vocab=131072, dim=1024, dtype="bf16", train=False),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    cap = rng.choice([0.0, 0.0, 20.0, 50.0])
    if rng.random() < 0.55:
        nmax = _log_uniform(rng, 16, 1500)
        nmin = rng.randint(1, nmax)
        kv = rng.choice([1, 2, 4])
        heads = kv * rng.choice([1, 2])
        budget = 1.2e8  # graphs x heads x longest^2 (the plain form pads)
        most = max(1, min(512, int(budget / (heads * nmax * nmax))))
        layout = rng.choice(["ragged", "ragged", "dense"])
        kind = rng.random()
        case = dict(op="attention", layout=layout, graphs=_log_uniform(rng, 1, most), nmin=nmin,
                    nmax=nmax, kmin=0, kmax=0, heads=heads, kv_heads=kv,
                    dim=rng.choice([16, 24, 32, 40, 64, 96, 128]), dtype=dtype,
                    pos=rng.choice([0, 2, 3, 3]), cap=cap, train=rng.random() < 0.6)
        if layout == "ragged" and kind < 0.35:  # queries and keys of their own lengths
            case["kmax"] = _log_uniform(rng, 16, 1500)
            case["kmin"] = rng.randint(1, case["kmax"])
            most = max(1, min(512, int(budget / (heads * nmax * case["kmax"]))))
            case["graphs"] = _log_uniform(rng, 1, most)
        elif layout == "ragged" and kind < 0.5:  # single queries, long keys
            case.update(nmin=1, nmax=1, kmax=_log_uniform(rng, 64, 100000), train=False)
            case["kmin"] = rng.randint(1, case["kmax"])
            case["graphs"] = _log_uniform(rng, 1, max(1, min(512, 200000 // case["kmax"])))
        return case
    rows = _log_uniform(rng, 1, 20000)
    vocab = _log_uniform(rng, 100, 140000)
    if rows * vocab > 5e8:
        vocab = max(100, int(5e8 / rows))
    return dict(op="cross_entropy", rows=rows, vocab=vocab,
                dim=rng.choice([64, 100, 128, 256, 264, 512, 768]), dtype=dtype, cap=cap,
                train=rng.random() < 0.6)


def _sizes(lo, hi, n):
    """n sizes spread evenly over lo..hi (the same for every seed)."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case):
    q = _sizes(case["nmin"], case["nmax"], case["graphs"])
    k = _sizes(case["kmin"], case["kmax"], case["graphs"]) if case["kmax"] else q
    return q, k


def _shuffled(sizes, perm):
    return [sizes[i] for i in perm]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * scale

    st = {"case": case}
    if case["op"] == "cross_entropy":
        n, v, d = case["rows"], case["vocab"], case["dim"]
        st["x"] = randn(n, d).to(dt)
        st["w"] = randn(v, d, scale=2.0 / math.sqrt(d)).to(dt)
        t = torch.randint(0, v, (n,), generator=gen, device=dev)
        if n > 1:  # some rows have no label
            t[torch.rand(n, generator=gen, device=dev) < 0.05] = _IGNORE
            t[0] = 0
        st["target"] = t
        for name in ("x", "w"):
            st[name].requires_grad_(case["train"])
        return st

    P, H, HK, D, C = (case[k] for k in ("graphs", "heads", "kv_heads", "dim", "pos"))
    perm = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
    nq, nk = _lengths(case)
    nq, nk = _shuffled(nq, perm), _shuffled(nk, perm)
    if case["layout"] == "dense":
        # padded clouds: the tail is masked and holds whatever was there, a
        # few valid places are masked too, one cloud is empty where there are many
        N = case["nmax"]
        lens = torch.tensor(nq, device=dev)
        mask = torch.arange(N, device=dev)[None] < lens[:, None]
        mask &= torch.rand(P, N, generator=gen, device=dev) > 0.02
        if P > 8:
            mask[seed % P] = False
        shape_q, shape_k = (P, N), (P, N)
        st["mask"] = mask
    else:
        shape_q, shape_k = (sum(nq),), (sum(nk),)
        st["q_ptr"] = torch.tensor([0] + nq, device=dev).cumsum(0)
        st["k_ptr"] = torch.tensor([0] + nk, device=dev).cumsum(0)
        st["max_q"], st["max_k"] = max(nq), max(nk)
    st["q"] = randn(*shape_q, H, D).to(dt)
    st["k"] = randn(*shape_k, HK, D).to(dt)
    st["v"] = randn(*shape_k, HK, D).to(dt)
    if case["layout"] == "dense":
        for name in ("q", "k", "v"):
            st[name][~mask] = math.nan
    same = case["kmax"] == 0
    st["q_pos"] = st["k_pos"] = st["sigma"] = None
    if C:
        st["q_pos"] = randn(*shape_q, C)
        st["k_pos"] = st["q_pos"].clone() if same else randn(*shape_k, C)
        st["sigma"] = torch.tensor([0.25 * 2.0 ** (i % 4) for i in range(H)], device=dev)
    st["g"] = randn(*shape_q, H, D).to(dt)
    st["inputs"] = [n for n in ("q", "k", "v", "q_pos", "k_pos", "sigma") if st[n] is not None]
    for name in st["inputs"]:
        st[name].requires_grad_(case["train"])
    if own and case["layout"] == "ragged":
        import rapidalign_b200 as ra
        st["segments"] = ra.attention_segments(st["q_ptr"], st["k_ptr"])
    return st


# ---- plain forms -------------------------------------------------------------

def _padded(t, ptr, longest):
    """(graphs, longest, ...) rows of each graph, zeros behind its end."""
    place = torch.arange(longest, device=ptr.device)[None] + ptr[:-1, None]
    valid = place < ptr[1:, None]
    rows = t[place.clamp(max=max(t.shape[0] - 1, 0))]
    return torch.where(valid.reshape(valid.shape + (1,) * (t.dim() - 1)), rows,
                       torch.zeros((), device=t.device)), valid


def _plain_attention(st, q, k, v, q_pos, k_pos, sigma):
    case = st["case"]
    zero = torch.zeros((), device=q.device)
    if case["layout"] == "dense":
        vq = vk = st["mask"]
        q, k, v = (torch.where(st["mask"][:, :, None, None], t, zero) for t in (q, k, v))
        pq, pk = q_pos, k_pos
    else:
        (q, vq), (k, vk) = (_padded(q, st["q_ptr"], st["max_q"]),
                            _padded(k, st["k_ptr"], st["max_k"]))
        v = _padded(v, st["k_ptr"], st["max_k"])[0]
        pq = None if q_pos is None else _padded(q_pos, st["q_ptr"], st["max_q"])[0]
        pk = None if k_pos is None else _padded(k_pos, st["k_ptr"], st["max_k"])[0]
    group = case["heads"] // case["kv_heads"]
    k = k.repeat_interleave(group, dim=2)
    v = v.repeat_interleave(group, dim=2)
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))  # graphs, heads, rows, dim
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(case["dim"]))
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    if pq is not None:
        r2 = ((pq[:, :, None] - pk[:, None]) ** 2).sum(-1)
        s = s - r2[:, None] / (2.0 * sigma * sigma)[None, :, None, None]
    keep = vq[:, None, :, None] & vk[:, None, None, :]
    s = torch.where(keep, s, torch.full((), -1e30, device=s.device))
    e = torch.exp(s - s.amax(-1, keepdim=True).detach()) * keep
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.transpose(1, 2)
    return out if case["layout"] == "dense" else out[vq]


def _plain_cross_entropy(st, x, w):
    z = torch.matmul(x, w.t())
    cap = st["case"]["cap"]
    if cap:
        z = cap * torch.tanh(z / cap)
    top = z.amax(-1, keepdim=True).detach()
    lse = torch.log(torch.exp(z - top).sum(-1)) + top[:, 0]
    t = st["target"]
    labelled = t != _IGNORE
    at = z.gather(1, torch.where(labelled, t, 0)[:, None])[:, 0]
    rows = torch.where(labelled, lse - at, torch.zeros_like(lse))
    return rows.sum() / labelled.sum(), lse


# ---- one pass ----------------------------------------------------------------

def run(st):
    case = st["case"]
    if case["op"] == "cross_entropy":
        with torch.set_grad_enabled(case["train"]):
            if own:
                import rapidalign_b200 as ra
                loss, lse = ra.linear_cross_entropy(st["x"], st["w"], st["target"],
                                                    softcap=case["cap"], ignore_index=_IGNORE)
            else:
                loss, lse = _plain_cross_entropy(st, st["x"].float(), st["w"].float())
        out = {"loss": loss.detach(), "lse": lse.detach()}
        if case["train"]:
            out["dx"], out["dw"] = torch.autograd.grad(loss, [st["x"], st["w"]])
        return out

    leaves = [st[n] for n in st["inputs"]]
    with torch.set_grad_enabled(case["train"]):
        if own:
            import rapidalign_b200 as ra
            kw = dict(q_pos=st["q_pos"], k_pos=st["k_pos"], sigma=st["sigma"],
                      softcap=case["cap"])
            if case["layout"] == "dense":
                o = ra.kernel_attention_dense(st["q"], st["k"], st["v"], st["mask"], st["mask"],
                                              **kw)
            else:
                o = ra.pyg_kernel_attention(st["q"], st["k"], st["v"],
                                            segments=st["segments"], **kw)
        else:
            o = _plain_attention(st, st["q"].float(), st["k"].float(), st["v"].float(),
                                 st["q_pos"], st["k_pos"], st["sigma"]).to(st["q"].dtype)
    out = {"out": o.detach()}
    if case["train"]:
        grads = torch.autograd.grad(o, leaves, st["g"])
        out.update({"d" + n: g for n, g in zip(st["inputs"], grads)})
    return out


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "cross_entropy":
        n, v, d = case["rows"], case["vocab"], case["dim"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * size * d * (n + v) + 12 * n,
                "flops": (6 if case["train"] else 2) * n * v * d}
    nq, nk = _lengths(case)
    H, HK, D = case["heads"], case["kv_heads"], case["dim"]
    pairs = H * sum(a * b for a, b in zip(nq, nk))
    if case["layout"] == "dense":  # the padding is written (zeros), not read
        out_rows = case["graphs"] * case["nmax"]
    else:
        out_rows = sum(nq)
    moved = size * D * (H * (sum(nq) + out_rows) + 2 * HK * sum(nk))
    moved += 4 * case["pos"] * (sum(nq) + sum(nk))
    if case["train"]:
        moved += size * D * (H * (sum(nq) + out_rows) + 2 * HK * sum(nk))
        moved += 4 * case["pos"] * (sum(nq) + sum(nk))
    return {"bytes": moved, "flops": (12 if case["train"] else 4) * D * pairs}


# ---- the definition in 64 bits -------------------------------------------------

def _exact_cross_entropy(case, st):
    x, w, t = st["x"].detach().double(), st["w"].detach().double(), st["target"]
    n, cap, train = x.shape[0], case["cap"], case["train"]
    count = int((t != _IGNORE).sum())
    lse = torch.empty(n, dtype=torch.float64, device=x.device)
    total = torch.zeros((), dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    step = max(1, int(2e8) // w.shape[0])
    for a in range(0, n, step):
        b = min(n, a + step)
        z = x[a:b] @ w.T
        if cap:
            z = torch.tanh(z / cap) * cap
        lse[a:b] = torch.logsumexp(z, 1)
        rows = torch.nonzero(t[a:b] != _IGNORE)[:, 0]
        cols = t[a:b][rows]
        total += (lse[a:b][rows] - z[rows, cols]).sum()
        if train:
            g = torch.zeros_like(z)
            g[rows] = torch.exp(z[rows] - lse[a:b][rows, None]) / count
            g[rows, cols] -= 1.0 / count
            if cap:
                g *= 1.0 - (z / cap) ** 2
            dx[a:b] = g @ w
            dw += g.T @ x[a:b]
            del g
        del z
    out = {"loss": total / count, "lse": lse}
    if train:
        out.update(dx=dx, dw=dw)
    return out


def _exact_attention(case, st):
    names = st["inputs"]
    val = {n: st[n].detach().double() for n in names}
    g = st["g"].double()
    grads = {n: torch.zeros_like(val[n]) for n in names}
    out = torch.zeros_like(g)
    P, H, HK = case["graphs"], case["heads"], case["kv_heads"]
    a, cap = 1.0 / math.sqrt(case["dim"]), case["cap"]
    if case["layout"] == "dense":
        places = [torch.nonzero(st["mask"][p])[:, 0] for p in range(P)]
    else:
        qp, kp = st["q_ptr"].tolist(), st["k_ptr"].tolist()
    head = torch.arange(H, device=g.device) // (H // HK)
    for p in range(P):
        if case["layout"] == "dense":
            iq = ik = (p, places[p])
            if places[p].numel() == 0:
                continue
        else:
            iq, ik = slice(qp[p], qp[p + 1]), slice(kp[p], kp[p + 1])
        q = val["q"][iq].transpose(0, 1)
        k = val["k"][ik].transpose(0, 1)[head]
        v = val["v"][ik].transpose(0, 1)[head]
        u = torch.einsum("hid,hjd->hij", q, k) * a
        s = torch.tanh(u / cap) * cap if cap else u
        slope = 1.0 - (s / cap) ** 2 if cap else None
        if "sigma" in val:
            diff = val["q_pos"][iq][:, None] - val["k_pos"][ik][None]
            r2 = diff.square().sum(-1)
            sig = val["sigma"][:, None, None]
            s = s - r2 / (2.0 * sig ** 2)
        prob = torch.softmax(s, -1)
        o = prob @ v
        out[iq] = o.transpose(0, 1)
        if not case["train"]:
            continue
        go = g[iq].transpose(0, 1)
        ds = prob * (go @ v.transpose(1, 2) - (go * o).sum(-1, keepdim=True))
        if "sigma" in val:
            grads["sigma"] += (ds * r2).sum((1, 2)) / val["sigma"] ** 3
            per = torch.einsum("hij,h->ij", ds, val["sigma"] ** -2)
            grads["q_pos"][iq] = -(per[:, :, None] * diff).sum(1)
            grads["k_pos"][ik] = (per[:, :, None] * diff).sum(0)
        if slope is not None:
            ds = ds * slope
        grads["q"][iq] = (ds @ k * a).transpose(0, 1)
        dk = ds.transpose(1, 2) @ q * a
        dv = prob.transpose(1, 2) @ go
        grads["k"][ik] = dk.reshape(HK, H // HK, *dk.shape[1:]).sum(1).transpose(0, 1)
        grads["v"][ik] = dv.reshape(HK, H // HK, *dv.shape[1:]).sum(1).transpose(0, 1)
    res = {"out": out}
    if case["train"]:
        res.update({"d" + n: grads[n] for n in names})
    return res


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "cross_entropy":
        return _exact_cross_entropy(case, st)
    return _exact_attention(case, st)
