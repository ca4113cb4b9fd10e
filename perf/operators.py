"""Cases of the decoder's dense operators: attention with biased, capped and masked scores
(forward, backward, and for a few queries over many keys) and LayerNorm with its gradients.

With ``own`` false every case is computed in its plain form, from elementary torch operations in
fp32 and rounded once at the end; with ``own`` true by this package's operators.  ``exact`` is
the definition in 64 bits, its gradients by automatic differentiation.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _norm(name, dtype, rows, width):
    return {"name": name, "kind": "norm", "dtype": dtype, "rows": rows, "width": width}


def _attn(name, dtype, batch, queries, keys, heads, kv_heads, dim, train=False, pos=0, slopes="none", cap=0.0,
          documents=0, lens=False):
    """``pos`` coordinates per token for the distance bias (0: none), ``slopes`` "head" (one per
    head) or "row" (one per query and head), ``documents`` > 0 masks across that many documents,
    ``lens`` gives every batch entry its own number of valid keys."""
    return {"name": name, "kind": "attention", "dtype": dtype, "batch": batch, "queries": queries, "keys": keys,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "train": train, "pos": pos, "slopes": slopes,
            "cap": cap, "documents": documents, "lens": lens}


def listed():
    return [
        # One frame's decoder norm in training: 900 instances of 256 features, forward and gradients.
        _norm("norm_frame", "f32", 900, 256),
        # The pre-norm of the asymmetric FFN over a batch of 32 frames, forward and gradients.
        _norm("norm_batch", "f32", 28800, 512),
        # Rows that are no multiple of a vector load, in half precision.
        _norm("norm_odd", "f16", 7213, 1001),
        # Many wide rows in bf16: a training batch of a wide model.
        _norm("norm_wide", "bf16", 16384, 4096),
        # The decoder's self-attention for one frame with a ground-plane distance bias.
        _attn("frame", "bf16", 1, 900, 900, 8, 8, 64, pos=2, slopes="head"),
        # The same over a batch of 32 frames.
        _attn("batch", "bf16", 32, 900, 900, 8, 8, 64, pos=2, slopes="head"),
        # Training at the 1,800 anchors of the high-resolution configuration, a learned slope for
        # every query and head.
        _attn("highres_train", "bf16", 4, 1800, 1800, 8, 8, 64, train=True, pos=2, slopes="row"),
        # Training with groups that may not see one another (900 instances and denoising groups
        # behind them, the last tokens padding).
        _attn("groups_train", "bf16", 8, 1437, 1437, 8, 8, 64, train=True, documents=6),
        # Shared heads, capped scores, ragged numbers of valid keys.
        _attn("capped", "f16", 2, 4096, 4096, 16, 4, 128, cap=30.0, lens=True),
        # A long sequence in training with shared heads and a distance bias along it.
        _attn("long_train", "bf16", 1, 8192, 8192, 16, 8, 64, train=True, pos=1, slopes="head"),
        # One query against a long cache.
        _attn("one_long", "bf16", 4, 1, 65536, 32, 8, 128, pos=1, slopes="head"),
        # A few queries against the 600 cached instances of each frame, some frames with none.
        _attn("few_cached", "bf16", 6, 13, 600, 8, 8, 64, lens=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.35:
        width = _log(rng, 32, 4096)
        rows = max(1, min(_log(rng, 200, 60000), (16384 * 4096) // width))
        return _norm("", rng.choice(["f32", "bf16", "f16"]) if rows * width < 30_000_000 else "bf16", rows, width)
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 3, 4])
    dim = rng.choice([64, 64, 128, 32, 40, 96])
    pos = rng.choice([0, 1, 2])
    slopes = "none" if pos == 0 else rng.choice(["head", "row"])
    cap = rng.choice([0.0, 0.0, 20.0, 50.0])
    if rng.random() < 0.3:  # a few queries over many keys
        keys = _log(rng, 200, 50000)
        batch = max(1, min(_log(rng, 1, 8), 200_000 // keys))
        return _attn("", rng.choice(["bf16", "f16"]), batch, _log(rng, 1, 16), keys, heads, kv, dim, pos=pos,
                     slopes=slopes, cap=cap, lens=rng.random() < 0.5)
    train = rng.random() < 0.5
    queries = _log(rng, 100, 6000)
    documents = rng.choice([0, 0, 3, 9])
    keys = queries if documents or rng.random() < 0.5 else _log(rng, 100, 6000)
    batch = max(1, min(_log(rng, 1, 24), 500_000_000 // (queries * keys * heads * (2 if train else 1)),
                       50_000_000 // ((queries + keys) * heads * dim)))
    return _attn("", "bf16" if train else rng.choice(["bf16", "f16"]), batch, queries, keys, heads, kv, dim,
                 train=train, pos=pos, slopes=slopes, cap=cap, documents=documents,
                 lens=not documents and rng.random() < 0.4)


# ---- inputs ---------------------------------------------------------------------------------


def _document_sizes(tokens, documents):
    """Tokens of each document: the first holds about five eighths, the others uneven shares of the
    rest, and about one token in forty at the end is padding."""
    pad = tokens // 40
    first = (tokens - pad) * 5 // 8
    rest, sizes = tokens - pad - first, [first]
    weights = [2 + i % 3 for i in range(documents - 1)]
    for i, w in enumerate(weights):
        sizes.append(rest * w // sum(weights) if i + 1 < len(weights) else rest - sum(sizes[1:]))
    return sizes


def _valid_keys(case):
    """Valid keys of every batch entry: all of them in the first, none in every eighth."""
    return [case["keys"] * ((b * 5 + 7) % 8) // 7 for b in range(case["batch"])]


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device=dev) * std + mean).to(dtype)

    if case["kind"] == "norm":
        r, n = case["rows"], case["width"]
        return {"x": normal(r, n, std=1.7, mean=0.4), "dy": normal(r, n),
                "weight": normal(n, std=0.2, mean=1.0, dtype=torch.float32),
                "bias": normal(n, std=0.2, dtype=torch.float32)}
    B, Nq, Nk, H, G, D = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    st = {"q": normal(B, Nq, H, D), "k": normal(B, Nk, G, D), "v": normal(B, Nk, G, D), "slopes": None,
          "q_pos": None, "k_pos": None, "q_segment": None, "k_segment": None, "k_len": None}
    if case["train"]:
        st["dout"] = normal(B, Nq, H, D)
    if case["pos"] == 1:  # places along a sequence, the queries at its end
        kp = torch.arange(Nk, device=dev, dtype=torch.float32)
        st["k_pos"] = kp[None, :, None].expand(B, -1, -1).contiguous()
        qp = torch.arange(Nk - Nq, Nk, device=dev, dtype=torch.float32)
        st["q_pos"] = qp[None, :, None].expand(B, -1, -1).contiguous()
    elif case["pos"] == 2:  # metres in the ground plane
        st["k_pos"] = torch.rand(B, Nk, 2, generator=gen, device=dev) * 100 - 50
        st["q_pos"] = (st["k_pos"].clone() if Nq == Nk
                       else torch.rand(B, Nq, 2, generator=gen, device=dev) * 100 - 50)
    unit = 0.5 if case["pos"] == 2 else 0.25
    if case["slopes"] == "head":
        st["slopes"] = unit * torch.exp2(-6.0 * torch.arange(H, device=dev, dtype=torch.float32) / H)
        st["slopes"] = st["slopes"] * (0.5 + torch.rand(H, generator=gen, device=dev))
    elif case["slopes"] == "row":
        st["slopes"] = unit * torch.rand(B, Nq, H, generator=gen, device=dev)
    if case["documents"]:
        seg = torch.full((Nk,), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(_document_sizes(Nk, case["documents"])):
            seg[at:at + n] = i
            at += n
        st["q_segment"] = st["k_segment"] = seg[None].expand(B, -1).contiguous().to(dev)
    if case["lens"]:
        st["k_len"] = torch.tensor(_valid_keys(case), dtype=torch.int32, device=dev)
    return st


def prepare(case, seed):
    return dict(case=case, **_inputs(case, seed))


# ---- one pass -------------------------------------------------------------------------------


def _own_norm(s):
    from sparse4d_tt_b200 import decoder_norm_backward, decoder_norm_forward

    y, mean, rstd = decoder_norm_forward(s["x"], s["weight"], s["bias"], 1e-5)
    dx, dw, db = decoder_norm_backward(s["dy"], s["x"], s["weight"], mean, rstd)
    return y, dx, dw, db


def _plain_norm(s):
    x, dy = s["x"].float(), s["dy"].float()
    d = x - x.mean(-1, keepdim=True)
    rstd = ((d * d).mean(-1, keepdim=True) + 1e-5).rsqrt()
    n = d * rstd
    y = n * s["weight"] + s["bias"]
    g = dy * s["weight"]
    dx = (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True)) * rstd
    dt = s["x"].dtype
    return y.to(dt), dx.to(dt), (dy * n).sum(0), dy.sum(0)


BIAS = ("slopes", "q_pos", "k_pos", "q_segment", "k_segment", "k_len")


def _own_attention(s):
    from sparse4d_tt_b200 import decoder_attention_backward, decoder_attention_forward

    how = dict({k: s[k] for k in BIAS}, softcap=s["case"]["cap"])
    out, lse = decoder_attention_forward(s["q"], s["k"], s["v"], **how)
    if not s["case"]["train"]:
        return out
    dq, dk, dv, dslopes = decoder_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **how)
    return (out, dq, dk, dv) if dslopes is None else (out, dq, dk, dv, dslopes)


def _plain_part(s, b, g):
    """Batch entries ``b`` and shared heads ``g`` (slices): out, and the gradients in training."""
    c = s["case"]
    rep, D = c["heads"] // c["kv_heads"], c["dim"]
    hs = slice(g.start * rep, g.stop * rep)
    G, B = g.stop - g.start, b.stop - b.start
    Nq, Nk = c["queries"], c["keys"]

    def by_head(t, part):  # [B, N, heads, D] -> [B, G, heads / G * N, D] in fp32
        return t[b, :, part].float().transpose(1, 2).reshape(B, G, -1, D)

    def back(t, n):  # and back
        return t.reshape(B, -1, n, D).transpose(1, 2)

    q, k, v = by_head(s["q"], hs), by_head(s["k"], g), by_head(s["v"], g)
    x = (q @ k.transpose(-1, -2)) * D ** -0.5
    if c["cap"]:
        t = torch.tanh(x / c["cap"])
        x = t * c["cap"]
    x = x.reshape(B, G, rep, Nq, Nk)
    if c["pos"]:
        d2 = 0
        for i in range(c["pos"]):
            d = s["q_pos"][b, :, None, i] - s["k_pos"][b, None, :, i]
            d2 = d2 + d * d
        dist = torch.sqrt(d2)[:, None, None]
        slope = s["slopes"] if c["slopes"] == "row" else s["slopes"][None, None].expand(c["batch"], Nq, -1)
        x = x - slope[b, :, hs].transpose(1, 2).reshape(B, G, rep, Nq, 1) * dist
    ok = None
    if c["documents"]:
        qs, ks = s["q_segment"][b, :, None], s["k_segment"][b, None, :]
        ok = ((qs == ks) & (qs >= 0))[:, None, None]
    if c["lens"]:
        ok = (torch.arange(Nk, device=x.device)[None] < s["k_len"][b, None])[:, None, None, None]
    if ok is None:
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    else:
        x = torch.where(ok, x, x.new_full((), -math.inf))
        m = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
        z = p.sum(-1, keepdim=True)
        p = p / torch.where(z == 0, torch.ones_like(z), z)
    p = p.reshape(B, G, rep * Nq, Nk)
    o = p @ v
    if not c["train"]:
        return (back(o, Nq),)
    do = by_head(s["dout"], hs)
    dv = p.transpose(-1, -2) @ do
    dx = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    dslope = ()
    if c["pos"]:
        dslope = (-(dx.reshape(B, G, rep, Nq, Nk) * dist).sum(-1).reshape(B, G * rep, Nq).transpose(1, 2),)
    if c["cap"]:
        dx = dx * (1 - t * t)
    dx = dx * D ** -0.5
    return (back(o, Nq), back(dx @ k, Nq), back(dx.transpose(-1, -2) @ q, Nk), back(dv, Nk)) + dslope


def _plain_attention(s):
    c = s["case"]
    per_group = c["queries"] * c["keys"] * c["heads"] // c["kv_heads"]
    most = 1 << 28  # scores held at a time
    step = max(1, min(c["batch"], most // (per_group * c["kv_heads"])))
    heads = c["kv_heads"] if step * per_group * c["kv_heads"] <= most else 1
    rows = []
    for b in range(0, c["batch"], step):
        parts = [_plain_part(s, slice(b, min(b + step, c["batch"])), slice(g, g + heads))
                 for g in range(0, c["kv_heads"], heads)]
        rows.append([torch.cat(p, 2) for p in zip(*parts)])
    outs = [torch.cat(p, 0) for p in zip(*rows)]
    dt = DTYPES[c["dtype"]]
    res = [o.to(dt).contiguous() for o in outs[:4]]
    if len(outs) > 4:
        res.append(outs[4].sum((0, 1)) if c["slopes"] == "head" else outs[4].contiguous())
    return tuple(res) if c["train"] else res[0]


def run(state):
    if state["case"]["kind"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_attention(state) if own else _plain_attention(state)


# ---- work -----------------------------------------------------------------------------------


def _pairs(case):
    """Query-key pairs that the masks allow, over the batch, for one head."""
    if case["documents"]:
        return case["batch"] * sum(n * n for n in _document_sizes(case["keys"], case["documents"]))
    if case["lens"]:
        return case["queries"] * sum(_valid_keys(case))
    return case["batch"] * case["queries"] * case["keys"]


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "norm":
        n = case["rows"] * case["width"]
        return {"bytes": 4 * n * size + 4 * 4 * case["width"], "flops": 20 * n}
    keys = sum(_valid_keys(case)) if case["lens"] else case["batch"] * case["keys"]
    q = case["batch"] * case["queries"] * case["heads"] * case["dim"]
    kv = keys * case["kv_heads"] * case["dim"]
    pairs = _pairs(case) * case["heads"]
    tokens = case["batch"] * (case["queries"] + case["keys"])
    extra = 4 * case["pos"] * tokens + (4 * tokens if case["documents"] else 0)
    if case["slopes"] == "row":
        extra += 4 * case["batch"] * case["queries"] * case["heads"] * (2 if case["train"] else 1)
    if not case["train"]:
        return {"bytes": (2 * q + 2 * kv) * size + extra, "flops": 4 * case["dim"] * pairs}
    return {"bytes": (4 * q + 4 * kv) * size + extra, "flops": 14 * case["dim"] * pairs}


# ---- the definition in 64 bits -------------------------------------------------------------


def _exact_norm(s):
    x = s["x"].double().requires_grad_()
    w, b = (s[k].double().requires_grad_() for k in ("weight", "bias"))
    mean = x.mean(1)
    var = (x * x).mean(1) - mean * mean
    y = (x - mean[:, None]) / torch.sqrt(var + 1e-5)[:, None] * w + b
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return y.detach(), dx, dw, db


def _exact_attention(case, s):
    B, Nq, Nk, H, G, D = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    train, rep = case["train"], H // G
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dslopes = torch.zeros(B, Nq, H, dtype=torch.float64, device=q.device)
    for b in range(B):
        seen = torch.ones(Nq, Nk, dtype=torch.bool, device=q.device)
        if s["k_len"] is not None:
            seen[:, int(s["k_len"][b]):] = False
        if s["k_segment"] is not None:
            seen &= s["q_segment"][b][:, None].eq(s["k_segment"][b][None]) & s["k_segment"][b][None].ge(0)
        some = seen.any(1)
        if not bool(some.any()):
            continue
        if case["pos"]:
            gap = (s["q_pos"][b].double()[:, None] - s["k_pos"][b].double()[None]).norm(dim=-1)
        for h in range(H):
            with torch.set_grad_enabled(train):
                qh, kh, vh = (t.detach().clone().requires_grad_(train)
                              for t in (q[b, :, h], k[b, :, h // rep], v[b, :, h // rep]))
                z = torch.einsum("id,jd->ij", qh, kh) / math.sqrt(D)
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                leaves = [qh, kh, vh]
                if case["pos"]:
                    sl = s["slopes"][b, :, h] if case["slopes"] == "row" else s["slopes"][h].expand(Nq)
                    sl = sl.double().clone().requires_grad_(train)
                    z = z - sl[:, None] * gap
                    leaves.append(sl)
                z = z.masked_fill(~seen, -math.inf)
                w = torch.exp(z - torch.logsumexp(z, 1, keepdim=True).masked_fill(~some[:, None], 0.0))
                o = torch.einsum("ij,jd->id", w, vh)
            out[b, :, h] = o.detach()
            if train:
                grads = torch.autograd.grad(o, leaves, s["dout"][b, :, h].double())
                # a row without a key has no gradient: its softmax is a quotient of zeros
                dq[b, :, h] = torch.nan_to_num(grads[0])
                dk[b, :, h // rep] += grads[1]
                dv[b, :, h // rep] += grads[2]
                if case["pos"]:
                    dslopes[b, :, h] = grads[3]
    if not train:
        return out
    res = (out, dq, dk, dv)
    if case["pos"]:
        res += (dslopes.sum((0, 1)) if case["slopes"] == "head" else dslopes,)
    return res


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_norm(s) if case["kind"] == "norm" else _exact_attention(case, s)
