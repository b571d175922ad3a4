"""Work that the attention and layer-norm operators are measured on.

Every case is one pass a program makes: a training step through an operator (output and gradients), a prompt, one decoded
token per sequence over a cache, a normalisation of rows.  ``run`` computes it with elementary torch operations in 32 bits
(``own`` false) or with the package's public functions (``own`` true); ``exact`` gives the definition in 64 bits.
"""
import math

import torch

own = False

#: the kinds of passes: ``train`` (attention, forward and backward), ``prompt`` (attention, forward), ``token`` (attention of
#: single tokens over a cache), ``norm`` (layer norm, forward), ``norm_train`` (layer norm, forward and backward)
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _attn(name, kind, dtype, b, nq, nk, hq, hk, d, causal=True, cap=0.0, bias=False, docs=0, pad=0, prefix=0, shortest=0):
    c = {"kind": kind, "dtype": dtype, "b": b, "nq": nq, "nk": nk, "hq": hq, "hk": hk, "d": d, "causal": causal, "cap": cap,
         "bias": bias, "docs": docs, "pad": pad, "prefix": prefix, "shortest": shortest}
    return dict(c, name=name) if name else c


def _norm(name, kind, dtype, rows, d, stride, wide):
    c = {"kind": kind, "dtype": dtype, "rows": rows, "d": d, "stride": stride, "wide": wide}
    return dict(c, name=name) if name else c


def listed():
    return [
        # pre-training on packed documents: grouped heads, capped scores, a row of several documents, padding at its end
        _attn("train_documents_cap", "train", "bf16", 1, 8192, 8192, 16, 2, 128, cap=50.0, docs=7, pad=150),
        # training with a distance bias, 64-wide heads, one sequence per batch entry
        _attn("train_distance_bias", "train", "bf16", 4, 2048, 2048, 12, 12, 64, bias=True),
        # fine-tuning on a short odd length in fp16
        _attn("train_short_odd", "train", "fp16", 3, 777, 777, 8, 2, 128),
        # a small smoother trained in the package's own data type
        _attn("train_fp32", "train", "fp32", 2, 1000, 1000, 4, 4, 64, causal=False, cap=30.0),
        # a prompt whose first part is read in both directions
        _attn("prompt_prefix", "prompt", "bf16", 2, 6000, 6000, 16, 8, 128, prefix=1100),
        # a piece of a prompt behind a long cache
        _attn("prompt_piece", "prompt", "fp16", 1, 300, 20000, 32, 8, 128, cap=30.0, bias=True),
        # one request, a short cache: latency
        _attn("token_single", "token", "bf16", 1, 1, 900, 16, 4, 128, shortest=900),
        # an ordinary batch of ragged caches with a distance bias
        _attn("token_ragged", "token", "fp16", 24, 1, 5001, 16, 16, 64, bias=True, shortest=1),
        # a large batch of long caches
        _attn("token_long", "token", "bf16", 32, 1, 32768, 32, 8, 128, cap=50.0, shortest=16384),
        # the query and key heads of a packed projection, normalised head by head
        _norm("norm_heads", "norm", "bf16", 300000, 128, 384, False),
        # a few rows between two layers of a decoding step, with their gradient: latency
        _norm("norm_train_few", "norm_train", "fp32", 37, 1537, 1537, True),
        # a training step's activations
        _norm("norm_train_wide", "norm_train", "bf16", 16384, 8192, 8192, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one(rng):
    kind = rng.choice(["train", "prompt", "token", "norm", "norm_train"])
    if kind in ("norm", "norm_train"):
        d = _log(rng, 8, 16000)
        rows = _log(rng, 1, 300000)
        return _norm(None, kind, rng.choice(["bf16", "fp16", "fp32"]), rows, d, d + rng.choice([0, 0, 8, d]), rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    hk = rng.choice([1, 2, 3, 4, 8])
    hq = hk * rng.choice([1, 2, 4, 5, 8])
    d = rng.choice([32, 64, 64, 80, 96, 128, 128])
    cap, bias = rng.choice([0.0, 0.0, 30.0, 50.0]), rng.random() < 0.4
    if kind == "token":
        nk = _log(rng, 1, 32768)
        return _attn(None, kind, dtype, _log(rng, 1, 48), 1, nk, hq, hk, d, True, cap, bias, shortest=rng.randint(0, nk))
    n = _log(rng, 1, 8192 if dtype != "fp32" else 1500)
    b = _log(rng, 1, 8)
    if kind == "train":
        docs = rng.choice([0, 0, 1, 3, 9]) if n > 64 else 0
        return _attn(None, kind, dtype, b, n, n, hq, hk, d, rng.random() < 0.8, cap, bias, docs, rng.randint(0, n // 16) if docs else 0)
    nk = n + rng.choice([0, _log(rng, 1, 12000 if dtype != "fp32" else 1500)])
    return _attn(None, kind, dtype, b, n, nk, hq, hk, d, True, cap, bias, prefix=rng.choice([0, nk // 3]))


def draw(rng):
    top = [work(c) for c in listed()]
    big = {"flops": max(w["flops"] for w in top), "bytes": max(w["bytes"] for w in top)}
    while True:
        c = _one(rng)
        w = work(c)
        if c["kind"] in ("norm", "norm_train"):
            fits = c["rows"] * c["d"] <= 16384 * 8192 // 4
        else:
            fits = c["b"] * c["hq"] * c["nq"] * c["nk"] <= 16 * 8192 * 8192 * (1 if c["dtype"] != "fp32" else 1 / 16)
        if fits and w["flops"] <= big["flops"] and w["bytes"] <= big["bytes"]:
            return c


def _doc_lengths(c):
    """Lengths of the documents of a row: growing in equal steps, together all tokens that are not padding."""
    n = c["nk"] - c["pad"]
    w = [i + 1 for i in range(c["docs"])]
    out = [n * x // sum(w) for x in w]
    out[-1] += n - sum(out)
    return out


def _cache_lengths(c):
    lo, b = c["shortest"], c["b"]
    return [lo + (c["nk"] - lo) * (i + 1) // b for i in range(b)] if c["kind"] == "token" else [c["nk"]] * b


def work(case):
    c, size = case, {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if c["kind"] in ("norm", "norm_train"):
        n, par = c["rows"] * c["d"], c["d"] * (4 if c["wide"] else size)
        if c["kind"] == "norm":
            return {"bytes": 2 * n * size + 2 * par, "flops": 8 * n}
        return {"bytes": 4 * n * size + 4 * par, "flops": 20 * n}
    qs, ks = c["nq"] * c["hq"] * c["d"] * size, c["hk"] * c["d"] * size
    if c["kind"] == "token":
        lens = _cache_lengths(c)
        return {"bytes": 2 * c["b"] * qs + 2 * sum(lens) * ks, "flops": 4 * c["d"] * c["hq"] * sum(lens)}
    if c["docs"]:
        pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in _doc_lengths(c))
    elif c["causal"]:
        first = c["nk"] - c["nq"] + 1  # keys that the first query sees
        p = c["prefix"]
        few = min(c["nq"], max(0, p - first))  # queries that see the prefix and no key behind it
        pairs = few * p + (first + few + c["nk"]) * (c["nq"] - few) // 2
    else:
        pairs = c["nq"] * c["nk"]
    flops, nbytes = 4 * c["d"] * c["b"] * c["hq"] * pairs, c["b"] * (2 * qs + 2 * c["nk"] * ks)
    if c["kind"] == "train":
        flops, nbytes = flops * 7 // 2, c["b"] * (4 * qs + 4 * c["nk"] * ks)
    return {"bytes": nbytes, "flops": flops}


def prepare(case, seed):
    c, dev, dt = case, torch.device("cuda"), _TYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=dt)

    s = {"case": c}
    if c["kind"] in ("norm", "norm_train"):
        wt = torch.float32 if c["wide"] else dt
        x = normal(c["rows"], c["stride"])[:, : c["d"]]
        x = x.mul_(2).add_(0.5)
        w = torch.randn(c["d"], device=dev, generator=g, dtype=torch.float32).mul_(0.2).add_(1).to(wt)
        bias = torch.randn(c["d"], device=dev, generator=g, dtype=torch.float32).mul_(0.2).to(wt)
        train = c["kind"] == "norm_train"
        s.update(x=x.requires_grad_(train), w=w.requires_grad_(train), bias=bias.requires_grad_(train), eps=1e-5)
        if train:
            s["dy"] = normal(c["rows"], c["d"])
        return s
    b, hq, hk, d = c["b"], c["hq"], c["hk"], c["d"]
    train = c["kind"] == "train"
    s["kv_lens"] = s["documents"] = s["prefix_lens"] = s["slopes"] = None
    if c["nq"] == c["nk"]:  # the views of one packed projection
        packed = normal(b, c["nq"], hq + 2 * hk, d)
        s["q"], s["k"], s["v"] = packed[:, :, :hq], packed[:, :, hq:hq + hk], packed[:, :, hq + hk:]
    else:
        s["q"], s["k"], s["v"] = normal(b, c["nq"], hq, d), normal(b, c["nk"], hk, d), normal(b, c["nk"], hk, d)
    s["q"].mul_(1.5)
    if c["kind"] == "token":
        lens = torch.tensor(_cache_lengths(c))[torch.randperm(b, generator=host)].to(torch.int32).to(dev)
        s["kv_lens"] = lens
        behind = torch.arange(c["nk"], device=dev) >= lens[:, None]
        for t in (s["k"], s["v"]):  # what lies behind a sequence in its cache was never written
            t.masked_fill_(behind[:, :, None, None], float("nan"))
    if c["docs"]:
        rows = []
        for _ in range(b):
            lens = [_doc_lengths(c)[i] for i in torch.randperm(c["docs"], generator=host).tolist()]
            ids = torch.arange(c["docs"]).repeat_interleave(torch.tensor(lens))
            rows.append(torch.cat([ids, torch.full((c["pad"],), -1)]))
        s["documents"] = torch.stack(rows).to(torch.int32).to(dev)
    if c["prefix"]:
        s["prefix_lens"] = torch.full((b,), c["prefix"], dtype=torch.int32, device=dev)
    if c["bias"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, hq + 1, device=dev, dtype=torch.float32) / hq)
    if train:
        for n in ("q", "k", "v"):
            s[n].requires_grad_(True)
        s["do"] = normal(b, c["nq"], hq, d)
    return s


def _visible(s):
    """Which keys each query may see, (b, nq, nk) truth values, and how far they lie from it, in 32 bits."""
    c, dev = s["case"], s["q"].device
    j = torch.arange(c["nk"], device=dev)
    lens = s["kv_lens"].long() if s["kv_lens"] is not None else torch.full((c["b"],), c["nk"], device=dev)
    at = torch.arange(c["nq"], device=dev)[None, :] + (lens - c["nq"])[:, None]
    see = (j < lens[:, None])[:, None, :].expand(c["b"], c["nq"], c["nk"])
    if c["causal"]:
        early = j[None, None, :] <= at[:, :, None]
        if s["prefix_lens"] is not None:
            early = early | (j < s["prefix_lens"][:, None])[:, None, :]
        see = see & early
    if s["documents"] is not None:
        see = see & (s["documents"][:, :, None] == s["documents"][:, None, :]) & (s["documents"][:, :, None] >= 0)
    return see, (at[:, :, None] - j).abs().float()


def _plain_attention(s):
    c = s["case"]
    b, nq, nk, hk, d = c["b"], c["nq"], c["nk"], c["hk"], c["d"]
    grp = c["hq"] // hk
    scale = 1.0 / math.sqrt(d)
    q = s["q"].detach().float().reshape(b, nq, hk, grp, d).permute(0, 2, 3, 1, 4).reshape(b, hk, grp * nq, d)
    k = s["k"].detach().float().permute(0, 2, 1, 3)
    v = s["v"].detach().float().permute(0, 2, 1, 3)
    see, far = _visible(s)
    if s["kv_lens"] is not None:
        held = (torch.arange(nk, device=q.device) < s["kv_lens"][:, None])[:, None, :, None]
        k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    sc = (q @ k.transpose(2, 3)).mul_(scale).view(b, hk, grp, nq, nk)
    t = None
    if c["cap"]:
        t = sc.div_(c["cap"]).tanh_()
        sc = t * c["cap"]
    if s["slopes"] is not None:
        sc = sc - s["slopes"].view(1, hk, grp, 1, 1) * far[:, None, None]
    sc = sc.masked_fill(~see[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    tot = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(tot == 0, 1.0, tot)).view(b, hk, grp * nq, nk)
    o = p @ v

    def heads(x, n, h):
        return x.view(b, hk, h // hk, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(s["q"].dtype)

    if c["kind"] != "train":
        return heads(o, nq, c["hq"])
    do = s["do"].float().reshape(b, nq, hk, grp, d).permute(0, 2, 3, 1, 4).reshape(b, hk, grp * nq, d)
    dv = p.transpose(2, 3) @ do
    ds = (do @ v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if t is not None:
        ds = ds * (1 - t * t).view(ds.shape)
    ds = ds * scale
    return heads(o, nq, c["hq"]), heads(ds @ k, nq, c["hq"]), heads(ds.transpose(2, 3) @ q, nk, hk), heads(dv, nk, hk)


def _plain_norm(s):
    x, w, bias = (s[n].detach().float() for n in ("x", "w", "bias"))
    xc = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + s["eps"])
    xh = xc * rstd
    y = (xh * w + bias).to(s["x"].dtype)
    if s["case"]["kind"] == "norm":
        return y
    dy = s["dy"].float()
    g = dy * w
    dx = (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) * rstd
    return y, dx.to(s["x"].dtype), (dy * xh).sum(0).to(s["w"].dtype), dy.sum(0).to(s["bias"].dtype)


def _own_attention(s):
    from falkon_b200 import mmv_ops

    c = s["case"]
    o = mmv_ops.attention(s["q"], s["k"], s["v"], causal=c["causal"], softcap=c["cap"], slopes=s["slopes"],
                          prefix_lens=s["prefix_lens"], documents=s["documents"], kv_lens=s["kv_lens"])
    if c["kind"] != "train":
        return o
    return (o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"]))


def _own_norm(s):
    from falkon_b200 import mmv_ops

    y = mmv_ops.layer_norm(s["x"], s["w"], s["bias"], eps=s["eps"])
    if s["case"]["kind"] == "norm":
        return y
    return (y, *torch.autograd.grad(y, (s["x"], s["w"], s["bias"]), s["dy"]))


def run(state):
    norm = state["case"]["kind"] in ("norm", "norm_train")
    if own:
        return _own_norm(state) if norm else _own_attention(state)
    return _plain_norm(state) if norm else _plain_attention(state)


def _exact_head(s, i, h):
    """Output and gradients of one query head of one sequence, in 64 bits: (o, dq, dk, dv)."""
    c = s["case"]
    kv = h // (c["hq"] // c["hk"])
    n = int(s["kv_lens"][i]) if s["kv_lens"] is not None else c["nk"]
    q, k, v = s["q"][i, :, h].detach().double(), s["k"][i, :n, kv].detach().double(), s["v"][i, :n, kv].detach().double()
    row = torch.arange(c["nq"], device=q.device)[:, None] + n - c["nq"]
    col = torch.arange(n, device=q.device)[None, :]
    see = torch.ones(c["nq"], n, dtype=torch.bool, device=q.device)
    if c["causal"]:
        see &= (col <= row) | (col < (int(s["prefix_lens"][i]) if s["prefix_lens"] is not None else 0))
    if s["documents"] is not None:
        ids = s["documents"][i]
        see &= (ids[:, None] == ids[None, :]) & (ids[:, None] >= 0)
    score = torch.einsum("id,jd->ij", q, k) / c["d"] ** 0.5
    slope_of_cap = 1.0
    if c["cap"]:
        t = torch.tanh(score / c["cap"])
        score, slope_of_cap = c["cap"] * t, 1 - t * t
    if s["slopes"] is not None:
        score = score - s["slopes"][h].double() * (row - col).abs()
    weight = torch.where(see, score, torch.full_like(score, -1e300))
    if n:
        weight = torch.where(see, torch.exp(weight - weight.max(1, keepdim=True).values), 0.0)
    weight = weight / weight.sum(1, keepdim=True).clamp_min(1e-300)
    o = torch.einsum("ij,jd->id", weight, v)
    if c["kind"] != "train":
        return o, None, None, None
    do = s["do"][i, :, h].double()
    dp = torch.einsum("id,jd->ij", do, v)
    ds = weight * (dp - (weight * dp).sum(1, keepdim=True)) * slope_of_cap / c["d"] ** 0.5
    return o, torch.einsum("ij,jd->id", ds, k), torch.einsum("ij,id->jd", ds, q), torch.einsum("ij,id->jd", weight, do)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] in ("norm", "norm_train"):
        x, w, bias = (s[n].detach().double() for n in ("x", "w", "bias"))
        var, mean = torch.var_mean(x, dim=-1, keepdim=True, unbiased=False)
        sd = (var + s["eps"]).sqrt()
        xh = (x - mean) / sd
        y = torch.addcmul(bias, xh, w)
        if c["kind"] == "norm":
            return y
        dy = s["dy"].double()
        g = dy * w
        dx = (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) / sd
        return y, dx, (dy * xh).sum(0), dy.sum(0)
    o = torch.zeros(c["b"], c["nq"], c["hq"], c["d"], dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(c["b"], c["nk"], c["hk"], c["d"], dtype=torch.float64, device="cuda") for _ in "kv")
    for i in range(c["b"]):
        for h in range(c["hq"]):
            kv = h // (c["hq"] // c["hk"])
            o[i, :, h], *grads = _exact_head(s, i, h)
            if c["kind"] == "train":
                dq[i, :, h] = grads[0]
                dk[i, :, kv] += grads[1]
                dv[i, :, kv] += grads[2]
    return (o, dq, dk, dv) if c["kind"] == "train" else o
