"""Cases of the token-side operators: LayerNorm, the scaled token embedding and
per-token log probabilities, each with its gradient.

``run`` computes a case in its plain form (elementary torch operations in 32
bits) or, with ``own``, through ``spikingtransformer_b200.ops``.  ``exact`` is
the operator's definition in 64 bits.  A case is a dict: ``op`` names the
operator, ``train`` adds the backward pass (the gradients are outputs), the
rest are sizes and types.
"""

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
IGNORE = -100


def listed():
    return [
        # LayerNorm of one decoding step of 64 sequences at the OCR model's width: latency
        {"name": "layer_norm step", "op": "layer_norm", "train": False, "rows": 64, "D": 384, "dtype": "bf16",
         "pitch": 384, "half_w": False},
        # the residual stream of an encoder forward: 4 steps x 256 images x 256 tokens
        {"name": "layer_norm encoder", "op": "layer_norm", "train": False, "rows": 262144, "D": 384, "dtype": "bf16",
         "pitch": 384, "half_w": False},
        # training rows of a decoder in fp32 at the default width: 4 steps x 64 images x 64 tokens
        {"name": "layer_norm train fp32", "op": "layer_norm", "train": True, "rows": 16384, "D": 512, "dtype": "fp32",
         "pitch": 512, "half_w": False},
        # the MLP's hidden width at the training batch: 4 steps x 64 images x 256 tokens
        {"name": "layer_norm train wide", "op": "layer_norm", "train": True, "rows": 65536, "D": 1536, "dtype": "bf16",
         "pitch": 1536, "half_w": False},
        # an odd width read out of a wider projection (a column slice), fp16 weights
        {"name": "layer_norm train odd", "op": "layer_norm", "train": True, "rows": 5001, "D": 515, "dtype": "fp16",
         "pitch": 643, "half_w": True},
        # the next token of 64 sequences, byte vocabulary
        {"name": "embedding step", "op": "embedding", "train": False, "n": 64, "V": 256, "D": 384, "dtype": "fp32",
         "skew": 1.0, "pad": 0.0},
        # a training batch of text lines: 64 x 64 byte tokens, a quarter of them padding
        {"name": "embedding train lines", "op": "embedding", "train": True, "n": 4096, "V": 256, "D": 384,
         "dtype": "fp32", "skew": 2.0, "pad": 0.25},
        # a large vocabulary with a long-tailed token distribution
        {"name": "embedding train large", "op": "embedding", "train": True, "n": 131072, "V": 65536, "D": 1024,
         "dtype": "bf16", "skew": 4.0, "pad": 0.0},
        # scoring 256 lines of 64 byte tokens: logits of 4 steps, five alternatives a token
        {"name": "logprobs score lines", "op": "logprobs", "train": False, "T": 4, "rows": 16384, "V": 256,
         "dtype": "fp32", "top_k": 5, "masked": False, "ignored": 0.0},
        # one decoding step of 32 sequences over a large vocabulary, eight alternatives, part of it barred
        {"name": "logprobs step large", "op": "logprobs", "train": False, "T": 1, "rows": 32, "V": 65536,
         "dtype": "bf16", "top_k": 8, "masked": True, "ignored": 0.0},
        # training on log probabilities and entropy with the default 10 steps and 1000 symbols
        {"name": "logprobs train default", "op": "logprobs", "train": True, "T": 10, "rows": 1003, "V": 1000,
         "dtype": "fp32", "top_k": 0, "masked": False, "ignored": 0.1},
        # the same over a large vocabulary: 1 GB of logits
        {"name": "logprobs train large", "op": "logprobs", "train": True, "T": 1, "rows": 8192, "V": 65536,
         "dtype": "bf16", "top_k": 0, "masked": False, "ignored": 0.1},
    ]


def _log_between(rng, lo, hi):
    """An integer in [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["layer_norm", "embedding", "logprobs"])
    dtype = rng.choice(["fp32", "fp16", "bf16"])
    train = rng.random() < 0.6
    if op == "layer_norm":
        D = _log_between(rng, 32, 8192)
        if rng.random() < 0.5:
            D = max(32, D // 8 * 8)
        rows = _log_between(rng, 1, min(262144, (1 << 26) // D))
        pitch = D if rng.random() < 0.6 else D + rng.randint(1, 128)
        return {"op": op, "train": train, "rows": rows, "D": D, "dtype": dtype, "pitch": pitch,
                "half_w": rng.random() < 0.3}
    if op == "embedding":
        D = _log_between(rng, 32, 2048)
        if rng.random() < 0.6:
            D = max(32, D // 8 * 8)
        V = _log_between(rng, 64, min(65536, (1 << 26) // D))
        n = _log_between(rng, 1, min(131072, (1 << 26) // D))
        return {"op": op, "train": train, "n": n, "V": V, "D": D, "dtype": dtype,
                "skew": rng.choice([1.0, 2.0, 4.0]), "pad": rng.choice([0.0, 0.0, 0.25])}
    dtype = rng.choice(["fp32", "bf16"])
    T = rng.choice([1, 1, 4, 10])
    V = _log_between(rng, 64, 131072)
    top_k = rng.choice([0, 0, 1, 5, 20])
    most = (1 << 24) if top_k else (1 << 27)  # the plain form sorts whole rows
    rows = _log_between(rng, 1, max(1, min(65536, most // (V * T))))
    return {"op": op, "train": train, "T": T, "rows": rows, "V": V, "dtype": dtype, "top_k": top_k,
            "masked": rng.random() < 0.3, "ignored": rng.choice([0.0, 0.1])}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    s = {"case": case}
    if case["op"] == "layer_norm":
        rows, D = case["rows"], case["D"]
        wide = randn(rows, case["pitch"]) * (0.5 + torch.rand(rows, 1, generator=g, device=dev)) + randn(rows, 1)
        wdt = dt if case["half_w"] else torch.float32
        s["x"] = wide.to(dt)[:, :D]
        s["w"] = (1.0 + 0.2 * randn(D)).to(wdt)
        s["b"] = (0.2 * randn(D)).to(wdt)
        leaves = ("x", "w", "b")
        if case["train"]:
            s["g"] = randn(rows, D).to(dt)
    elif case["op"] == "embedding":
        n, V, D = case["n"], case["V"], case["D"]
        rank = (torch.rand(n, generator=g, device=dev, dtype=torch.float64) ** case["skew"] * V).long().clamp(max=V - 1)
        tok = torch.randperm(V, generator=g, device=dev)[rank]
        tok[torch.rand(n, generator=g, device=dev) < case["pad"]] = 0
        s["tokens"], s["scale"] = tok, D ** 0.5
        s["pad"] = 0 if case["pad"] > 0 else None
        s["w"] = randn(V, D).to(dt)
        leaves = ("w",)
        if case["train"]:
            s["g"] = randn(n, D).to(dt)
    else:
        T, rows, V = case["T"], case["rows"], case["V"]
        s["logits"] = randn(T, rows, V, dtype=dt).mul_(3.0)
        if case["masked"]:  # symbols that the vocabulary's user has barred, the same for every row
            barred = torch.rand(V, generator=g, device=dev) < 0.3
            barred[:32] = False
            s["logits"].masked_fill_(barred, float("-inf"))
        s["tokens"] = torch.randint(0, min(32, V) if case["masked"] else V, (rows,), generator=g, device=dev)
        s["tokens"][torch.rand(rows, generator=g, device=dev) < case["ignored"]] = IGNORE
        leaves = ("logits",)
        if case["train"]:
            s["g_logp"], s["g_entropy"] = randn(rows), 0.1 * randn(rows)
    if case["train"]:
        for k in leaves:
            s[k].requires_grad_(True)
    return s


def work(case):
    e = DTYPES[case["dtype"]].itemsize
    train = case["train"]
    if case["op"] == "layer_norm":
        n, we = case["rows"] * case["D"], e if case["half_w"] else 4
        return {"bytes": n * e * (4 if train else 2) + case["D"] * we * (4 if train else 2),
                "flops": n * (20 if train else 8)}
    if case["op"] == "embedding":
        n, V, D = case["n"], case["V"], case["D"]
        used = V * (1.0 - (1.0 - 1.0 / V) ** n)  # rows that n uniform draws touch: no more are read
        return {"bytes": 8 * n + used * D * e + n * D * e + ((n * D + V * D) * e if train else 0),
                "flops": n * D * (2 if train else 1)}
    n = case["T"] * case["rows"] * case["V"]
    rows = case["rows"]
    return {"bytes": n * e * (2 if train else 1) + rows * (8 + 8 + 12 * case["top_k"] + (8 if train else 0)),
            "flops": n * (12 if train else 5)}


# ------------------------------------------------------------------ plain forms


def _plain_layer_norm(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    h = xc * rstd
    y = (h * w + b).to(s["x"].dtype)
    if "g" not in s:
        return {"y": y}
    g = s["g"].float()
    a = g * w
    gx = rstd * (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True))
    return {"y": y, "gx": gx.to(s["x"].dtype), "gw": (g * h).sum(0).to(s["w"].dtype),
            "gb": g.sum(0).to(s["b"].dtype)}


def _plain_embedding(s):
    w, tok = s["w"], s["tokens"]
    out = (w[tok].float() * s["scale"]).to(w.dtype)
    if "g" not in s:
        return {"out": out}
    g = s["g"].float()
    if s["pad"] is not None:
        g = g * (tok != s["pad"]).unsqueeze(1)
    gw = torch.zeros(w.shape, device=w.device).index_add_(0, tok, g) * s["scale"]
    return {"out": out, "gw": gw.to(w.dtype)}


def _plain_logprobs(s):
    x, tok, K = s["logits"], s["tokens"], s["case"]["top_k"]
    T = x.shape[0]
    # the mean over the steps in 64 bits: the order of the alternatives hangs on its last bit
    z = x[0].float() if T == 1 else x.double().mean(0).float()
    used = tok != IGNORE
    y = tok.clamp(min=0).unsqueeze(1)
    u = z - z.amax(-1, keepdim=True)
    e = torch.exp(u)
    total = e.sum(-1, keepdim=True)
    p, lp = e / total, u - torch.log(total)
    plp = torch.where(p > 0, p * lp, 0.0)
    H = -plp.sum(-1)
    out = {"logp": torch.where(used, lp.gather(1, y).squeeze(1), 0.0), "entropy": torch.where(used, H, 0.0)}
    if K:
        idx = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :K]
        out["top_logp"] = torch.where(used.unsqueeze(1), lp.gather(1, idx), 0.0)
        out["top_idx"] = torch.where(used.unsqueeze(1), idx, -1)
    if "g_logp" in s:
        gl = (s["g_logp"] * used).unsqueeze(1)
        gh = (s["g_entropy"] * used).unsqueeze(1)
        dz = -gl * p - gh * (plp + p * H.unsqueeze(1))
        dz.scatter_add_(1, y, gl)
        out["glogits"] = (dz / T).to(x.dtype).expand(x.shape).contiguous()
    return out


def run(s):
    op = s["case"]["op"]
    if not own:
        with torch.no_grad():
            return {"layer_norm": _plain_layer_norm, "embedding": _plain_embedding,
                    "logprobs": _plain_logprobs}[op](s)
    from spikingtransformer_b200 import ops
    if op == "layer_norm":
        y = ops.layer_norm(s["x"], s["w"], s["b"], EPS)
        if "g" not in s:
            return {"y": y}
        gx, gw, gb = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["g"])
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    if op == "embedding":
        out, _ = ops.embedding(s["tokens"], s["w"], s["scale"], padding_idx=s["pad"])
        if "g" not in s:
            return {"out": out}
        return {"out": out, "gw": torch.autograd.grad(out, s["w"], s["g"])[0]}
    K = s["case"]["top_k"]
    logp, entropy, top_logp, top_idx, _ = ops.token_logprobs(s["logits"], s["tokens"], top_k=K, ignore_index=IGNORE)
    out = {"logp": logp, "entropy": entropy}
    if K:
        out["top_logp"], out["top_idx"] = top_logp, top_idx
    if "g_logp" in s:
        out["glogits"], = torch.autograd.grad((logp, entropy), s["logits"], (s["g_logp"], s["g_entropy"]))
    return out


# ------------------------------------------------------------------ definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    train = case["train"]
    if case["op"] == "layer_norm":
        x, w, b = (s[k].detach().double().requires_grad_(train) for k in ("x", "w", "b"))
        mu = x.mean(-1, keepdim=True)
        y = (x - mu) * torch.rsqrt(x.var(-1, unbiased=False, keepdim=True) + EPS) * w + b
        out = {"y": y.detach()}
        if train:
            out["gx"], out["gw"], out["gb"] = torch.autograd.grad(y, (x, w, b), s["g"].double())
        return out
    if case["op"] == "embedding":
        tok, scale = s["tokens"], s["scale"]
        w = s["w"].detach().double()
        out = {"out": w.index_select(0, tok) * scale}
        if train:
            keep = torch.ones_like(tok, dtype=torch.bool) if s["pad"] is None else tok != s["pad"]
            order = torch.argsort(tok[keep], stable=True)
            rows = s["g"].double()[keep][order]
            ends = torch.cumsum(torch.bincount(tok[keep], minlength=case["V"]), 0)
            sums = torch.cat([rows.new_zeros(1, rows.shape[1]), torch.cumsum(rows, 0)])
            gw = sums[ends]
            gw[1:] -= sums[ends[:-1]]
            out["gw"] = gw * scale
        return out
    x, tok = s["logits"].detach(), s["tokens"]
    T, rows, V = x.shape
    per = max(1, (1 << 26) // V)
    parts = []
    for a in range(0, rows, per):  # a slice of the rows at a time: eight bytes a value
        z = x[:, a:a + per].double().mean(0)
        z = torch.where(z == float("-inf"), -1e4, z).requires_grad_(train)  # exp(-1e4) is 0 in 64 bits too
        t = tok[a:a + per]
        lsm = torch.log_softmax(z, -1)
        used = (t != IGNORE).double()
        lp = lsm.gather(1, t.clamp(min=0).unsqueeze(1)).squeeze(1) * used
        H = torch.special.entr(torch.softmax(z, -1)).sum(-1) if not train else -(lsm.exp() * lsm).sum(-1)
        H = H * used
        part = {"logp": lp.detach(), "entropy": H.detach()}
        if case["top_k"]:
            best = torch.sort(lsm.detach(), dim=-1, descending=True, stable=True).values[:, :case["top_k"]]
            best = torch.where(best < -9e3, float("-inf"), best)
            part["top_logp"] = best * used.unsqueeze(1) if used.all() else torch.where(used.unsqueeze(1) > 0, best, 0.0)
        if train:
            gz, = torch.autograd.grad((lp, H), z, (s["g_logp"][a:a + per].double(), s["g_entropy"][a:a + per].double()))
            part["glogits"] = gz / T
        parts.append(part)
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if train:
        out["glogits"] = out["glogits"].expand(T, rows, V)
    if case["top_k"]:
        out["top_idx"] = None
    return out
