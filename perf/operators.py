"""Cases of three operators of the SEDD training and sampling path, their plain forms and their calls.

  sample  truncated categorical sampling: temperature, top-k, top-p and min-p from given uniform numbers
          (catsample.sample_logits), alone and inside the ancestral update of the absorbing graph (Absorbing.ancestral_step)
  norm    the gated residual of a block whose branch output is normalised too, fused with the next sub-layer's
          LayerNorm-modulate, forward and backward (ops.post_norm_residual_fwd / _bwd)
  clip    the norm of the gradients over many tensors and their clipping in place (ops.clip_grad_norm_)
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-5  # LayerNorm
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # ---- sampling.  One position of one request: the smallest call, all latency
        {"name": "sample one protein row", "op": "sample", "B": 1, "L": 1, "V": 26, "dtype": "fp32", "temperature": 0.8,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0, "per_request": False, "step": False},
        # one ancestral update in the middle of a sampling run at the sampler's shard (512 sequences of 1024 residues):
        # half of the positions are still masked, every request has its own temperature and top-p
        {"name": "sample protein step", "op": "sample", "B": 512, "L": 1024, "V": 26, "dtype": "bf16", "temperature": 0.9,
         "top_k": 0, "top_p": 0.95, "min_p": 0.0, "per_request": True, "step": True},
        # the ligand vocabulary, all truncations on
        {"name": "sample ligand rows", "op": "sample", "B": 16, "L": 1024, "V": 2365, "dtype": "bf16", "temperature": 1.1,
         "top_k": 50, "top_p": 0.9, "min_p": 0.02, "per_request": False, "step": False},
        # a vocabulary of tens of thousands of tokens for a few requests, fp32 logits, an odd size
        {"name": "sample wide rows", "op": "sample", "B": 8, "L": 61, "V": 32003, "dtype": "fp32", "temperature": 0.7,
         "top_k": 0, "top_p": 0.8, "min_p": 0.0, "per_request": True, "step": False},
        # ---- norms around a block.  One token: a sampler step of a single short sequence
        {"name": "norm one token fwd", "op": "norm", "B": 1, "L": 1, "D": 768, "dtype": "bf16", "next": True, "scale": 1.0,
         "back": False},
        # the training step's shape (64 sequences of 512), both directions
        {"name": "norm train fwd", "op": "norm", "B": 64, "L": 512, "D": 768, "dtype": "bf16", "next": True, "scale": 1.0,
         "back": False},
        {"name": "norm train bwd", "op": "norm", "B": 64, "L": 512, "D": 768, "dtype": "bf16", "next": True, "scale": 1.0,
         "back": True},
        # fp32 compute, a wider block, a ragged length, no norm behind it (a block that runs by itself)
        {"name": "norm fp32 ragged bwd", "op": "norm", "B": 5, "L": 333, "D": 1024, "dtype": "fp32", "next": False,
         "scale": 0.875, "back": True},
        # ---- clipping.  A small model's gradients: many tiny tensors, launch-bound
        {"name": "clip small model", "op": "clip", "width": 64, "blocks": 3, "dtype": "fp32", "max_norm": 1.0, "packed": False},
        # a mid-sized model in fp32
        {"name": "clip model", "op": "clip", "width": 640, "blocks": 12, "dtype": "fp32", "max_norm": 1.0, "packed": False},
        # a large one whose matrices have bf16 gradients and whose vectors fp32 ones, packed end to end as in a
        # communication bucket, so that few of them begin at a multiple of 16 bytes
        {"name": "clip large mixed packed", "op": "clip", "width": 1280, "blocks": 16, "dtype": "mixed", "max_norm": 0.5,
         "packed": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "norm", "clip"])
    if op == "sample":
        V = _log_int(rng, 3, 32003)
        rows = min(_log_int(rng, 1, 500000), 38000000 // V)
        L = min(rows, _log_int(rng, 1, 1100))
        k = rng.choice([0, 0, 1, _log_int(rng, 2, V), _log_int(rng, 2, V)])
        return {"op": op, "B": max(1, rows // L), "L": L, "V": V, "dtype": rng.choice(["fp32", "bf16"]),
                "temperature": round(rng.uniform(0.3, 1.5), 3), "top_k": k,
                "top_p": rng.choice([1.0, round(rng.uniform(0.1, 0.99), 3), round(rng.uniform(0.1, 0.99), 3)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.005, 0.3), 4)]), "per_request": rng.random() < 0.5,
                "step": rng.random() < 0.4}
    if op == "norm":
        D = 4 * _log_int(rng, 8, 512)
        rows = min(_log_int(rng, 1, 33000), 25000000 // D)
        L = min(rows, _log_int(rng, 1, 1100))
        return {"op": op, "B": max(1, rows // L), "L": L, "D": D, "dtype": rng.choice(["fp32", "bf16"]),
                "next": rng.random() < 0.7, "scale": rng.choice([1.0, round(rng.uniform(0.5, 1.1), 3)]),
                "back": rng.random() < 0.6}
    return {"op": op, "width": _log_int(rng, 17, 1200), "blocks": rng.randint(1, 12),
            "dtype": rng.choice(["fp32", "bf16", "mixed"]), "max_norm": round(math.exp(rng.uniform(-3, 4)), 4),
            "packed": rng.random() < 0.5}


# --------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _grad_shapes(c):
    """The trainable tensors of a SEDD model: embedding, per block two norms, qkv, out, two MLP layers with biases and the
    modulation layer, then the output layer."""
    w, cond = c["width"], 128
    block = [(w,), (3 * w, w), (w, w), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,), (6 * w, cond), (6 * w,)]
    return [(26, w)] + block * c["blocks"] + [(w,), (26, w), (26,)]


def _prepare_sample(c, seed):
    g = _gen(seed)
    B, L, V = c["B"], c["L"], c["V"]
    # with "step" the last column of the log-scores is the mask token's and that of the noise decides who moves
    lead = torch.randn(B, L, 1, generator=g, device=DEV) * 0.5 + 2.0
    logits = (torch.randn(B, L, V, generator=g, device=DEV) * lead).to(DT[c["dtype"]])
    if not c["step"] and V > 8:
        logits[..., 1] = -math.inf  # a token that is never sampled (padding)
    s = {"logits": logits, "u": torch.rand(B, L, V, generator=g, device=DEV), "top_k": c["top_k"]}
    for name in ("temperature", "top_p", "min_p"):
        s[name] = c[name]
    if c["per_request"]:
        s["temperature"] = c["temperature"] * (0.75 + 0.5 * torch.rand(B, generator=g, device=DEV))
        if c["top_p"] < 1:
            s["top_p"] = (c["top_p"] - 0.05 + 0.1 * torch.rand(B, generator=g, device=DEV)).clamp(0.02, 1.0)
    if c["step"]:
        masked = torch.rand(B, L, generator=g, device=DEV) < 0.5
        tokens = torch.randint(0, V - 1, (B, L), generator=g, device=DEV)
        s["x"] = torch.where(masked, torch.full_like(tokens, V - 1), tokens)
        s["move"] = 0.2 + 0.6 * torch.rand(B, generator=g, device=DEV)
    return s


def _prepare_norm(c, seed):
    g = _gen(seed)
    B, L, D, T = c["B"], c["L"], c["D"], DT[c["dtype"]]
    mod = (torch.randn(B, 6 * D, generator=g, device=DEV) * 0.3).to(T)
    s = {"residual": torch.randn(B, L, D, generator=g, device=DEV) * 1.5,
         "a": (torch.randn(B, L, D, generator=g, device=DEV) * 0.7 + 0.1).to(T),
         "post_w": 1 + 0.1 * torch.randn(D, generator=g, device=DEV),
         "gate": mod[:, 2 * D:3 * D], "shift": mod[:, 3 * D:4 * D], "scale": mod[:, 4 * D:5 * D],
         "w": 1 + 0.1 * torch.randn(D, generator=g, device=DEV)}
    if c["back"]:  # what the forward pass left behind, and the gradients that come in
        x1, _, (s["pmean"], s["prstd"], s["mean"], s["rstd"]) = _norm_fwd(s, c["scale"], True)
        s["x1"] = x1
        s["dx1"] = torch.randn(B, L, D, generator=g, device=DEV) * 0.5
        s["dh"] = (torch.randn(B, L, D, generator=g, device=DEV) * 0.5).to(T)
    return s


def _prepare_clip(c, seed):
    g = _gen(seed)
    shapes = _grad_shapes(c)
    kinds = [torch.float32 if c["dtype"] == "fp32" or (c["dtype"] == "mixed" and len(s) == 1) else torch.bfloat16
             for s in shapes]
    align = 1 if c["packed"] else 128
    arenas, grads = {}, []
    for T in (torch.float32, torch.bfloat16):
        n = sum(-(-math.prod(s) // align) * align for s, k in zip(shapes, kinds) if k == T)
        if n:
            arenas[T] = (torch.randn(n, generator=g, device=DEV) * 0.003).to(T)
    at = dict.fromkeys(arenas, 0)
    for s, k in zip(shapes, kinds):
        n = math.prod(s)
        grads.append(arenas[k][at[k]:at[k] + n].view(s))
        at[k] += -(-n // align) * align
    return {"grads": grads, "arenas": list(arenas.values())}


def prepare(case, seed):
    s = {"sample": _prepare_sample, "norm": _prepare_norm, "clip": _prepare_clip}[case["op"]](case, seed)
    s["case"] = case
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _per_row(v, B, like):
    """a parameter for all requests, or one for each, as the 32-bit number that it is, in 64 bits, by request"""
    v = v if torch.is_tensor(v) else torch.tensor(float(v), dtype=torch.float32, device=like.device)
    return v.double().reshape(-1, 1, 1).expand(B, 1, 1)


def _sample_plain(logits, u, temperature, top_k, top_p, min_p):
    """[B, L, V] -> [B, L].  In 64 bits: what is kept turns on sums next to a border, and whole numbers come out."""
    B, V = logits.shape[0], logits.shape[-1]
    z = logits.double()
    top = z.amax(-1, keepdim=True)
    p = torch.exp((z - top) / _per_row(temperature, B, z))
    order = torch.argsort(z, dim=-1, descending=True, stable=True)  # ties: the lowest index first
    ps = p.gather(-1, order)
    if 0 < top_k < V:
        ps[..., top_k:] = 0
    before = ps.cumsum(-1) - ps
    P = _per_row(top_p, B, z)
    kept = (before < P * ps.sum(-1, keepdim=True)) | (P >= 1)
    kept &= (ps > 0) & (ps >= _per_row(min_p, B, z))
    noise = (u + 1e-10).clamp(max=1.0).double()
    e = 1e-10 - torch.log(noise)
    keep = torch.zeros_like(kept).scatter_(-1, order, kept)
    return torch.where(keep, p / e, -1.0).argmax(-1)


def _layer_norm(v):
    mean = v.mean(-1, keepdim=True)
    rstd = ((v - mean).square().mean(-1, keepdim=True) + EPS).rsqrt()
    return (v - mean) * rstd, mean, rstd


def _norm_fwd(s, alpha, nxt):
    n, pmean, prstd = _layer_norm(s["a"].float())
    x1 = alpha * s["residual"] + s["gate"].float()[:, None] * (n * s["post_w"])
    if not nxt:
        return x1, None, (pmean, prstd)
    xh, mean, rstd = _layer_norm(x1)
    h = xh * s["w"] * (1 + s["scale"].float()[:, None]) + s["shift"].float()[:, None]
    return x1, h.to(s["a"].dtype), tuple(t.reshape(-1).contiguous() for t in (pmean, prstd, mean, rstd))


def _layer_norm_bwd(g, xh, rstd):
    return rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))


def _norm_bwd(s, alpha, nxt):
    B, L, D = s["a"].shape
    rows = lambda t: t.view(B, L, 1)  # noqa: E731
    out = {}
    d = s["dx1"]
    if nxt:
        xh = (s["x1"] - rows(s["mean"])) * rows(s["rstd"])
        dh, sc = s["dh"].float(), 1 + s["scale"].float()[:, None]
        out["dshift"], out["dscale"] = dh.sum(1), (dh * xh * s["w"]).sum(1)
        out["dw"] = (dh * sc * xh).sum((0, 1))
        d = d + _layer_norm_bwd(dh * sc * s["w"], xh, rows(s["rstd"]))
    ah = (s["a"].float() - rows(s["pmean"])) * rows(s["prstd"])
    dn = d * s["gate"].float()[:, None]
    out["dgate"] = (d * ah * s["post_w"]).sum(1)
    out["dpost_w"] = (dn * ah).sum((0, 1))
    da = _layer_norm_bwd(dn * s["post_w"], ah, rows(s["prstd"]))
    out["dx"], out["da"], out["dbias"] = alpha * d, da.to(s["a"].dtype), da.sum((0, 1))
    return out


def _clip_plain(grads, max_norm):
    norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt()
    coef = (max_norm / (norm + 1e-6)).clamp(max=1.0).float()
    [g.mul_(coef) for g in grads]
    return norm.float()


# ------------------------------------------------------------------------------------------------------------ runs
def _run_sample(s):
    c = s["case"]
    if own:
        from protein_lig_sedd_amd import catsample, graph_lib
        kw = {k: s[k] for k in ("temperature", "top_k", "top_p", "min_p")}
        if c["step"]:
            return graph_lib.Absorbing(c["V"] - 1).ancestral_step(s["logits"], s["x"], s["move"], u=s["u"], **kw)
        return catsample.sample_logits(s["logits"], u=s["u"], **kw)
    a = (s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    if not c["step"]:
        return _sample_plain(s["logits"], s["u"], *a)
    x, u = s["x"], s["u"]
    go = (x == c["V"] - 1) & (u[..., -1] < s["move"][:, None])
    return torch.where(go, _sample_plain(s["logits"][..., :-1], u[..., :-1], *a), x)


def _run_norm(s):
    c = s["case"]
    if not own:
        if c["back"]:
            return _norm_bwd(s, c["scale"], c["next"])
        x1, h, _ = _norm_fwd(s, c["scale"], c["next"])
        return {"x1": x1, "h": h}
    from protein_lig_sedd_amd import ops
    if not c["back"]:
        x1, h, _ = ops.post_norm_residual_fwd(s["residual"], s["a"], s["post_w"], s["gate"], res_scale=c["scale"],
                                              norm=(s["w"], s["shift"], s["scale"]) if c["next"] else None)
        return {"x1": x1, "h": h}
    B, L, D = s["a"].shape
    dmod = torch.empty(B, 3 * D, dtype=torch.float32, device=DEV)
    dvec = torch.zeros(3, D, dtype=torch.float32, device=DEV)
    out = {"dgate": dmod[:, :D], "dpost_w": dvec[0], "dbias": dvec[1]}
    norm = None
    if c["next"]:
        out.update(dshift=dmod[:, D:2 * D], dscale=dmod[:, 2 * D:], dw=dvec[2])
        norm = (s["dh"], s["x1"], s["w"], s["scale"], out["dw"], out["dshift"], out["dscale"])
    stats = (s["pmean"], s["prstd"], s["mean"], s["rstd"])
    out["dx"], out["da"] = ops.post_norm_residual_bwd(s["dx1"], s["a"], s["post_w"], s["gate"], stats, out["dgate"],
                                                      out["dpost_w"], dbias=out["dbias"], res_scale=c["scale"], norm=norm)
    return out


def _run_clip(s):
    if own:
        from protein_lig_sedd_amd import ops
        # (the coefficient as each tensor's type holds it, as in the plain form's mul_)
        norm = ops.clip_grad_norm_(s["grads"], s["case"]["max_norm"], round_coef=True)
    else:
        norm = _clip_plain(s["grads"], s["case"]["max_norm"])
    return {"norm": norm, "grads": s["arenas"]}


def run(state):
    return {"sample": _run_sample, "norm": _run_norm, "clip": _run_clip}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    c, size = case, {"fp32": 4, "bf16": 2, "mixed": 2}[case["dtype"]]
    if c["op"] == "sample":
        rows, V = c["B"] * c["L"], c["V"]
        if c["step"]:  # the masked rows (half) read a move number, half of those their scores and noise
            return {"bytes": rows * 16 + rows // 2 * 4 + rows // 4 * (V - 1) * (size + 4), "flops": rows // 4 * V * 12}
        return {"bytes": rows * (V * (size + 4) + 8), "flops": rows * V * 12}
    if c["op"] == "norm":
        n, rows, B, D = c["B"] * c["L"] * c["D"], c["B"] * c["L"], c["B"], c["D"]
        if not c["back"]:
            return {"bytes": n * (8 + size + (size if c["next"] else 0)) + B * D * size * (3 if c["next"] else 1)
                    + 8 * D + 16 * rows, "flops": n * (20 if c["next"] else 10)}
        return {"bytes": n * (8 + 2 * size + (4 + size if c["next"] else 0)) + B * D * (size + 4) * 3 + 20 * D + 16 * rows,
                "flops": n * (50 if c["next"] else 25)}
    n = sum(math.prod(s) for s in _grad_shapes(c))
    return {"bytes": 2 * n * size, "flops": 3 * n}


# ----------------------------------------------------------------------------------------------------------- exact
def _exact_sample(c, s):
    """By elimination, without sorting or running sums: the largest of weight / noise among what is left is taken if it
    is kept; if not, all that does not come before it is dropped."""
    z = s["logits"].double()
    u, V = s["u"], c["V"]
    go = torch.ones(z.shape[:2], dtype=torch.bool, device=z.device)
    x = torch.full(z.shape[:2], -1, dtype=torch.int64, device=z.device)
    if c["step"]:
        x = s["x"]
        go = (x == V - 1) & (u[..., -1] < s["move"][:, None])
        z, u = z[..., :-1], u[..., :-1]
    B, L, V = z.shape
    z, u = z[go], u[go]
    by = [(t if torch.is_tensor(t) else torch.full((B,), t, device=z.device, dtype=torch.float32)).double()[:, None].expand(B, L)[go]
          for t in (s["temperature"], s["top_p"], s["min_p"])]
    q = torch.exp((z - z.amax(-1, keepdim=True)) / by[0][:, None])
    score = torch.log(q) - torch.log(1e-10 - torch.log((u + 1e-10).clamp(max=1.0).double()))
    score[z == -math.inf] = -math.inf
    k = c["top_k"] if 0 < c["top_k"] < V else V
    edge = torch.topk(z, k, dim=-1).values[:, -1:]
    more = (z > edge).sum(-1, keepdim=True)
    mass = torch.where(z > edge, q, 0.0).sum(-1) + (k - more[:, 0]) * torch.where(z == edge, q, 0.0).amax(-1)
    got = torch.full((z.shape[0],), -1, dtype=torch.int64, device=z.device)
    left = torch.arange(z.shape[0], device=z.device)
    at = torch.arange(V, device=z.device)
    while left.numel():
        w = score[left].argmax(-1, keepdim=True)
        zl, ql = z[left], q[left]
        zw, qw = zl.gather(-1, w), ql.gather(-1, w)[:, 0]
        before = (zl > zw) | ((zl == zw) & (at < w))
        rank, S = before.sum(-1), torch.where(before, ql, 0.0).sum(-1)
        ok = (rank < k) & ((S < by[1][left] * mass[left]) | (by[1][left] >= 1)) & (qw >= by[2][left])
        got[left[ok]] = w[ok, 0]
        score[left[~ok]] = torch.where(before[~ok], score[left[~ok]], -math.inf)
        left = left[~ok]
    x = x.clone()
    x[go] = got
    return x


def _exact_norm(c, s):
    """The forward pass in 64 bits; the gradients by differentiating it."""
    d = {k: v.double() if torch.is_tensor(v) else v for k, v in s.items()}
    leaf = {k: d[k].clone().requires_grad_(c["back"]) for k in ("residual", "a", "post_w", "gate", "w", "shift", "scale")}

    def norm(v):
        v = v - v.mean(-1, keepdim=True)
        return v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + EPS)

    x1 = c["scale"] * leaf["residual"] + leaf["gate"].unsqueeze(1) * norm(leaf["a"]) * leaf["post_w"]
    h = norm(x1) * leaf["w"] * (1 + leaf["scale"].unsqueeze(1)) + leaf["shift"].unsqueeze(1) if c["next"] else None
    if not c["back"]:
        return {"x1": x1, "h": h}
    total = (x1 * d["dx1"]).sum()
    if c["next"]:
        total = total + (h * d["dh"]).sum()
    names = ["residual", "a", "post_w", "gate"] + (["w", "shift", "scale"] if c["next"] else [])
    g = dict(zip(names, torch.autograd.grad(total, [leaf[n] for n in names])))
    out = {"dx": g["residual"], "da": g["a"], "dpost_w": g["post_w"], "dgate": g["gate"]}
    if c["next"]:
        out.update(dw=g["w"], dshift=g["shift"], dscale=g["scale"])
    out["dbias"] = out["da"].sum((0, 1))  # of da before it is rounded to its type
    return out


def _exact_clip(c, s):
    arenas = [a.double() for a in s["arenas"]]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.double()) for g in s["grads"]]))
    scale = min(1.0, c["max_norm"] / (float(norm) + 1e-6))
    inside = [torch.zeros_like(a, dtype=torch.bool) for a in s["arenas"]]
    for g in s["grads"]:  # what lies between the tensors stays as it is
        k = [a.dtype for a in s["arenas"]].index(g.dtype)
        inside[k][g.storage_offset():g.storage_offset() + g.numel()] = True
    return {"norm": norm, "grads": [torch.where(i, a * scale, a) for a, i in zip(arenas, inside)]}


def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _exact_sample, "norm": _exact_norm, "clip": _exact_clip}[case["op"]](case, s)
