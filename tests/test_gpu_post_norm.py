"""Norms before and after a block fused with its gate and residual scale (ops.post_norm_residual_fwd / _bwd, DDiTBlock with
post_norm) against 64-bit formulas, those against autograd and differences.

Tolerances.  Inputs are taken as the stored values, so errors are those of the kernel's own fp32 roundings (2^-24 each) and of
storing results.  A row value passes two LayerNorms: at most 48 roundings one after the other (two sums of up to 2048 terms, 8 in
a lane and 6 across: 14 each; 20 in between) of terms no larger than the row's own size, and a mean that is subtracted can
lose as much again: norm-wise 96 x 2^-24 forward, twice that backward, whose means subtract once more.  What is centred
(ahat, xhat, d, da) has an error relative to its ROW's size, not to its own value, which a subtraction may have left as small as
one likes: with |f - f'| <= e (|f| + rms f) for both factors of a product, the product is off by at most
2 e (|f| + rms f)(|g| + rms g).  So a column sum of n products is off by (2 x 96 + n) x 2^-24 of the sum of those sizes: n for its
adds.  bf16 results add half a step, 2^-8 of the value."""
import math
import types

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E32 = 2.0 ** -24
FWD, BWD = 96 * E32, 192 * E32


def ln(v):
    mean = v.mean(-1, keepdim=True)
    rstd = ((v - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    return (v - mean) * rstd, mean, rstd


def make(B, L, D, dtype, seed=0, mod_dtype=None):
    g = torch.Generator().manual_seed(seed + 1000 * D + L)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    mod = (0.4 * r(B, 3 * D)).to(mod_dtype or dtype).to(DEV)
    return dict(residual=(1.5 * r(B, L, D)).to(DEV), a=(0.8 * r(B, L, D) + 0.2).to(dtype).to(DEV),
                post_w=(1 + 0.2 * r(D)).to(DEV), w=(1 + 0.2 * r(D)).to(DEV), gate=mod[:, :D], shift=mod[:, D:2 * D],
                scale=mod[:, 2 * D:], dx1=r(B, L, D).to(DEV), dh=(0.7 * r(B, L, D)).to(dtype).to(DEV))


def fwd64(s, alpha, nxt, keep=None):
    d = {k: v.cpu().double() for k, v in s.items()}
    n, pm, pr = ln(d["a"])
    n = n * d["post_w"]
    if keep is not None:
        n = n * keep
    x1 = alpha * d["residual"] + d["gate"][:, None] * n
    if not nxt:
        return x1, None, (pm, pr)
    xh, mu, rs = ln(x1)
    return x1, xh * d["w"] * (1 + d["scale"][:, None]) + d["shift"][:, None], (pm, pr, mu, rs)


def bwd64(s, alpha, nxt, keep=None, dx1=True, x1=None):
    """-> ({name: value}, {name: sum of the terms' sizes} for the column sums).  x1: the stored one that the kernel sees."""
    d = {k: v.cpu().double() for k, v in s.items()}
    back = lambda g, xh, rs: rs * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))  # noqa: E731
    out, size = {}, {}

    def col(name, terms, dims, sizes):
        out[name], size[name] = terms.sum(dims), sizes.sum(dims)

    def sz(f):  # what a row value's error is relative to
        return f.abs() + f.square().mean(-1, keepdim=True).sqrt()

    t = d["dx1"] if dx1 else torch.zeros_like(d["dx1"])
    if nxt:
        xh, _, rs = ln(fwd64(s, alpha, False, keep)[0] if x1 is None else x1.cpu().double())
        sc = 1 + d["scale"][:, None]
        col("dshift", d["dh"], 1, d["dh"].abs())
        col("dscale", d["dh"] * xh * d["w"], 1, (d["dh"] * d["w"]).abs() * sz(xh))
        col("dw", d["dh"] * sc * xh, (0, 1), (d["dh"] * sc).abs() * sz(xh))
        t = t + back(d["dh"] * sc * d["w"], xh, rs)
    ah, _, pr = ln(d["a"])
    dk = t if keep is None else t * keep
    col("dgate", dk * ah * d["post_w"], 1, sz(dk) * sz(ah) * d["post_w"].abs())
    dn = dk * d["gate"][:, None]
    col("dpost_w", dn * ah, (0, 1), sz(dk) * d["gate"][:, None].abs() * sz(ah))
    out["da"] = back(dn * d["post_w"], ah, pr)
    col("dbias", out["da"], (0, 1), sz(out["da"]))
    out["dx"] = alpha * t
    return out, size


def near(got, want, tol, what):
    got, want = got.cpu().double(), want.reshape(got.shape)
    if got.dtype != torch.float64 or got.numel() == 0:
        return
    rms = float(want.norm()) / max(want.numel(), 1) ** 0.5
    err = (got - want).abs()
    bound = tol["half"] * want.abs() + tol["rel"] * (want.abs() + 4 * rms) + 1e-30
    assert bool((err <= bound).all()), f"{what}: {float((err / bound).max()):.2f} of the bound, |err| {float(err.max()):.3e}"


def half(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else E32


def run_fwd(s, alpha, nxt, keep=None, inv=1.0):
    from protein_lig_sedd_amd import ops
    return ops.post_norm_residual_fwd(s["residual"], s["a"], s["post_w"], s["gate"], keep, inv, alpha,
                                      norm=(s["w"], s["shift"], s["scale"]) if nxt else None)


def run_bwd(s, alpha, nxt, x1, stats, keep=None, inv=1.0, dx1=True):
    from protein_lig_sedd_amd import ops
    B, L, D = s["a"].shape
    wide = torch.full((B, 5 * D), 7.0, device=DEV)
    vec = torch.full((3, D), 0.5, device=DEV)
    out = dict(dgate=wide[:, D:2 * D], dshift=wide[:, 2 * D:3 * D], dscale=wide[:, 3 * D:4 * D], dpost_w=vec[0], dbias=vec[1],
               dw=vec[2])
    norm = (s["dh"], x1, s["w"], s["scale"], out["dw"], out["dshift"], out["dscale"]) if nxt else None
    out["dx"], out["da"] = ops.post_norm_residual_bwd(s["dx1"] if dx1 else None, s["a"], s["post_w"], s["gate"], stats,
                                                      out["dgate"], out["dpost_w"], keep, inv, alpha, norm, out["dbias"])
    torch.cuda.synchronize()
    assert bool((wide[:, :D] == 7).all()) and bool((wide[:, 4 * D:] == 7).all())
    if not nxt:
        assert bool((wide[:, 2 * D:] == 7).all()) and bool((vec[2] == 0.5).all())
    for k in ("dpost_w", "dbias", "dw"):
        out[k] = out[k] - 0.5  # (accumulated; the sums are far larger than 0.5, so the shift costs a rounding at most)
    return out


def check(B, L, D, dtype, nxt, alpha, seed=0, mod_dtype=None, keep=None, inv=1.0, mask=None, dx1=True):
    s = make(B, L, D, dtype, seed, mod_dtype)
    x1, h, stats = run_fwd(s, alpha, nxt, keep, inv)
    want = fwd64(s, alpha, nxt, mask)
    near(x1, want[0], dict(half=0, rel=FWD), "x1")
    if nxt:
        # h is the norm of the x1 that was stored
        xh, mu, rs = ln(x1.cpu().double())
        d = {k: s[k].cpu().double() for k in ("w", "scale", "shift")}
        near(h, xh * d["w"] * (1 + d["scale"][:, None]) + d["shift"][:, None], dict(half=half(dtype), rel=FWD), "h")
        assert h.dtype == dtype
    got = run_bwd(s, alpha, nxt, x1, stats, keep, inv, dx1)
    ref, size = bwd64(s, alpha, nxt, mask, dx1, x1 if nxt else None)
    near(got["dx"], ref["dx"], dict(half=0, rel=BWD), "dx")
    near(got["da"], ref["da"], dict(half=half(dtype), rel=BWD), "da")
    n = {"dgate": L, "dshift": L, "dscale": L}
    for k in size:
        bound = (192 + n.get(k, B * L)) * E32 * size[k] + 2 * E32  # (2 E32: the 0.5 that the buffers held)
        err = (got[k].cpu().double() - ref[k]).abs()
        assert bool((err <= bound).all()), f"{k}: {float((err / bound).max()):.2f} of the bound"
    return s, got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [4, 32, 100, 252, 256, 260, 512, 516, 768, 1020, 1024, 1028, 1536, 2048])
def test_widths(D, dtype):
    for L, nxt, alpha in ((1, True, 1.0), (37, True, 0.9), (37, False, 1.1)):
        check(3, L, D, dtype, nxt, alpha)


@pytest.mark.parametrize("B,L", [(1, 1), (1, 2), (7, 1), (1, 31), (2, 32), (2, 33), (3, 65), (1, 400), (40, 420)])
def test_lengths(B, L):
    """chunks of 4 to 32 rows, whole and cut off"""
    check(B, L, 64, torch.bfloat16, True, 1.0)
    check(B, L, 64, torch.float32, False, 0.5)
    check(B, L, 64, torch.float32, True, 1.0, dx1=False)


@pytest.mark.parametrize("B,L,D", [(11, 1, 1028), (9, 2, 96), (5, 3, 64), (30001, 1, 32), (16003, 3, 32), (16000, 2, 100)])
def test_short_batch_elements(B, L, D):
    """several whole batch elements to a chunk, the last chunk not full; 5 x 3: one to a chunk"""
    check(B, L, D, torch.bfloat16, True, 1.0)
    check(B, L, D, torch.float32, False, 0.5)


@pytest.mark.parametrize("D", [36, 256, 516, 768, 1024, 1484, 2048])
def test_next_norm_is_the_plain_norm_to_the_bit(D):
    """blocks that are joined at their boundary and blocks that are not give the same activations"""
    from protein_lig_sedd_amd import ops
    for dtype in (torch.float32, torch.bfloat16):
        s = make(4, 300, D, dtype)
        x1, h, (_, _, mean, rstd) = run_fwd(s, 0.9, True)
        y, m, r = ops.ln_modulate_fwd(x1, s["w"], s["shift"], s["scale"], out_dtype=dtype)
        assert torch.equal(h.view(-1), y.view(-1)) and torch.equal(mean, m.view(-1)) and torch.equal(rstd, r.view(-1))


def test_types_of_activations_and_modulation():
    for dtype in (torch.float32, torch.bfloat16):
        for mod in (torch.float32, torch.bfloat16):
            check(2, 9, 96, dtype, True, 1.0, mod_dtype=mod)


def test_rows_that_are_constant_and_large_offsets():
    """a row without variance (its norm is 0 / sqrt(eps)), and one whose mean is far larger than its spread: the two passes over
    the row in registers lose nothing, a sum of squares minus a squared mean would"""
    s = make(2, 6, 64, torch.float32)
    s["a"][0, 0] = 3.25
    s["a"][0, 1] = 0.0
    x1, _, (pm, pr) = run_fwd(s, 1.0, False)[0], None, run_fwd(s, 1.0, False)[2][:2]
    assert float(pm[0]) == 3.25 and abs(float(pr[0]) * 1e-5 ** 0.5 - 1) < 4 * E32
    assert torch.equal(x1[0, :2], s["residual"][0, :2])
    # the mean, an fp32 number that is saved for the backward, is a sum of terms of about 1000: it is off by up to 14 x 2^-24 x 1000
    # (the roundings of its adds) where the spread is 0.8; a variance taken as a difference of squares would be off by 1000 as much
    s["a"][1] = 1000.0 + s["a"][1]
    near(run_fwd(s, 1.0, False)[0], fwd64(s, 1.0, False)[0], dict(half=0, rel=FWD + 14 * E32 * 1000 / 0.8), "x1")


def test_dropout_masks_agree():
    """the mask of a DropSeed, read off a forward pass whose other factors are 1, holds in forward and backward"""
    from protein_lig_sedd_amd import ops
    B, L, D, p = 2, 21, 192, 0.25
    s = make(B, L, D, torch.float32)
    keep = ops.DropSeed(p, seed=12345)
    inv = 1 / (1 - p)
    z = dict(s, residual=torch.zeros_like(s["residual"]), gate=torch.ones(B, D, device=DEV), post_w=torch.ones(D, device=DEV))
    n = run_fwd(z, 1.0, False)[0]
    m = run_fwd(z, 1.0, False, keep, inv)[0]
    mask = (m != 0).cpu().double() * inv
    assert abs(float((m != 0).float().mean()) - (1 - p)) < 5 * (p * (1 - p) / n.numel()) ** 0.5
    for nxt in (True, False):
        check(B, L, D, torch.float32, nxt, 0.9, keep=keep, inv=inv, mask=mask)


def test_gradients_against_differences():
    """d/dt of the scalar sum(x1 dx1) + sum(h dh) along a random direction of every input, by central differences of the fp32
    kernel's forward (summed in 64 bits) with step 2^-6.  The truncation error is (2^-12 / 6) of the third derivative, at most a
    few units per element of the terms' sizes; rounding is FWD x sizes / 2^-6: both below 2^-9 of the sum of the sizes'
    root of squares, which is what random signs leave."""
    s = make(2, 5, 64, torch.float32)
    alpha, t = 0.8, 2.0 ** -6
    x1, h, stats = run_fwd(s, alpha, True)
    got = run_bwd(s, alpha, True, x1, stats)
    names = dict(residual="dx", a="da", post_w="dpost_w", gate="dgate", w="dw", scale="dscale", shift="dshift")
    for name, gname in names.items():
        v = torch.randn(s[name].shape, generator=torch.Generator().manual_seed(3)).to(DEV)
        v = v / v.norm()  # (a unit direction: the inputs move by 2^-6 in all)
        f = []
        for sign in (1, -1):
            q = dict(s)
            q[name] = (s[name] + sign * t * v)
            if name in ("gate", "scale", "shift"):
                mod = torch.cat([q["gate"], q["shift"], q["scale"]], 1)
                q["gate"], q["shift"], q["scale"] = mod.chunk(3, 1)
            y1, yh, _ = run_fwd(q, alpha, True)
            f.append(float((y1.double() * s["dx1"].double()).sum() + (yh.double() * s["dh"].double()).sum()))
        num = (f[0] - f[1]) / (2 * t)
        ana = float((got[gname].double() * v.double()).sum())
        size = float(got[gname].double().norm())
        assert abs(num - ana) <= 2.0 ** -9 * size + FWD * 640 * 4 / t ** 0.5, (name, num, ana)


def test_formulas_against_autograd():
    """the 64-bit formulas themselves (CPU)"""
    s = {k: v.cpu() for k, v in make(2, 7, 32, torch.float32).items()}
    leaf = {k: s[k].double().clone().requires_grad_() for k in ("residual", "a", "post_w", "gate", "w", "shift", "scale")}
    n = torch.nn.functional.layer_norm(leaf["a"], (32,), leaf["post_w"])
    x1 = 0.9 * leaf["residual"] + leaf["gate"][:, None] * n
    h = torch.nn.functional.layer_norm(x1, (32,), leaf["w"]) * (1 + leaf["scale"][:, None]) + leaf["shift"][:, None]
    ((x1 * s["dx1"].double()).sum() + (h * s["dh"].double()).sum()).backward()
    ref, _ = bwd64(s, 0.9, True)
    for k, g in dict(residual="dx", a="da", post_w="dpost_w", gate="dgate", w="dw", shift="dshift", scale="dscale").items():
        assert float((leaf[k].grad - ref[g]).abs().max()) < 1e-12
    assert float((fwd64(s, 0.9, True)[1] - h.detach()).abs().max()) < 1e-12


def test_runs_repeat_and_capture():
    s = make(3, 50, 768, torch.bfloat16)
    x1, h, stats = run_fwd(s, 1.0, True)
    first = run_bwd(s, 1.0, True, x1, stats)
    graphs = []
    from protein_lig_sedd_amd import ops
    D = 768
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        dmod, vec = torch.zeros(3, 3 * D, device=DEV), torch.zeros(3, D, device=DEV)
        with torch.cuda.graph(gr):
            y1, yh, st = run_fwd(s, 1.0, True)
            vec.zero_()
            dx, da = ops.post_norm_residual_bwd(s["dx1"], s["a"], s["post_w"], s["gate"], st, dmod[:, :D], vec[0],
                                                norm=(s["dh"], y1, s["w"], s["scale"], vec[2], dmod[:, D:2 * D], dmod[:, 2 * D:]),
                                                dbias=vec[1])
        graphs.append((gr, y1, yh, dx, da, dmod, vec))
    side = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for g in graphs:
            for t in g[1:]:
                t.fill_(9.0)
        torch.cuda.synchronize()
        for st, g in zip(side, graphs):
            with torch.cuda.stream(st):
                g[0].replay()
        again = run_bwd(s, 1.0, True, x1, stats)
        torch.cuda.synchronize()
        for k in first:
            assert torch.equal(first[k], again[k]), k
        for _, y1, yh, dx, da, dmod, vec in graphs:
            assert torch.equal(y1, x1) and torch.equal(yh, h) and torch.equal(dx, first["dx"]) and torch.equal(da, first["da"])
            assert torch.equal(dmod[:, :D], first["dgate"]) and torch.equal(dmod[:, 2 * D:], first["dscale"])
            assert float((vec[0] - first["dpost_w"]).abs().max()) <= 2.0 ** -22 * float(vec[0].abs().max())


def test_empty():
    from protein_lig_sedd_amd import ops
    for B, L in ((0, 5), (2, 0)):
        s = make(B, L, 64, torch.float32)
        x1, h, stats = run_fwd(s, 1.0, True)
        assert x1.shape == h.shape == (B, L, 64)
        dmod = torch.full((B, 64), 3.0, device=DEV)
        dx, da = ops.post_norm_residual_bwd(s["dx1"], s["a"], s["post_w"], s["gate"], stats, dmod, None)
        assert dx.shape == da.shape == (B, L, 64) and not dmod.any()


def test_refusals():
    from protein_lig_sedd_amd import ops
    s = make(2, 3, 64, torch.float32)
    ok = dict(residual=s["residual"], a=s["a"], post_w=s["post_w"], gate=s["gate"])
    for k, v in (("residual", s["residual"].bfloat16()), ("residual", s["residual"][0]), ("residual", s["residual"].transpose(0, 1)),
                 ("a", s["a"][:, :2]), ("a", s["a"].transpose(0, 1).contiguous().transpose(0, 1)), ("post_w", s["post_w"][:32]),
                 ("post_w", s["post_w"].bfloat16()), ("gate", s["gate"][:1]), ("gate", s["gate"].t().contiguous().t())):
        with pytest.raises(ValueError):
            ops.post_norm_residual_fwd(**dict(ok, **{k: v}))
    with pytest.raises(ValueError):
        ops.post_norm_residual_fwd(**ok, norm=(s["w"], s["shift"].contiguous(), s["scale"]))  # another row stride
    with pytest.raises(ValueError):
        ops.post_norm_residual_fwd(**ok, keep=torch.ones(2, 3, 64, dtype=torch.uint8, device=DEV))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.post_norm_residual_fwd(**dict(ok, a=s["a"].cpu()))
    st = run_fwd(s, 1.0, False)[2]
    with pytest.raises(ValueError, match="dx1"):
        ops.post_norm_residual_bwd(None, s["a"], s["post_w"], s["gate"], st, None, None)
    with pytest.raises(ValueError, match="post_mean"):
        ops.post_norm_residual_bwd(s["dx1"], s["a"], s["post_w"], s["gate"], (st[0][:3], st[1]), None, None)


# ------------------------------------------------------------------------------------------------------ the model
def config(post=True, scale=0.9, D=64, blocks=3):
    ns = types.SimpleNamespace
    return ns(tokens=25, graph=ns(type="absorb"),
              model=ns(hidden_size=D, cond_dim=32, n_heads=2, n_blocks=blocks, dropout=0.0, scale_by_sigma=False, post_norm=post,
                       residual_scale=scale))


def seeded(model, seed=0):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n, p in sorted(model.named_parameters()):
            r = torch.randn(p.shape, generator=g)
            p.copy_((1 + 0.1 * r) if p.dim() == 1 and "norm" in n else r * (0.3 / max(p.shape[-1], 1) ** 0.5 if p.dim() > 1 else 0.05))
    return model


def model64(sd, x, sigma, cfg):
    """the model in plain torch on the CPU, 64 bits"""
    F = torch.nn.functional
    m = cfg.model
    D, H, alpha = m.hidden_size, m.n_heads, m.residual_scale
    d = D // H
    P = lambda n: sd[n]  # noqa: E731
    lin = lambda v, n: F.linear(v, P(n + ".weight"), sd.get(n + ".bias"))  # noqa: E731
    h = P("vocab_embed.embedding.weight")[x]
    k = torch.arange(128, dtype=torch.float64)
    arg = sigma.double()[:, None] * torch.exp(-torch.log(torch.tensor(10000.0, dtype=torch.float64)) * k / 128)
    c = F.silu(lin(F.silu(lin(torch.cat([arg.cos(), arg.sin()], -1), "sigma_map.mlp.0")), "sigma_map.mlp.2"))
    f = 1.0 / (10000 ** (torch.arange(0, d, 2).double() / d))
    ang = torch.arange(x.shape[1]).double()[:, None] * f
    co, si = ang.cos()[None, :, None], ang.sin()[None, :, None]

    def rot(t):
        a, b = t[..., :d // 2], t[..., d // 2:]
        return torch.cat([a * co - b * si, b * co + a * si], -1)

    for i in range(m.n_blocks):
        b = f"blocks.{i}."
        mod = lin(c, b + "adaLN_modulation")[:, None].chunk(6, -1)
        n1 = F.layer_norm(h, (D,), P(b + "norm1.weight")) * (1 + mod[1]) + mod[0]
        q, kk, v = lin(n1, b + "attn_qkv").view(*x.shape, 3, H, d).unbind(2)
        q, kk = rot(q), rot(kk)
        w = torch.softmax(torch.einsum("blhd,bmhd->bhlm", q, kk) / d ** 0.5, -1)
        o = lin(torch.einsum("bhlm,bmhd->blhd", w, v).reshape(*x.shape, D), b + "attn_out")
        h = alpha * h + mod[2] * F.layer_norm(o, (D,), P(b + "post_norm1.weight"))
        n2 = F.layer_norm(h, (D,), P(b + "norm2.weight")) * (1 + mod[4]) + mod[3]
        y = lin(F.gelu(lin(n2, b + "mlp.0"), approximate="tanh"), b + "mlp.2")
        h = alpha * h + mod[5] * F.layer_norm(y, (D,), P(b + "post_norm2.weight"))
    sh, sc = lin(c, "output_layer.adaLN_modulation")[:, None].chunk(2, -1)
    out = lin(F.layer_norm(h, (D,), P("output_layer.norm_final.weight")) * (1 + sc) + sh, "output_layer.linear")
    return out.scatter(-1, x[..., None], 0.0)


@pytest.mark.parametrize("chained", [True, False])
@pytest.mark.parametrize("sinks", [True, False])
def test_model_gradients(chained, sinks, monkeypatch):
    """logits and every gradient of a model with post_norm and a residual scale, with the boundary fusion and without it, into
    gradient buffers that exist (accumulated) and fresh ones.  fp32 compute, three blocks: the bar of the repository's fp32 model
    tests, 1e-4 relative per tensor."""
    from protein_lig_sedd_amd.model import layers
    from protein_lig_sedd_amd.model.transformer import _SEDD
    monkeypatch.setattr(layers, "BLOCK_CHAIN", chained)
    cfg = config()
    model = seeded(_SEDD(cfg, compute_dtype=torch.float32)).to(DEV)
    g = torch.Generator().manual_seed(5)
    x, sigma = torch.randint(0, 26, (3, 20), generator=g), torch.rand(3, generator=g) + 0.1
    up = torch.randn(3, 20, 26, generator=g)
    sd = {k: v.detach().cpu().double().requires_grad_(v.is_floating_point() and "inv_freq" not in k)
          for k, v in model.state_dict().items()}
    want = model64(sd, x, sigma, cfg)
    (want * up.double()).sum().backward()
    if sinks:
        for p in model.parameters():
            p.grad = torch.full_like(p, 0.25)
    out = model(x.to(DEV), sigma.to(DEV))
    (out * up.to(DEV)).sum().backward()
    err = float((out.detach().cpu().double() - want.detach()).norm() / want.detach().norm())
    assert err < 1e-4, err
    for n, p in model.named_parameters():
        got = p.grad.cpu().double() - (0.25 if sinks else 0.0)
        ref = sd[n].grad
        err = float((got - ref).norm() / ref.norm().clamp_min(1e-6))
        assert err < 1e-4, (n, err)


def test_residual_scale_one_and_no_post_norm_are_the_old_model():
    from protein_lig_sedd_amd.model.transformer import _SEDD
    g = torch.Generator().manual_seed(1)
    x, sigma = torch.randint(0, 26, (2, 16), generator=g).to(DEV), torch.rand(2, generator=g).to(DEV)
    cfg = config(post=False, scale=1.0)
    a = seeded(_SEDD(cfg)).to(DEV)
    del cfg.model.post_norm, cfg.model.residual_scale
    b = _SEDD(cfg).to(DEV)
    b.load_state_dict(a.state_dict())
    assert torch.equal(a(x, sigma), b(x, sigma))


def test_bf16_chained_equals_unchained(monkeypatch):
    """the boundary fusion changes where gradients meet, not what they are: bf16 compute, D 256, dropout on (same seeds)"""
    from protein_lig_sedd_amd import ops
    from protein_lig_sedd_amd.model import layers
    from protein_lig_sedd_amd.model.transformer import _SEDD
    cfg = config(D=256, blocks=2, scale=1.0)
    cfg.model.dropout = 0.1
    model = seeded(_SEDD(cfg)).to(DEV)
    model.train()
    g = torch.Generator().manual_seed(5)
    x, sigma = torch.randint(0, 26, (4, 96), generator=g).to(DEV), torch.rand(4, generator=g).to(DEV)
    got = []
    for chain in (True, False):
        monkeypatch.setattr(layers, "BLOCK_CHAIN", chain)
        ops.DropSeed._counter = 40
        model.zero_grad(set_to_none=True)
        out = model(x, sigma)
        out.float().square().mean().backward()
        got.append((out.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}))
    assert torch.equal(got[0][0], got[1][0])
    for n, v in got[0][1].items():
        # (sums in another order: fp32 roundings of bf16 gradients, half a bf16 step where one of them flips)
        assert float((v - got[1][1][n]).norm()) <= 2.0 ** -8 * float(v.norm()) + 1e-12, n


@pytest.mark.parametrize("cdt", [torch.float32, torch.bfloat16])
def test_trainer_eager_captured_and_with_a_second_stream(cdt):
    """the trainer's fused step on a post-norm model: one captured step replayed, and weight gradients on a second stream, leave
    the bits of the eager steps"""
    from protein_lig_sedd_amd import graph_lib, noise_lib
    from protein_lig_sedd_amd.model.transformer import _SEDD
    from protein_lig_sedd_amd.train import SEDDTrainer
    B, L, steps = 4, 48, 6
    graph, noise = graph_lib.Absorbing(25), noise_lib.LogLinearNoise(eps=1e-3).to(DEV)
    g = torch.Generator().manual_seed(9)
    xs = [torch.randint(0, 25, (B, L), generator=g).to(DEV) for _ in range(steps)]
    ts = [(torch.rand(B, generator=g) * 0.9 + 0.05).to(DEV) for _ in range(steps)]
    us = [torch.rand(B, L, generator=g).to(DEV) for _ in range(steps)]

    def run(**kw):
        model = seeded(_SEDD(config(D=128, blocks=2), compute_dtype=cdt)).to(DEV)
        tr = SEDDTrainer(model, noise, graph, dict(lr=1e-3, warmup=3, grad_clip=1.0, weight_decay=0.01), world_size=1, **kw)
        losses = [float(tr.train_step(xs[i], t=ts[i], u=us[i])) for i in range(steps)]
        torch.cuda.synchronize()
        return losses, tr

    eager, te = run()
    assert eager[-1] != eager[0] and all(map(math.isfinite, eager))
    for kw in (dict(hip_graph=True), dict(wgrad_stream=True)):
        losses, tr = run(**kw)
        assert losses == eager, kw
        for name in ("p", "m", "v", "ema"):
            assert torch.equal(getattr(tr.flat, name), getattr(te.flat, name)), (kw, name)


# ------------------------------------------------------------------------------------- the three operators together
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_train_clip_and_sample(dtype):
    """a post-norm model trained by a torch optimiser with clipping over its gradient tensors, then sampled with truncation"""
    from protein_lig_sedd_amd import graph_lib, losses, noise_lib, sampling
    from protein_lig_sedd_amd.model.transformer import _SEDD
    ns = types.SimpleNamespace
    B, L, steps = 4, 32, 4
    cfg = config(scale=1.0, blocks=2)
    cfg.model.scale_by_sigma = True
    cfg.optim = ns(lr=1e-3, warmup=0, grad_clip=1e-3)
    torch.manual_seed(0)
    model = seeded(_SEDD(cfg, compute_dtype=dtype)).to(DEV)
    graph, noise = graph_lib.Absorbing(25), noise_lib.LogLinearNoise(eps=1e-3).to(DEV)
    loss_fn = losses.get_loss_fn(noise, graph)
    params = list(model.parameters())
    opt = torch.optim.SGD(params, lr=1.0)
    optimize = losses.optimization_manager(cfg)
    batch = torch.randint(0, 25, (B, L), device=DEV)
    for step in range(1, 4):
        opt.zero_grad()
        loss = loss_fn(model, batch)
        loss.backward()
        before = [p.detach().clone() for p in params]
        g = [p.grad.double() for p in params if p.grad is not None]
        norm = float(torch.stack([t.square().sum() for t in g]).sum().sqrt())
        optimize(opt, None, params, step, lr=1.0)
        moved = float(torch.stack([(p.detach() - b).double().square().sum() for p, b in zip(params, before)]).sum().sqrt())
        # SGD with lr 1 moves the weights by the clipped gradient: its norm is min(norm, grad_clip); fp32 weights of size about 1
        # hold the difference to 2^-24 each
        n = sum(p.numel() for p in params)
        assert torch.isfinite(loss) and abs(moved - min(norm, 1e-3)) <= 1e-3 * 2.0 ** -20 + n ** 0.5 * 2.0 ** -24
    us = [torch.rand(B, L, 26, device=DEV) for _ in range(steps)] + [torch.rand(B, L, 25, device=DEV)]
    run = sampling.get_pc_sampler(graph, noise, (B, L), "ancestral", steps, device=DEV, temperature=0.8, top_k=10, top_p=0.9)
    out = run(model, noise_seq=us)
    assert out.shape == (B, L) and int(out.min()) >= 0 and int(out.max()) < 25
    assert torch.equal(out, run(model, noise_seq=us))
    # the last step, redone by hand
    plain = sampling.get_pc_sampler(graph, noise, (B, L), "ancestral", steps, denoise=False, device=DEV, temperature=0.8,
                                    top_k=10, top_p=0.9)
    x = plain(model, noise_seq=us)
    with torch.no_grad():
        s = model(x, noise(torch.full((B, 1), 1e-5, device=DEV))[0].reshape(-1))
    from test_gpu_sample_truncated import ref
    tok = ref(s[..., :-1], us[-1], 0.8, 10, 0.9).to(DEV)
    assert torch.equal(out, torch.where(x == 25, tok, x))
