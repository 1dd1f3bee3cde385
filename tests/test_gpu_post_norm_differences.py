"""The gradients of post_norm_residual_bwd along their own direction against differences of the 64-bit formula of the forward pass.

f(t) = sum(x1 dx1) + sum(h dh) along v = g / |g| for a gradient g of the kernel: f'(0) is g64 . v and g . v = |g|, so they differ by
at most |g - g64|, and v leaves nothing of g out.  |g - g64| is bounded by the norm of the elements' bounds that
test_gpu_post_norm.py derives, with twice the roundings, as the kernel's backward starts from an x1 and statistics that its
forward has rounded: about 2^-13 |g|.  f' comes from five points 2^-8 apart, in 64 bits: h^4 / 30 of the fifth derivative, which
is below 5! (1 / 6.4)^5 x 640 along a unit direction (rows of 64 with a spread of 0.8): 10^-9 of a |g| of about 10."""
import pytest
import torch

from test_gpu_post_norm import BWD, E32, bwd64, fwd64, half, make, run_bwd, run_fwd

pytestmark = pytest.mark.gpu
NAMES = dict(residual="dx", a="da", post_w="dpost_w", gate="dgate", w="dw", scale="dscale", shift="dshift")


def along(s, name, v, alpha, nxt, dx1):
    d = {k: t.cpu().double() for k, t in s.items()}
    at = d[name]

    def f(t):
        d[name] = at + t * v
        x1, h, _ = fwd64(d, alpha, nxt)
        return float(((x1 * d["dx1"]).sum() if dx1 else 0.0) + ((h * d["dh"]).sum() if nxt else 0.0))

    e = 2.0 ** -8
    return (8 * (f(e) - f(-e)) - (f(2 * e) - f(-2 * e))) / (12 * e)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,D,nxt,alpha,dx1", [(2, 5, 64, True, 0.8, True), (2, 5, 64, False, 1.0, True), (3, 1, 64, True, 1.0, False),
                                                 (1, 41, 100, True, 1.1, True), (30, 3, 72, True, 0.9, True), (2, 70, 516, True, 1.0, True)])
def test_along_the_gradient(B, L, D, nxt, alpha, dx1, dtype):
    s = make(B, L, D, dtype, 17, torch.float32)
    x1, _, stats = run_fwd(s, alpha, nxt)
    got = run_bwd(s, alpha, nxt, x1, stats, dx1=dx1)
    ref, size = bwd64(s, alpha, nxt, None, dx1)
    n = {"dgate": L, "dshift": L, "dscale": L}
    for name, gname in NAMES.items():
        if gname not in ref:
            continue
        g = got[gname].cpu().double().reshape(s[name].shape)
        v = g / g.norm()
        if gname in size:
            bound = (2 * 192 + n.get(gname, B * L)) * E32 * size[gname] + 2 * E32
        else:
            r = ref[gname]
            rms = r.square().mean().sqrt()
            bound = 2 * BWD * (r.abs() + 4 * rms) + (half(dtype) * r.abs() if gname == "da" else 0.0)
        num, ana, tol = along(s, name, v, alpha, nxt, dx1), float(g.norm()), float(bound.norm()) + 1e-8 * float(g.norm())
        assert tol <= 2.0 ** -7 * ana, (gname, tol, ana)  # (the comparison says something)
        assert abs(num - ana) <= tol, (gname, num, ana, tol)
