"""Truncated sampling where top-k and top-p act together and the mass before an entry lies within a rounding of its border: rows
that 32-bit arithmetic cannot decide, in every form of the kernel, against the definition in 64 bits on the CPU.  Tokens are
compared for equality: two 64-bit evaluations differ only where two sums agree to 1e-15, and the borders here are fp32 numbers,
about 1e-8 away from the sums."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def want(x, u, k, P):
    """x, u [R, V], P [R] -> tokens, from the definition"""
    z, order = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    z, order = z[:, :k], order[:, :k]
    q = torch.exp(z - z[:, :1])
    S, W = q.cumsum(-1) - q, q.sum(-1, keepdim=True)
    kept = S < P.double()[:, None] * W
    kept[:, 0] = True
    e = 1e-10 - torch.log((u.gather(-1, order) + 1e-10).clamp(max=1.0).double())
    r = torch.where(kept, q / e, -1.0)
    return torch.where(r == r.amax(-1, keepdim=True), order, x.shape[1]).amin(-1)


def border_rows(rows, V, k, dtype, seed, shift):
    """scores around `shift`, top-p at the fp32 number at, below or above the mass before some rank 1 .. k - 1, and noise that
    makes the entry of that rank win if it is kept"""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=g) * 2.0 + shift).to(dtype)
    z, order = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    q = torch.exp(z[:, :k] - z[:, :1])
    rank = torch.randint(1, k, (rows, 1), generator=g)
    P = ((q.cumsum(-1) - q) / q.sum(-1, keepdim=True)).gather(-1, rank)[:, 0].float()
    step = torch.randint(-1, 2, (rows,), generator=g)
    P = torch.where(step < 0, torch.nextafter(P, torch.zeros(())), torch.where(step > 0, torch.nextafter(P, torch.ones(())), P))
    u = torch.full((rows, V), 0.5)
    u.scatter_(1, order.gather(-1, rank), 1.0 - 2.0 ** -20)
    return x, u, P


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,rows", [(26, 300), (64, 300), (150, 60), (300, 60), (700, 60), (1500, 60), (1500, 520), (2365, 60),
                                    (2365, 520), (2900, 520), (3500, 60), (6000, 40), (6000, 260), (12000, 40), (12000, 260),
                                    (20000, 40), (33001, 20)])
def test_top_p_at_a_border_under_top_k(V, rows, dtype):
    from protein_lig_sedd_amd import ops
    for k in (2, 3, 5, 10, 40):
        if k >= V:
            continue
        for i, shift in enumerate((0.0, 30.0, -30.0)):  # (scores of both signs, all above zero, all below)
            x, u, P = border_rows(rows, V, k, dtype, 1000 * V + 10 * k + i, shift)
            ref = want(x, u, k, P)
            got = ops.sample_truncated(x.to(DEV), u.to(DEV), top_k=k, top_p=P.to(DEV)).cpu()
            bad = (got != ref).nonzero()
            assert bad.numel() == 0, f"{len(bad)} of {rows} tokens differ: k {k}, shift {shift}, first at {bad[0].tolist()}"


@pytest.mark.parametrize("V", [300, 2365, 6000, 20000])
def test_two_entries_above_many_equal_ones(V):
    """top-k 2 whose second entry begins exactly at the mass that top-p keeps: it is out, whatever the rest of the row weighs"""
    from protein_lig_sedd_amd import ops
    x = torch.full((1, V), 0.5)
    x[0, 0], x[0, 100] = 2.0, 1.0
    u = torch.full((1, V), 0.5)
    u[0, 100] = 0.9999
    P = torch.tensor(1 / (1 + math.exp(-1)), dtype=torch.float32)
    for p, token in ((torch.nextafter(P, torch.zeros(())), 0), (torch.nextafter(P, torch.ones(())), 100)):
        assert want(x, u, 2, p.reshape(1)).tolist() == [token]
        for dtype in (torch.float32, torch.bfloat16):
            assert ops.sample_truncated(x.to(dtype).to(DEV), u.to(DEV), top_k=2, top_p=float(p)).tolist() == [token]
