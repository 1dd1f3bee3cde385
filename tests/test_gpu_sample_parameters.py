"""Truncated sampling with per-request parameters outside the range that numbers are held to.  Tensors are not read on the host, so
the definition covers every value: T <= 0 and NaN take the first maximum, top_k <= 0 or >= V, top_p >= 1 or NaN and min_p <= 0 or NaN
switch a truncation off, top_p <= 0 and min_p > 1 leave the first maximum alone.  Against that definition in 64 bits on the CPU."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def want(x, u, T, k, P, m):
    z, order = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    V = x.shape[1]
    T, P, m = (v.float().double()[:, None] for v in (T, P, m))
    q = torch.where(z > -math.inf, torch.exp((z - z[:, :1]) / torch.where(T > 0, T, 1.0)), 0.0)
    k = torch.where((k <= 0) | (k > V), V, k)[:, None]
    place = torch.arange(V)
    W = torch.where(place < k, q, 0.0).sum(-1, keepdim=True)
    S = q.cumsum(-1) - q
    kept = (z > -math.inf) & (place < k) & (~(P < 1) | (S < P * W)) & ~(q < m)
    kept &= T > 0
    kept[:, 0] = True
    e = 1e-10 - torch.log((u.gather(-1, order) + 1e-10).clamp(max=1.0).double())
    r = torch.where(kept, q / e, -1.0)
    return torch.where(r == r.amax(-1, keepdim=True), order, V).amin(-1)


CASES = [dict(m=1.5), dict(m=1.0078125), dict(m=math.inf), dict(m=-0.5), dict(m=math.nan), dict(P=-0.25), dict(P=0.0), dict(P=1.5),
         dict(P=math.inf), dict(P=math.nan), dict(T=-1.0), dict(T=0.0), dict(T=math.nan), dict(k=-3), dict(k=0), dict(k=10 ** 6),
         dict(m=1.5, P=0.9), dict(m=1.5, k=5), dict(m=math.inf, k=5, P=0.9), dict(m=1.5, T=1e-3), dict(m=1.5, T=1e6),
         dict(P=-1.0, k=5), dict(P=2.0, k=5, m=0.05)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,copies", [(26, 4), (64, 4), (300, 4), (1500, 2), (1500, 25), (2365, 2), (2365, 25), (3500, 2), (6000, 1),
                                      (6000, 12), (12000, 1), (12000, 12), (20000, 1), (33001, 1)])
def test_values_outside_their_range(V, copies, dtype):
    from protein_lig_sedd_amd import ops
    cases = CASES * copies
    R = len(cases)
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(R, V, generator=g) * 2.5).to(dtype)
    x[:, 0] = -math.inf  # (a token that is never sampled)
    u = torch.rand(R, V, generator=g)
    col = lambda name, off, t: torch.tensor([c.get(name, off) for c in cases], dtype=t)  # noqa: E731
    T, k, P, m = (col("T", 1.0, torch.float32), col("k", 0, torch.int32), col("P", 1.0, torch.float32), col("m", 0.0, torch.float32))
    ref = want(x, u, T, k, P, m)
    got = ops.sample_truncated(x.to(DEV), u.to(DEV), T.to(DEV), k.to(DEV), P.to(DEV), m.to(DEV)).cpu()
    bad = (got != ref).nonzero()[:, 0].tolist()
    assert not bad, [(cases[i], int(got[i]), int(ref[i])) for i in bad[:8]]
    for i, c in enumerate(CASES):  # one request at a time
        one = [v[i:i + 1].to(DEV) for v in (T, k, P, m)]
        assert int(ops.sample_truncated(x[i:i + 1].to(DEV), u[i:i + 1].to(DEV), *one)) == int(ref[i]), c
