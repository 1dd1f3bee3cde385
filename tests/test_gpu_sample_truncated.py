"""Truncated sampling (ops.sample_truncated, catsample.sample_logits, Absorbing.ancestral_step, the "ancestral" predictor)
against a plain 64-bit evaluation of its definition on the CPU.  The results are token indices, so every comparison is for
equality: the kernels decide as 64-bit arithmetic does, and two 64-bit evaluations differ only where two sums agree to 1e-15."""
import math
import types

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ref_row(x, u, T, k, P, m):
    """one row, straight from the definition: sort, running sums, arg-max"""
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    V = len(x)
    cand = x > -np.inf
    if not cand.any():
        return -1
    top = x.max()
    if not T > 0:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore", over="ignore"):
        q = np.exp((x - top) / np.float64(np.float32(T)))
    q = np.where(x == top, 1.0, np.where(np.isinf(top), 0.0, q))
    order = sorted(np.nonzero(cand)[0], key=lambda j: (-x[j], j))
    if 0 < k < V:
        order = order[:int(k)]
    W, S, kept = math.fsum(q[order]), 0.0, []
    P, m = np.float64(np.float32(P)), np.float64(np.float32(m))
    for r, j in enumerate(order):
        if r == 0 or ((P >= 1 or S < P * W) and q[j] >= m):
            kept.append(j)
        S += q[j]
    w = np.minimum(np.float32(u) + np.float32(1e-10), np.float32(1)).astype(np.float64)
    kept = sorted(kept)
    r = q[kept] / (1e-10 - np.log(w[kept]))
    return int(kept[int(np.argmax(r))])


def ref(logits, u, T=1.0, k=0, P=1.0, m=0.0):
    x = logits.detach().float().cpu().numpy().reshape(-1, logits.shape[-1])
    un = u.detach().cpu().numpy().reshape(-1, u.shape[-1])
    B = logits.shape[0] if logits.dim() > 1 else 1
    per = lambda v, i: float(v.reshape(-1)[i * B // len(x) if v.numel() > 1 else 0]) if torch.is_tensor(v) else v  # noqa: E731
    cpu = [v.cpu() if torch.is_tensor(v) else v for v in (T, k, P, m)]
    out = [ref_row(x[i], un[i][:x.shape[1]], *[per(v, i) for v in cpu]) for i in range(len(x))]
    return torch.tensor(out, dtype=torch.int64).reshape(logits.shape[:-1])


def data(shape, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*shape, generator=g) * spread).to(dtype)
    return x.to(DEV), torch.rand(*shape, generator=g).to(DEV)


CUTS = [dict(), dict(temperature=0.6), dict(top_k=1), dict(top_k=7), dict(top_p=0.7), dict(min_p=0.1),
        dict(temperature=1.3, top_k=11, top_p=0.85, min_p=0.02)]


def check(x, u, **c):
    from protein_lig_sedd_amd import ops
    got = ops.sample_truncated(x, u, **c).cpu()
    want = ref(x, u, c.get("temperature", 1.0), c.get("top_k", 0), c.get("top_p", 1.0), c.get("min_p", 0.0))
    bad = (got != want).nonzero()
    assert bad.numel() == 0, f"{len(bad)} of {got.numel()} tokens differ, first at {bad[0].tolist()}: {c}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 25, 26, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 300, 511, 513])
def test_small_vocabularies(V, dtype):
    x, u = data((3, 90, V), dtype, V)
    for c in CUTS:
        check(x, u, **c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,rows", [(1000, 24), (2365, 16), (2397, 16), (4096, 6), (4097, 6), (9001, 5), (16385, 4), (32768, 3),
                                    (33001, 3), (70001, 2)])
def test_wide_vocabularies(V, rows, dtype):
    x, u = data((rows, V), dtype, V)
    for c in CUTS + [dict(top_k=V - 1, top_p=0.999), dict(top_k=V // 2, top_p=0.5)]:
        check(x, u, **c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,rows", [(1025, 600), (2047, 600), (2365, 513), (2600, 600), (3000, 600), (3001, 600), (4097, 300), (8200, 260),
                                    (12001, 257), (16384, 257)])
def test_wide_vocabularies_in_many_rows(V, rows, dtype):
    """what many rows decide is what the formulas say of some of them, and what few rows at a time decide of all"""
    from protein_lig_sedd_amd import ops
    x, u = data((rows, V), dtype, V)
    some = [0, 1, rows // 2, rows - 1]
    for c in CUTS + [dict(top_k=V // 2, top_p=0.5)]:
        got = ops.sample_truncated(x, u, **c)
        want = ref(x[some], u[some], c.get("temperature", 1.0), c.get("top_k", 0), c.get("top_p", 1.0), c.get("min_p", 0.0))
        assert torch.equal(got[some].cpu(), want), c
        parts = [ops.sample_truncated(x[i:i + 100], u[i:i + 100], **c) for i in range(0, rows, 100)]
        assert torch.equal(got, torch.cat(parts)), c


@pytest.mark.parametrize("V", [26, 64, 300, 5000])
def test_many_rows_and_one(V):
    for rows in (1, 255, 256, 257, 2000 if V < 1000 else 40):
        x, u = data((rows, V), torch.bfloat16, rows)
        check(x, u, temperature=0.9, top_p=0.9, top_k=20)
    x, u = data((V,), torch.float32, 5)  # a single row without a leading dimension
    check(x, u, top_p=0.8)


@pytest.mark.parametrize("V", [5, 26, 64, 200, 3000])
def test_ties_and_equal_rows(V):
    """equal scores: the order goes by index, and with equal weights the sums before a border are whole numbers"""
    g = torch.Generator().manual_seed(V)
    u = torch.rand(64, V, generator=g).to(DEV)
    for x in (torch.zeros(64, V), torch.randint(0, 3, (64, V), generator=g).float(), torch.full((64, V), -7.25)):
        for c in (dict(), dict(top_p=0.5), dict(top_p=0.25, top_k=4), dict(top_k=3), dict(min_p=1.0), dict(top_p=1e-6)):
            check(x.to(DEV), u, **c)
    for dtype in (torch.float32, torch.bfloat16):  # equal scores across the border of the k, above and below zero
        x = torch.randint(-5, 4, (96, V), generator=g).to(dtype).to(DEV) * 0.75
        uu = torch.rand(96, V, generator=g).to(DEV)
        for k in (2, 3, 5, max(V // 3, 1), max(V - 2, 1)):
            for P in (0.3, 0.6, 0.9):
                check(x, uu, top_k=k, top_p=P)
    x = torch.zeros(8, V)
    x[:, V // 2:] = -0.0  # both zeros are one value
    check(x.to(DEV), u[:8], top_k=max(V // 2, 1), top_p=0.9)
    u1 = torch.full((4, V), 0.5, device=DEV)  # equal noise too: the lowest index
    check(torch.zeros(4, V, device=DEV), u1)
    check(torch.ones(4, V, device=DEV), u1, top_k=2)


@pytest.mark.parametrize("V,rows", [(40, 5), (300, 5), (700, 3), (1500, 3), (1500, 520), (2365, 3), (2365, 520), (2900, 520), (3500, 3),
                                    (6000, 3), (6000, 260), (12000, 3), (12000, 260), (20000, 2), (33000, 2)])
def test_rows_decided_by_a_tie(V, rows):
    """the two best ratios equal to the bit (equal scores and noise), alone and where a border runs through them"""
    from protein_lig_sedd_amd import ops
    x, u = data((rows, V), torch.float32, V)
    u[:] = 0.5
    top, i = x.topk(3, dim=-1)
    x.scatter_(1, i[:, 1:2], top[:, :1])
    some = [0, rows - 1]
    for c in (dict(), dict(top_k=1), dict(top_k=2), dict(top_k=20, top_p=0.9), dict(top_p=0.3), dict(top_k=200, top_p=0.999, min_p=0.01),
              dict(temperature=3.0, min_p=0.5)):
        got = ops.sample_truncated(x, u, **c)
        assert torch.equal(got[some].cpu(), ref(x[some], u[some], c.get("temperature", 1.0), c.get("top_k", 0), c.get("top_p", 1.0),
                                                c.get("min_p", 0.0))), c
        assert torch.equal(got, i[:, :2].amin(-1)), c  # the lower index of the two


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3, 26, 64, 150, 4500])
def test_masks_and_non_finite(V, dtype):
    x, u = data((12, V), dtype, V + 1)
    low = torch.finfo(dtype).min
    x[0] = -math.inf
    x[1] = math.nan
    x[2, :] = -math.inf
    x[2, V - 1] = -3.0
    x[3, ::2] = -math.inf
    x[4] = low
    x[5, 1:] = low
    x[6, V // 2] = math.inf
    x[7, V // 2] = math.inf
    x[7, V - 1] = math.inf
    x[8, ::2] = math.nan
    x[9] = low
    x[9, V - 1] = torch.finfo(dtype).max
    x[10, 0] = math.nan
    x[10, 1:] = -math.inf
    for c in (dict(), dict(temperature=0.3), dict(top_k=2), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=0.0),
              dict(temperature=1.1, top_k=3, top_p=0.9, min_p=0.01)):
        check(x, u, **c)
    from protein_lig_sedd_amd import ops
    got = ops.sample_truncated(x, u, top_p=0.9)
    assert got[0] == -1 and got[1] == -1 and got[10] == -1 and got[2] == V - 1


@pytest.mark.parametrize("V", [26, 64, 700])
def test_extreme_parameters_and_noise(V):
    x, u = data((40, V), torch.float32, 3)
    for c in (dict(temperature=1e-30), dict(temperature=1e-42), dict(temperature=1e-3), dict(temperature=3e38),
              dict(temperature=50.0), dict(top_p=0.0), dict(top_p=1e-30), dict(min_p=1.0), dict(top_k=10 ** 9), dict(top_k=V)):
        check(x, u, **c)
    u[:, ::3] = 0.0
    u[:, 1] = 1.0
    u[:, 2 % V] = 1.0 - 2.0 ** -24
    for c in CUTS:
        check(x, u, **c)
    check(x * 1e30, u, top_p=0.9)
    check(x * 1e-30, u, top_p=0.9, temperature=1e-30)


def test_values_at_the_border():
    """rows whose decision turns on differences far below 32-bit accuracy"""
    g = torch.Generator().manual_seed(1)
    for V in (26, 300):
        x = torch.randn(200, V, generator=g)
        u = torch.rand(200, V, generator=g)
        q = torch.exp(x.double() - x.double().amax(-1, keepdim=True))
        # top_p at the very sum before some entry, as near as 32 bits come
        order = torch.argsort(x.double(), dim=-1, descending=True, stable=True)
        qs = q.gather(-1, order)
        before = (qs.cumsum(-1) - qs) / qs.sum(-1, keepdim=True)
        P = before[torch.arange(200), torch.randint(1, 12, (200,), generator=g)].float()
        check(x.to(DEV), u.to(DEV), top_p=P.to(DEV))
        # min_p at the weight of some entry
        m = qs[torch.arange(200), torch.randint(1, 12, (200,), generator=g)].float()
        check(x.to(DEV), u.to(DEV), min_p=m.to(DEV))
        # two entries whose weight / noise agree to a few parts in 1e8
        u2 = u.clone()
        j = torch.argmax(q / -torch.log(u.double()), -1)
        i = (j + 1) % V
        r = torch.arange(200)
        e = -torch.log(u.double()[r, j]) * q[r, i] / q[r, j]
        u2[r, i] = torch.exp(-e).float()
        check(x.to(DEV), u2.to(DEV), top_p=0.999)


def test_per_request_parameters_layouts_and_types():
    B, L, V = 5, 9, 26
    x, u = data((B, L, V), torch.bfloat16, 11)
    g = torch.Generator().manual_seed(2)
    T = (0.3 + torch.rand(B, generator=g)).to(DEV)
    T[2] = 0.0
    k = torch.tensor([0, 3, 26, 1, 100])
    P = torch.tensor([1.0, 0.5, 0.9, 0.0, 0.7], dtype=torch.float64)
    m = torch.tensor([0.0, 0.1, 0.0, 0.3, 0.05]).to(DEV)
    check(x, u, temperature=T, top_k=k.to(DEV), top_p=P.to(DEV), min_p=m)
    check(x, u, temperature=T, top_k=k, top_p=0.8)  # (a parameter in host memory)
    check(x, u, temperature=torch.tensor(0.7), top_p=torch.tensor([0.6]))
    # views: the last column cut off, a transposed batch, odd offsets, an expanded row, a 64-bit noise tensor
    check(x[..., :-1], u[..., 1:], top_p=0.9)
    check(x[:, 1:], u[:, 1:], top_k=4)
    check(x.transpose(0, 1), u.transpose(0, 1), top_p=0.9)
    check(x.transpose(1, 2).contiguous().transpose(1, 2), u, top_p=0.9)
    flat = torch.randn(1 + 7 * 26, device=DEV).bfloat16()
    check(flat[1:].view(7, 26), u.reshape(-1, V)[:7], top_p=0.9)
    check(x[:1, :1].expand(4, L, V), u[:4], top_p=0.9)
    check(x, u.double(), top_p=0.9)
    wide = torch.randn(6, 700, device=DEV)
    check(wide[:, 3:600], torch.rand(6, 700, device=DEV)[:, 1:598], top_p=0.9, top_k=90)


def test_empty_and_long():
    from protein_lig_sedd_amd import ops
    for shape in ((0, 26), (3, 0, 26), (0, 4, 26)):
        assert ops.sample_truncated(torch.zeros(shape, device=DEV), torch.zeros(shape, device=DEV)).shape == shape[:-1]
    # more rows than one launch has waves, and offsets beyond 2^31 bytes
    M, V = 1100003, 26
    x, u = torch.randn(M, V, device=DEV), torch.rand(M, V, device=DEV)
    got = ops.sample_truncated(x, u, temperature=0.8, top_p=0.9, top_k=9)
    pick = torch.cat([torch.arange(40), torch.arange(M - 40, M)])
    assert torch.equal(got[pick].cpu(), ref(x[pick], u[pick], 0.8, 9, 0.9))
    x = torch.randn(300000, 2050, device=DEV).bfloat16()
    u = torch.rand(300000, 2050, device=DEV)
    got = ops.sample_truncated(x, u, top_k=30, top_p=0.9)
    pick = torch.cat([torch.arange(6), torch.arange(300000 - 6, 300000)])
    assert torch.equal(got[pick].cpu(), ref(x[pick], u[pick], 1.0, 30, 0.9))


def test_frequencies():
    """what is drawn follows the truncated distribution: n draws of one row, each count within 5 standard deviations (of
    about 30 counts: a false alarm once in 60000 seeds; the seed is fixed)"""
    from protein_lig_sedd_amd import ops
    for V in (26, 300):
        g = torch.Generator(device=DEV).manual_seed(V)
        n = 200000
        x = torch.randn(V, generator=g, device=DEV) * 1.5
        got = ops.sample_truncated(x.expand(n, V), torch.rand(n, V, generator=g, device=DEV), temperature=0.9, top_k=12, top_p=0.9)
        p = torch.softmax(x.double() / 0.9, -1)
        v, i = p.sort(descending=True)
        v[12:] = 0
        v = v / v.sum()
        v[(v.cumsum(0) - v) >= 0.9] = 0
        p = torch.zeros_like(p).scatter(0, i, v / v.sum())
        cnt = torch.bincount(got, minlength=V).double()
        assert bool((cnt[p == 0] == 0).all())
        assert bool(((cnt - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt() + 1e-9).all())


# ------------------------------------------------------------------------------------------------ masked positions
@pytest.mark.parametrize("V", [26, 64, 2365])
def test_ancestral_step_moves_only_masked_positions(V):
    from protein_lig_sedd_amd import graph_lib
    graph = graph_lib.Absorbing(V - 1)
    g = torch.Generator().manual_seed(V)
    B, L = 6, 50
    s = torch.randn(B, L, V, generator=g).bfloat16().to(DEV)
    x = torch.randint(0, V - 1, (B, L), generator=g)
    x[torch.rand(B, L, generator=g) < 0.6] = V - 1
    x[0] = V - 1
    x[1] = 3 % (V - 1)
    u = torch.rand(B, L, V, generator=g)
    move = torch.tensor([0.5, 0.5, 0.0, 1.0, 0.3, 0.9])
    s[4, :, :-1] = -math.inf  # nothing to sample: the position stays masked
    x, u, move = x.to(DEV), u.to(DEV), move.to(DEV)
    kw = dict(temperature=0.8, top_k=6, top_p=0.9)
    tok = ref(s[..., :-1], u, 0.8, 6, 0.9)
    tok[tok < 0] = V - 1
    for mv, uu in ((move, u), (0.4, u), (None, u[..., :-1])):
        got = graph.ancestral_step(s, x, mv, u=uu, **kw).cpu()
        go = x.cpu() == V - 1
        if mv is not None:
            go &= u[..., -1].cpu() < (mv.cpu()[:, None] if torch.is_tensor(mv) else torch.tensor(mv))
        assert torch.equal(got, torch.where(go, tok, x.cpu()))
    from protein_lig_sedd_amd import ops
    ph = ops.PhiloxNoise(77, 3)
    want = graph.ancestral_step(s, x, move, u=ops.philox_uniform(ph, (B, L, V), DEV), **kw)
    assert torch.equal(graph.ancestral_step(s, x, move, u=ph, **kw), want)


class _Model(torch.nn.Module):
    """stands in for a score model: fixed log-scores that depend on the position and on how much is masked"""

    def __init__(self, B, L, V):
        super().__init__()
        self.base = torch.randn(B, L, V, generator=torch.Generator().manual_seed(4)).to(DEV)
        self.V = V

    def forward(self, x, sigma):
        return self.base * (1 + (x == self.V - 1).float().mean(-1)[:, None, None]) + sigma.float()[:, None, None]


@pytest.mark.parametrize("hip_graph", [False, True])
def test_sampler_with_truncation(hip_graph):
    """the whole loop with given noise, against the same loop in 64 bits; replayed as a graph too"""
    from protein_lig_sedd_amd import graph_lib, noise_lib, sampling
    B, L, V, steps = 4, 32, 26, 6
    graph, noise = graph_lib.Absorbing(V - 1), noise_lib.LogLinearNoise(eps=1e-3).to(DEV)
    model = _Model(B, L, V)
    g = torch.Generator().manual_seed(9)
    us = [torch.rand(B, L, V, generator=g).to(DEV) for _ in range(steps)] + [torch.rand(B, L, V - 1, generator=g).to(DEV)]
    cut = dict(temperature=0.7, top_k=8, top_p=0.9, min_p=0.01)
    run = sampling.get_pc_sampler(graph, noise, (B, L), "ancestral", steps, device=DEV, hip_graph=hip_graph, **cut)
    x = torch.full((B, L), V - 1, dtype=torch.int64, device=DEV)
    ts, dt = torch.linspace(1, 1e-5, steps + 1, device=DEV), (1 - 1e-5) / steps
    for i in range(steps + 1):
        t = ts[i] * torch.ones(B, 1, device=DEV)
        tok = ref(model(x, noise(t)[0].reshape(-1))[..., :-1], us[i], 0.7, 8, 0.9, 0.01).to(DEV)
        go = x == V - 1
        if i < steps:
            s0, s1 = noise(t)[0], noise(t - dt)[0]
            go &= us[i][..., -1] < torch.expm1(s0 - s1) / torch.expm1(s0)
        x = torch.where(go, tok, x)
    for _ in range(3):  # (with hip_graph: a capture and its replays, eager work in between)
        got = run(model, noise_seq=us)
        torch.cuda.synchronize()
        assert torch.equal(got, x)
        torch.randn(1000, device=DEV).sum()
    assert bool((got != V - 1).all())
    one = sampling.get_pc_sampler(graph, noise, (B, L), "none", 2, device=DEV, top_k=1)(model)
    assert torch.equal(one, model(torch.full_like(x, V - 1), noise(ts[-1] * torch.ones(B, 1, device=DEV))[0].reshape(-1))[..., :-1].argmax(-1))


def test_sampler_reads_its_configuration():
    from protein_lig_sedd_amd import graph_lib, noise_lib, sampling
    ns = types.SimpleNamespace
    cfg = ns(sampling=ns(predictor="ancestral", steps=3, noise_removal=True, top_k=1))
    B, L, V = 2, 16, 26
    model = _Model(B, L, V)
    run = sampling.get_sampling_fn(cfg, graph_lib.Absorbing(V - 1), noise_lib.LogLinearNoise().to(DEV), (B, L), 1e-5, DEV)
    out = run(model)
    assert torch.equal(out, model.base[..., :-1].argmax(-1))  # top_k 1: whenever a position moves, to its best token


def test_captured_and_on_other_streams():
    """two captured graphs and eager work side by side, replayed several times: every result is the eager one"""
    from protein_lig_sedd_amd import ops
    cases = [data((n, V), torch.bfloat16, n) + (dict(temperature=0.9, top_k=9, top_p=0.9),) for n, V in ((700, 26), (90, 900))]
    want = [ops.sample_truncated(x, u, **c) for x, u, c in cases]
    graphs, outs = [], []
    for x, u, c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.sample_truncated(x, u, **c))
        graphs.append(gr)
    side = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        for o in outs:
            o.fill_(-5)
        torch.cuda.synchronize()
        for st, gr in zip(side, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        eager = [ops.sample_truncated(x, u, **c) for x, u, c in cases]
        torch.cuda.synchronize()
        for o, e, w in zip(outs, eager, want):
            assert torch.equal(o, w) and torch.equal(e, w)


def test_refusals():
    from protein_lig_sedd_amd import graph_lib, noise_lib, ops, sampling
    x, u = data((2, 3, 26), torch.float32, 1)
    tok = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    bad = [(dict(temperature=-1.0), ValueError), (dict(temperature=math.nan), ValueError), (dict(temperature=math.inf), ValueError),
           (dict(top_k=-1), ValueError), (dict(top_k=1.5), ValueError), (dict(top_p=1.5), ValueError), (dict(top_p=-0.1), ValueError),
           (dict(min_p=2.0), ValueError), (dict(top_p=torch.ones(3, device=DEV)), ValueError), (dict(x=tok), ValueError),
           (dict(mask_id=3), ValueError), (dict(move=0.5), ValueError), (dict(x=tok[:1], mask_id=25), ValueError),
           (dict(x=tok, mask_id=25, move=0.5), ValueError)]
    for kw, err in bad:
        with pytest.raises(err):
            ops.sample_truncated(x, u, **kw)
    with pytest.raises(ValueError):
        ops.sample_truncated(x, u[..., :-1])
    with pytest.raises(TypeError):
        ops.sample_truncated(x.half(), u)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.sample_truncated(x, u.cpu())
    noise = noise_lib.LogLinearNoise().to(DEV)
    for pred in ("euler", "analytic"):
        with pytest.raises(ValueError, match="ancestral"):
            sampling.get_pc_sampler(graph_lib.Absorbing(25), noise, (2, 4), pred, 2, device=DEV, top_p=0.9)
    with pytest.raises(ValueError, match="absorbing"):
        sampling.get_pc_sampler(graph_lib.Uniform(26), noise, (2, 4), "ancestral", 2, device=DEV)
    with pytest.raises(ValueError, match="states"):
        graph_lib.Absorbing(30).ancestral_step(x, tok)
