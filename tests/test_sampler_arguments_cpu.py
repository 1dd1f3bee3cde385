"""get_pc_sampler's arguments that go together; nothing is launched."""
import types

import pytest
import torch


def test_truncation_that_nothing_would_apply():
    """predictor "none" draws tokens in the denoising step alone"""
    from protein_lig_sedd_amd import graph_lib, noise_lib, sampling
    g, n = graph_lib.Absorbing(25), noise_lib.LogLinearNoise()
    for cut in (dict(top_p=0.9), dict(top_k=3), dict(min_p=0.1), dict(temperature=0.5), dict(top_p=torch.tensor([0.9]))):
        with pytest.raises(ValueError, match="denois"):
            sampling.get_pc_sampler(g, n, (1, 4), "none", 2, denoise=False, **cut)
        assert callable(sampling.get_pc_sampler(g, n, (1, 4), "none", 2, **cut))
        assert callable(sampling.get_pc_sampler(g, n, (1, 4), "ancestral", 2, denoise=False, **cut))
    assert callable(sampling.get_pc_sampler(g, n, (1, 4), "none", 2, denoise=False))
    ns = types.SimpleNamespace
    with pytest.raises(ValueError, match="denois"):
        sampling.get_sampling_fn(ns(sampling=ns(predictor="none", steps=2, noise_removal=False, top_k=2)), g, n, (1, 4), 1e-5, "cpu")


class _Recorder:
    """stands in for the graph: keeps the move probabilities of the update"""

    def ancestral_step(self, log_score, x, move=None, u=None, **kw):
        self.move = move
        return x


class _Zeros(torch.nn.Module):
    def forward(self, x, sigma):
        return torch.zeros(*x.shape, 26)


@pytest.mark.parametrize("sigma_max", [1.0, 20.0, 79.0, 85.0, 88.0, 90.0, 200.0, 1e6])
def test_move_probability_of_the_ancestral_update(sigma_max):
    """(m(t) - m(t - dt)) / m(t), m = 1 - e^-sigma, in 64 bits from the fp32 sigmas, also where e^sigma leaves the range of fp32.
    Relative: sigma - sigma' is rounded, (1 + sigma) 2^-24 of its expm1; two expm1 of a step (2^-23) each and the division, 2^-24.
    Where sigma is above 80 it may be taken for 80: e^-80 absolute."""
    from protein_lig_sedd_amd import noise_lib, sampling
    noise, graph = noise_lib.GeometricNoise(1e-3, sigma_max), _Recorder()
    pred = sampling.AncestralPredictor(graph, noise)
    model = _Zeros()
    t = torch.tensor([1.0, 0.97, 0.9, 0.6, 0.3, 0.1])[:, None]
    for dt in (0.01, 0.1):
        pred.update_fn(score_model=model, x=torch.full((6, 4), 25), t=t, step_size=dt)
        s1, s0 = noise(t)[0].double().reshape(-1), noise(t - dt)[0].double().reshape(-1)
        want = torch.exp(-s0) * torch.expm1(-(s1 - s0)) / torch.expm1(-s1)
        err = (graph.move.double() - want).abs()
        assert graph.move.shape == (6,) and bool((err <= (2.0 ** -21 + 2.0 ** -24 * s1.clamp(max=80.0)) * want + 2e-35).all()), (dt, graph.move, want)
        keep = (torch.expm1(noise(t)[0] - noise(t - dt)[0]) / torch.expm1(noise(t)[0])).reshape(-1)
        low = s1 <= 80
        assert torch.equal(graph.move[low], keep[low])
