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
