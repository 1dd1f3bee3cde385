"""The clip coefficient: max_norm / (norm + 1e-6) in 64 bits, rounded once to fp32, for any max_norm that a Python number holds.
n^2 ones have the norm n to the last bit, so what is left in them is the coefficient itself."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
LIMITS = (0.1, 0.3, 1e-3, 0.7, 1.1, 0.375)


@pytest.mark.parametrize("max_norm", LIMITS)
def test_coefficient_is_rounded_once(max_norm):
    from protein_lig_sedd_amd import ops
    for n in range(2, 60):
        g = torch.ones(n * n, device=DEV)
        assert float(ops.clip_grad_norm_([g[:n], g[n:]], max_norm)) == n
        coef = (torch.tensor(max_norm, dtype=torch.float64) / (n + 1e-6)).float()
        assert torch.equal(g.cpu(), coef.expand(n * n)), (n, max_norm)


@pytest.mark.parametrize("max_norm", LIMITS)
def test_loop_over_the_tensors(max_norm):
    """round_coef: bit for bit what a loop of grad.mul_(coef) gives, for both types"""
    from protein_lig_sedd_amd import ops
    for n in range(2, 60):
        gen = torch.Generator().manual_seed(n)
        # (values +-1: the norm is exact, and a product is the coefficient as the type holds it)
        grads = [(1 - 2 * torch.randint(0, 2, (size,), generator=gen)).to(t).to(DEV)
                 for size, t in ((n, torch.float32), (n * n - 2 * n, torch.bfloat16), (n, torch.bfloat16))]
        copy = [g.clone() for g in grads]
        norm = ops.clip_grad_norm_(grads, max_norm, round_coef=True)
        coef = (max_norm / (norm.double() + 1e-6)).clamp(max=1.0).float()
        for g, c in zip(grads, copy):
            assert torch.equal(g, c.mul_(coef)), (n, max_norm, g.dtype)
