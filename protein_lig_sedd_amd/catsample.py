"""Drop-in for protlig_dd/utils/catsample.py: Gumbel-max categorical sampling on the HIP kernel.

`u=` (new, optional) supplies the uniform noise so that identical noise gives bit-identical indices."""
import torch

from . import ops


def sample_categorical(categorical_probs, method="hard", u=None):
    """catsample.py:10-15"""
    if method == "hard":
        if u is None:
            u = torch.rand(categorical_probs.shape, dtype=torch.float32, device=categorical_probs.device)
        return ops.gumbel_argmax(categorical_probs, u)
    raise ValueError(f"Method {method} for sampling categorical variables is not valid.")


def sample_logits(logits, u=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens from unnormalised log-weights [..., V], truncated by temperature, top-k, top-p and min-p: what
    sample_categorical draws from softmax(logits / temperature) restricted to the kept entries and with the same form of
    noise, u [..., V] uniform (None: torch.rand).  Parameters are numbers, or tensors with one value per leading entry
    (ops.sample_truncated)."""
    if u is None:
        u = torch.rand(logits.shape, dtype=torch.float32, device=logits.device)
    return ops.sample_truncated(logits, u, temperature, top_k, top_p, min_p)
