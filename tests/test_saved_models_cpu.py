"""Whole models that were saved before a block had post_norm and residual_scale."""
import io

import torch


def test_a_block_saved_without_the_new_attributes():
    from protein_lig_sedd_amd.model import layers
    from protein_lig_sedd_amd.model.transformer import _SEDD
    m = dict(hidden_size=64, cond_dim=32, n_heads=2, n_blocks=2, dropout=0.0, scale_by_sigma=False)
    model = _SEDD(dict(tokens=25, graph=dict(type="absorb"), model=m))
    for blk in model.blocks:  # (what such a file holds)
        for name in ("residual_scale", "param_names"):
            blk.__dict__.pop(name, None)
    buf = io.BytesIO()
    torch.save(model, buf)
    buf.seek(0)
    for blk in torch.load(buf, weights_only=False).blocks:  # (written above)
        assert blk.param_names == layers.BLOCK_PARAMS and blk.residual_scale == 1.0
