"""ops.philox_uniform without a GPU: where it may write, and on which device's stream it launches."""
import pytest
import torch


def test_host_memory_is_refused():
    """the kernel would write through the host address of the tensor"""
    from protein_lig_sedd_amd import graph_lib, ops
    noise = ops.PhiloxNoise(5, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.philox_uniform(noise, (2, 3, 26), "cpu")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        graph_lib.Absorbing(25).ancestral_step(torch.zeros(2, 3, 26), torch.full((2, 3), 25), 0.5, u=noise)
