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


def test_launched_on_the_device_of_its_tensor(monkeypatch):
    """between entering and leaving the tensor's device, so that the reader of the noise, which goes there too, comes behind"""
    from protein_lig_sedd_amd import ops
    log = []

    class On:
        def __init__(self, t):
            log.append(("of", t))

        def __enter__(self):
            log.append("enter")

        def __exit__(self, *exc):
            log.append("leave")

    class Lib:
        @staticmethod
        def sedd_philox_uniform(*args):
            log.append("launch")
            return 0

    monkeypatch.setattr(ops, "_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_on_device", On)
    monkeypatch.setattr(ops, "_stream", lambda: log.append("stream"))
    monkeypatch.setattr(ops, "lib", lambda: Lib)
    u = ops.philox_uniform(ops.PhiloxNoise(5, 1), (2, 3, 26), "cpu")
    assert log[0][1] is u and log[1:] == ["enter", "stream", "launch", "leave"]
