"""Where post_norm_residual_bwd may write the gradients of gate, shift and scale."""
import pytest
import torch

from test_gpu_post_norm import make, run_bwd, run_fwd

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("which", ["dgate", "dshift", "dscale"])
def test_rows_that_overlap_are_refused(which):
    """the gradient of a modulation that all batch elements share is a row each, summed by the caller: blocks write rows at once"""
    from protein_lig_sedd_amd import ops
    B, L, D = 3, 5, 64
    s = make(B, L, D, torch.float32)
    x1, _, stats = run_fwd(s, 1.0, True)
    for bad in (torch.zeros(1, D, device=DEV).expand(B, D), torch.zeros(B * D, device=DEV).as_strided((B, D), (D // 2, 1))):
        out = {n: bad if n == which else torch.zeros(B, D, device=DEV) for n in ("dgate", "dshift", "dscale")}
        with pytest.raises(ValueError, match="rows"):
            ops.post_norm_residual_bwd(s["dx1"], s["a"], s["post_w"], s["gate"], stats, out["dgate"], None,
                                       norm=(s["dh"], x1, s["w"], s["scale"], None, out["dshift"], out["dscale"]))


def test_a_shared_modulation():
    """gate, shift and scale of one row for all batch elements: the gradients are those of copies of it"""
    B, L, D = 3, 5, 64
    s = make(B, L, D, torch.float32)
    one = {n: s[n][:1].contiguous() for n in ("gate", "shift", "scale")}
    shared, copied = ({**s, **{n: t.expand(B, D) if e else t.repeat(B, 1) for n, t in one.items()}} for e in (True, False))
    out = []
    for q in (shared, copied):
        x1, h, stats = run_fwd(q, 0.9, True)
        out.append((x1, h, run_bwd(q, 0.9, True, x1, stats)))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    for k, t in out[0][2].items():
        assert torch.equal(t, out[1][2][k]), k


def test_one_batch_element_of_any_row_stride():
    from protein_lig_sedd_amd import ops
    L, D = 5, 64
    s = make(1, L, D, torch.float32)
    x1, _, stats = run_fwd(s, 1.0, False)
    want = run_bwd(s, 1.0, False, x1, stats)["dgate"]
    dgate = torch.zeros(D, device=DEV).as_strided((1, D), (0, 1))
    ops.post_norm_residual_bwd(s["dx1"], s["a"], s["post_w"], s["gate"], stats, dgate, None)
    assert torch.equal(dgate, want)


def test_modulation_of_one_batch_element_and_any_row_stride():
    """one row has no next one, so its stride means nothing"""
    L, D = 5, 64
    s = make(1, L, D, torch.float32)
    odd = {n: torch.cat([s[n], torch.zeros(1, 1, device=DEV)], 1)[:, :D] for n in ("gate", "shift", "scale")}
    assert all(t.stride(0) == D + 1 for t in odd.values())
    x1, h, stats = run_fwd(s, 1.0, True)
    y1, g, other = run_fwd({**s, **odd}, 1.0, True)
    assert torch.equal(x1, y1) and torch.equal(h, g)
    want, got = run_bwd(s, 1.0, True, x1, stats), run_bwd({**s, **odd}, 1.0, True, y1, other)
    assert all(torch.equal(want[k], got[k]) for k in want)
