"""Argument checks of the truncated sampling, post-norm residual and many-tensor clipping entry points that need no GPU: bad
arguments are refused before anything is launched, empty problems need no pointers."""
import ctypes
import math

import pytest
import torch


def _lib():
    from protein_lig_sedd_amd import _lib
    return _lib.lib()


@pytest.fixture()
def ptr():
    buf = ctypes.create_string_buffer(128)
    yield (ctypes.addressof(buf) + 63) // 64 * 64
    del buf


def _sample(L, p, dtype=0, ld=26, ldu=26, T=1.0, k=0, P=1.0, m=0.0, x=None, move=None, M=4, Ln=2, V=26):
    return L.sedd_sample_truncated(p, dtype, ld, p, ldu, None, None, None, None, T, k, P, m, x, 25, move, p, M, Ln, V, None)


def test_sample_truncated_refusals(ptr):
    L = _lib()
    for kw in (dict(dtype=7), dict(M=5), dict(Ln=0), dict(V=0), dict(V=2 ** 30 + 1, ld=2 ** 30 + 1, ldu=2 ** 30 + 1), dict(M=-1), dict(ld=25), dict(ldu=25), dict(T=-1.0),
               dict(T=math.nan), dict(T=math.inf), dict(P=1.5), dict(P=math.nan), dict(m=-0.5), dict(k=-2), dict(move=ptr),
               dict(x=ptr, move=ptr), dict(x=ptr)):  # (the last two: no column for the move numbers; out is x)
        assert _sample(L, ptr, **kw) == -1, kw
        assert b"sample_truncated" in L.sedd_last_error()
    assert _sample(L, None) == -1 and b"null" in L.sedd_last_error()
    assert _sample(L, None, M=0) == 0
    # more rows than one launch has threads for
    assert _sample(L, ptr, M=1 << 26, Ln=1 << 26, V=65, ld=65, ldu=65) == -1 and b"rows" in L.sedd_last_error()
    assert _sample(L, ptr, M=1 << 32, Ln=1 << 32) == -1 and b"rows" in L.sedd_last_error()


def _fwd(L, p, a_dtype=0, mod_dtype=0, stride=64, p_drop=0.0, w=None, nxt=None, M=4, Ln=2, D=64):
    return L.sedd_post_norm_residual_fwd(p, p, a_dtype, p, p, nxt, nxt, mod_dtype, stride, 1.0, 1.0, 0, p_drop, w, p, nxt, p, p,
                                         nxt, nxt, M, Ln, D, None)


def _bwd(L, p, dh=None, a_dtype=0, mod_dtype=0, stride=64, p_drop=0.0, M=4, Ln=2, D=64, dx1=0, x1=None, ws=0):
    return L.sedd_post_norm_residual_bwd(p if dx1 == 0 else dx1, dh, x1, x1, x1, x1, x1, p, a_dtype, p, p, mod_dtype, stride, p, p,
                                         1.0, 1.0, 0, p_drop, p, p, p, 64, None, None, 64, None, None, None,
                                         p if ws == 0 else ws, M, Ln, D, None)


def test_post_norm_refusals(ptr):
    L = _lib()
    for fn in (_fwd, _bwd):
        for kw, rc in ((dict(a_dtype=3), -1), (dict(mod_dtype=-1), -1), (dict(p_drop=1.0), -1), (dict(p_drop=-0.1), -1),
                       (dict(M=5), -1), (dict(Ln=0), -1), (dict(D=0), -2), (dict(D=62), -2), (dict(D=2052), -2),
                       (dict(stride=66), -2)):
            assert fn(L, ptr, **kw) == rc, (fn, kw)
            assert b"post_norm_residual" in L.sedd_last_error()
        assert fn(L, None) == -1 and fn(L, ptr + 4) == -1  # null, misaligned
        assert fn(L, ptr, M=1 << 26) == -1 and b"rows" in L.sedd_last_error()
        assert fn(L, None, M=0) == 0
    assert _fwd(L, ptr, w=ptr) == -1 and _bwd(L, ptr, dh=ptr) == -1  # a next norm without its tensors
    assert _bwd(L, ptr, dx1=None) == -1                              # neither gradient
    assert _bwd(L, ptr, ws=None) == -1
    assert L.sedd_post_norm_chunks(0, 4, 64) == 0 and L.sedd_post_norm_chunks(4, 0, 64) == 0
    assert L.sedd_post_norm_chunks(64 * 1024, 1024, 768) == 64 * 32  # parts of a batch element
    assert L.sedd_post_norm_chunks(64 * 1024, 4, 768) == 64 * 32     # several to a chunk


def test_multi_tensor_refusals(ptr):
    L = _lib()

    def norm(ptrs, sizes, kinds, max_norm=1.0, ws=ptr, nws=5000, out=ptr, n=None):
        k = len(ptrs)
        return L.sedd_multi_norm_clip((ctypes.c_void_p * k)(*ptrs), (ctypes.c_int64 * k)(*sizes), (ctypes.c_int32 * k)(*kinds),
                                      k if n is None else n, max_norm, ws, nws, out, None)

    for args, kw in ((([None], [4], [0]), {}), (([ptr], [-1], [0]), {}), (([ptr], [4], [2]), {}), (([ptr + 2], [4], [0]), {}),
                     (([ptr + 1], [4], [1]), {}), (([ptr], [4], [0]), dict(max_norm=-1.0)),
                     (([ptr], [4], [0]), dict(max_norm=math.nan)), (([ptr], [4], [0]), dict(nws=4096)),
                     (([ptr], [4], [0]), dict(ws=None)), (([ptr], [4], [0]), dict(out=None)), (([ptr], [4], [0]), dict(n=-1))):
        assert norm(*args, **kw) == -1, (args, kw)
        assert b"multi_norm_clip" in L.sedd_last_error()
    one = ((ctypes.c_void_p * 1)(ptr), (ctypes.c_int64 * 1)(4), (ctypes.c_int32 * 1)(0), 1)
    assert L.sedd_multi_scale(*one, None, 0, None) == -1
    assert L.sedd_multi_scale(None, None, None, 0, ptr, 0, None) == 0  # nothing to scale


def test_host_refusals():
    from protein_lig_sedd_amd import graph_lib, noise_lib, ops, sampling
    from protein_lig_sedd_amd.model.transformer import DDiTBlock
    t = torch.zeros(2, 3, 26)
    for call in (lambda: ops.sample_truncated(t, t), lambda: ops.clip_grad_norm_([torch.zeros(3)], 1.0),
                 lambda: ops.grad_norm([torch.zeros(3)]),
                 lambda: ops.post_norm_residual_fwd(t, t, torch.ones(26), torch.zeros(2, 26))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    assert float(ops.clip_grad_norm_([], 1.0)) == 0.0 and float(ops.grad_norm([])) == 0.0
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            ops.clip_grad_norm_([torch.zeros(3)], bad)
    with pytest.raises(ValueError):
        DDiTBlock(64, 2, 32, residual_scale=0.5)
    for dim in (62, 2052):
        with pytest.raises(ValueError):
            DDiTBlock(dim, 2, 32, post_norm=True)
    g, n = graph_lib.Absorbing(25), noise_lib.LogLinearNoise()
    with pytest.raises(ValueError, match="ancestral"):
        sampling.get_pc_sampler(g, n, (1, 4), "euler", 2, temperature=0.5)
    with pytest.raises(ValueError, match="absorbing"):
        sampling.get_pc_sampler(graph_lib.Uniform(25), n, (1, 4), "none", 2, top_k=3)
    assert sampling.get_predictor("ancestral") is sampling.AncestralPredictor


def test_block_parameters_and_names():
    from protein_lig_sedd_amd.model.transformer import DDiTBlock, _SEDD
    plain, post = DDiTBlock(64, 2, 32), DDiTBlock(64, 2, 32, post_norm=True, residual_scale=0.9)
    extra = set(dict(post.named_parameters())) - set(dict(plain.named_parameters()))
    assert extra == {"post_norm1.weight", "post_norm2.weight"}
    import types
    ns = types.SimpleNamespace
    m = dict(hidden_size=64, cond_dim=32, n_heads=2, n_blocks=2, dropout=0.0, scale_by_sigma=False)
    a = _SEDD(ns(tokens=25, graph=ns(type="absorb"), model=ns(**m)))
    b = _SEDD(ns(tokens=25, graph=ns(type="absorb"), model=ns(**m, post_norm=True, residual_scale=0.5)))
    assert not any("post_norm" in k for k in a.state_dict()) and a.blocks[0].residual_scale == 1.0
    assert "blocks.1.post_norm2.weight" in b.state_dict() and b.blocks[1].residual_scale == 0.5


def test_the_dual_track_model_refuses_what_it_has_not():
    from protein_lig_sedd_amd.model.transformers_protlig_cross import DualTrackDiffusionTransformer
    for extra in (dict(post_norm=True), dict(residual_scale=0.9)):
        with pytest.raises(ValueError, match="dual-track"):
            DualTrackDiffusionTransformer(dict(model=dict(hidden_size=64, cond_dim=32, n_heads=2, n_blocks=1, dropout=0.0, **extra)), 26, 26)
