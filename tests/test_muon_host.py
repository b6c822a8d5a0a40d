"""Argument checks of the orthogonalised updates on the CPU: nothing is launched."""
import ctypes

import pytest
import torch

BUF = 4096  # any non-NULL address: refused before it is looked at


def coef(*v):
    return (ctypes.c_float * len(v))(*v)


def test_cpu_tensors_are_refused():
    from phoneme_contrast_amd.optim import FusedMuon, muon_step, orthogonalize
    x = torch.randn(4, 5)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        orthogonalize(x)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        muon_step([x], [x], [x], lr=0.1)
    p = torch.nn.Parameter(x)
    p.grad = torch.ones_like(x)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        FusedMuon([p]).step()


def test_orthogonalize_refuses_before_any_launch():
    from phoneme_contrast_amd import _lib
    lib = _lib.lib()

    def call(dt=0, batch=1, rows=8, cols=8, x=BUF, out=BUF, steps=1, c=coef(3.0, -4.0, 2.0), eps=1e-7, ws=BUF, nws=1 << 30):
        return lib.pcx_orthogonalize(dt, batch, rows, cols, x, 64, 8, 1, out, steps, c, eps, ws, nws, None)
    for rc in (call(dt=3), call(batch=-1), call(rows=0), call(cols=0), call(rows=1 << 21), call(rows=20000, cols=20000),
               call(x=None), call(out=None), call(steps=0), call(steps=65), call(c=None), call(c=coef(float("nan"), 0, 0)),
               call(c=coef(0, float("inf"), 0)), call(c=coef(9.0, 0, 0)), call(eps=0.0), call(eps=float("nan")), call(eps=-1.0)):
        assert rc == _lib.PCX_EINVAL and _lib.last_error()
    assert call(ws=None) == _lib.PCX_EWORKSPACE and call(nws=64) == _lib.PCX_EWORKSPACE
    assert call(batch=0) == _lib.PCX_OK
    # growing steps: the bound follows the iteration
    assert call(steps=3, c=coef(*(3.0, 0, 0) * 3)) == _lib.PCX_EINVAL
    assert lib.pcx_orthogonalize_workspace_bytes(1, 0, 4) == 0 and lib.pcx_orthogonalize_workspace_bytes(0, 4, 4) == 0
    assert lib.pcx_orthogonalize_workspace_bytes(3, 400, 300) > lib.pcx_orthogonalize_workspace_bytes(1, 400, 300) > 0
    assert lib.pcx_orthogonalize_workspace_bytes(3, 100, 40) > 0


def test_muon_step_refuses_before_any_launch():
    from phoneme_contrast_amd import _lib
    lib = _lib.lib()
    c = coef(3.0, -4.0, 2.0)

    def call(mats, n=None, lr=0.1, mu=0.9, steps=1, cf=c, eps=1e-7, ws=BUF, nws=1 << 30):
        arr = (_lib.MuonMatrix * max(1, len(mats)))(*mats)
        return lib.pcx_muon_step(arr, len(mats) if n is None else n, lr, mu, 1, 0.0, 1.0, steps, cf, eps, ws, nws, None)
    ok = (BUF, BUF, BUF, 8, 9, 1.0)
    for rc in (call([ok], n=-1), call([ok], mu=1.0), call([ok], mu=-0.1), call([ok], mu=float("nan")), call([ok], steps=0),
               call([ok], eps=0.0), call([(BUF, BUF, BUF, 0, 9, 1.0)]), call([ok] * 30 + [(None, BUF, BUF, 8, 9, 1.0)]),
               call([(BUF, None, BUF, 8, 9, 1.0)]), call([(BUF, BUF, None, 8, 9, 1.0)]), call([ok], cf=coef(50.0, 0, 0)),
               lib.pcx_muon_step(None, 2, 0.1, 0.9, 1, 0.0, 1.0, 1, c, 1e-7, BUF, 1 << 30, None)):
        assert rc == _lib.PCX_EINVAL and _lib.last_error()
    assert call([ok], ws=None) == _lib.PCX_EWORKSPACE and call([ok], nws=100) == _lib.PCX_EWORKSPACE
    assert call([]) == _lib.PCX_OK
    arr = (_lib.MuonMatrix * 2)(ok, (BUF, BUF, BUF, -3, 9, 1.0))
    assert lib.pcx_muon_workspace_bytes(arr, 2) == 0 and lib.pcx_muon_workspace_bytes(arr, 1) > 0
    assert lib.pcx_muon_workspace_bytes(None, 1) == 0


def test_adam_segments_refuses_before_any_launch():
    from phoneme_contrast_amd import _lib
    lib = _lib.lib()

    def call(segs, p=BUF, step=1):
        arr = (_lib.Segment * max(1, len(segs)))(*segs)
        return lib.pcx_adam_segments(p, BUF, BUF, BUF, arr, len(segs), step, 0.1, 0.9, 0.999, 1e-8, 0.0, 1.0, None)
    for rc in (call([(0, 0, 4)], p=None), call([(0, 0, 4)], step=0), call([(-1, 0, 4)]), call([(0, -2, 4)]), call([(0, 0, -4)]),
               call([(0, 0, 1 << 40)])):
        assert rc == _lib.PCX_EINVAL
    assert call([]) == _lib.PCX_OK and call([(5, 5, 0)]) == _lib.PCX_OK


def test_which_parameters_are_matrices():
    from phoneme_contrast_amd.optim import _is_matrix, _matrix_shape, _update_scale
    assert _matrix_shape(torch.empty(64, 32, 3, 3)) == (64, 288)
    assert _is_matrix(torch.empty(32, 1, 3, 3)) and _is_matrix(torch.empty(2, 2))
    assert not any(_is_matrix(torch.empty(s)) for s in ((5,), (1, 512, 1, 1), (7, 1), (0, 4), ()))
    assert _update_scale("rms", 64, 576) == pytest.approx(0.2 * 24) and _update_scale("spectral", 64, 16) == 2.0
    assert _update_scale("spectral", 16, 64) == 1.0 and _update_scale(None, 3, 4) == 1.0


def test_workspaces_off_their_boundary_are_refused():
    from phoneme_contrast_amd import _lib
    lib = _lib.lib()
    c = coef(3.0, -4.0, 2.0)
    arr = (_lib.MuonMatrix * 1)((BUF, BUF, BUF, 8, 9, 1.0))
    for ws in (BUF + 128, BUF + 1):
        assert lib.pcx_orthogonalize(0, 1, 8, 8, BUF, 64, 8, 1, BUF, 1, c, 1e-7, ws, 1 << 30, None) == _lib.PCX_EWORKSPACE
        assert lib.pcx_muon_step(arr, 1, 0.1, 0.9, 1, 0.0, 1.0, 1, c, 1e-7, ws, 1 << 30, None) == _lib.PCX_EWORKSPACE
        assert "boundary" in _lib.last_error()


def test_the_state_of_another_muon_is_refused():
    """torch.optim.Muon's groups have ns_steps, but neither the fields nor the state of FusedMuon's."""
    from phoneme_contrast_amd.optim import FusedAdam, FusedMuon
    if not hasattr(torch.optim, "Muon"):
        pytest.skip("this torch has none")

    def weight():
        return [torch.nn.Parameter(torch.ones(4, 5))]
    other = torch.optim.Muon(weight()).state_dict()
    for opt in (FusedMuon(weight()), FusedAdam(weight())):
        before = dict(opt.param_groups[0])
        with pytest.raises(ValueError, match="another optimizer"):
            opt.load_state_dict(other)
        assert opt.param_groups[0] == before
        opt.load_state_dict(opt.state_dict())
