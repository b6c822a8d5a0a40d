"""Argument checks of the layer norm on the CPU: nothing is launched."""
import pytest
import torch


def test_cpu_tensors_are_refused():
    from phoneme_contrast_amd.layers import LayerNorm, layer_norm
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        layer_norm(torch.randn(2, 8), 8)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        LayerNorm(8)(torch.randn(2, 8))


def test_c_entry_points_refuse_before_any_launch():
    from phoneme_contrast_amd import _lib
    lib = _lib.lib()
    buf = 4096  # any non-NULL address: refused before it is looked at

    def fwd(dt=0, wdt=0, rows=4, D=8, x=buf, xs=8, eps=1e-5, y=buf):
        return lib.pcx_layernorm_forward(dt, wdt, rows, D, x, xs, None, None, eps, y, None, None)

    def bwd(dt=0, wdt=0, rows=4000, D=8, xs=8, dys=8, stats=buf, dx=buf, dw=buf, ws=buf, nws=1 << 20, eps=1e-5):
        return lib.pcx_layernorm_backward(dt, wdt, rows, D, buf, xs, None, eps, stats, buf, dys, dx, dw, None, ws, nws, None)
    for rc in (fwd(dt=3), fwd(dt=-1), fwd(dt=0, wdt=1), fwd(dt=1, wdt=2), fwd(rows=-1), fwd(D=0), fwd(D=32769), fwd(x=None),
               fwd(y=None), fwd(xs=7), fwd(eps=0.0), fwd(eps=-1.0), fwd(eps=float("nan")), fwd(eps=float("inf")),
               bwd(dt=7), bwd(rows=0), bwd(xs=3), bwd(dys=7), bwd(stats=None), bwd(D=40000)):
        assert rc == _lib.PCX_EINVAL and _lib.last_error()
    assert bwd(ws=None) == _lib.PCX_EWORKSPACE
    assert bwd(nws=8) == _lib.PCX_EWORKSPACE and "needed" in _lib.last_error()
    assert fwd(rows=0) == _lib.PCX_OK          # nothing to do
    assert bwd(dx=None, dw=None) == _lib.PCX_OK
    assert lib.pcx_layernorm_workspace_bytes(0, 4096, 128) > 0
    assert lib.pcx_layernorm_workspace_bytes(0, 4096, 1 << 20) == 0 and lib.pcx_layernorm_workspace_bytes(9, 4, 8) == 0


def test_the_torch_operator_calls_the_library_that_is_loaded(tmp_path):
    """PCX_LIB_PATH names another build: no second copy of the library comes with the torch operators."""
    import os
    import shutil
    import subprocess
    import sys
    from phoneme_contrast_amd import _lib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    here = os.path.join(os.path.dirname(_lib.__file__), "libpcx.so")
    other = str(tmp_path / "other.so")
    shutil.copy(here, other)
    code = ("from phoneme_contrast_amd import _lib; _lib.torch_ops(); "
            "print(sorted({l.split()[-1] for l in open('/proc/self/maps') if '.so' in l and 'pcx' in l or 'other.so' in l}))")
    out = subprocess.run([sys.executable, "-c", code], cwd=root, env={**os.environ, "PCX_LIB_PATH": other},
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    mapped = out.stdout
    assert other in mapped and "libpcx_torch.so" in mapped and "libpcx.so" not in mapped, mapped


def test_the_torch_operator_alone_says_what_it_lacks():
    import subprocess
    import sys
    from phoneme_contrast_amd import _lib
    code = (f"import torch; torch.ops.load_library({_lib.TORCH_OPS_PATH!r})\n"
            "try: torch.ops.pcx.layer_norm(torch.ones(2, 8), (8,), None, None, 1e-5)\n"
            "except RuntimeError as e: print(e)")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "has not loaded libpcx.so" in out.stdout, out.stdout + out.stderr


def test_make_without_torch_and_with_another_one(tmp_path):
    """The C library needs no torch; libpcx_torch.so is built anew when torch's version is another."""
    import glob
    import os
    import shutil
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if not shutil.which("make"):
        pytest.skip("no make")

    def plan(*args):
        out = subprocess.run(["make", "-n", *args], cwd=root, capture_output=True, text=True, timeout=120)
        assert out.returncode == 0, out.stderr
        return out.stdout
    none = plan("-B", "PYTHON=false", f"BUILD={tmp_path}/obj")
    assert "adam.hip" in none and "libpcx.so" in none and "torch_ops.cpp" not in none
    assert "torch_ops.cpp" in plan("-B", f"BUILD={tmp_path}/obj")
    lib = "phoneme_contrast_amd/libpcx_torch.so"
    if not (os.path.exists(os.path.join(root, lib)) and glob.glob(os.path.join(root, "build", "torch-*"))):
        pytest.skip("built elsewhere")
    assert "torch_ops.cpp" not in plan(lib)
    assert "torch_ops.cpp" in plan("TORCH=1.0 /somewhere", lib)


def test_a_config_of_the_older_layout_is_read_to_its_end_alone():
    """pcx_net_config has no size or version: what lies behind the ten fields a caller may have been built with is not read."""
    import ctypes
    from phoneme_contrast_amd import _lib
    lib = _lib.lib()
    assert ctypes.sizeof(_lib.NetConfig) == 40

    def plan(behind, norm=None):
        raw = (ctypes.c_int * 12)(0, 1, 128, 1, 64, 128, 256, 512, 1, 0, behind, behind)
        cfg = ctypes.cast(raw, ctypes.POINTER(_lib.NetConfig))
        p = lib.pcx_net_create(cfg, 4, 40, 100) if norm is None else lib.pcx_net_create_norm(cfg, norm, 4, 40, 100)
        assert p, _lib.last_error()
        nbn = ctypes.c_int()
        assert lib.pcx_net_info(p, None, ctypes.byref(nbn), None, None) == _lib.PCX_OK
        ws = lib.pcx_net_workspace_bytes(p)
        lib.pcx_net_destroy(p)
        return nbn.value, ws
    first = plan(0)
    assert first[0] == 7 and plan(1) == first and plan(-77) == first and plan(5, norm=0) == first
    assert plan(0, norm=1)[0] == 6
    cfg = _lib.NetConfig(0, 1, 128, 1, (64, 128, 256, 512), 1, 0)
    for norm in (-1, 2):
        assert not lib.pcx_net_create_norm(ctypes.byref(cfg), norm, 4, 40, 100) and "proj_norm" in _lib.last_error()


@pytest.mark.parametrize("kind", ["phoneme_cnn", "phoneme_cnn_deep"])
def test_a_model_saved_before_the_choice_of_norm(kind):
    """A whole module unpickled from an older file has no projection_norm of its own."""
    from phoneme_contrast_amd.models import model_registry
    m = model_registry.create(kind, {})
    del m.__dict__["projection_norm"]
    assert m.projection_norm == "batch" and m._plan(4, 40, 100).nbn == len(m._bn_modules())


@pytest.mark.parametrize("kind,F,T,fits", [(0, 7, 6, False), (0, 7, 8, True), (0, 40, 4, True), (1, 16, 16, False), (1, 16, 17, True),
                                           (1, 1, 9, False)])
def test_one_sample_whose_last_plane_is_one_pixel(kind, F, T, fits):
    """With the layer norm a training batch of one is allowed, where every BatchNorm2d still sees two values."""
    import ctypes
    from phoneme_contrast_amd import _lib
    lib = _lib.lib()
    last = (F // 4) * (T // 4) if kind == 0 else ((F + 15) // 16) * ((T + 15) // 16)
    assert (last > 1) is fits
    cfg = _lib.NetConfig(kind, 1, 128, 1, (16, 32, 64, 128), 1, 0)
    p = lib.pcx_net_create_norm(ctypes.byref(cfg), 1, 1, F, T)
    assert p, _lib.last_error()
    if not fits:  # (refused before anything is launched)
        buf = (ctypes.c_void_p * 64)()
        rc = lib.pcx_net_forward(p, buf, buf, buf, 4096, None, 1, 4096, 4096, lib.pcx_net_workspace_bytes(p), None)
        assert rc == _lib.PCX_EINVAL and "more than 1 value" in _lib.last_error()
    lib.pcx_net_destroy(p)
