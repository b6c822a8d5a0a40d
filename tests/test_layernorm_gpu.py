"""Layer norm kernels against the formulas in float64 (phoneme_contrast_amd.layers, csrc/layernorm.hip).

Error bounds (u = 2^-24, h = half a step of the output's type, first order): a thread adds at most 32 values, then at
most 10 levels of partial sums follow, so a row sum of v is off by at most 45 u sum|v|.  With A = mean|x| and
S = |xhat| + rstd A, xhat is off by at most 64 u S (45 u of the mean through rstd A; half of 47 u of the variance, the
root and three products through |xhat|).  Hence
    |d y|  <= 64 u |w| S + 2 u (|w xhat| + |b|) + h |y|
    |d dx| <= 128 u rstd (|g| + mean|g| + 2 S mean(|g| S)) + h |dx|      (c1, c2 each a row sum; S >= |xhat|)
    |d dw| <= (128 + n) u sum|dy| S + h |dw|,  |d db| <= (64 + n) u sum|dy| + h |db|   (n additions in a thread)
Rows of up to 32 values are computed in float64: h of the result alone, and its float64 error 2^-40 of the terms."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(t):
    return torch.finfo(t).eps / 2


def reference(x, w, b, dy, eps):
    """float64 formulas -> y, dx, dw, db and the bounds above without the output's rounding."""
    D = x.shape[-1]
    x, dy = x.double().reshape(-1, D), dy.double().reshape(-1, D)
    w = torch.ones(D, dtype=torch.float64) if w is None else w.double().reshape(D)
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.double().reshape(D)
    mean = x.mean(1, keepdim=True)
    u = x - mean
    rstd = 1 / torch.sqrt((u * u).mean(1, keepdim=True) + eps)
    xh = u * rstd
    y = xh * w + b
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    dw, db = (dy * xh).sum(0), dy.sum(0)
    k = 1.0 if D > 32 else 2.0 ** -16  # (float64 rows)
    S = xh.abs() + rstd * x.abs().mean(1, keepdim=True)
    n = 64 + x.shape[0] / 64
    tol = (k * U * (64 * w.abs() * S + 2 * ((w * xh).abs() + b.abs())),
           k * 128 * U * rstd * (g.abs() + g.abs().mean(1, keepdim=True) + 2 * S * (g.abs() * S).mean(1, keepdim=True)),
           (128 * k + n) * U * (dy.abs() * S).sum(0) if D > 32 else (k * 128 + 2) * U * (dy.abs() * S).sum(0),
           (64 * k + n) * U * dy.abs().sum(0) if D > 32 else (k * 64 + 2) * U * dy.abs().sum(0))
    return (y, dx, dw, db), tol


def close(got, ref, tol, what):
    got = got.detach().cpu()
    limit = tol + half(got.dtype) * (1 + 2 ** -6) * ref.abs() + torch.finfo(got.dtype).tiny
    off = (got.double().reshape(ref.shape) - ref).abs()
    assert torch.isfinite(got).all(), what
    worst = (off - limit).max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: over its bound by {worst:.3e} at {int((off - limit).argmax())}"


def inputs(rows, D, t, wt, seed, shift=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, D, generator=gen) * torch.exp(0.5 * torch.randn(D, generator=gen)) + shift).to(t)
    w = (1 + 0.1 * torch.randn(D, generator=gen)).to(wt)
    b = (0.1 * torch.randn(D, generator=gen)).to(wt)
    dy = (0.01 * torch.randn(rows, D, generator=gen)).to(t)
    return x, w, b, dy


def check(x, w, b, dy, eps=1e-5):
    from phoneme_contrast_amd.layers import layer_norm
    xd = x.cuda().requires_grad_(True)
    wd = w.cuda().requires_grad_(True) if w is not None else None
    bd = b.cuda().requires_grad_(True) if b is not None else None
    y = layer_norm(xd, x.shape[-1], wd, bd, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    leaves = [t for t in (xd, wd, bd) if t is not None]
    grads = dict(zip([n for n, t in (("dx", xd), ("dw", wd), ("db", bd)) if t is not None],
                     torch.autograd.grad(y, leaves, dy.cuda())))
    (ry, rdx, rdw, rdb), tol = reference(x, w, b, dy, eps)
    close(y, ry, tol[0], "y")
    close(grads["dx"], rdx, tol[1], "dx")
    if w is not None:
        assert grads["dw"].dtype == w.dtype
        close(grads["dw"], rdw, tol[2], "dw")
    if b is not None:
        close(grads["db"], rdb, tol[3], "db")
    with torch.no_grad():
        assert torch.equal(layer_norm(x.cuda(), x.shape[-1], wd, bd, eps), y.detach())


DIMS = [1, 2, 3, 31, 32, 33, 40, 64, 127, 128, 257, 504, 512, 520, 1000, 1024, 1025, 1537, 2048, 2056, 4096, 4104, 8191,
        8192, 8200, 16384, 16392, 20001, 32768]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("D", DIMS)
def test_every_row_width(D, t):
    rows = 5 if D > 4096 else 67
    check(*inputs(rows, D, TYPES[t], TYPES[t], D))


@pytest.mark.parametrize("rows,D", [(1, 128), (2, 5), (24, 128), (4096, 128), (4097, 33), (9001, 7), (1003, 1537),
                                    (700, 4096), (3000, 8192)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_row_counts(rows, D, t):
    check(*inputs(rows, D, TYPES[t], TYPES[t], rows))


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("D", [20, 129, 256, 4096, 5001])
def test_float32_weights_for_narrower_rows(D, t):
    check(*inputs(33, D, TYPES[t], torch.float32, 3))


@pytest.mark.parametrize("use_w,use_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("D", [16, 128, 1001, 4096])
@pytest.mark.parametrize("wt", ["f32", "bf16"])
def test_without_weight_or_bias(D, use_w, use_b, wt):
    x, w, b, dy = inputs(19, D, torch.bfloat16, TYPES[wt], 4)
    check(x, w if use_w else None, b if use_b else None, dy)


@pytest.mark.parametrize("D,shift", [(128, 1e4), (1000, -3e3), (4096, 1e3), (2, 1e4)])
def test_rows_far_from_zero(D, shift):
    check(*inputs(40, D, torch.float32, torch.float32, 5, shift))


@pytest.mark.parametrize("D", [1, 7, 128, 1025, 4096])
def test_constant_rows_give_the_bias(D):
    from phoneme_contrast_amd.layers import layer_norm
    x = torch.tensor([0.0, 1.0, -3.25, 1024.0]).view(4, 1).expand(4, D).contiguous().cuda()
    w, b = torch.full((D,), 2.0, device="cuda"), torch.linspace(-1, 1, D, device="cuda")
    y = layer_norm(x, D, w, b)
    # a constant row whose D-fold sum is exact has mean x exactly, else within 45 u |x|: |xhat| <= 45 u |x| / sqrt(eps)
    tol = 2 * 45 * U * 1024 / 1e-5 ** 0.5 if D == 1025 else 0.0
    assert (y - b).abs().max().item() <= tol


@pytest.mark.parametrize("D", [24, 128, 1000, 4096])
def test_strided_rows_and_gradients_that_are_not_contiguous(D):
    from phoneme_contrast_amd.layers import layer_norm
    gen = torch.Generator().manual_seed(6)
    big = torch.randn(6, 5, D + 24, generator=gen)
    w, b = torch.randn(D, generator=gen), torch.randn(D, generator=gen)
    views = {"padded": lambda t: t[..., 8:8 + D], "odd": lambda t: t[..., 3:3 + D], "last": lambda t: t[:, -1, :D],
             "transposed": lambda t: t[..., :D].transpose(0, 1), "columns": lambda t: t[0, :, :D].t().contiguous().t(),
             "expanded": lambda t: t[:, :1, :D].expand(6, 5, D), "broadcast_last": lambda t: t[..., :1].expand(6, 5, D)}
    for name, view in views.items():
        leaf = big.cuda().requires_grad_(True)
        x = view(leaf)
        xr = view(big)
        y = layer_norm(x, D, w.cuda(), b.cuda())
        dy = torch.randn(xr.shape, generator=gen)
        (ry, rdx, _, _), tol = reference(xr.reshape(-1, D), w, b, dy, 1e-5)
        close(y, ry, tol[0], name)
        (dx,) = torch.autograd.grad(y, x, dy.cuda(), retain_graph=True)
        close(dx, rdx, tol[1], name)
        # a sum's gradient has stride 0 everywhere
        (dx,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
        (_, rdx, _, _), tol = reference(xr.reshape(-1, D), w, b, torch.ones(xr.shape), 1e-5)
        close(dx, rdx, tol[1], name + " (sum)")
        dyt = torch.randn(*xr.shape[:-1], 2 * D, generator=gen)[..., ::2]
        (dx,) = torch.autograd.grad(y, x, dyt.cuda())
        (_, rdx, _, _), tol = reference(xr.reshape(-1, D), w, b, dyt, 1e-5)
        close(dx, rdx, tol[1], name + " (strided)")


def test_trailing_axes_empty_batches_and_the_module():
    from phoneme_contrast_amd.layers import LayerNorm, layer_norm
    gen = torch.Generator().manual_seed(7)
    x, dy = torch.randn(3, 4, 5, 8, generator=gen), torch.randn(3, 4, 5, 8, generator=gen)
    m, ref = LayerNorm((5, 8)).cuda(), torch.nn.LayerNorm((5, 8))
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.1 * torch.randn(p.shape, generator=gen).cuda())
    ref.load_state_dict(m.state_dict())
    assert list(m.state_dict()) == ["weight", "bias"]
    xd = x.cuda().requires_grad_(True)
    m(xd).backward(dy.cuda())
    w, b = ref.weight.detach().view(-1), ref.bias.detach().view(-1)
    (ry, rdx, rdw, rdb), tol = reference(x.view(-1, 40), w, b, dy.view(-1, 40), 1e-5)
    close(m(xd), ry, tol[0], "y")
    close(xd.grad, rdx, tol[1], "dx")
    assert m.weight.grad.shape == (5, 8)
    close(m.weight.grad.view(-1), rdw, tol[2], "dw")
    close(m.bias.grad.view(-1), rdb, tol[3], "db")
    e = torch.empty(0, 40, device="cuda", requires_grad=True)
    wd = w.cuda().requires_grad_(True)
    y = layer_norm(e, 40, wd)
    assert y.shape == (0, 40)
    dx, dw = torch.autograd.grad(y.sum(), (e, wd))
    assert dx.shape == (0, 40) and not dw.any()


def test_only_the_wanted_gradients():
    from phoneme_contrast_amd.layers import layer_norm
    x, w, b, dy = (t.cuda() for t in inputs(50, 300, torch.float32, torch.float32, 8))
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(full[0], 300, full[1], full[2]), full, dy)
    for want in ((0,), (1,), (2,), (0, 1), (1, 2)):
        leaves = [t.clone().requires_grad_(i in want) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(layer_norm(leaves[0], 300, leaves[1], leaves[2]), [leaves[i] for i in want], dy)
        for i, g in zip(want, got):
            assert torch.equal(g, grads[i])


@pytest.mark.parametrize("D", [8, 128, 4096])
def test_non_finite_rows_stay_their_own(D):
    x, w, b, dy = inputs(6, D, torch.float32, torch.float32, 9)
    from phoneme_contrast_amd.layers import layer_norm
    bad = x.clone()
    bad[1, 0], bad[3, D // 2] = float("nan"), float("inf")
    outs = []
    for t in (x, bad):
        leaf = t.cuda().requires_grad_(True)
        y = layer_norm(leaf, D, w.cuda(), b.cuda())
        outs.append((y.detach().cpu(), torch.autograd.grad(y, leaf, dy.cuda())[0].cpu()))
    keep = [0, 2, 4, 5]
    for a, c in zip(*outs):
        assert torch.equal(a[keep], c[keep])
        assert torch.isnan(c[1]).all() and torch.isnan(c[3]).any()


def test_directional_differences():
    """The gradients against central differences of the operator itself.  f = sum y dy has second differences of size
    |f'''| h^2 <= 50 h^2 here; f is a sum of 200 float32 results of size 1, off by 2^-20 at most after averaging, so a
    difference over 2 h = 2^-5 is off by at most 2^-20 * 2^5 * 2 = 2^-14 ... and 50 * 2^-12 by the third order."""
    from phoneme_contrast_amd.layers import layer_norm
    gen = torch.Generator().manual_seed(10)
    t = [torch.randn(5, 40, generator=gen), 1 + 0.1 * torch.randn(40, generator=gen), torch.randn(40, generator=gen)]
    dy = torch.randn(5, 40, generator=gen).cuda() / 14
    leaves = [v.cuda().requires_grad_(True) for v in t]
    grads = torch.autograd.grad(layer_norm(leaves[0], 40, leaves[1], leaves[2]), leaves, dy)
    h = 2.0 ** -6
    for i in range(3):
        d = torch.randn(t[i].shape, generator=gen).cuda()
        d /= d.norm()

        def f(s):
            v = [x.detach() for x in leaves]
            v[i] = v[i] + s * d
            return (layer_norm(v[0], 40, v[1], v[2]) * dy).double().sum().item()
        num, ana = (f(h) - f(-h)) / (2 * h), (grads[i] * d).double().sum().item()
        assert abs(num - ana) <= 2.0 ** -14 + 50 * h * h, (i, num, ana)


def test_same_bits_every_time_and_on_another_stream():
    from phoneme_contrast_amd.layers import layer_norm
    x, w, b, dy = (t.cuda() for t in inputs(2000, 1024, torch.bfloat16, torch.bfloat16, 11))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def go():
        y = layer_norm(leaves[0], 1024, leaves[1], leaves[2])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    first = go()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = go()
    torch.cuda.current_stream().wait_stream(s)
    for a, c, e in zip(first, second, go()):
        assert torch.equal(a, c) and torch.equal(a, e)


def test_captured_and_replayed():
    from phoneme_contrast_amd.layers import layer_norm
    x, w, b, dy = (t.cuda() for t in inputs(300, 640, torch.float32, torch.float32, 12))

    def go():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = layer_norm(leaves[0], 640, leaves[1], leaves[2])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        go()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):  # two graphs of one pool: their workspaces may share memory
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            out = go()
        graphs.append((g, out))
    gen = torch.Generator().manual_seed(13)
    for i in range(3):
        x.copy_(torch.randn(300, 640, generator=gen))
        want = go()
        torch.cuda.synchronize()
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, want):
            assert torch.equal(a, c)


def test_refusals_on_the_device():
    from phoneme_contrast_amd.layers import layer_norm
    x = torch.randn(4, 8, device="cuda")
    for bad in (lambda: layer_norm(x, 9), lambda: layer_norm(x, (4, 9)), lambda: layer_norm(x, (2, 4, 8)),
                lambda: layer_norm(x, 8, torch.ones(7, device="cuda")),
                lambda: layer_norm(x, 8, torch.ones(8, device="cuda", dtype=torch.float16)),
                lambda: layer_norm(x.bfloat16(), 8, torch.ones(8, device="cuda"),
                                   torch.ones(8, device="cuda", dtype=torch.bfloat16)),
                lambda: layer_norm(x.double(), 8), lambda: layer_norm(x.int(), 8), lambda: layer_norm(x, 8, eps=0.0),
                lambda: layer_norm(x, 8, eps=float("nan")),
                lambda: layer_norm(torch.zeros(1, 32769, device="cuda"), 32769),
                lambda: layer_norm(torch.zeros(1, 0, device="cuda"), 0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        layer_norm(x, 8, torch.ones(8))


def test_autograd_contract():
    """A second derivative is refused, an input changed before its backward pass is noticed, a result may be changed."""
    from phoneme_contrast_amd.layers import layer_norm
    x, w, b, dy = (t.cuda() for t in inputs(6, 40, torch.float32, torch.float32, 15))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    (gx,) = torch.autograd.grad(layer_norm(x, 40, w, b), [x], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(gx.square().sum(), [x])
    plain = torch.autograd.grad(layer_norm(x, 40, w, b), leaves, dy)
    y = layer_norm(x, 40, w, b)
    y.mul_(2.0)
    for a, c in zip(plain, torch.autograd.grad(y, leaves, dy)):
        assert torch.equal(2 * a, c)  # (a power of two goes through every rounding)
    for t in (x, w):
        h, y = t * 1, None
        y = layer_norm(h if t is x else x, 40, h if t is w else w, b)
        h.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(y, [x], dy)
    with torch.inference_mode():
        assert torch.equal(layer_norm(x, 40, w, b), layer_norm(x.detach(), 40, w, b))
    twice = layer_norm(x, 40, w, w)  # one tensor in both places: its gradient is the sum
    assert torch.equal(torch.autograd.grad(twice, [w], dy)[0], plain[1] + plain[2])


@pytest.mark.parametrize("D", [128, 8192, 8193, 16384, 16392, 32768])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_writes_stay_inside_their_tensors(D, t):
    """Rows between guards, input and gradient in views of wider buffers off 16-byte alignment."""
    from phoneme_contrast_amd.layers import layer_norm
    x, w, b, dy = inputs(3, D, TYPES[t], TYPES[t], 16)
    wide = torch.full((3, 2 * D + 6), 3.0, dtype=TYPES[t])
    wide[:, 1:D + 1], wide[:, D + 3:2 * D + 3] = x, dy
    wide = wide.cuda()
    before = wide.clone()
    vx, vdy = wide[:, 1:D + 1].requires_grad_(True), wide[:, D + 3:2 * D + 3]
    wd, bd = w.cuda().requires_grad_(True), b.cuda().requires_grad_(True)
    y = layer_norm(vx, D, wd, bd)
    got = [y.detach(), *torch.autograd.grad(y, [vx, wd, bd], vdy)]
    assert torch.equal(wide.detach(), before)
    for a, r, tol, what in zip(got, *reference(x, w, b, dy, 1e-5), ("y", "dx", "dw", "db")):
        close(a, r, tol, what)


@pytest.mark.parametrize("D", [33, 39, 65, 250, 513, 1030, 4097, 9001])
@pytest.mark.parametrize("t,wt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
def test_slices_off_every_boundary(D, t, wt):
    """Rows, gradients and weights that start at each element of a 16-byte group."""
    from phoneme_contrast_amd.layers import layer_norm
    x, w, b, dy = inputs(5, D, TYPES[t], TYPES[wt], 17)
    ref, tol = reference(x, w, b, dy, 1e-5)
    n = 16 // x.element_size()
    first = None
    for off in range(n):
        wide = torch.zeros(5, 2 * D + 2 * n + 1, dtype=TYPES[t], device="cuda")
        wide[:, off:off + D], wide[:, D + n:2 * D + n] = x.cuda(), dy.cuda()
        flat = torch.zeros(2, D + n, dtype=TYPES[wt], device="cuda")
        flat[0, off:off + D], flat[1, n - off:n - off + D] = w.cuda(), b.cuda()
        vx = wide[:, off:off + D].requires_grad_(True)
        vw, vb = flat[0, off:off + D].requires_grad_(True), flat[1, n - off:n - off + D].requires_grad_(True)
        y = layer_norm(vx, D, vw, vb)
        got = [y.detach(), *torch.autograd.grad(y, [vx, vw, vb], wide[:, D + n:2 * D + n])]
        for a, r, lim, what in zip(got, ref, tol, ("y", "dx", "dw", "db")):
            close(a, r, lim, what)
        first = first or got
        for a, c in zip(first, got):
            assert torch.equal(a, c)  # where a row lies does not change it


@pytest.mark.parametrize("rows,D", [(600000, 4096), (70000, 32768)])
def test_offsets_that_pass_32_bits(rows, D):
    from phoneme_contrast_amd.layers import layer_norm
    x = torch.empty(rows, D, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    w = torch.linspace(0.5, 1.5, D).bfloat16()
    b = torch.linspace(-1, 1, D).bfloat16()
    x.requires_grad_(True)
    y = layer_norm(x, D, w.cuda(), b.cuda())
    dy = torch.flip(y.detach(), (0,))
    (dx,) = torch.autograd.grad(y, [x], dy)
    pick = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1])
    ref, tol = reference(x[pick.cuda()].detach().cpu(), w, b, dy[pick.cuda()].cpu(), 1e-5)
    close(y[pick.cuda()], ref[0], tol[0], "y")
    close(dx[pick.cuda()], ref[1], tol[1], "dx")


def test_transforms():
    """Nothing is dropped in silence: forward mode, torch.func.grad and tensors without memory raise."""
    import torch.autograd.forward_ad as fwd
    from torch._subclasses.fake_tensor import FakeTensorMode
    from phoneme_contrast_amd.layers import layer_norm
    x, w, b, dy = (t.cuda() for t in inputs(6, 40, torch.float32, torch.float32, 18))
    with fwd.dual_level():
        for i in range(3):
            for leaf in (False, True):
                args = [t.clone() for t in (x, w, b)]
                args[i] = fwd.make_dual(args[i].requires_grad_(leaf), torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    layer_norm(args[0], 40, args[1], args[2])
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            layer_norm(fwd.make_dual(x, dy), 40, w, b)
        layer_norm(x, 40, w, b)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: layer_norm(t, 40, w, b), (x,), (dy,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: layer_norm(t, 40, w, b).sum())(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: layer_norm(t, 40, w.clone().requires_grad_(True), b))(x.view(2, 3, 40))
    # without gradients torch maps the operator slice by slice
    rows = torch.func.vmap(lambda t: layer_norm(t, 40, w, b))(x.view(2, 3, 40))
    assert torch.equal(rows.view(6, 40), layer_norm(x, 40, w, b))
    weights = torch.func.vmap(lambda u: layer_norm(x, 40, u, b))(torch.stack([w, b]))
    assert torch.equal(weights[0], layer_norm(x, 40, w, b)) and torch.equal(weights[1], layer_norm(x, 40, b, b))
    with FakeTensorMode() as mode, pytest.raises((RuntimeError, ValueError)):
        layer_norm(mode.from_tensor(x), 40)


FAR = [(t, v) for t, vs in (("f32", (1.0, 16384.0, 60000.0, -0.1, 1e15, 3e38)), ("f16", (16384.0, 60000.0)),
                            ("bf16", (16384.0, 0.1))) for v in vs]


@pytest.mark.parametrize("t,v", FAR)
def test_constant_rows_of_any_value(t, v):
    """A constant row has xhat = 0: y is the bias, dw 0 and dx = rstd (g - c1), whatever the value and the width.  c1 is
    off by the row sum (at most 32 additions in a thread, 6 in a wave, 16 over waves) and two roundings, rstd by four."""
    from phoneme_contrast_amd.layers import layer_norm
    for D in (33, 40, 100, 513, 1025, 1172, 1228, 1537, 2056, 4097, 5000, 8191, 9001, 16383, 20001, 32767):
        gen = torch.Generator().manual_seed(D)
        x = torch.full((3, D), v, dtype=TYPES[t]).cuda().requires_grad_(True)
        w = torch.randn(D, generator=gen).cuda().requires_grad_(True)
        b = torch.randn(D, generator=gen).cuda().requires_grad_(True)
        if t == "f32" and D % 2:
            dy = torch.randn(3, D, generator=gen)
        else:
            dy = torch.randn(3, D, generator=gen).to(TYPES[t])
        y = layer_norm(x, D, w, b)
        assert torch.equal(y, b.detach().to(TYPES[t]).expand(3, D)), D
        dx, dw = torch.autograd.grad(y, [x, w], dy.cuda())
        assert not dw.any(), D
        g = dy.double() * w.detach().cpu().double()
        ref = (g - g.mean(1, keepdim=True)) / 1e-5 ** 0.5
        tol = (8 * U * (g.abs() + g.abs().mean(1, keepdim=True)) + 56 * U * g.abs().mean(1, keepdim=True)) / 1e-5 ** 0.5
        close(dx, ref, tol, f"dx {D}")


@pytest.mark.parametrize("base", [60000.0, -16384.0, 3e7])
@pytest.mark.parametrize("D", [40, 1025, 1172, 1537, 4100, 20001])
def test_rows_a_few_steps_wide(base, D):
    """Values on float32's own grid around a far base: x - m is exact, and y as exact as for rows at zero.  A row sum is off
    by 54 u (32 additions in a thread, 6 in a wave, 16 over waves at most) and its mean by 55 u; the variance is at least
    half of sum d^2 / D, so off by 110 u, rstd by 57 u; d - e by one rounding and 55 u of e, which is at most half a step;
    two more roundings to the result: 60 u |xhat w| + 28 u rstd step |w| + u |y|."""
    from phoneme_contrast_amd.layers import layer_norm
    gen = torch.Generator().manual_seed(D)
    step = 2.0 ** (np.floor(np.log2(abs(base))) - 23)
    x = (base + step * torch.randint(-3, 4, (4, D), generator=gen).double()).float()
    x[0], x[0, 0] = base, base + step  # one value off
    w, b = torch.randn(D, generator=gen), torch.randn(D, generator=gen)
    xd = x.double()
    u = xd - xd.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((u * u).mean(1, keepdim=True) + 1e-5)
    ref = u * rstd * w.double() + b.double()
    tol = U * (64 * (u.abs() * rstd + rstd * step) * w.double().abs() + 2 * b.double().abs())
    close(layer_norm(x.cuda(), D, w.cuda(), b.cuda()), ref, tol, "y")


@pytest.mark.parametrize("D", [1, 24, 300])
def test_pending_negation(D):
    """The imaginary part of a conjugate is a view of the other sign's memory."""
    from phoneme_contrast_amd.layers import layer_norm
    gen = torch.Generator().manual_seed(19)
    z = torch.randn(5, D, dtype=torch.complex64, generator=gen).cuda()
    w, b, dy = (t.cuda() for t in inputs(5, D, torch.float32, torch.float32, 20)[1:])
    views = [(z.conj().imag, w, b, dy), (torch._neg_view(z.real.contiguous()), w, b, dy)]
    views += [(z.real, torch._neg_view(w), torch._neg_view(b), dy), (z.real, w, b, torch._neg_view(dy))]
    for args in views:
        assert any(t.is_neg() for t in args)
        got, want = [], []
        for out, src in ((got, args), (want, [torch.neg(torch.neg(t)) for t in args])):
            leaves = [t.detach().requires_grad_(True) for t in src[:3]]
            y = layer_norm(leaves[0], D, leaves[1], leaves[2])
            out += [y.detach(), *torch.autograd.grad(y, leaves, src[3])]
            with torch.no_grad():
                out.append(layer_norm(src[0], D, src[1], src[2]))
        for a, c in zip(got, want):
            assert torch.equal(a.resolve_neg(), c.resolve_neg())


def test_column_sums_join_in_64_bits():
    """db of 4096 x 128 float32 rows: 128 blocks sum 32 rows each in float32 (4 in a lane, 2 lanes, 4 waves), the rest is in
    64 bits.  Of dy ~ N(0, s^2) a block's sum is about 6 s, in [4 s, 8 s): an addition rounds it by 2^-23 4 s / sqrt(12) =
    1.4e-7 s rms, the smaller ones before it make that 1.6 times as much, 128 blocks 2.5e-6 s; db is 64 s, so 4e-8 of it,
    and 3.4e-8 (at most) from its own rounding: 5.3e-8, tested with half as much again.  (Joined in float32: 1.2e-7.)"""
    from phoneme_contrast_amd.layers import layer_norm
    off = size = 0.0
    for seed in range(8):
        x, w, b, dy = inputs(4096, 128, torch.float32, torch.float32, 100 + seed)
        leaf = b.cuda().requires_grad_(True)
        (db,) = torch.autograd.grad(layer_norm(x.cuda(), 128, w.cuda(), leaf), [leaf], dy.cuda())
        ref = dy.double().sum(0)
        off += (db.cpu().double() - ref).square().sum().item()
        size += ref.square().sum().item()
    assert (off / size) ** 0.5 <= 8e-8


@pytest.mark.parametrize("D", [1, 2, 7, 32])
def test_narrow_rows_sum_their_columns_in_64_bits(D):
    """dw and db of rows of up to 32 values are rounded once, also where the sums of many blocks cancel: every block's dy is
    followed by almost its negative.  40000 additions in 64 bits are off by 2^-37 of the sum of the terms' sizes at most."""
    from phoneme_contrast_amd.layers import layer_norm
    x, w, b, dy = inputs(20000, D, torch.float32, torch.float32, 30)
    x, dy = torch.cat([x, x]), torch.cat([dy, -dy * (1 + 2.0 ** -14)])
    leaves = [t.cuda().requires_grad_(True) for t in (w, b)]
    got = torch.autograd.grad(layer_norm(x.cuda(), D, *leaves), leaves, dy.cuda())
    ref, _ = reference(x, w, b, dy, 1e-5)
    xh = (ref[0] - b.double()) / w.double()
    for g, r, size in zip(got, ref[2:], ((dy.double() * xh).abs().sum(0), dy.double().abs().sum(0))):
        close(g, r, 2.0 ** -37 * size + 2.0 ** -45 * dy.double().abs().sum(0), "columns")


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("D", [20, 33, 40, 100, 128, 250, 513, 1025, 5000, 20001])
def test_a_row_has_the_same_bits_among_any_others(D, t):
    """Rows of one wave take different numbers of turns about their means: constant ones, far ones, not finite ones."""
    from phoneme_contrast_amd.layers import layer_norm
    gen = torch.Generator().manual_seed(D)
    rows = torch.randn(24, D, generator=gen)
    rows[1], rows[5], rows[9] = 60000.0, -0.1, 3e37
    rows[2] = 16384 + torch.randint(0, 2, (D,), generator=gen)
    rows[6, 0], rows[7, D // 2] = float("nan"), float("inf")
    rows[11] *= 1e-30
    rows[13] = 1e6 + rows[13]
    x = rows.to(TYPES[t]).cuda()
    w, b = torch.randn(D, generator=gen).cuda(), torch.randn(D, generator=gen).cuda()
    dy = torch.randn(24, D, generator=gen).to(TYPES[t]).cuda()

    def go(pick):
        leaf = x[pick].requires_grad_(True)
        y = layer_norm(leaf, D, w, b)
        return y.detach(), torch.autograd.grad(y, leaf, dy[pick])[0]
    whole = go(torch.arange(24))
    for pick in (torch.randperm(24, generator=gen), torch.arange(24)[::2], *(torch.tensor([i]) for i in range(24))):
        for a, c in zip(go(pick), whole):
            assert torch.equal(torch.nan_to_num(a, 7.0), torch.nan_to_num(c[pick.cuda()], 7.0)), pick
    ok = [i for i in range(24) if i not in (6, 7)]
    assert all(torch.isfinite(v[ok]).all() for v in whole) and torch.isnan(whole[0][[6, 7]]).all()
