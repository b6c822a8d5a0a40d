"""Newton-Schulz orthogonalisation, the optimiser step on it and FusedMuon against float64 (csrc/muon.hip, optim.py).

Error bound.  One step maps X to p(X) = a X + (b A + c A A) X with every product summed in float32 from operands held to
2^-24, the lo lo terms (2^-24) dropped: a K-term sum is off by at most g = (4 + 2 sqrt(K)) 2^-24 of the product of its
operands' Frobenius and spectral norms (roundings of random sign).  With s the largest singular value before the step
and f = |X|_F, the step adds at most g f (|a| + 3 |b| s^2 + 5 |c| s^4), and later steps multiply an error by at most
max |p'| over the singular values on the way: the sum over the steps of the one times the other bounds the result's
Frobenius error (`bound`), from the float64 singular values of the case itself.  The sharper claim of the documentation,
float32's own accuracy, is tested against the float32 iteration on the CPU."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def triples(coef, steps):
    return [coef] * steps if not isinstance(coef[0], (tuple, list)) else list(coef)


def iterate(x, coef=COEF, steps=5, eps=1e-7):
    """The definition, in x's type, on the shorter side."""
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    norm = x.double().square().sum((-1, -2), keepdim=True).sqrt()
    x = (x.double() / (norm + eps)).to(x.dtype)
    for a, b, c in triples(coef, steps):
        g = x @ x.mT.contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT.contiguous() if tall else x


def bound(x, coef=COEF, steps=5, eps=1e-7):
    """Largest Frobenius error of the iteration for one float64 matrix."""
    if x.shape[0] > x.shape[1]:
        x = x.mT
    g = (4 + 2 * math.sqrt(max(x.shape))) * 2.0 ** -24
    s = torch.linalg.svdvals(x / (torch.linalg.vector_norm(x) + eps))
    err = 2.0 ** -23 * s.norm().item()  # the scaled input: two roundings
    for a, b, c in triples(coef, steps):
        slope = (a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max().item()
        top, f = s.max().item(), s.norm().item()
        err = err * max(slope, 1e-3) + g * f * (abs(a) + 3 * abs(b) * top ** 2 + 5 * abs(c) * top ** 4)
        s = (a * s + b * s ** 3 + c * s ** 5).abs()
    return err


def gradient(rows, cols, seed, n=96, noise=0.1):
    """A minibatch gradient: n samples' outer products of falling weight, and noise."""
    gen = torch.Generator().manual_seed(seed)
    w = torch.arange(1, n + 1).float().pow(-0.5)[:, None]
    g = (torch.randn(n, rows, generator=gen) * w).T @ torch.randn(n, cols, generator=gen)
    return 1e-2 * (g + noise * torch.randn(rows, cols, generator=gen))


def close(got, x, coef=COEF, steps=5, eps=1e-7):
    """got (any type) against the float64 iteration of x (float64, one matrix)."""
    ref = iterate(x, coef, steps, eps)
    off = torch.linalg.vector_norm(got.detach().cpu().double() - ref).item()
    h = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 2.0 ** -24
    limit = bound(x, coef, steps, eps) * (1 + h) + h * torch.linalg.vector_norm(ref).item()
    assert off <= limit, (off, limit)
    return off


SHAPES = [(1, 1), (1, 2), (2, 1), (1, 300), (300, 1), (2, 3), (3, 5), (9, 32), (31, 33), (63, 64), (64, 64), (65, 64), (64, 129),
          (65, 65), (128, 128), (100, 577), (577, 100), (128, 1152), (200, 1001), (333, 129), (512, 512), (257, 2305)]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_shapes_and_types(rows, cols, t):
    from phoneme_contrast_amd.optim import orthogonalize
    x = gradient(rows, cols, rows * 7 + cols).to(TYPES[t])
    out = orthogonalize(x.cuda())
    assert out.dtype == x.dtype and out.shape == x.shape and out.is_contiguous()
    close(out, x.double())


@pytest.mark.parametrize("rows,cols", [(64, 576), (128, 128), (200, 333), (512, 1024), (640, 640)])
def test_as_exact_as_float32_arithmetic(rows, cols):
    """Twice the float32 iteration's own error: its operands and sums round at 2^-24 as these do, and the dropped
    lo lo terms and the rescaled input add no more than as much again."""
    from phoneme_contrast_amd.optim import orthogonalize
    for seed in range(3):
        x = gradient(rows, cols, seed)
        ref = iterate(x.double())
        err32 = torch.linalg.vector_norm(iterate(x).double() - ref)
        err = torch.linalg.vector_norm(orthogonalize(x.cuda()).cpu().double() - ref)
        assert err <= 2 * err32, (err.item(), err32.item())


def test_result_is_nearly_orthogonal():
    """Five steps take singular values in [0.01, 1] of the normalised matrix into [0.68, 1.21] (the polynomial's own
    range, by its definition); a well-conditioned matrix of 64 rows starts above 0.05."""
    from phoneme_contrast_amd.optim import orthogonalize
    x = torch.randn(64, 400, generator=torch.Generator().manual_seed(1))
    s = torch.linalg.svdvals(orthogonalize(x.cuda()).cpu().double())
    assert 0.68 < s.min() and s.max() < 1.21


@pytest.mark.parametrize("steps,coef", [(1, COEF), (2, COEF), (3, COEF), (8, COEF), (6, (1.875, -1.25, 0.375)),
                                        (4, ((4.0, -6.0, 2.5), (3.0, -3.5, 1.4), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0)))])
def test_steps_and_coefficients(steps, coef):
    from phoneme_contrast_amd.optim import orthogonalize
    x = gradient(90, 150, 5)
    close(orthogonalize(x.cuda(), ns_steps=steps, ns_coefficients=coef), x.double(), coef, steps)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-7, 1e4, 1e18, 1e30])
def test_any_size_of_input(scale):
    """Sums of squares have no range to leave (float64); below eps the matrix is only scaled up, to |x| / eps."""
    from phoneme_contrast_amd.optim import orthogonalize
    x = gradient(70, 130, 6) * scale
    close(orthogonalize(x.cuda()), x.double())


def test_strides_views_and_batches():
    from phoneme_contrast_amd.optim import orthogonalize
    big = torch.stack([gradient(80, 220, s) for s in range(6)]).view(2, 3, 80, 220)
    dev = big.cuda()
    views = {"transposed": lambda t: t.mT, "sliced": lambda t: t[..., 3:70, 5:205], "every second": lambda t: t[..., ::2, ::3],
             "swapped batch": lambda t: t.transpose(0, 1), "expanded": lambda t: t[:1].expand(4, 3, 80, 220),
             "one": lambda t: t[1, 2], "rows of one": lambda t: t[..., :1, :], "uneven batch": lambda t: t[:, :2]}
    for name, view in views.items():
        x, out = view(big), orthogonalize(view(dev))
        assert out.shape == x.shape and out.is_contiguous()
        for i, (m, o) in enumerate(zip(x.reshape(-1, *x.shape[-2:]), out.reshape(-1, *x.shape[-2:]))):
            close(o, m.double())
    assert torch.equal(orthogonalize(dev)[1, 1], orthogonalize(dev[1, 1]))  # a batch changes nothing


def test_empty_zero_and_non_finite_matrices():
    from phoneme_contrast_amd.optim import orthogonalize
    for shape in ((0, 5, 6), (3, 0, 6), (3, 5, 0), (0, 0)):
        assert orthogonalize(torch.empty(shape, device="cuda")).shape == shape
    x = torch.stack([gradient(70, 100, s) for s in range(5)])
    clean = orthogonalize(x.cuda())
    x[1], x[2, 3, 4], x[3, 69, 99] = 0, float("nan"), float("inf")
    out = orthogonalize(x.cuda())
    assert torch.equal(out[0], clean[0]) and torch.equal(out[4], clean[4])
    assert not out[1].any() and torch.isnan(out[2]).all() and torch.isnan(out[3]).all()


def test_no_gradient_and_repeats_on_any_stream():
    from phoneme_contrast_amd.optim import orthogonalize
    x = gradient(300, 500, 8).cuda().requires_grad_(True)
    a = orthogonalize(x)
    assert not a.requires_grad
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = orthogonalize(x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, b) and torch.equal(a, orthogonalize(x))


def test_two_captured_graphs():
    from phoneme_contrast_amd.optim import orthogonalize
    x = gradient(130, 260, 9).cuda()
    y = gradient(260, 130, 10).cuda()
    orthogonalize(x), orthogonalize(y)
    torch.cuda.synchronize()
    graphs = []
    for t in (x, y):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            out = orthogonalize(t)
        graphs.append((g, t, out))
    for i in range(4):
        g, t, out = graphs[i % 2]
        t.copy_(gradient(*t.shape, 20 + i))
        want = orthogonalize(t)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals():
    from phoneme_contrast_amd.optim import FusedMuon, muon_step, orthogonalize
    x = torch.randn(8, 9, device="cuda")
    for bad in (lambda: orthogonalize(x[0]), lambda: orthogonalize(x.double()), lambda: orthogonalize(x.int()),
                lambda: orthogonalize(x, ns_steps=0), lambda: orthogonalize(x, ns_steps=65), lambda: orthogonalize(x, eps=0.0),
                lambda: orthogonalize(x, eps=float("nan")), lambda: orthogonalize(x, ns_coefficients=(1.0, 2.0)),
                lambda: orthogonalize(x, ns_coefficients=((1.0, 2.0, 3.0),) * 4),
                lambda: orthogonalize(x, ns_coefficients=(10.0, 0.0, 0.0)),
                lambda: orthogonalize(x, ns_coefficients=(float("nan"), 0.0, 0.0)),
                lambda: orthogonalize(torch.empty(1, 1, device="cuda").expand(20000, 20000))):
        with pytest.raises(ValueError):
            bad()
    p, g, m = (torch.randn(8, 9, device="cuda") for _ in range(3))

    def step(ps=(p,), gs=(g,), ms=(m,), **kw):
        muon_step(ps, gs, ms, **{"lr": 0.1, **kw})
    before = p.clone()
    for bad in (lambda: step(gs=()), lambda: step(ps=(p, p), gs=(g, g), ms=(m, m.clone())), lambda: step(ms=(p,)),
                lambda: step(ps=(p, p.clone()), gs=(g, g), ms=(m, m)), lambda: step(gs=(g[:, :8],)), lambda: step(gs=(g.half(),)),
                lambda: step(ps=(p.T.contiguous().T,)), lambda: step(ps=(p[0],), gs=(g[0],), ms=(m[0],)), lambda: step(lr=-1.0),
                lambda: step(momentum=1.0), lambda: step(weight_decay=-0.1), lambda: step(eps=0.0), lambda: step(adjust="no"),
                lambda: FusedMuon([torch.nn.Parameter(p)], momentum=1.5), lambda: FusedMuon([torch.nn.Parameter(p)], lr=-1.0),
                lambda: FusedMuon([torch.nn.Parameter(p)], adjust="x"), lambda: FusedMuon([torch.nn.Parameter(p)], ns_steps=0)):
        with pytest.raises(ValueError):
            bad()
    assert torch.equal(p, before)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        step(gs=(g.cpu(),))
    step(ps=(), gs=(), ms=())


def reference_step(p, g, m, lr, momentum, nesterov, wd, adjust, gs=1.0, **kw):
    """float64 -> new parameter, new momentum, and the bound on the parameter's error."""
    p, g, m = (t.cpu().double() for t in (p, g, m))
    m = momentum * m + (1 - momentum) * gs * g
    u = ((1 - momentum) * gs * g + momentum * m if nesterov else m).reshape(p.shape[0], -1)
    rows, cols = u.shape
    k = {"rms": 0.2 * math.sqrt(max(rows, cols)), "spectral": math.sqrt(max(1, rows / cols)), None: 1.0}[adjust]
    o = iterate(u, **kw)
    # u itself carries three float32 roundings; the iteration multiplies them as it does the input's
    tol = 3 * bound(u, **kw) * lr * k + 3 * 2.0 ** -24 * (p.norm().item() + lr * k * o.norm().item())
    return (1 - lr * wd) * p - lr * k * o.view_as(p), m, tol


@pytest.mark.parametrize("nesterov,adjust,wd,gs", [(True, "rms", 0.1, 1.0), (False, "spectral", 0.0, 0.125), (True, None, 1e-2, 4.0)])
def test_step_of_a_list(nesterov, adjust, wd, gs):
    """More matrices than one launch takes, of every kind of shape."""
    from phoneme_contrast_amd.optim import muon_step
    shapes = [(32, 1, 3, 3), (64, 32, 3, 3), (128, 128), (96, 200), (200, 96), (5, 2), (2, 70), (1, 40), (40, 1), (130, 64, 1, 1)]
    shapes = shapes * 3 + [(256, 600)]
    gen = torch.Generator().manual_seed(2)
    p = [torch.randn(s, generator=gen) for s in shapes]
    g = [gradient(s[0], math.prod(s[1:]), i).view(s) for i, s in enumerate(shapes)]
    m = [gradient(s[0], math.prod(s[1:]), 100 + i).view(s) for i, s in enumerate(shapes)]
    dp, dg, dm = ([t.cuda() for t in ts] for ts in (p, g, m))
    for _ in range(2):
        ref = [reference_step(a, b, c, 0.02, 0.9, nesterov, wd, adjust, gs) for a, b, c in zip(dp, dg, dm)]
        muon_step(dp, dg, dm, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=wd, adjust=adjust, grad_scale=gs)
        for a, c, (ra, rc, tol) in zip(dp, dm, ref):
            assert (a.cpu().double() - ra).norm().item() <= tol
            assert ((c.cpu().double() - rc).abs() <= 3 * 2.0 ** -24 * (rc.abs() + c.cpu().abs().max())).all()
    for a, b in zip(dg, g):
        assert torch.equal(a.cpu(), b)


def small_model(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Conv2d(3, 20, 3), torch.nn.BatchNorm2d(20), torch.nn.Conv2d(20, 1, 1),
                               torch.nn.Flatten(), torch.nn.Linear(36, 50), torch.nn.Linear(50, 7, bias=False)).cuda()


def set_grads(model, seed):
    gen = torch.Generator().manual_seed(seed)
    for p in model.parameters():
        p.grad = torch.randn(p.shape, generator=gen).cuda() * 0.1


def adam_reference(p, g, m, v, step, lr, wd, betas=(0.9, 0.999), eps=1e-8):
    g = g + wd * p
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    den = v.sqrt() / math.sqrt(1 - betas[1] ** step) + eps
    return p - lr / (1 - betas[0] ** step) * m / den, m, v


@pytest.mark.parametrize("flat", [False, True])
def test_optimizer_matches_the_formulas(flat):
    from phoneme_contrast_amd.optim import FusedMuon
    model = small_model()
    opt = FusedMuon(model.parameters(), lr=0.01, weight_decay=0.05)
    names = [n for n, _ in model.named_parameters()]
    mats = {"0.weight", "4.weight", "5.weight"}  # the 1 x 20 convolution, norms and biases take Adam
    state = {n: (torch.zeros_like(p).cpu().double(), torch.zeros_like(p).cpu().double()) for n, p in model.named_parameters()}
    for step in range(1, 4):
        set_grads(model, step)
        before = {n: p.detach().cpu().double() for n, p in model.named_parameters()}
        grads = {n: p.grad.cpu().double() for n, p in model.named_parameters()}
        if flat:  # the summed gradients of two ranks, averaged in the step
            fg = torch.cat([2 * p.grad.reshape(-1) for p in model.parameters()])
            opt.step(flat_grads=[fg], grad_scale=0.5)
        else:
            opt.step()
        for n, p in model.named_parameters():
            got = p.detach().cpu().double()
            m, v = state[n]
            if n in mats:
                ref, m2, tol = reference_step(before[n].float(), grads[n].float(), m.float(), 0.01, 0.95, True, 0.05, "rms")
                assert (got - ref).norm().item() <= tol, n
                state[n] = (m2, v)
            else:
                ref, m2, v2 = adam_reference(before[n], grads[n], m, v, step, 0.01, 0.05)
                # eight float32 operations on an update of size lr and on p
                assert ((got - ref).abs() <= 16 * 2.0 ** -24 * (ref.abs() + 0.01 * 4)).all(), n
                state[n] = (m2, v2)
    sd = opt.state_dict()
    for i, n in enumerate(names):
        s = sd["state"][i]
        assert set(s) == ({"step", "momentum_buffer"} if n in mats else {"step", "exp_avg", "exp_avg_sq"}) and int(s["step"]) == 3
        own = s["momentum_buffer" if n in mats else "exp_avg"].cpu().double()
        assert ((own - state[n][0]).abs() <= 16 * 2.0 ** -24 * (state[n][0].abs() + 0.2)).all()


def test_optimizer_state_moves_on(tmp_path):
    """Save, load and go on; parameters bound anew behind the optimizer's back; a group of Adam only; a schedule."""
    from phoneme_contrast_amd.optim import FusedAdam, FusedMuon
    a, b = small_model(1), small_model(1)
    oa, ob = FusedMuon(a.parameters(), lr=0.02), FusedMuon(b.parameters(), lr=0.02)
    for k in range(2):
        set_grads(a, k), set_grads(b, k)
        oa.step(), ob.step()
    torch.save({"o": ob.state_dict(), "m": b.state_dict()}, tmp_path / "c.pt")
    c = small_model(2)
    saved = torch.load(tmp_path / "c.pt", weights_only=True, map_location="cuda")
    c.load_state_dict(saved["m"])
    oc = FusedMuon(c.parameters(), lr=0.5)
    oc.load_state_dict(saved["o"])
    a.cpu(), a.cuda()  # re-bound: new storages
    sched = torch.optim.lr_scheduler.StepLR(oa, 1, 0.5)
    for k in range(2, 4):
        for mdl, o in ((a, oa), (c, oc)):
            o.param_groups[0]["lr"] = 0.02
            set_grads(mdl, k)
            o.step()
    for p, q in zip(a.parameters(), c.parameters()):
        assert torch.equal(p, q)
    oa.param_groups[0]["lr"] = sched.base_lrs[0]
    sched.step()
    assert oa.param_groups[0]["lr"] == 0.01
    fa = FusedAdam(small_model(3).parameters())
    with pytest.raises(ValueError, match="another optimizer"):
        oc.load_state_dict(fa.state_dict())
    d, e = small_model(4), small_model(4)
    od, oe = FusedMuon([{"params": d.parameters(), "muon": False}], lr=0.01, weight_decay=0.1), FusedAdam(e.parameters(), 0.01, weight_decay=0.1)
    for k in range(2):
        set_grads(d, k), set_grads(e, k)
        od.step(), oe.step()
    for p, q in zip(d.parameters(), e.parameters()):
        assert ((p - q).abs() <= 4 * 2.0 ** -24 * (q.abs() + 0.02)).all()  # (two kernels: contractions may differ)
    assert oc.step() is None  # (no further gradients set: the last ones again)
    with pytest.raises(ValueError, match="flat gradient"):
        oc.step(flat_grads=[torch.zeros(3, device="cuda")])


def test_step_in_a_captured_graph():
    from phoneme_contrast_amd.optim import muon_step
    shapes = [(32, 9), (64, 288), (128, 128)]
    p = [gradient(*s, 1).cuda() for s in shapes]
    m = [gradient(*s, 2).cuda() for s in shapes]
    g = [gradient(*s, 3).cuda() for s in shapes]
    p2, m2 = [t.clone() for t in p], [t.clone() for t in m]
    warm = [t.clone() for t in p], [t.clone() for t in m]
    muon_step(warm[0], g, warm[1], lr=0.01)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step(p, g, m, lr=0.01)
    for k in range(3):
        for i, s in enumerate(shapes):
            g[i].copy_(gradient(*s, 10 + k))
        graph.replay()
        muon_step(p2, g, m2, lr=0.01)
        torch.cuda.synchronize()
        for a, b in zip(p + m, p2 + m2):
            assert torch.equal(a, b)


@pytest.mark.parametrize("batch,rows,cols", [
    (3, 1100, 2100), (3, 2100, 1100),  # 128 x 128 tiles over ragged edges, in every product
    (1, 1856, 1856),                   # more 64 x 64 tiles than the card holds at a time: the last ones in parts
    (1, 2900, 2900),                   # the same of 128 x 128 tiles
    (1, 600, 5000), (1, 5000, 600),    # parts of a long K
    (40, 150, 90), (7, 40, 3000)])     # many small ones, and short sides of a long K
def test_every_way_to_cut_the_products(batch, rows, cols):
    from phoneme_contrast_amd.optim import orthogonalize
    x = torch.stack([gradient(rows, cols, 50 + i) for i in range(batch)])
    out = orthogonalize(x.cuda())
    for i in sorted({0, batch - 1}):
        close(out[i], x[i].double(), steps=5)
    assert torch.equal(out, orthogonalize(x.cuda()))


def test_memory_shared_between_the_tensors_of_a_step():
    from phoneme_contrast_amd.optim import muon_step
    flat = torch.randn(400, device="cuda")
    p, g, m = flat[:72].view(8, 9), flat[72:144].view(8, 9), flat[144:216].view(8, 9)
    near = flat[180:252].view(8, 9)  # half of m
    before = flat.clone()
    for ps, gs, ms in (([p], [m], [m]), ([p], [p], [m]), ([p], [near], [m]), ([p, near], [g, g], [m, flat[300:372].view(8, 9)]),
                       ([p], [g], [g]), ([p], [g], [flat[36:108].view(8, 9)])):
        with pytest.raises(ValueError, match="shares memory"):
            muon_step(ps, gs, ms, lr=0.1)
    assert torch.equal(flat, before)
    q, n = flat[216:288].view(8, 9), flat[288:360].view(8, 9)
    ref = [reference_step(a, g, b, 0.1, 0.95, True, 0.0, "rms") for a, b in ((p, m), (q, n))]
    muon_step([p, q], [g, g], [m, n], lr=0.1)  # neighbours, and one gradient for two
    for a, (r, _, tol) in zip((p, q), ref):
        assert (a.cpu().double() - r).norm().item() <= tol
    assert torch.equal(g, before[72:144].view(8, 9)) and torch.equal(flat[360:], before[360:])


def test_writes_stay_inside_their_tensors():
    """Views between guards of a flat buffer, at offsets off every alignment but float32's."""
    from phoneme_contrast_amd.optim import muon_step
    for rows, cols in ((31, 65), (130, 700), (700, 130), (1, 9)):
        n = rows * cols
        flat = torch.full((3 * n + 100,), 7.0, device="cuda")
        views = [flat[17 + i * (n + 13):17 + i * (n + 13) + n].view(rows, cols) for i in range(3)]
        p, g, m = (gradient(rows, cols, s) for s in range(3))
        for v, t in zip(views, (p, g, m)):
            v.copy_(t)
        ref, _, tol = reference_step(p, g, m, 0.1, 0.95, True, 0.0, "rms")
        muon_step([views[0]], [views[1]], [views[2]], lr=0.1)
        assert (views[0].cpu().double() - ref).norm().item() <= tol
        assert torch.equal(views[1].cpu(), g)
        guard = torch.ones_like(flat, dtype=torch.bool)
        for i in range(3):
            guard[17 + i * (n + 13):17 + i * (n + 13) + n] = False
        assert (flat[guard] == 7.0).all()


def test_states_of_the_two_optimizers_are_told_apart():
    from phoneme_contrast_amd.optim import FusedAdam, FusedMuon
    a, b = small_model(1), small_model(1)
    oa, ob = FusedAdam(a.parameters()), FusedMuon(b.parameters())
    for mdl, o in ((a, oa), (b, ob)):
        set_grads(mdl, 0)
        o.step()
    for o, other in ((oa, ob), (ob, oa)):
        before = [t.clone() for t in (a if o is oa else b).parameters()]
        with pytest.raises(ValueError, match="another optimizer"):
            o.load_state_dict(other.state_dict())
        for p, q in zip(before, (a if o is oa else b).parameters()):
            assert torch.equal(p, q)
        o.load_state_dict(o.state_dict())
    plain = torch.optim.Adam([torch.nn.Parameter(p.detach().clone()) for p in a.parameters()])
    oa.load_state_dict(plain.state_dict())
    plain.load_state_dict(oa.state_dict())


def test_offsets_that_pass_32_bits():
    """The longest side there is (planes of 2^32 numbers), both ways round, and batches far apart in memory."""
    from phoneme_contrast_amd.optim import orthogonalize
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(512, 1 << 20, device="cuda", generator=gen).bfloat16()
    ref = x.double()
    ref /= torch.linalg.vector_norm(ref) + 1e-7
    gram = ref @ ref.T.contiguous()
    # `bound` needs the singular values alone; every step's polynomial in X X^T acts on the left
    small = torch.diag(torch.linalg.eigvalsh(gram.cpu()).clamp(min=0).sqrt())
    g = (4 + 2 * math.sqrt(1 << 20)) / (4 + 2 * math.sqrt(512))
    left = torch.eye(512, dtype=torch.float64, device="cuda")
    for _ in range(5):
        a = left @ gram @ left.T.contiguous()
        left = COEF[0] * left + (COEF[1] * a + COEF[2] * (a @ a)) @ left
    ref = left @ ref
    limit = g * bound(small, eps=0.0) + (2.0 ** -8 + 2.0 ** -20) * torch.linalg.vector_norm(ref).item()
    for t in (x, x.T):
        out = orthogonalize(t)
        out = out if t is x else out.T
        off = sum(torch.linalg.vector_norm(out[i:i + 64].double() - ref[i:i + 64]).item() ** 2 for i in range(0, 512, 64)) ** 0.5
        assert off <= limit, (off, limit)
        assert torch.isfinite(out[-1, -1]) and (out[-1, -4096:].double() - ref[-1, -4096:]).abs().max() <= 2.0 ** -7 * ref.abs().max()
    del x, ref, out
    far = torch.empty(2 * ((1 << 31) + 7) + 40000, dtype=torch.float16, device="cuda")
    view = far.as_strided((3, 90, 110), ((1 << 31) + 7, 1, 301))
    values = torch.stack([gradient(90, 110, s) for s in range(3)]).half()
    view.copy_(values)
    for o, v in zip(orthogonalize(view), values):
        close(o, v.double())


def test_two_streams_at_once():
    from phoneme_contrast_amd.layers import layer_norm
    from phoneme_contrast_amd.optim import muon_step, orthogonalize
    xs = [gradient(300, 2000, 1).cuda(), gradient(700, 130, 2).cuda()]
    want = [orthogonalize(x) for x in xs]
    norms = [layer_norm(x, x.shape[-1]) for x in xs]
    start = [[gradient(*s, 3).cuda() for s in ((64, 288), (128, 1152), (40, 9))] for _ in range(3)]
    p, g, m = ([t.clone() for t in ts] for ts in start)
    muon_step(p, g, m, lr=0.1)
    sides = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, (s, x) in enumerate(zip(sides, xs)):
            with torch.cuda.stream(s):
                lists = [[t.clone() for t in ts] for ts in start]
                muon_step(*lists, lr=0.1)
                got[i].append((orthogonalize(x), layer_norm(x, x.shape[-1]), lists))
    torch.cuda.synchronize()
    for i in range(2):
        for o, y, lists in got[i]:
            assert torch.equal(o, want[i]) and torch.equal(y, norms[i])
            for a, b in zip(lists[0] + lists[2], p + m):
                assert torch.equal(a, b)


TINY = torch.finfo(torch.float32).tiny


@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 3), (8, 9), (64, 64), (128, 128), (200, 333)])  # one block; products
@pytest.mark.parametrize("eps", [TINY, 2.0 ** -149])
def test_tiny_eps(rows, cols, eps):
    """The scale 1 / (|x|_F + eps) leaves float32's range: a zero matrix stays zero on every route, a tiny one is scaled."""
    from phoneme_contrast_amd.optim import muon_step, orthogonalize
    x = gradient(rows, cols, 3)
    x *= 1e-36 / x.norm()
    batch = torch.stack([torch.zeros_like(x), x, gradient(rows, cols, 4)])
    out = orthogonalize(batch.cuda(), eps=eps)
    assert not out[0].any()
    close(out[1], batch[1].double(), eps=eps)
    close(out[2], batch[2].double(), eps=eps)
    # a layer without a gradient is decayed alone
    if rows == 1:
        return
    p = [gradient(rows, cols, 5).cuda() for _ in range(2)]
    g, m = [torch.zeros_like(p[0]), x.cuda()], [torch.zeros_like(p[0]) for _ in range(2)]
    want = (p[0].double() * (1 - 0.1 * 0.5)).cpu()
    muon_step(p, g, m, lr=0.1, weight_decay=0.5, eps=eps)
    assert ((p[0].cpu().double() - want).abs() <= 2.0 ** -22 * want.abs()).all()
    assert torch.isfinite(p[1]).all() and not m[0].any()


@pytest.mark.parametrize("rows,cols", [(5, 7), (130, 260)])
def test_pending_negation(rows, cols):
    """The imaginary part of a conjugate is a view of the other sign's memory."""
    from phoneme_contrast_amd.optim import muon_step, orthogonalize
    z = torch.randn(2, rows, cols, dtype=torch.complex64, generator=torch.Generator().manual_seed(1)).cuda()
    x = z.conj().imag
    assert x.is_neg() and torch.equal(orthogonalize(x), orthogonalize(torch.neg(z.imag)))
    n = torch._neg_view(z[0].real.contiguous())
    assert torch.equal(orthogonalize(n), orthogonalize(-z[0].real))
    t = [torch.randn(rows, cols, device="cuda") for _ in range(3)]
    for i in range(3):
        with pytest.raises(ValueError, match="in memory"):
            muon_step(*[[n if k == i else t[k]] for k in range(3)], lr=0.1)


def rms_errors(shapes, run, seeds=40):
    """Per shape: rms relative errors of `run` (a list of matrices -> theirs orthogonalised) and of the float32 iteration."""
    own, f32 = [0.0] * len(shapes), [0.0] * len(shapes)
    for seed in range(seeds):
        xs = [gradient(r, c, 7 * seed + i) for i, (r, c) in enumerate(shapes)]
        for i, (x, o) in enumerate(zip(xs, run(xs))):
            ref = iterate(x.double())
            own[i] += ((o.cpu().double() - ref).norm() / ref.norm()).item() ** 2
            f32[i] += ((iterate(x).double() - ref).norm() / ref.norm()).item() ** 2
    return [((a / seeds) ** 0.5, (b / seeds) ** 0.5) for a, b in zip(own, f32)]


SHORT = [(1, 1), (1, 2), (1, 50), (2, 3), (3, 5), (200, 3), (5, 5), (8, 30), (32, 9), (16, 100), (24, 24), (31, 33), (32, 32),
         (288, 32), (32, 288), (32, 700), (20, 1000)]


def by_step(xs):
    """The same through a step: without momentum, decay or a scale a parameter of 0 becomes minus its gradient's."""
    from phoneme_contrast_amd.optim import muon_step
    p = [torch.zeros_like(x, device="cuda") for x in xs]
    muon_step(p, [x.cuda() for x in xs], [torch.zeros_like(t) for t in p], lr=1.0, momentum=0.0, nesterov=False, adjust=None)
    return [-t for t in p]


def test_short_sides_are_as_exact_as_float32():
    """Matrices whose short side is one tile are computed in float32 throughout, alone, in batches and in lists that blocks
    hold: as many roundings as the float32 iteration has, in another order.  Of 40 draws an rms is known to 1 / sqrt(80) =
    11 %, two to 16 %: half as much again is allowed (operands of 22 bits: 1.9 times at 1 x 50 and 3 x 5)."""
    from phoneme_contrast_amd.optim import orthogonalize
    routes = {"alone": lambda xs: [orthogonalize(x.cuda()) for x in xs],
              "batch": lambda xs: [orthogonalize(torch.stack([x, x]).cuda())[1] for x in xs],
              "list": lambda xs: by_step(xs[:9]) + by_step(xs[9:]),
              "mixed list": lambda xs: by_step(xs[:9] + [gradient(64, 64, 1)])[:9] + by_step(xs[9:] + [gradient(96, 300, 1)])[:-1]}
    for name, run in routes.items():
        for shape, (own, f32) in zip(SHORT, rms_errors(SHORT, run)):
            assert own <= 1.5 * f32, (name, shape, own, f32)


def test_short_sides_among_the_products():
    """In a list with others that blocks do not hold, operands have 22 bits: twice the float32
    iteration's error where sums are short, with the 22 % that two rms of 20 draws may be off; long ones alone have not."""
    from phoneme_contrast_amd.optim import orthogonalize
    shapes = [(1, 2000), (3, 2000), (20, 1500), (32, 1100)]
    for shape, (own, f32) in zip(shapes, rms_errors(shapes, lambda xs: [orthogonalize(x.cuda()) for x in xs], 20)):
        assert own <= 2 * f32, (shape, own, f32)
    shapes = SHORT[:15]
    for shape, (own, f32) in zip(shapes, rms_errors(shapes, lambda xs: by_step(xs + [gradient(200, 300, 1)])[:-1], 20)):
        assert own <= 2.5 * f32, (shape, own, f32)


def test_a_graph_that_holds_the_old_weights_is_noticed():
    """A weight that changes between a forward pass and its backward pass is an error, as with torch's own optimizers."""
    from phoneme_contrast_amd.optim import FusedMuon, muon_step
    x = torch.randn(6, 9, device="cuda", requires_grad=True)
    p, g, m = (torch.randn(8, 9, device="cuda") for _ in range(3))
    y, z = (x @ p.T).sum(), (x[:, 0] * m[:6, 0]).sum()
    muon_step([p], [g], [m], lr=0.1)
    for out in (y, z):
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(out, [x])
    torch.autograd.grad((x @ p.T).sum(), [x])
    with torch.inference_mode():  # (such tensors have no version)
        muon_step([p.clone()], [g], [m.clone()], lr=0.1)
    model = small_model()
    opt = FusedMuon(model.parameters())
    set_grads(model, 0)
    opt.step()  # (the first step moves the weights into the flat buffer)
    set_grads(model, 1)
    ys = [(x[0, 0] * q).sum() for q in model.parameters()]
    opt.step()
    for y in ys:
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(y, [x])


LONG = [(1, 1025), (1, 2000), (1, 7600), (2, 4700), (4, 3999), (3000, 5), (7, 2700), (32, 1100), (20, 1500), (2059, 4)]


def test_long_matrices_of_few_rows_are_as_exact_as_float32():
    """As test_short_sides_are_as_exact_as_float32, behind 1024 values of the long side; 20 draws: two rms to 22 %."""
    from phoneme_contrast_amd.optim import orthogonalize
    routes = {"alone": lambda xs: [orthogonalize(x.cuda()) for x in xs],
              "list": lambda xs: by_step(xs[:4] + [gradient(8, 30, 1), gradient(32, 32, 1)])[:4] + by_step(xs[4:])}
    for name, run in routes.items():
        for shape, (own, f32) in zip(LONG, rms_errors(LONG, run, 20)):
            assert own <= 1.5 * f32, (name, shape, own, f32)


@pytest.mark.parametrize("rows,cols", [(1, 1025), (32, 1056), (31, 1057), (1057, 31), (5, 16384), (16385, 9), (17, 131073), (40001, 32)])
@pytest.mark.parametrize("t", list(TYPES))
def test_long_matrices_of_few_rows(rows, cols, t):
    from phoneme_contrast_amd.optim import orthogonalize
    x = gradient(rows, cols, rows + cols).to(TYPES[t])
    out = orthogonalize(x.cuda())
    close(out, x.double())
    assert torch.equal(out, orthogonalize(x.cuda()))
    view = torch.zeros(cols + 3, 2 * rows + 1, dtype=x.dtype, device="cuda")[2:2 + cols, 1::2].t()  # any strides
    view.copy_(x)
    assert torch.equal(out, orthogonalize(view))


def test_long_matrices_in_batches_and_lists():
    """Batches with zero and not finite matrices, tiny eps, steps of lists with others that blocks hold, guards, graphs."""
    from phoneme_contrast_amd.optim import muon_step, orthogonalize
    x = torch.stack([gradient(9, 1500, s) for s in range(6)])
    clean = orthogonalize(x.cuda())
    x[1], x[2, 3, 4], x[3, 8, 1499], x[4] = 0, float("nan"), float("inf"), x[4] * 1e-30
    for eps in (1e-7, TINY):
        out = orthogonalize(x.cuda(), eps=eps)
        assert not out[1].any() and torch.isnan(out[2]).all() and torch.isnan(out[3]).all()
        close(out[4], x[4].double(), eps=eps)
        close(out[0], x[0].double(), eps=eps)
    assert torch.equal(orthogonalize(x.cuda())[[0, 5]], clean[[0, 5]])
    for coef, steps in ((COEF, 1), (COEF, 2), ((1.875, -1.25, 0.375), 7)):
        close(orthogonalize(x[0].cuda(), ns_steps=steps, ns_coefficients=coef), x[0].double(), coef, steps)
    shapes = [(32, 9), (4, 3, 20, 20), (2000, 3), (1, 1300), (30, 30), (1300, 1)]
    sizes = [math.prod(s) for s in shapes]
    flat = torch.full((3 * sum(sizes) + 7 * 40,), 7.0, device="cuda")
    mask = torch.ones_like(flat, dtype=torch.bool)
    lists, at = ([], [], []), 5
    for i, s in enumerate(shapes):
        for k in range(3):
            lists[k].append(flat[at:at + sizes[i]].view(s))
            lists[k][-1].copy_(gradient(s[0], sizes[i] // s[0], 10 * i + k).view(s))
            mask[at:at + sizes[i]] = False
            at += sizes[i] + 13
    p, g, m = lists
    twin = [[t.clone() for t in ts] for ts in lists]
    ref = [reference_step(a, b, c, 0.02, 0.9, True, 0.1, "rms") for a, b, c in zip(p, g, m)]
    muon_step(p, g, m, lr=0.02, momentum=0.9, weight_decay=0.1)
    for a, c, (ra, rc, tol) in zip(p, m, ref):
        assert (a.cpu().double() - ra).norm().item() <= tol
        assert ((c.cpu().double() - rc).abs() <= 3 * 2.0 ** -24 * (rc.abs() + c.cpu().abs().max())).all()
    assert (flat[mask] == 7.0).all()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        muon_step(*twin, lr=0.02, momentum=0.9, weight_decay=0.1)
    for k in range(3):
        graph.replay()
        if k:
            muon_step(p, g, m, lr=0.02, momentum=0.9, weight_decay=0.1)
        torch.cuda.synchronize()
        for a, b in zip(twin[0] + twin[2], p + m):
            assert torch.equal(a, b)
