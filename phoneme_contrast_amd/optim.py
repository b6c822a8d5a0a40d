"""Fused optimizers over one flat parameter buffer, and the orthogonalisation they use.

FusedAdam — drop-in for the reference's optimizer.

The reference builds `torch.optim.Adam(model.parameters(), lr, weight_decay)` (scripts/train.py:
129-133): coupled L2 decay, betas (0.9, 0.999), eps 1e-8, bias correction.  FusedAdam keeps that
exact update but re-homes every parameter of a group into one contiguous fp32 buffer and runs a
single libpcx kernel (pcx_adam_step) per step instead of one torch kernel chain per tensor.
`state_dict()` is laid out like torch.optim.Adam's (per-parameter step / exp_avg / exp_avg_sq),
so checkpoints written by the trainer load into either optimizer.

FusedMuon updates weight matrices by their orthogonalised momentum and everything else as FusedAdam does
(`accel.optimizer: muon` in scripts/train.py); `muon_step` is the same update for a list of tensors and `orthogonalize`
the Newton-Schulz iteration alone (csrc/muon.hip).
"""
import ctypes
import functools
import math

import torch

from . import _lib


class FusedAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        self._check_adam(lr, betas, eps, weight_decay)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._flat = [None] * len(self.param_groups)

    @staticmethod
    def _check_adam(lr, betas, eps, weight_decay):
        if lr < 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if eps < 0.0:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"Invalid beta parameters: {betas}")
        if weight_decay < 0.0:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")

    # ------------------------------------------------------------------ flat storage
    def _group_flat(self, gi):
        group = self.param_groups[gi]
        ps = group["params"]
        st = self._flat[gi]
        if st is not None and self._bound(st, ps):
            return st
        dev = ps[0].device
        _lib.require_gpu(ps[0], what="FusedAdam")
        n = sum(p.numel() for p in ps)
        flat = torch.empty(n, device=dev, dtype=torch.float32)
        m = torch.zeros(n, device=dev, dtype=torch.float32)
        v = torch.zeros(n, device=dev, dtype=torch.float32)
        step = 0
        off = 0
        # parameters re-bound behind the optimizer's back (model.to(), load_state_dict(assign=True)):
        # the moments and step count of the previous flat buffers carry over; state loaded through
        # load_state_dict (which drops the flat buffers) comes from self.state
        prev = st if st is not None and st["n"] == n else None
        for p in ps:
            k = p.numel()
            flat[off:off + k].copy_(p.detach().reshape(-1))
            s = self.state.get(p)
            if prev is not None:
                m[off:off + k].copy_(prev["m"][off:off + k])
                v[off:off + k].copy_(prev["v"][off:off + k])
                step = prev["step"]
            elif s and "exp_avg" in s:
                m[off:off + k].copy_(s["exp_avg"].reshape(-1))
                v[off:off + k].copy_(s["exp_avg_sq"].reshape(-1))
                step = int(s["step"])
            p.data = flat[off:off + k].view_as(p)
            off += k
        st = {"flat": flat, "m": m, "v": v, "step": step, "n": n, "stage": None}
        self._flat[gi] = st
        return st

    @staticmethod
    def _bound(st, ps):
        base = st["flat"].data_ptr()
        off = 0
        for p in ps:
            if p.data_ptr() != base + 4 * off:
                return False
            off += p.numel()
        return True

    @staticmethod
    def _flat_grad(st, ps):
        """The group's gradients as one flat tensor: a zero-copy view when the backward produced
        them contiguously in parameter order (libpcx does), else one gather copy."""
        g0 = ps[0].grad
        # zero-copy only when the view starts 16-byte aligned (pcx_adam_step's vector loads): a
        # second parameter group's gradients can sit at any offset of the backward's flat buffer
        if g0 is not None and g0.is_contiguous() and g0.data_ptr() % 16 == 0:
            base, sto = g0.data_ptr(), g0.untyped_storage().data_ptr()
            off, ok = 0, True
            for p in ps:
                g = p.grad
                if (g is None or not g.is_contiguous() or g.data_ptr() != base + 4 * off
                        or g.untyped_storage().data_ptr() != sto or g.dtype != torch.float32):
                    ok = False
                    break
                off += p.numel()
            if ok:
                return torch.empty(0, device=g0.device).set_(g0.untyped_storage(), g0.storage_offset(),
                                                             (st["n"],), (1,))
        if st["stage"] is None:
            st["stage"] = torch.empty_like(st["flat"])
        buf, off = st["stage"], 0
        for p in ps:
            k = p.numel()
            if p.grad is None:
                raise RuntimeError("FusedAdam: every parameter of a group needs a gradient")
            buf[off:off + k].copy_(p.grad.reshape(-1))
            off += k
        return buf

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None, flat_grads=None, grad_scale=1.0):
        """Adam step.  `flat_grads` (one flat tensor per group, e.g. after an all-reduce) bypasses
        the p.grad gather; `grad_scale` multiplies the gradient first (1/world_size)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _lib.lib()
        for gi, group in enumerate(self.param_groups):
            ps = group["params"]
            if not ps:
                continue
            st = self._group_flat(gi)
            if flat_grads is not None:
                g = flat_grads[gi]
            else:
                if all(p.grad is None for p in ps):
                    continue
                g = self._flat_grad(st, ps)
            st["step"] += 1
            b1, b2 = group["betas"]
            _lib.check(lib.pcx_adam_step(_lib.ptr(st["flat"]), _lib.ptr(g), _lib.ptr(st["m"]),
                                         _lib.ptr(st["v"]), st["n"], st["step"], float(group["lr"]),
                                         float(b1), float(b2), float(group["eps"]),
                                         float(group["weight_decay"]), float(grad_scale),
                                         _lib.stream_of(st["flat"])), "pcx_adam_step")
        return loss

    def flat_grad_views(self):
        """Flat gradient tensors (one per group), zero-copy when possible — for all-reduce."""
        out = []
        for gi, group in enumerate(self.param_groups):
            st = self._group_flat(gi)
            out.append(self._flat_grad(st, group["params"]))
        return out

    # ------------------------------------------------------------------ torch.optim.Adam-style state
    def state_dict(self):
        for gi, group in enumerate(self.param_groups):
            st = self._flat[gi]
            if st is None:
                continue
            off = 0
            for p in group["params"]:
                k = p.numel()
                self.state[p] = {"step": torch.tensor(float(st["step"])),
                                 "exp_avg": st["m"][off:off + k].view_as(p).clone(),
                                 "exp_avg_sq": st["v"][off:off + k].view_as(p).clone()}
                off += k
        return super().state_dict()

    def load_state_dict(self, state_dict):
        own = isinstance(self, FusedMuon)  # (torch.optim.Muon's groups have ns_steps too)
        if any(("ns_eps" in g) != own or ("ns_steps" in g) != own for g in state_dict["param_groups"]):
            raise ValueError(f"{type(self).__name__}: this is the state of another optimizer")
        super().load_state_dict(state_dict)
        self._flat = [None] * len(self.param_groups)


# ----------------------------------------------------------------------------- orthogonalised updates
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # five steps take singular values in [0.01, 1] into [0.7, 1.2]


@functools.lru_cache(maxsize=32)
def _ns_coefficients(coefficients, steps):
    """(a, b, c), or one such triple per step, as the C array of 3 * steps floats."""
    if not 1 <= steps <= 64:
        raise ValueError(f"ns_steps must be 1 to 64, got {steps}")
    if len(coefficients) == 3 and all(isinstance(v, (int, float)) for v in coefficients):
        coefficients = (coefficients,) * steps
    if len(coefficients) != steps or any(len(t) != 3 for t in coefficients):
        raise ValueError("ns_coefficients must be three numbers, or as many triples as ns_steps")
    flat = [float(v) for t in coefficients for v in t]
    return (ctypes.c_float * len(flat))(*flat)


def _coefficients(coefficients, steps):
    return _ns_coefficients(tuple(tuple(t) if isinstance(t, (list, tuple)) else t for t in coefficients), int(steps))


@functools.lru_cache(maxsize=256)
def _orthogonalize_bytes(batch, rows, cols):
    n = _lib.lib().pcx_orthogonalize_workspace_bytes(batch, rows, cols)
    if n == 0:
        raise ValueError(f"orthogonalize: {batch} matrices of {rows} x {cols} are not supported")
    return n


@torch.no_grad()
def orthogonalize(x, ns_steps=5, ns_coefficients=NS_COEFFICIENTS, eps=1e-7):
    """The matrices of x ([..., rows, cols]; float32, bfloat16 or float16, any strides) with their singular values taken
    to about 1 by `ns_steps` Newton-Schulz steps: X = x / (|x|_F + eps), then X <- a X + (b A + c A A) X, A = X X^T.

    `ns_coefficients`: (a, b, c), or one triple per step.  Computed for every type with sums in float32 and rounded once to
    x's: in float32 throughout where the short side is at most 32, else from operands of 22 bits, whose error is below float32
    arithmetic's own (but for a matrix whose norm is under a hundredth of eps: below 5e-6, where float32 arithmetic has 1e-7).
    A zero matrix stays zero, one with a value that is not finite becomes NaN.  Not differentiable (the result
    carries no gradient)."""
    _lib.require_gpu(x, what="orthogonalize")
    if x.dtype not in _lib.DTYPES:
        raise ValueError(f"orthogonalize: float32, bfloat16 or float16 expected, got {x.dtype}")
    if x.dim() < 2:
        raise ValueError(f"orthogonalize: matrices expected, got a tensor of shape {tuple(x.shape)}")
    coef = _coefficients(ns_coefficients, ns_steps)
    if not 0.0 < float(eps) < float("inf"):
        raise ValueError(f"orthogonalize: eps must be positive, got {eps}")
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return out
    x = x.resolve_neg()  # (the kernels read memory)
    rows, cols = x.shape[-2:]
    if x.dim() == 2:
        batch, bstride = 1, 0
    else:
        x = x.reshape(-1, rows, cols)  # (a copy where the leading axes are not evenly spaced)
        batch, bstride = x.shape[0], x.stride(0)
    nws = _orthogonalize_bytes(batch, rows, cols)
    ws = torch.empty(nws, dtype=torch.uint8, device=x.device)
    with _lib.on_device(x):
        _lib.check(_lib.lib().pcx_orthogonalize(_lib.DTYPES[x.dtype], batch, rows, cols, x.data_ptr(), bstride,
                                                x.stride(-2), x.stride(-1), out.data_ptr(), int(ns_steps), coef,
                                                float(eps), ws.data_ptr(), nws, _lib.raw_stream(x)),
                   "pcx_orthogonalize")
    return out


def _matrix_shape(p):
    """(rows, cols) of a weight: the first axis against the rest."""
    return p.shape[0], p.numel() // p.shape[0]


def _is_matrix(p):
    return p.dim() >= 2 and p.numel() > 0 and min(_matrix_shape(p)) > 1


def _update_scale(adjust, rows, cols):
    if adjust == "rms":  # an orthogonal rows x cols matrix has an RMS of 1 / sqrt(max): 0.2 is that of an Adam update
        return 0.2 * math.sqrt(max(rows, cols))
    if adjust == "spectral":
        return math.sqrt(max(1.0, rows / cols))
    if adjust is None:
        return 1.0
    raise ValueError(f'adjust must be "rms", "spectral" or None, got {adjust!r}')


def _check_muon(lr, momentum, weight_decay, eps):
    if not lr >= 0.0:
        raise ValueError(f"Invalid learning rate: {lr}")
    if not 0.0 <= momentum < 1.0:
        raise ValueError(f"Invalid momentum value: {momentum}")
    if not weight_decay >= 0.0:
        raise ValueError(f"Invalid weight_decay value: {weight_decay}")
    if not 0.0 < eps < float("inf"):
        raise ValueError(f"Invalid epsilon value: {eps}")


@torch.no_grad()
def muon_step(params, grads, momentum_buffers, *, lr, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="rms",
              ns_steps=5, ns_coefficients=NS_COEFFICIENTS, eps=1e-7, grad_scale=1.0):
    """One update of a list of weights by their orthogonalised momentum, in place, all of them in the same launches:

        buffer <- momentum buffer + (1 - momentum) grad_scale grad
        u       = (1 - momentum) grad_scale grad + momentum buffer   (nesterov), or buffer
        param  <- (1 - lr weight_decay) param - lr k orthogonalize(u)

    with k = 0.2 sqrt(max(rows, cols)) (adjust "rms": the size of an Adam update, so that its learning rate and decay
    serve), sqrt(max(1, rows / cols)) ("spectral") or 1 (None).  A weight of more than two axes is the matrix of its
    first axis against the rest.  Accuracy as in `orthogonalize`, except that short sides up to 32 take operands of 22
    bits too, with up to twice float32 arithmetic's error, in a list with others (each 16 in order count) unless all are small
    enough for one block (128 x 128, 64 x 512, 32 x 1024).  All tensors float32, contiguous and on one GPU; no parameter or buffer shares memory
    with another tensor of the call (a gradient may appear twice)."""
    params, grads, buffers = list(params), list(grads), list(momentum_buffers)
    if not len(params) == len(grads) == len(buffers):
        raise ValueError(f"muon_step: {len(params)} parameters, {len(grads)} gradients, {len(buffers)} momentum buffers")
    _check_muon(lr, momentum, weight_decay, eps)
    coef = _coefficients(ns_coefficients, ns_steps)
    _update_scale(adjust, 1, 1)
    if not params:
        return
    _lib.require_gpu(params[0], what="muon_step")
    dev = params[0].device
    mats = (_lib.MuonMatrix * len(params))()
    spans = []
    for i, (p, g, m) in enumerate(zip(params, grads, buffers)):
        if p.dim() < 2 or p.numel() == 0:
            raise ValueError(f"muon_step: parameter {i} of shape {tuple(p.shape)} is no matrix")
        for name, t in (("parameter", p), ("gradient", g), ("momentum buffer", m)):
            if t.device != dev:
                _lib.require_gpu(t, what="muon_step")
                raise RuntimeError(f"muon_step: {name} {i} is on {t.device}, parameter 0 on {dev}")
            if t.shape != p.shape:
                raise ValueError(f"muon_step: {name} {i} has shape {tuple(t.shape)}, {tuple(p.shape)} expected")
            if t.dtype != torch.float32 or not t.is_contiguous() or t.is_neg():
                raise ValueError(f"muon_step: {name} {i} must be contiguous float32 in memory")
            spans.append((t.data_ptr(), t.data_ptr() + 4 * t.numel(), name != "gradient"))
        rows, cols = _matrix_shape(p)
        e = mats[i]
        e.param, e.grad, e.momentum, e.rows, e.cols = p.data_ptr(), g.data_ptr(), m.data_ptr(), rows, cols
        e.scale = _update_scale(adjust, rows, cols)
    any_end = written_end = 0  # (gradients are read again once the buffers are written: only they may share memory)
    for start, end, is_written in sorted(spans):
        if start < written_end or (is_written and start < any_end):
            raise ValueError("muon_step: a parameter or momentum buffer shares memory with another tensor of the call")
        any_end = max(any_end, end)
        written_end = max(written_end, end) if is_written else written_end
    _muon_launch(mats, len(params), params[0], lr, momentum, nesterov, weight_decay, grad_scale, ns_steps, coef, eps)
    torch.autograd.graph.increment_version(params + buffers)  # (autograd cannot see the kernels' writes)


def _muon_launch(mats, n, at, lr, momentum, nesterov, weight_decay, grad_scale, ns_steps, coef, eps, nws=None):
    lib = _lib.lib()
    if nws is None:
        nws = lib.pcx_muon_workspace_bytes(mats, n)
    if nws == 0:
        raise ValueError(_lib.last_error())
    ws = torch.empty(nws, dtype=torch.uint8, device=at.device)
    with _lib.on_device(at):
        _lib.check(lib.pcx_muon_step(mats, n, float(lr), float(momentum), 1 if nesterov else 0, float(weight_decay),
                                     float(grad_scale), int(ns_steps), coef, float(eps), ws.data_ptr(), nws,
                                     _lib.raw_stream(at)), "pcx_muon_step")


class FusedMuon(FusedAdam):
    """Orthogonalised momentum for the weight matrices (`muon_step`), FusedAdam's update for the other parameters.

    A parameter of two or more axes whose rows and columns both number more than one is a matrix; biases, norms and the
    1 x C attention weight take Adam with `betas` and `eps`.  A group with `muon=False` takes Adam throughout.  One `lr`
    serves both with adjust="rms" (see muon_step); `weight_decay` is decoupled for matrices and coupled for the rest, as
    in FusedAdam.  Parameters, gradients and momentum live in one flat float32 buffer per group, in parameter order, so
    the trainer's clipping, all-reduce buckets and `flat_grads` work as with FusedAdam."""

    def __init__(self, params, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="rms", ns_steps=5,
                 ns_coefficients=NS_COEFFICIENTS, ns_eps=1e-7, betas=(0.9, 0.999), eps=1e-8):
        self._check_adam(lr, betas, eps, weight_decay)
        _check_muon(lr, momentum, weight_decay, ns_eps)
        _coefficients(ns_coefficients, ns_steps)
        _update_scale(adjust, 1, 1)
        torch.optim.Optimizer.__init__(self, params, dict(
            lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, adjust=adjust,
            ns_steps=ns_steps, ns_coefficients=ns_coefficients, ns_eps=ns_eps, muon=True))
        self._flat = [None] * len(self.param_groups)

    def _group_flat(self, gi):
        group = self.param_groups[gi]
        ps = group["params"]
        st = self._flat[gi]
        if st is not None and self._bound(st, ps):
            return st
        _lib.require_gpu(ps[0], what="FusedMuon")
        dev = ps[0].device
        n = sum(p.numel() for p in ps)
        kinds = [bool(group["muon"]) and _is_matrix(p) for p in ps]
        prev = st if st is not None and st["n"] == n and st["kinds"] == kinds else None
        flat = torch.empty(n, device=dev, dtype=torch.float32)
        m = torch.zeros(n, device=dev, dtype=torch.float32)  # momentum of matrices, exp_avg of the rest
        v = torch.zeros(sum(p.numel() for p, k in zip(ps, kinds) if not k), device=dev, dtype=torch.float32)
        step, off, voff, places, segs = 0, 0, 0, [], []
        for p, is_mat in zip(ps, kinds):
            k, s = p.numel(), self.state.get(p)
            flat[off:off + k].copy_(p.detach().reshape(-1))
            if prev is None and s and "step" in s:
                step = int(s["step"])
                m[off:off + k].copy_(s["momentum_buffer" if is_mat else "exp_avg"].reshape(-1))
                if not is_mat:
                    v[voff:voff + k].copy_(s["exp_avg_sq"].reshape(-1))
            if is_mat:
                places.append((off, *_matrix_shape(p)))
            else:
                if segs and segs[-1][0] + segs[-1][2] == off:
                    segs[-1][2] += k
                else:
                    segs.append([off, voff, k])
                voff += k
            p.data = flat[off:off + k].view_as(p)
            off += k
        if prev is not None:  # parameters re-bound behind the optimizer's back: its own state carries over
            m.copy_(prev["m"])
            v.copy_(prev["v"])
            step = prev["step"]
        mats = (_lib.MuonMatrix * len(places))()
        for e, (o, rows, cols) in zip(mats, places):
            e.param, e.momentum, e.rows, e.cols = flat.data_ptr() + 4 * o, m.data_ptr() + 4 * o, rows, cols
        st = {"flat": flat, "m": m, "v": v, "step": step, "n": n, "stage": None, "kinds": kinds, "places": places,
              "mats": mats, "segs": (_lib.Segment * len(segs))(*[tuple(s) for s in segs]),
              "nws": _lib.lib().pcx_muon_workspace_bytes(mats, len(places)) if places else 0}
        if places and st["nws"] == 0:
            raise ValueError(_lib.last_error())
        self._flat[gi] = st
        return st

    @torch.no_grad()
    def step(self, closure=None, flat_grads=None, grad_scale=1.0):
        """One step; `flat_grads` and `grad_scale` as in FusedAdam.step."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _lib.lib()
        for gi, group in enumerate(self.param_groups):
            ps = group["params"]
            if not ps or (flat_grads is None and all(p.grad is None for p in ps)):
                continue
            st = self._group_flat(gi)
            g = flat_grads[gi] if flat_grads is not None else self._flat_grad(st, ps)
            if g.numel() != st["n"] or g.dtype != torch.float32 or not g.is_contiguous() or g.device != st["flat"].device:
                raise ValueError(f"FusedMuon: flat gradient of group {gi} must be {st['n']} contiguous float32 values on "
                                 f"{st['flat'].device}")
            st["step"] += 1
            base = g.data_ptr()
            if st["places"]:
                for e, (o, rows, cols) in zip(st["mats"], st["places"]):
                    e.grad, e.scale = base + 4 * o, _update_scale(group["adjust"], rows, cols)
                _muon_launch(st["mats"], len(st["places"]), st["flat"], group["lr"], group["momentum"], group["nesterov"],
                             group["weight_decay"], grad_scale, group["ns_steps"],
                             _coefficients(group["ns_coefficients"], group["ns_steps"]), group["ns_eps"], st["nws"])
            if len(st["segs"]):
                b1, b2 = group["betas"]
                with _lib.on_device(st["flat"]):
                    _lib.check(lib.pcx_adam_segments(st["flat"].data_ptr(), base, st["m"].data_ptr(), st["v"].data_ptr(),
                                                     st["segs"], len(st["segs"]), st["step"], float(group["lr"]),
                                                     float(b1), float(b2), float(group["eps"]),
                                                     float(group["weight_decay"]), float(grad_scale),
                                                     _lib.raw_stream(st["flat"])), "pcx_adam_segments")
            torch.autograd.graph.increment_version(ps)  # (as in muon_step)
        return loss

    # ------------------------------------------------------------------ state: momentum_buffer, or Adam's moments
    def state_dict(self):
        for gi, group in enumerate(self.param_groups):
            st = self._flat[gi]
            if st is None:
                continue
            off = voff = 0
            for p, is_mat in zip(group["params"], st["kinds"]):
                k = p.numel()
                own = st["m"][off:off + k].view_as(p).clone()
                if is_mat:
                    self.state[p] = {"step": torch.tensor(float(st["step"])), "momentum_buffer": own}
                else:
                    self.state[p] = {"step": torch.tensor(float(st["step"])), "exp_avg": own,
                                     "exp_avg_sq": st["v"][voff:voff + k].view_as(p).clone()}
                    voff += k
                off += k
        return torch.optim.Optimizer.state_dict(self)
