"""Layer norm (fc3d.ops.layer_norm, fc3d_layer_norm_fwd / _bwd) against its formula in 64 bits.

Tolerances, with u = 2^-24 and r the half step of the output's type (eps / 2 relative to the value):
a sum of n terms added along chains of at most k additions is off by k u sum|terms|.  The longest chain of the
kernels' channel sums is below 48 additions for the sizes here (16 values a lane, 6 steps across a wavefront, 16
wavefronts; 18 + 18 in the long form), of the sums over positions below 128 (5 rounds, 32 row groups, 32 + 32
partial sums).  The statistics, the normalised value and the results follow by adding the terms' bounds."""
import pytest
import torch

U = 2.0 ** -24
KC, KP = 48 * U, 128 * U          # channel sums, position sums


def half_step(dt):
    return torch.finfo(dt).eps / 2


def formula(x, w, b, dy, dim, eps, mask=None):
    """y, dx, dw, db and their bounds (without the output's own rounding) in 64 bits; tensors on the CPU."""
    x = x.double().movedim(dim, -1)
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    d = x - mu
    rs = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    h = d * rs
    # x - mu: the mean's error, then one rounding; 1 / sqrt(var + eps): relative KC for the sum, 4 U for the rest
    eh = rs * KC * x.abs().mean(-1, keepdim=True) + h.abs() * (KC + 6 * U)
    y = h * w + b
    ey = w.abs() * eh + 2 * U * (y.abs() + (h * w).abs())
    if mask is not None:
        y = torch.where(y > 0, y, torch.zeros_like(y))
    out = dict(y=y.movedim(-1, dim), ey=ey.movedim(-1, dim))
    if dy is not None:
        g = dy.double().movedim(dim, -1)
        if mask is not None:
            g = g * mask.movedim(dim, -1)
        gw = g * w
        m1, m2 = gw.mean(-1, keepdim=True), (gw * h).mean(-1, keepdim=True)
        e1 = (KC + 2 * U) * gw.abs().mean(-1, keepdim=True)
        e2 = (KC + 3 * U) * (gw * h).abs().mean(-1, keepdim=True) + (gw.abs() * eh).mean(-1, keepdim=True)
        dx = rs * (gw - m1 - h * m2)
        edx = rs * (e1 + eh * m2.abs() + h.abs() * e2 + 4 * U * (gw.abs() + m1.abs() + (h * m2).abs())) + dx.abs() * (KC + 6 * U)
        pos = tuple(range(g.dim() - 1))
        out.update(dx=dx.movedim(-1, dim), edx=edx.movedim(-1, dim), dw=(g * h).sum(pos), db=g.sum(pos),
                   edw=(KP * (g * h).abs() + g.abs() * eh).sum(pos), edb=KP * g.abs().sum(pos))
    return out


def close(got, ref, bound, dt, what):
    got, ref = got.detach().cpu().double(), ref.to(torch.float64)
    assert got.shape == ref.shape, what
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    tol = bound + half_step(dt) * (ref.abs() + bound) + tiny
    off = (got - ref).abs()
    bad = ~(off <= tol)
    bad = torch.where(torch.isnan(ref), ~torch.isnan(got), bad)      # an infinite input leaves NaN in its position
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.2f} of the bound"


def inputs(shape, dim, dt, wdt, seed, wide=1.0):
    g = torch.Generator().manual_seed(seed)
    lead = list(shape)
    lead[dim] = 1
    x = (wide * torch.randn(shape, generator=g) + torch.randn(lead, generator=g)).to(dt)
    w = None if wdt is None else (1 + 0.3 * torch.randn(shape[dim], generator=g)).to(wdt)
    b = None if wdt is None else (0.3 * torch.randn(shape[dim], generator=g)).to(wdt)
    dy = torch.randn(shape, generator=g).to(dt)
    return x, w, b, dy


# rows: one value, one row, rows shorter than a vector, odd lengths, every number of lanes per row, beyond the registers;
# planes: odd and tiny planes, one position, every number of channel groups, single values, beyond the registers
SHAPES = [((1, 1), -1), ((3, 2), -1), ((1, 1024), -1), ((70, 3), -1), ((513, 51), -1), ((4097, 96), -1), ((130, 500), -1),
          ((2000, 777), -1), ((2, 3, 1000), -1), ((1030, 2048), -1), ((9, 4099), -1), ((3, 16384), -1), ((5, 16390), -1),
          ((2, 32, 16, 16), 1), ((3, 200, 5, 7), 1), ((1, 1, 9, 9), 1), ((2, 5, 1, 3), 1), ((2, 64, 33, 31), 1),
          ((2, 512, 8, 12), 1), ((2, 700, 3, 5), 1), ((1, 1100, 3, 5), 1), ((6, 16, 1, 1), 1), ((4, 7, 130), 1),
          ((40, 6, 5, 3), 0), ((3, 128, 45, 77), 1), ((40, 32, 32, 32), 1)]
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, None), (F32, None)]


# ---- on the CPU: the formula itself, and what is refused -----------------------------------------------------

def test_formula_against_differences():
    torch.manual_seed(0)
    x, w, b = (torch.randn(s, dtype=torch.float64, requires_grad=True) for s in ((4, 7, 5), (7,), (7,)))

    def f(x, w, b):
        xm = x.movedim(1, -1)
        d = xm - xm.mean(-1, keepdim=True)
        return (d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5) * w + b).movedim(-1, 1)
    assert torch.autograd.gradcheck(f, (x, w, b), eps=1e-6, atol=1e-7)
    dy = torch.randn(4, 7, 5, dtype=torch.float64)
    dx, dw, db = torch.autograd.grad(f(x, w, b), (x, w, b), dy)
    r = formula(x.detach(), w.detach(), b.detach(), dy, 1, 1e-5)
    for a, k in ((dx, "dx"), (dw, "dw"), (db, "db")):
        assert torch.allclose(a, r[k], rtol=1e-12, atol=1e-12), k


def test_refusals():
    from fc3d import _native, ops
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.layer_norm(x)
    lib = _native.load()
    one = 16
    fwd = lambda **k: lib.fc3d_layer_norm_fwd(None, *[{**dict(x=one, t=0, w=None, b=None, wt=0, outer=2, C=8, inner=1, st=8,  # noqa: E731
                                                               eps=1e-5, relu=0, y=one, m=None, r=None), **k}[n] for n in
                                                       ("x", "t", "w", "b", "wt", "outer", "C", "inner", "st", "eps", "relu", "y", "m", "r")])
    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(t=3) == -1 and fwd(t=-1) == -1
    assert fwd(t=1, wt=2) == -1                                   # weights in another 16-bit type
    assert fwd(C=0) == -1 and fwd(inner=0) == -1 and fwd(outer=-1) == -1 and fwd(st=-1) == -1
    assert fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1
    assert fwd(m=one) == -1                                       # one of the two statistics
    assert fwd(outer=1 << 20, inner=1 << 12) == -2 and fwd(C=1 << 24) == -2 and fwd(outer=1 << 40) == -2
    assert fwd(x=18) == -3 and fwd(t=1, wt=1, x=17) == -3 and fwd(w=18) == -3
    assert fwd(outer=0, x=None, y=None) == 0                      # nothing to do, nothing launched
    bwd = lambda **k: lib.fc3d_layer_norm_bwd(None, *[{**dict(dy=one, x=one, t=0, w=None, b=None, wt=0, m=one, r=one, outer=2, C=8,  # noqa: E731
                                                               inner=1, gst=8, st=8, relu=0, dx=one, dw=None, db=None, ws=None), **k}[n]
                                                       for n in ("dy", "x", "t", "w", "b", "wt", "m", "r", "outer", "C", "inner", "gst",
                                                                 "st", "relu", "dx", "dw", "db", "ws")])
    assert bwd(dy=None) == -1 and bwd(m=None) == -1 and bwd(dw=one) == -1 and bwd(gst=-1) == -1 and bwd(dx=18) == -3
    assert bwd(dx=None) == 0
    assert lib.fc3d_layer_norm_bwd_workspace(0, 0, 8, 1) == 0 and lib.fc3d_layer_norm_bwd_workspace(0, 5, 0, 1) == 0
    assert lib.fc3d_layer_norm_bwd_workspace(0, 5, 4096, 1) == 5 * 2 * 4096 * 4         # a row per workgroup
    n = lib.fc3d_layer_norm_bwd_workspace(0, 1 << 20, 64, 1)                            # bounded, however many rows
    assert n % (2 * 64 * 4) == 0 and 256 <= n // (2 * 64 * 4) <= 2048


def test_strides_of_merged_axes():
    from fc3d.ops import _one_stride
    t = torch.empty(4, 5, 6)
    assert _one_stride(t.shape, t.stride()) == 1
    assert _one_stride(t[:, :, ::2].shape, t[:, :, ::2].stride()) == 2
    v = t[:, :4]
    assert _one_stride(v.shape, v.stride()) is None and _one_stride(v.shape[1:], v.stride()[1:]) == 1
    e = torch.empty(1, 6).expand(4, 6)
    assert _one_stride(e.shape, e.stride()) is None and _one_stride((4,), (0,)) == 0 and _one_stride((1, 1), (9, 9)) == 0


# ---- on the GPU -----------------------------------------------------------------------------------------------

gpu = pytest.mark.gpu


def run(ops, x, w, b, dy, dim, relu, eps=1e-5):
    leaves = [t.cuda().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = ops.layer_norm(*leaves, eps=eps, dim=dim, relu=relu)
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dy.cuda())
    return y, list(got) + [None] * (3 - len(got))


@gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(v).replace("torch.", "") for v in t))
@pytest.mark.parametrize("shape,dim", SHAPES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else None)
def test_against_formula(shape, dim, types):
    from fc3d import ops
    dt, wdt = types
    for relu in (False, True):
        x, w, b, dy = inputs(shape, dim, dt, wdt, 11)
        y, (dx, dw, db) = run(ops, x, w, b, dy, dim, relu)
        mask = None
        if relu:                         # which values passed is the forward's decision, checked by y itself
            mask = (y.detach().cpu() > 0).double()
        r = formula(x, w, b, dy, dim, 1e-5, mask)
        close(y, r["y"], r["ey"], dt, f"y relu={relu}")
        close(dx, r["dx"], r["edx"], dt, f"dx relu={relu}")
        if wdt is not None:
            close(dw, r["dw"], r["edw"], wdt, f"dw relu={relu}")
            close(db, r["db"], r["edb"], wdt, f"db relu={relu}")
        with torch.no_grad():            # the call without statistics gives the same bits
            assert torch.equal(ops.layer_norm(x.cuda(), None if w is None else w.cuda(), None if b is None else b.cuda(),
                                              dim=dim, relu=relu), y)


@gpu
def test_partial_gradients_and_single_parameters():
    from fc3d import ops
    x, w, b, dy = inputs((37, 129), -1, F32, F32, 3)
    r = formula(x, w, None, dy, -1, 1e-5)
    xd, wd = x.cuda(), w.cuda().requires_grad_()
    y = ops.layer_norm(xd, wd)                                   # a weight alone, x without gradient
    (dw,) = torch.autograd.grad(y, wd, dy.cuda())
    close(y, r["y"], r["ey"], F32, "y")
    close(dw, r["dw"], r["edw"], F32, "dw")
    r = formula(x, None, b, dy, -1, 1e-5)
    bd = b.cuda().requires_grad_()
    y = ops.layer_norm(xd, bias=bd)
    (db,) = torch.autograd.grad(y, bd, dy.cuda())
    close(y, r["y"], r["ey"], F32, "y")
    close(db, r["db"], r["edb"], F32, "db")
    y = ops.layer_norm(xd.requires_grad_(), w.cuda(), b.cuda())  # frozen parameters
    (dx,) = torch.autograd.grad(y, xd, dy.cuda())
    r = formula(x, w, b, dy, -1, 1e-5)
    close(dx, r["dx"], r["edx"], F32, "dx")


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
def test_strides_and_alignment(dt):
    from fc3d import ops
    x, w, b, dy = inputs((3, 24, 10, 14), 1, dt, F32, 5)
    r = formula(x, w, b, dy, 1, 1e-5)
    base = torch.zeros(x.numel() + 1, dtype=dt, device="cuda")
    base[1:] = x.reshape(-1).cuda()
    off = base[1:].view(x.shape)                                   # starts in the middle of a vector
    wide = torch.full((3, 30, 10, 14), 7.0, dtype=dt, device="cuda")
    wide[:, 3:27] = x.cuda()
    cases = {"channels_last": x.cuda().contiguous(memory_format=torch.channels_last), "offset": off, "sliced": wide[:, 3:27],
             "transposed": x.cuda().transpose(2, 3).contiguous().transpose(2, 3)}
    for name, xs in cases.items():
        xs = xs.detach().requires_grad_()
        y = ops.layer_norm(xs, w.cuda(), b.cuda(), dim=1)
        (dx,) = torch.autograd.grad(y, xs, dy.cuda())
        close(y, r["y"], r["ey"], dt, name)
        close(dx, r["dx"], r["edx"], dt, name)
        if name == "channels_last":
            assert y.is_contiguous(memory_format=torch.channels_last) and dx.is_contiguous(memory_format=torch.channels_last)
    x, w, b, dy = inputs((6, 5, 65), -1, dt, F32, 6)
    rows = torch.zeros(6, 5, 70, dtype=dt, device="cuda")
    rows[..., 2:67] = x.cuda()
    for dyv in (dy, dy[:1, :1].expand(6, 5, 65), torch.ones((), dtype=dt).expand(6, 5, 65)):
        r = formula(x, w, b, dyv, -1, 1e-5)
        xs = rows[..., 2:67].detach().requires_grad_()
        y = ops.layer_norm(xs, w.cuda(), b.cuda())
        (dx,) = torch.autograd.grad(y, xs, dyv.cuda() if dyv is dy else dyv[:1, :1, :].cuda().expand(6, 5, 65))
        close(y, r["y"], r["ey"], dt, "rows of a wider tensor")
        close(dx, r["dx"], r["edx"], dt, "rows of a wider tensor")
    # the normalised axis contiguous in the middle, the others not walked with one stride, all sizes alike
    x, w, b, dy = inputs((4, 4, 4), 1, dt, F32, 7)
    r = formula(x, w, b, dy, 1, 1e-5)
    xs = torch.zeros(4, 6, 4, dtype=dt, device="cuda")
    xs[:, :4] = x.cuda().transpose(1, 2)
    xs = xs[:, :4].transpose(1, 2).detach().requires_grad_()
    y = ops.layer_norm(xs, w.cuda(), b.cuda(), dim=1)
    (dx,) = torch.autograd.grad(y, xs, dy.cuda())
    close(y, r["y"], r["ey"], dt, "middle axis")
    close(dx, r["dx"], r["edx"], dt, "middle axis")
    x = inputs((6, 5, 65), -1, dt, F32, 6)[0]
    w, b = inputs((6, 5, 65), -1, dt, F32, 6)[1:3]
    one = x[:1, :1].cuda().expand(6, 5, 65)
    r = formula(one.cpu(), w, b, None, -1, 1e-5)
    close(ops.layer_norm(one, w.cuda(), b.cuda()), r["y"], r["ey"], dt, "expanded input")


@gpu
@pytest.mark.parametrize("shape,dim", [((37, 51), -1), ((9, 4099), -1), ((3, 16400), -1), ((2, 33, 7, 9), 1), ((2, 1030, 3, 3), 1)])
@pytest.mark.parametrize("dt", [F32, F16])
def test_writes_nothing_beyond_its_outputs(shape, dim, dt):
    from fc3d import _native
    lib = _native.load()
    x, w, b, dy = inputs(shape, dim, dt, dt, 8)
    C, code, n = shape[dim], 0 if dt == F32 else 2, x.numel()
    outer, inner = (n // C, 1) if dim == -1 else (shape[0], n // shape[0] // C)
    d = {k: t.cuda() for k, t in dict(x=x, w=w, b=b, dy=dy).items()}
    pad = 64

    def guarded(count, t):
        return torch.full((count + 2 * pad,), 12288.0, dtype=t, device="cuda")
    y, dx, m, rs = guarded(n, dt), guarded(n, dt), guarded(outer * inner, F32), guarded(outer * inner, F32)
    dw, db = guarded(C, dt), guarded(C, dt)
    ws_n = lib.fc3d_layer_norm_bwd_workspace(code, outer, C, inner) // 4
    ws = guarded(ws_n, F32)
    at = lambda t: t.data_ptr() + pad * t.element_size()  # noqa: E731
    s = torch.cuda.current_stream().cuda_stream
    p = {k: t.data_ptr() for k, t in d.items()}
    assert lib.fc3d_layer_norm_fwd(s, p["x"], code, p["w"], p["b"], code, outer, C, inner, C * inner, 1e-5, 1, at(y), at(m), at(rs)) == 0
    assert lib.fc3d_layer_norm_bwd(s, p["dy"], p["x"], code, p["w"], p["b"], code, at(m), at(rs), outer, C, inner, C * inner,
                                   C * inner, 1, at(dx), at(dw), at(db), at(ws)) == 0
    torch.cuda.synchronize()
    for t in (y, dx, m, rs, dw, db, ws):
        assert bool((t[:pad] == 12288.0).all()) and bool((t[-pad:] == 12288.0).all())
    for t in (y, dx, m, rs, dw, db):
        assert not bool((t[pad:-pad] == 12288.0).any())


@gpu
def test_special_values_stay_in_their_positions():
    from fc3d import ops
    for shape, dim in (((9, 300), -1), ((2, 40, 3, 5), 1)):
        x, w, b, dy = inputs(shape, dim, F32, F32, 9)
        bad = x.clone().movedim(dim, -1).reshape(-1, x.shape[dim])
        bad[1, 3], bad[4, 0], bad[6, 2] = float("nan"), float("inf"), float("-inf")
        x2 = bad.reshape(x.movedim(dim, -1).shape).movedim(-1, dim).contiguous()
        for relu in (False, True):
            y = ops.layer_norm(x2.cuda(), w.cuda(), b.cuda(), dim=dim, relu=relu)
            ref = ops.layer_norm(x.cuda(), w.cuda(), b.cuda(), dim=dim, relu=relu)
            ym, rm = (t.movedim(dim, -1).reshape(-1, x.shape[dim]) for t in (y, ref))
            hit = torch.tensor([i in (1, 4, 6) for i in range(ym.shape[0])])
            assert bool(torch.isnan(ym[hit.cuda()]).all())
            assert torch.equal(ym[~hit.cuda()], rm[~hit.cuda()])
        # constant positions: nothing but eps under the root, and the result is the bias
        y = ops.layer_norm(torch.full(shape, 3.25, device="cuda"), w.cuda(), b.cuda(), dim=dim)
        assert torch.equal(y.movedim(dim, -1), b.cuda().expand_as(y.movedim(dim, -1)))
    # values whose squares pass the range of a 16-bit type (one of them, in the first row, passes the type's own: infinite)
    x = (torch.randn(4, 64, generator=torch.Generator().manual_seed(1)) * 2.0e4).to(F16)
    r = formula(x, None, None, None, -1, 1e-5)
    close(ops.layer_norm(x.cuda()), r["y"], r["ey"], F16, "large fp16")


@gpu
def test_empty_and_checks():
    from fc3d import ops
    w = torch.ones(8, device="cuda", requires_grad=True)
    b = torch.ones(8, device="cuda", requires_grad=True)
    for shape in ((0, 8), (3, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = ops.layer_norm(x, w, b)
        assert y.shape == shape
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert dx.shape == shape and not dw.any() and not db.any()
    x = torch.zeros(4, 8, device="cuda")
    for bad, err in ((dict(weight=w[:4]), ValueError), (dict(bias=b.double()), TypeError), (dict(eps=-1.0), ValueError),
                     (dict(dim=2), ValueError), (dict(weight=w.half()), TypeError), (dict(weight=w.cpu()), RuntimeError)):
        with pytest.raises(err):
            ops.layer_norm(x, **bad)
    with pytest.raises(TypeError):
        ops.layer_norm(x.half(), w.detach().half(), b.detach())
    with pytest.raises(TypeError):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError):
        ops.layer_norm(torch.zeros(4, 0, device="cuda"))
    y = ops.layer_norm(x.requires_grad_(), w, b)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):                              # differentiable once
        dx.sum().backward()


@gpu
def test_directional_differences():
    """(f(x + h v) - f(x - h v)) / 2h of the kernel's forward against <dx, v> of its backward.  The difference of the
    exact function has the same truncation, taken from the formula in 64 bits; the rest is the forward's rounding."""
    from fc3d import ops
    for shape, dim in (((16, 96), -1), ((2, 24, 6, 5), 1)):
        x, w, b, dy = inputs(shape, dim, F32, F32, 12)
        v = torch.randn(shape, generator=torch.Generator().manual_seed(13))
        h = 2.0 ** -6
        y, (dx, dw, db) = run(ops, x, w, b, dy, dim, False)
        sides = [(x + s * h * v) for s in (1, -1)]
        with torch.no_grad():
            got = [(ops.layer_norm(t.cuda(), w.cuda(), b.cuda(), dim=dim).cpu().double() * dy.double()).sum() for t in sides]
        exact = [formula(t, w, b, None, dim, 1e-5) for t in sides]
        ref = [(e["y"] * dy.double()).sum() for e in exact]
        noise = sum(((e["ey"] + half_step(F32) * e["y"].abs()) * dy.double().abs()).sum() for e in exact) / (2 * h)
        fd, fd64 = (got[0] - got[1]) / (2 * h), (ref[0] - ref[1]) / (2 * h)
        assert abs(fd - fd64) <= noise
        r = formula(x, w, b, dy, dim, 1e-5)
        slope, trunc = (r["dx"] * v.double()).sum(), abs(fd64 - (r["dx"] * v.double()).sum())
        off = (dx.cpu().double() * v.double()).sum()
        assert abs(off - slope) <= (r["edx"] * v.double().abs()).sum() + half_step(F32) * (r["dx"] * v.double()).abs().sum()
        assert abs(fd - off) <= noise + trunc + (r["edx"] * v.double().abs()).sum() + half_step(F32) * (r["dx"] * v.double()).abs().sum()


@gpu
def test_same_bits_every_time_and_on_another_stream():
    from fc3d import ops
    for shape, dim in (((5000, 130), -1), ((8, 64, 40, 41), 1)):
        x, w, b, dy = inputs(shape, dim, BF16, BF16, 14)
        first = run(ops, x, w, b, dy, dim, True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = run(ops, x, w, b, dy, dim, True)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(first[0], again[0])
        for a, c in zip(first[1], again[1]):
            assert torch.equal(a, c)


@gpu
def test_forward_and_backward_in_a_graph():
    """Captured once, replayed on new inputs with eager work in between; two graphs do not share what they work on."""
    from fc3d import ops

    def capture(shape, dim, seed):
        x, w, b, dy = (t.cuda() for t in inputs(shape, dim, F32, F32, seed))
        leaves = [x.requires_grad_(), w.requires_grad_(), b.requires_grad_()]

        def step():
            y = ops.layer_norm(*leaves, dim=dim, relu=True)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side, capture_error_mode="thread_local"):
            outs = step()
        return g, leaves, dy, outs, step
    a = capture((700, 96), -1, 20)
    c = capture((2, 48, 20, 21), 1, 21)
    for turn in range(4):
        for (g, leaves, dy, outs, step), shape, dim in ((a, (700, 96), -1), (c, (2, 48, 20, 21), 1)):
            new = [t.cuda() for t in inputs(shape, dim, F32, F32, 30 + turn)]
            with torch.no_grad():
                for t, v in zip((*leaves, dy), new):
                    t.copy_(v)
        a[0].replay()
        c[0].replay()
        torch.cuda.synchronize()
        for g, leaves, dy, outs, step in (a, c):
            eager = step()
            torch.cuda.synchronize()
            for got, ref in zip(outs, eager):
                assert torch.equal(got, ref)


@gpu
def test_offsets_beyond_32_bits():
    """Values more than 2^32 elements apart: the last rows of a long stride, the last image of large planes."""
    from fc3d import ops
    big = torch.empty((1 << 32) + 4096, dtype=torch.bfloat16, device="cuda")
    rows = big.as_strided((3, 512), (1 << 31, 1))
    x = inputs((3, 512), -1, BF16, None, 22)[0]
    rows.copy_(x.cuda())
    r = formula(x, None, None, None, -1, 1e-5)
    close(ops.layer_norm(rows), r["y"], r["ey"], BF16, "rows")
    planes = big.as_strided((3, 16, 8, 8), (1 << 31, 64, 8, 1))
    x = inputs((3, 16, 8, 8), 1, BF16, None, 23)[0]
    planes.copy_(x.cuda())
    r = formula(x, None, None, None, 1, 1e-5)
    close(ops.layer_norm(planes, dim=1), r["y"], r["ey"], BF16, "planes")


@gpu
def test_second_derivatives_are_refused():
    from fc3d import ops
    x = torch.randn(6, 20, device="cuda", requires_grad=True)
    w = torch.randn(20, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w)
    first, = torch.autograd.grad(y.square().sum(), x, create_graph=True)        # the first derivative itself is there
    plain, = torch.autograd.grad(ops.layer_norm(x, w).square().sum(), x)
    assert torch.equal(first, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), x)


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16], ids=lambda t: str(t).replace("torch.", ""))
def test_gradients_of_one_workgroup(dt):
    """Few rows or positions: the sums are written as gradients at once, in the parameters' type, one or both."""
    from fc3d import ops
    for shape, dim in (((5, 24), -1), ((1, 5000), -1), ((2, 1800), -1), ((2, 24, 3, 5), 1), ((1, 300, 2, 3), 1)):
        C = shape[dim]
        g = torch.Generator().manual_seed(C)
        x, dy = (torch.randn(shape, generator=g).to(dt) for _ in range(2))
        for pt in {dt, torch.float32}:
            w, b = (torch.randn(C, generator=g).to(pt) for _ in range(2))
            xr, wr, br = (t.double().requires_grad_() for t in (x, w, b))
            ref = torch.nn.functional.layer_norm(xr.movedim(dim, -1), (C,), wr, br, 1e-5).movedim(-1, dim)
            ref.backward(dy.double())
            for need_w, need_b in ((True, True), (True, False), (False, True)):
                xd, wd, bd = x.cuda().requires_grad_(), w.cuda().requires_grad_(need_w), b.cuda().requires_grad_(need_b)
                ops.layer_norm(xd, wd, bd, dim=dim).backward(dy.cuda())
                # a handful of terms each: sums of n <= 30 products in fp32 with h itself off by the norm's few half steps of
                # a value up to sqrt(C), n + 16 half steps of sum |dy h|; then the rounding to the parameters' type
                for t, r, need in ((wd, wr, need_w), (bd, br, need_b)):
                    if not need:
                        assert t.grad is None
                        continue
                    assert t.grad.dtype == pt
                    n = x.numel() // C
                    terms = (dy.double().abs() * (1 + x.double().abs())).movedim(dim, -1).reshape(-1, C).sum(0) * 4
                    tol = (n + 16) * 2.0 ** -24 * terms + torch.finfo(pt).eps / 2 * r.grad.abs() + 1e-7
                    assert bool(((t.grad.cpu().double() - r.grad).abs() <= tol).all()), (shape, dt, pt)


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("shape", [(1, 1025, 1, 3), (2, 2048, 3, 1), (3, 1500, 16, 17), (2, 16390, 2, 3), (2, 1100, 31, 33)])
def test_many_channels_of_planes(shape, dt):
    """More channels than the registers hold, few and many positions: forward, and all gradients, against 64 bits."""
    from fc3d import ops
    g = torch.Generator().manual_seed(shape[1])
    C = shape[1]
    x, dy = (torch.randn(shape, generator=g).to(dt) for _ in range(2))
    w, b = torch.randn(C, generator=g), torch.randn(C, generator=g)
    xr, wr, br = (t.double().requires_grad_() for t in (x, w, b))
    ref = torch.relu(torch.nn.functional.layer_norm(xr.movedim(1, -1), (C,), wr, br, 1e-5)).movedim(-1, 1)
    # values within rounding of the ReLU's edge may fall on either side: their gradient is taken out on both
    edge = torch.nn.functional.layer_norm(x.double().movedim(1, -1), (C,), w.double(), b.double(), 1e-5).movedim(-1, 1).abs() < 1e-4
    dy[edge] = 0
    ref.backward(dy.double())
    xd, wd, bd = (t.cuda().requires_grad_() for t in (x, w, b))
    y = ops.layer_norm(xd, wd, bd, dim=1, relu=True)
    y.backward(dy.cuda())
    half = torch.finfo(dt).eps / 2
    # sums of C (or of all positions) terms in fp32, in lanes and wavefronts: a few half steps times the sum's depth, 64 here,
    # relative to the 2-norm; one rounding to the type
    for got, want, own in ((y, ref, half), (xd.grad, xr.grad, half), (wd.grad, wr.grad, 0.0), (bd.grad, br.grad, 0.0)):
        off = float((got.detach().cpu().double() - want.detach()).norm() / want.detach().norm())
        assert off <= own + 64 * 2.0 ** -24, (shape, off)
    again = torch.autograd.grad(ops.layer_norm(xd, wd, bd, dim=1, relu=True), (xd, wd, bd), dy.cuda())
    for p, q in zip(again, (xd.grad, wd.grad, bd.grad)):
        assert torch.equal(p, q)


def test_tracers_and_tangents_go_through_autograd(monkeypatch):
    """Without a gradient too: a tracer records the call itself, not the kernel's empty output, and forward mode is refused
    as by the other operators.  On the CPU, with a stand-in for the launch."""
    import torch.autograd.forward_ad as fw
    import torch.nn.functional as F
    from fc3d import ops

    def stand_in(x, weight, bias, eps, dim, relu, want_stats):
        y = torch.empty_like(x)
        y.data.numpy()[:] = F.layer_norm(x.detach(), (8,), weight, bias, eps).numpy()      # behind the tracer's back
        return y, x, torch.zeros(1), None
    monkeypatch.setattr(ops, "_need_gpu_float", lambda t, what: 0)
    monkeypatch.setattr(ops, "_norm_forward", stand_in)
    w, b = torch.rand(8) + 0.5, torch.rand(8)
    x = torch.randn(4, 8)
    with torch.no_grad():
        traced = torch.jit.trace(lambda t: ops.layer_norm(t, w, b) * 2.0, (torch.randn(4, 8),), check_trace=False)
        assert "LayerNormFn" in str(traced.graph)
        assert torch.equal(traced(x), F.layer_norm(x, (8,), w, b, 1e-5) * 2.0)
    with fw.dual_level():
        assert torch.equal(ops.layer_norm(x, w, b), F.layer_norm(x, (8,), w, b, 1e-5))         # no tangent: nothing lost
        for args in ((fw.make_dual(x, torch.ones_like(x)), w, b), (x, fw.make_dual(w, torch.ones_like(w)), b)):
            with pytest.raises(NotImplementedError):
                ops.layer_norm(*args)


@gpu
@pytest.mark.parametrize("shape,dim", [((6, 40), -1), ((2, 16, 9, 7), 1)])
def test_traced_and_forward_mode_on_the_gpu(shape, dim):
    import torch.autograd.forward_ad as fw
    from fc3d import ops
    x, w, b, _ = (t.cuda() for t in inputs(shape, dim, F32, F32, 71))
    f = lambda t: ops.layer_norm(t, w, b, dim=dim, relu=True) + 1.0  # noqa: E731
    with torch.no_grad():
        traced = torch.jit.trace(f, (torch.zeros_like(x),), check_trace=False)
        for t in (x, 2.0 * x, x[:1], x.transpose(0, -1).contiguous().transpose(0, -1)):        # other values, sizes, orders
            assert torch.equal(traced(t), f(t))
    with fw.dual_level(), pytest.raises(NotImplementedError):
        f(fw.make_dual(x, x))


def test_empty_planes_have_no_position(monkeypatch):
    """What reaches the entry points of a tensor without values: no outer index, wherever the empty axis is.  On the CPU,
    with a stand-in for the launch, and the entry point itself (nothing is launched)."""
    from fc3d import _native, ops
    lib, seen = _native.load(), []

    class Lib:
        @staticmethod
        def fc3d_layer_norm_fwd(stream, *args):
            seen.append((args[5], args[6], args[7]))
            return lib.fc3d_layer_norm_fwd(None, *args)
    monkeypatch.setattr(ops, "_lib", Lib)
    monkeypatch.setattr(ops, "_need_gpu_float", lambda t, what: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "_get_device", lambda: -1)
    for shape in ((2, 8, 0, 5), (2, 8, 5, 0), (2, 8, 0), (0, 8, 3, 3), (0, 8)):
        for x in (torch.zeros(shape), torch.zeros(shape).transpose(0, -1).contiguous().transpose(0, -1)):
            assert ops.layer_norm(x, dim=1).shape == shape
            outer, C, inner = seen.pop()
            assert outer == 0 and C == 8 and inner >= 1


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("shape", [(2, 8, 0, 5), (2, 8, 5, 0), (2, 8, 0)])
def test_empty_planes(shape, dt):
    from fc3d import ops
    w, b = (torch.ones(8, device="cuda", dtype=dt, requires_grad=True) for _ in range(2))
    x = torch.zeros(shape, device="cuda", dtype=dt, requires_grad=True)
    for relu in (False, True):
        y = ops.layer_norm(x, w, b, dim=1, relu=relu)
        assert y.shape == shape and y.dtype == dt
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert dx.shape == shape and not dw.any() and not db.any()
    with torch.no_grad():
        assert ops.layer_norm(x, w, b, dim=1).shape == shape


@pytest.mark.parametrize("case", ["channels_last", "padded planes", "padded rows", "copied", "dense"])
def test_saved_tensors_in_another_memory_order(case, monkeypatch):
    """Hooks that keep saved tensors elsewhere hand them back dense, whatever their strides were: the backward pass has to
    read them as they come.  On the CPU, with the formula in place of the launches, its reads kept inside the tensors."""
    import ctypes
    from fc3d import ops
    room = {}                                                      # address -> values behind it

    def at(ptr, count):
        assert count <= room[ptr], f"{count} values read of {room[ptr]}"
        return torch.frombuffer((ctypes.c_float * count).from_address(ptr), dtype=F32)

    def normalised(ptr, outer, C, inner, step):
        t = at(ptr, step * (outer - 1) + C * inner if outer else 0).as_strided((outer, C, inner), (step, inner, 1))
        return t, t.mean(1, keepdim=True), t.var(1, unbiased=False, keepdim=True)

    class Lib:
        @staticmethod
        def fc3d_layer_norm_fwd(s, x, xt, w, b, wt, outer, C, inner, step, eps, relu, y, m, r):
            t, mu, var = normalised(x, outer, C, inner, step)
            ctypes.memmove(y, ((t - mu) / (var + eps).sqrt()).contiguous().data_ptr(), 4 * outer * C * inner)
            return 0

        @staticmethod
        def fc3d_layer_norm_bwd_workspace(*a):
            return 0

        @staticmethod
        def fc3d_layer_norm_bwd(s, dy, x, xt, w, b, wt, m, r, outer, C, inner, g_step, step, relu, dx, dw, db, ws):
            t, mu, var = normalised(x, outer, C, inner, step)
            g = at(dy, g_step * (outer - 1) + C * inner).as_strided((outer, C, inner), (g_step, inner, 1))
            rs = 1 / (var + 1e-5).sqrt()
            h = (t - mu) * rs
            out = rs * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
            ctypes.memmove(dx, out.contiguous().data_ptr(), 4 * outer * C * inner)
            return 0
    monkeypatch.setattr(ops, "_lib", Lib)
    monkeypatch.setattr(ops, "_need_gpu_float", lambda t, what: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "_get_device", lambda: -1)
    pointer = torch.Tensor.data_ptr

    def counted(t):
        room[pointer(t)] = (t.untyped_storage().nbytes() - 4 * t.storage_offset()) // t.element_size()
        return pointer(t)
    monkeypatch.setattr(torch.Tensor, "data_ptr", counted)
    base = torch.randn(3, 6, 4, 10)
    x, dim = {"channels_last": (base.contiguous(memory_format=torch.channels_last), 1), "padded planes": (base[:, :3], 1),
              "padded rows": (torch.randn(7, 20)[:, :9], -1), "copied": (base[:, :, :, ::2], 1), "dense": (base, 1)}[case]
    g = torch.randn(3, 6, 4, 10)[tuple(slice(n) for n in x.shape)] if x.dim() == 4 else torch.randn(x.shape)
    x = x.detach().requires_grad_()
    want = formula(x.detach(), None, None, g, dim, 1e-5)["dx"]
    for pack in (lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format)):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = ops.layer_norm(x, dim=dim)
        (dx,) = torch.autograd.grad(y, x, g)
        assert float((dx.double() - want).abs().max()) <= 1e-4
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.half()):
        y = ops.layer_norm(x, dim=dim)
    with pytest.raises(RuntimeError, match="came back"):
        torch.autograd.grad(y, x, g)


@gpu
@pytest.mark.parametrize("shape,dim,cut", [((2, 16, 9, 7), 1, None), ((2, 48, 9, 7), 1, 16), ((40, 96), -1, 50)])
def test_saved_tensors_on_the_host(shape, dim, cut):
    from fc3d import ops
    x, w, b, dy = (t.cuda() for t in inputs(shape, dim, F32, F32, 72))
    if cut is None:
        x = x.contiguous(memory_format=torch.channels_last)
    else:
        x, w, b, dy = x.narrow(dim, 0, cut), w[:cut], b[:cut], dy.narrow(dim, 0, cut)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(ops.layer_norm(*leaves, dim=dim, relu=True), leaves, dy)
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        y = ops.layer_norm(*leaves, dim=dim, relu=True)
    for a, c, r in zip(torch.autograd.grad(y, leaves, dy), want, (x, w, b)):
        # the same values in another order of the sums
        assert float((a - c).abs().max()) <= KP * 8 * float(c.abs().max()) and a.shape == r.shape


# Row lengths of the kernels that SHAPES leaves out: 2049 to 4096 (256 lanes a row forward, 512 backward), and 8193 to
# 16383 with rows that end inside a vector.
WIDTHS = [(600, 2560), (1030, 4096), (521, 3001), (700, 2049), (5, 9001), (3, 16383)]


@gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(v).replace("torch.", "") for v in t))
@pytest.mark.parametrize("shape", WIDTHS, ids=lambda v: "x".join(map(str, v)))
def test_more_row_lengths(shape, types):
    test_against_formula(shape, -1, types)


# More positions than the workgroups of a launch hold at a time, two to six rounds of them, for every number of lanes per
# row and of channel groups: the next row on its way, the LDS areas that take turns, the last round part full.
ROUNDS = [((90001, 33), -1), ((90001, 96), -1), ((50001, 200), -1), ((25001, 500), -1), ((12001, 1000), -1), ((6001, 2000), -1),
          ((3001, 3999), -1), ((3001, 5000), -1), ((2999, 9001), -1), ((1300, 16384), -1),
          ((5, 7, 601, 701), 1), ((5, 20, 301, 401), 1), ((5, 50, 201, 301), 1), ((5, 100, 101, 301), 1), ((5, 200, 101, 131), 1),
          ((5, 500, 81, 101), 1), ((5, 900, 61, 101), 1), ((3001, 40, 5), 1), ((2001, 300, 1, 2), 1)]


@gpu
@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F32)], ids=lambda t: "-".join(str(v).replace("torch.", "") for v in t))
@pytest.mark.parametrize("shape,dim", ROUNDS, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else None)
def test_several_rounds(shape, dim, types):
    """Chains of the sums over positions: six rounds of four positions a lane, 64 row groups or wavefronts, 32 + 32 partial
    sums: 128 at most, as above.  The formula on the device.

    Which values pass the ReLU is read off y, except where y is zero in fp16 and the value before it may be positive and
    below the type's range (half of 2^-24; among millions of values a few are).  The bounds bear both there: with d the
    gradients in question, dx moves by rs (|d w| + mean|d w| + |h| mean|d w h|), dw by the sum of |d h|, db by that of |d|."""
    from fc3d import ops
    dt, wdt = types
    x, w, b, dy = (t.cuda() for t in inputs(shape, dim, dt, wdt, 13))
    for relu in (False, True):
        y, (dx, dw, db) = run(ops, x, w, b, dy, dim, relu)
        mask = (y.detach() > 0).double() if relu else None
        r = formula(x, w, b, dy, dim, 1e-5, mask)
        if relu and dt == F16:
            pre = formula(x, w, b, None, dim, 1e-5)
            d = (dy.double() * ((y.detach() == 0) & (pre["y"] > -pre["ey"]))).abs().movedim(dim, -1)
            xm = x.double().movedim(dim, -1)
            rs = 1 / torch.sqrt(xm.var(-1, unbiased=False, keepdim=True) + 1e-5)
            h = (rs * (xm - xm.mean(-1, keepdim=True))).abs()
            gw = d * w.double().abs()
            r["edx"] += (rs * (gw + gw.mean(-1, keepdim=True) + h * (gw * h).mean(-1, keepdim=True))).movedim(-1, dim)
            pos = tuple(range(xm.dim() - 1))
            r["edw"] += (d * h).sum(pos)
            r["edb"] += d.sum(pos)
        for name, got, t in (("y", y, dt), ("dx", dx, dt), ("dw", dw, wdt), ("db", db, wdt)):
            close(got, r[name].cpu(), r["e" + name].cpu(), t, f"{name} relu={relu}")
