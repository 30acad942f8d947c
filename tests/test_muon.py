"""Newton-Schulz orthogonalisation and the Muon step (fc3d.ops.orthogonalize / muon_step, fc3d.optim.Muon) against
their definition in 64 bits.

Bounds, in the 2-norm of the whole result relative to the result's.  The operands are pairs of fp16 values: an operand
is off by 2^-23 of itself at most, the dropped product of the two lo planes by 2^-24 of the product: five half steps of
fp32 where fp32 products take their operands as they are and round in the sums alike.  So the error may be that of the
fp32 evaluation, taken on the same input, four times (its own share included), plus 2^-20 where that happens to be zero.
A 16-bit result adds its rounding, half a step, and the Gram form in one segment: a value of A is off by 2^-23 of
itself, A's spectrum by at most 2 * 2^-23 times a row's norm, which is 1 / sqrt(m) where the rows share the norm; a
singular value s of the result by s dP/dlambda <= 2.6e4 times that (the default polynomial's five steps): 6e-3 / sqrt(m)."""
import math

import pytest
import torch

COEFFS = (3.4445, -4.7750, 2.0315)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def ns(g, dt, steps=5, coeffs=COEFFS, eps=1e-7):
    """The definition, evaluated in type dt on the CPU."""
    a, b, c = coeffs
    x = g.to(dt).reshape(g.shape[0], -1)
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.t() if tall else x).reshape(g.shape)


def update(shape, kind, seed, dt=F32):
    g = torch.Generator().manual_seed(seed)
    m, n = shape[0], math.prod(shape[1:])
    x = torch.randn(m, n, generator=g)
    if kind == "low":                                # a few strong directions over a noise floor
        k = min(m, n, 4)
        x = torch.randn(m, k, generator=g) @ torch.randn(k, n, generator=g) + 0.01 * x
    return (1e-3 * x).reshape(shape).to(dt)


def bound(g, ref, steps=5, coeffs=COEFFS, eps=1e-7, dt=None):
    dt = g.dtype if dt is None else dt
    e32 = (ns(g, F32, steps, coeffs, eps).double() - ref).norm() / ref.norm()
    tol = 4 * float(e32) + 2.0 ** -20
    if dt != F32:
        tol += torch.finfo(dt).eps / 2 + 6e-3 / math.sqrt(min(g.shape[0], math.prod(g.shape[1:])))
    return tol


def near(got, g, what, steps=5, coeffs=COEFFS, eps=1e-7):
    ref = ns(g, torch.float64, steps, coeffs, eps)
    assert got.shape == ref.shape and got.dtype == g.dtype, what
    off = float((got.cpu().double() - ref).norm() / ref.norm())
    tol = bound(g, ref, steps, coeffs, eps)
    assert off <= tol, f"{what}: {off:.2e} of the result, {tol:.2e} allowed"


# ---- on the CPU -------------------------------------------------------------------------------------------------

def test_refusals():
    import ctypes
    from fc3d import _native, ops, optim
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.muon_step([torch.zeros(4, 4)], [torch.zeros(4, 4)], [torch.zeros(4, 4)])
    with pytest.raises(ValueError):
        ops.muon_step([torch.zeros(4, 4)], [], [])
    assert ops.orthogonalize([]) == []
    ops.muon_step([], [], [])
    for bad in (dict(steps=0), dict(steps=65), dict(eps=-1.0), dict(coefficients=(float("nan"), 0, 0))):
        with pytest.raises(ValueError):
            ops.orthogonalize([], **bad)
    for bad in (dict(momentum=1.5), dict(lr=float("inf")), dict(weight_decay=float("nan"))):
        with pytest.raises(ValueError):
            ops.muon_step([], [], [], **bad)
    p = torch.nn.Parameter(torch.zeros(4, 4))
    for bad in (dict(lr=-1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(steps=0), dict(scale="other")):
        with pytest.raises(ValueError):
            optim.Muon([p], **bad)
    with pytest.raises(ValueError, match="two axes"):
        optim.Muon([torch.nn.Parameter(torch.zeros(4))])
    lib = _native.load()
    I64, VP = ctypes.c_int64, ctypes.c_void_p
    one = 256

    def call(g=one, out=one, rows=4, cols=4, t=0, steps=5, co=COEFFS, eps=1e-7, ws=one, count=1):
        return lib.fc3d_orthogonalize(None, count, (VP * 1)(g), (VP * 1)(out), (I64 * 1)(rows), (I64 * 1)(cols), t, steps, *co, eps, ws)
    assert call(count=0) == 0 and call(count=-1) == -1
    assert call(g=None) == -1 and call(out=None) == -1 and call(ws=None) == -1 and call(rows=0) == -1 and call(cols=-3) == -1
    assert call(t=3) == -1 and call(steps=0) == -1 and call(steps=65) == -1 and call(eps=-1.0) == -1 and call(eps=float("nan")) == -1
    assert call(co=(float("inf"), 0, 0)) == -1
    assert call(co=(30.0, 0.0, 0.0)) == -2 and call(co=(2.0, 2.0, 2.0)) == -2           # singular values grow
    assert call(rows=1 << 24) == -2 and call(rows=1 << 20, cols=1 << 20) == -2
    assert call(g=one + 2) == -3 and call(out=one + 1, t=1) == -3 and call(ws=one + 16) == -3

    def step(mom=one, lr=0.1, beta=0.95, decay=1.0):
        return lib.fc3d_muon_step(None, 1, (VP * 1)(one), (VP * 1)(one), (VP * 1)(mom) if mom != 0 else None, (I64 * 1)(4), (I64 * 1)(4),
                                  (ctypes.c_float * 1)(lr), 0, 0, beta, 1, decay, 5, *COEFFS, 1e-7, None)
    assert step(mom=0) == -1 and step(mom=None) == -1 and step(beta=1.1) == -1 and step(beta=float("nan")) == -1
    assert step(decay=float("inf")) == -1 and step() == -1                               # no workspace
    ws = lambda r, c: lib.fc3d_orthogonalize_workspace(1, (I64 * 1)(r), (I64 * 1)(c))  # noqa: E731
    assert ws(0, 4) == 0 and ws(1 << 24, 4) == 0 and ws(4, 4) > 0 and ws(64, 64) == ws(4, 4)
    assert lib.fc3d_orthogonalize_workspace(0, None, None) == 0


def test_memory_orders_of_matrices():
    from fc3d.ops import _matrix_order, muon_scale
    t = torch.zeros(6, 5, 3, 3)
    assert _matrix_order(t) == (6, 45)
    assert _matrix_order(t.contiguous(memory_format=torch.channels_last)) == (6, 45)
    assert _matrix_order(torch.zeros(6, 4).t()) == (6, 4)                    # as the matrix that lies in memory
    assert _matrix_order(torch.zeros(6, 8)[:, :4]) is None and _matrix_order(torch.zeros(1, 4).expand(6, 4)) is None
    assert _matrix_order(torch.zeros(6, 1, 4).transpose(0, 2)) is None
    assert _matrix_order(torch.zeros(0, 4)) == (0, 0) and _matrix_order(torch.zeros(1, 4).t()) == (4, 1)
    with pytest.raises(ValueError):
        _matrix_order(torch.zeros(4))
    assert muon_scale((64, 16), "spectral") == 2.0 and muon_scale((16, 4, 4), "spectral") == 1.0
    assert muon_scale((4, 25, 4), "rms") == 2.0
    with pytest.raises(ValueError):
        muon_scale((4, 4), "x")


def test_five_steps_bring_singular_values_near_one():
    """What the definition is for; the coefficients' polynomial stays within 0.67 .. 1.21 from 0.02 on."""
    s = torch.linspace(0.02, 1, 1000, dtype=torch.float64)
    a, b, c = COEFFS
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    assert 0.66 < float(s.min()) and float(s.max()) < 1.21
    x = ns(update((24, 60), "gauss", 0), torch.float64)
    assert torch.linalg.svdvals(x).min() > 0.6


# ---- on the GPU -------------------------------------------------------------------------------------------------

gpu = pytest.mark.gpu

SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (9, 32), (32, 9), (64, 64), (64, 65), (65, 64), (63, 129), (130, 500), (300, 77),
          (100, 1000), (256, 256), (32, 32, 3, 3), (512, 700), (128, 128, 3, 3), (700, 65, 2)]


@gpu
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("kind", ["gauss", "low"])
def test_orthogonalize_against_definition(dt, kind):
    from fc3d import ops
    gs = [update(s, kind, 100 + i, dt) for i, s in enumerate(SHAPES)]
    together = ops.orthogonalize([g.cuda() for g in gs])
    for x, y in zip(together, ops.orthogonalize([g.cuda() for g in gs])):
        assert torch.equal(x, y)                                       # the same call: the same bits
    for g, x, shape in zip(gs, together, SHAPES):
        near(x, g, f"{shape} {dt} {kind}")
        near(ops.orthogonalize(g.cuda()), g, f"{shape} {dt} {kind} alone")      # with the kernels that suit it alone


@gpu
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 12])
def test_other_step_counts_and_coefficients(dt, steps):
    from fc3d import ops
    for shape in ((48, 60), (40, 200)):
        for coeffs in (COEFFS, (1.875, -1.25, 0.375)):                 # the second: cubic convergence to one
            g = update(shape, "gauss", steps, dt)
            near(ops.orthogonalize(g.cuda(), steps=steps, coefficients=coeffs), g, f"{shape} {steps} {coeffs}", steps, coeffs)


@gpu
@pytest.mark.parametrize("steps", [5, 10, 11, 16])
def test_rank_deficient_matrices_and_many_steps(steps):
    """Directions that the input lacks: what a step rounds there is amplified as a singular value would be."""
    from fc3d import ops
    for m, n in ((40, 200), (64, 90), (96, 300)):
        g = torch.Generator().manual_seed(steps * m)
        x = torch.randn(m, 6, generator=g) @ torch.randn(6, n, generator=g)
        near(ops.orthogonalize(x.cuda(), steps=steps), x, f"rank 6 of {m}, {steps} steps", steps)
        x[m // 2:] = 0.0
        near(ops.orthogonalize(x.cuda(), steps=steps), x, f"empty rows of {m}, {steps} steps", steps)


@gpu
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=lambda t: str(t).replace("torch.", ""))
def test_many_steps_keep_the_singular_values_bounded(dt):
    """The default polynomial maps [0, 1.21] into itself (1.203 at its maximum): whatever rounding leaves in directions that
    the input lacks grows to that and no further.  Bound: 1.21 and a 16-bit result's rounding."""
    from fc3d import ops
    for m, n in ((40, 200), (96, 300), (70, 75)):
        g = torch.Generator().manual_seed(m)
        x = torch.randn(m, 5, generator=g) @ torch.randn(5, n, generator=g)
        x[m // 2:] = 0.0
        for steps in (16, 30, 64):
            y = ops.orthogonalize(x.to(dt).cuda(), steps=steps).cpu().double()
            top = float(torch.linalg.svdvals(y)[0])
            assert 0.6 < top <= 1.21 * (1 + torch.finfo(dt).eps), (m, n, steps, top)


@gpu
@pytest.mark.parametrize("steps", [2, 3, 5])
def test_steep_coefficients(steps):
    """0.9 T_5(x), the Chebyshev polynomial: it multiplies small values by 4.5 and stays below one on [0, 1]."""
    from fc3d import ops
    coeffs = (4.5, -18.0, 14.4)
    a, b, c = coeffs
    lam = torch.linspace(0.0, 1.0, 20001, dtype=torch.float64, requires_grad=True)
    q0 = a + b * lam + c * lam * lam
    l1 = lam * q0 * q0
    (q0 * (a + b * l1 + c * l1 * l1)).sum().backward()
    slope = float((lam.detach().sqrt() * lam.grad.abs()).max())          # of two steps' factor, as for five above
    for m, n in ((40, 200), (96, 300), (130, 150)):
        g = update((m, n), "gauss", 300 + m)
        near(ops.orthogonalize(g.cuda(), steps=steps, coefficients=coeffs), g, f"{m} x {n}, {steps} steps", steps, coeffs)
        if steps == 2:
            h = g.bfloat16()
            ref = ns(h, torch.float64, steps, coeffs)
            tol = bound(h.float(), ref, steps, coeffs) + torch.finfo(BF16).eps / 2 + \
                slope * 2 * 2.0 ** -23 / math.sqrt(m) * math.sqrt(m) / float(ref.norm())
            off = float((ops.orthogonalize(h.cuda(), steps=steps, coefficients=coeffs).cpu().double() - ref).norm() / ref.norm())
            assert off <= tol, (m, n, off, tol)


@gpu
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=lambda t: str(t).replace("torch.", ""))
def test_workspace_holds_every_type_and_step_count(dt):
    """The workspace is sized by the matrices alone, what a call lays out in it depends on its types and steps too."""
    import ctypes
    from fc3d import _native
    lib = _native.load()
    I64, VP = ctypes.c_int64, ctypes.c_void_p
    code = {F32: 0, BF16: 1, F16: 2}[dt]
    for shapes in ([(64, 4000)], [(20, 30), (64, 64)], [(130, 9000)], [(300, 5000), (96, 200)], [(520, 4608), (64, 288), (32, 9)]):
        gs = [update(s, "gauss", 40 + i, dt).cuda() for i, s in enumerate(shapes)]
        k = len(shapes)
        r, c = (I64 * k)(*[s[0] for s in shapes]), (I64 * k)(*[s[1] for s in shapes])
        n = lib.fc3d_orthogonalize_workspace(k, r, c)
        ws = torch.full((n + 512,), 77, dtype=torch.uint8, device="cuda")
        base = ws.data_ptr() + 256
        assert base % 256 == 0
        at = (VP * k)(*[g.data_ptr() for g in gs])
        for steps in (1, 5, 12):
            out = [torch.empty_like(g) for g in gs]
            to = (VP * k)(*[o.data_ptr() for o in out])
            assert lib.fc3d_orthogonalize(torch.cuda.current_stream().cuda_stream, k, at, to, r, c, code, steps, *COEFFS, 1e-7, base) == 0
            torch.cuda.synchronize()
            assert bool((ws[:256] == 77).all()) and bool((ws[256 + n:] == 77).all()), (shapes, steps)
            assert all(bool(torch.isfinite(o).all()) for o in out)


@gpu
def test_scales_zeros_and_special_values():
    from fc3d import ops
    g = update((40, 100), "gauss", 5)
    x = ops.orthogonalize(g.cuda())
    for f in (2.0 ** 100, 2.0 ** 40, 2.0 ** -10):                       # only the eps feels the scale
        assert float((ops.orthogonalize((g * f).cuda(), eps=0.0) - ops.orthogonalize(g.cuda(), eps=0.0)).abs().max()) <= 2.0 ** -20
    h = update((40, 100), "gauss", 5, BF16)
    assert torch.equal(ops.orthogonalize((h * 2.0 ** 90).cuda(), eps=0.0), ops.orthogonalize(h.cuda(), eps=0.0))
    for dt in (F32, BF16, F16):
        z = torch.zeros(33, 70, dtype=dt, device="cuda")
        assert not ops.orthogonalize(z).any()
        assert bool(torch.isnan(ops.orthogonalize(z, eps=0.0)).all())
        for bad in (float("nan"), float("inf")):
            t = update((33, 70), "gauss", 6, dt).cuda()
            t[3, 4] = bad
            two = ops.orthogonalize([t, update((33, 70), "gauss", 6, dt).cuda()])
            assert bool(torch.isnan(two[0]).all()) and bool(torch.isfinite(two[1]).all())      # its own matrix alone
    assert torch.equal(ops.orthogonalize(g.cuda()), x)


@gpu
def test_lists_orders_and_empty_matrices():
    from fc3d import ops
    g = update((70, 40, 3, 3), "gauss", 7)
    plain = ops.orthogonalize(g.cuda())
    cl = ops.orthogonalize(g.cuda().contiguous(memory_format=torch.channels_last))
    assert cl.is_contiguous(memory_format=torch.channels_last)
    near(cl, g, "channels_last")
    near(plain, g, "dense")
    m = update((50, 90), "gauss", 8)
    t = ops.orthogonalize(m.cuda().t())
    near(t, m.t(), "transposed view")
    wide = torch.zeros(50, 100, device="cuda")
    wide[:, 5:95] = m.cuda()
    near(ops.orthogonalize(wide[:, 5:95]), m, "columns of a wider matrix")
    out = ops.orthogonalize([torch.zeros(0, 5, device="cuda"), m.cuda(), torch.zeros(5, 0, device="cuda", dtype=F16), m.bfloat16().cuda()])
    assert out[0].shape == (0, 5) and out[2].shape == (5, 0) and out[2].dtype == F16
    near(out[1], m, "among empty ones")
    near(out[3], m.bfloat16(), "among other types")
    # more than one group of launches takes
    many = [update((3 + i % 7, 5 + i % 11), "gauss", 200 + i) for i in range(101)]
    for x, v in zip(ops.orthogonalize([v.cuda() for v in many]), many):
        near(x, v, "one of many")
    with pytest.raises(ValueError, match="grow"):
        ops.orthogonalize(m.cuda(), coefficients=(30.0, 0.0, 0.0))
    with pytest.raises(TypeError):
        ops.orthogonalize(m.double().cuda())
    with pytest.raises(ValueError):
        ops.orthogonalize(torch.zeros(5, device="cuda"))


@gpu
def test_writes_nothing_beyond_its_outputs_and_works_in_place():
    import ctypes
    from fc3d import _native
    lib = _native.load()
    I64, VP = ctypes.c_int64, ctypes.c_void_p
    pad = 64
    for dt, code in ((F32, 0), (BF16, 1)):
        for shape in ((33, 70), (70, 33), (1, 129), (64, 64)):
            g = update(shape, "gauss", 9, dt)
            buf = torch.full((g.numel() + 2 * pad,), 512.0, dtype=dt, device="cuda")
            buf[pad:-pad] = g.reshape(-1).cuda()
            r, c = (I64 * 1)(shape[0]), (I64 * 1)(shape[1])
            n = lib.fc3d_orthogonalize_workspace(1, r, c)
            ws = torch.full((n + 512,), 77, dtype=torch.uint8, device="cuda")
            at = (VP * 1)(buf.data_ptr() + pad * buf.element_size())
            base = ws.data_ptr() + 256
            assert base % 256 == 0
            assert lib.fc3d_orthogonalize(torch.cuda.current_stream().cuda_stream, 1, at, at, r, c, code, 5, *COEFFS, 1e-7, base) == 0
            torch.cuda.synchronize()
            assert bool((buf[:pad] == 512.0).all()) and bool((buf[-pad:] == 512.0).all())
            assert bool((ws[:256] == 77).all()) and bool((ws[256 + n:] == 77).all())
            near(buf[pad:-pad].reshape(shape), g, f"in place {shape}")


def step_formula(w, g, m, lr, beta, nesterov, wd, scale_f, dt=torch.float64):
    w, g, m = w.to(dt), g.to(dt), m.to(dt)
    m = beta * m + (1 - beta) * g
    u = (1 - beta) * g + beta * m if nesterov else m
    return (1 - lr * wd) * w - lr * scale_f * ns(u, dt), m, u


@gpu
@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (BF16, F32)],
                         ids=lambda t: "-".join(str(v).replace("torch.", "") for v in t))
@pytest.mark.parametrize("nesterov,scale", [(True, "spectral"), (False, "rms")])
def test_step_against_definition(types, nesterov, scale):
    from fc3d import ops
    pt, gt = types
    shapes = [(40, 24, 3, 3), (24, 100), (100, 24), (65, 65), (1, 9), (128, 640)]
    w = [(torch.randn(s, generator=torch.Generator().manual_seed(i)) / 8).to(pt) for i, s in enumerate(shapes)]
    g = [update(s, "low", 30 + i, gt) for i, s in enumerate(shapes)]
    m = [update(s, "gauss", 60 + i) for i, s in enumerate(shapes)]
    wd, md = [t.cuda() for t in w], [t.cuda() for t in m]
    lr, beta, decay = 0.02, 0.9, 0.1
    ops.muon_step(wd, [t.cuda() for t in g], md, lr=lr, momentum=beta, nesterov=nesterov, weight_decay=decay, scale=scale)
    for i, s in enumerate(shapes):
        f = ops.muon_scale(s, scale)
        ref_w, ref_m, u = step_formula(w[i], g[i], m[i], lr, beta, nesterov, decay, f)
        # beta and 1 - beta rounded to fp32, a product and an fma: four half steps of the terms
        off = (md[i].cpu().double() - ref_m).abs()
        assert bool((off <= 4 * 2.0 ** -24 * (beta * m[i].double().abs() + (1 - beta) * g[i].double().abs()) + 2.0 ** -149).all()), s
        o = ns(u, torch.float64)
        # the update u comes with the same four half steps, which the steps amplify as they do fp32's own roundings
        tol = lr * f * float(o.norm()) * (bound(u.float(), o, dt=pt) + 2.0 ** -20)
        tol += (torch.finfo(pt).eps / 2 + 4 * 2.0 ** -24) * float(ref_w.norm() + (w[i].double() - ref_w).norm())
        assert float((wd[i].cpu().double() - ref_w).norm()) <= tol, s


@gpu
def test_step_checks():
    from fc3d import ops
    w, g, m = (torch.zeros(4, 6, device="cuda") for _ in range(3))
    v0 = w._version
    ops.muon_step([w], [g], [m])
    assert w._version > v0 and m._version > v0                        # seen by autograd's check of saved tensors
    for bad, err in ((([w, w], [g, g], [m, m.clone()]), ValueError), (([w, w.clone()], [g, g], [m, m]), ValueError),
                     (([w], [g], [m.half()]), TypeError), (([w], [g.t()], [m]), ValueError),
                     (([w], [g.cpu()], [m]), RuntimeError), (([w[:, :3]], [g[:, :3]], [m[:, :3]]), ValueError),
                     (([w.double()], [g], [m]), TypeError), (([w.t()], [g.t()], [m.t().contiguous()]), ValueError)):
        with pytest.raises(err):
            ops.muon_step(*bad)
    with pytest.raises(ValueError, match="grow"):
        ops.muon_step([w, w.half()], [g, g], [m, m.clone()], coefficients=(30.0, 0.0, 0.0))
    ops.muon_step([torch.zeros(0, 4, device="cuda")], [torch.zeros(0, 4, device="cuda")], [torch.zeros(0, 4, device="cuda")])


@gpu
def test_step_refuses_shared_memory():
    """Whatever is written may lie over nothing else; gradients may share among themselves."""
    from fc3d import ops
    flat = torch.arange(200, dtype=torch.float32, device="cuda") / 200
    at = lambda i, n=24: flat[i:i + n].view(4, n // 4)  # noqa: E731
    before = flat.clone()
    for p, g, m in (([at(0)], [at(0)], [at(48)]), ([at(0)], [at(48)], [at(48)]), ([at(0)], [at(20)], [at(48)]), ([at(0)], [at(48)], [at(8)]),
                    ([at(0), at(12)], [at(48), at(72)], [at(96), at(120)]), ([at(0), at(24)], [at(48), at(48)], [at(72), at(92)])):
        with pytest.raises(ValueError, match="share memory"):
            ops.muon_step(p, g, m)
    assert torch.equal(flat, before)
    ops.muon_step([at(0), at(24)], [at(48), at(48)], [at(72), at(96)])         # neighbours, and one gradient for two
    assert bool((flat[:48] != before[:48]).any()) and torch.equal(flat[48:72], before[48:72]) and torch.equal(flat[120:], before[120:])


@gpu
def test_step_of_weights_in_other_memory_orders():
    from fc3d import ops
    w, g, m = (update((24, 16, 3, 3), "gauss", 40 + i) for i in range(3))
    ref = [t.cuda() for t in (w, g, m)]
    ops.muon_step([ref[0]], [ref[1]], [ref[2]], weight_decay=0.1)
    cl = [t.cuda().contiguous(memory_format=torch.channels_last) for t in (w, g, m)]
    dense_g = g.cuda()                                                # the gradient in another order than its weight
    ops.muon_step([cl[0]], [dense_g], [cl[2]], weight_decay=0.1)
    assert float((cl[0] - ref[0]).abs().max()) <= 2.0 ** -18 * 0.02 and torch.equal(cl[2], ref[2])
    a, b, c = (update((60, 24), "gauss", 50 + i).cuda() for i in range(3))
    ta, tb, tc = a.clone(), b.clone(), c.clone()
    ops.muon_step([a], [b], [c], scale="rms")
    ops.muon_step([ta.t()], [tb.t()], [tc.t()], scale="rms")           # the factor is the same both ways round
    assert torch.equal(a, ta) and torch.equal(c, tc)


def test_groups_of_the_optimizer():
    from fc3d import optim
    opt = optim.Muon([torch.nn.Parameter(torch.zeros(4, 4))])
    with pytest.raises(ValueError, match="two axes"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4))]})
    assert len(opt.param_groups) == 1                                  # as it was
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4, 2))], "lr": 0.5})
    assert [g["lr"] for g in opt.param_groups] == [0.02, 0.5]
    assert opt.step() is None                                          # no gradients: nothing to do, on any device


@gpu
def test_optimizer_in_a_graph(monkeypatch):
    from fc3d import optim
    make = lambda: torch.nn.Parameter(update((40, 90), "gauss", 90).cuda())  # noqa: E731
    p, q = make(), make()
    opts = [optim.Muon([t]) for t in (p, q)]
    p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        opts[0].step()
    monkeypatch.undo()
    assert torch.equal(p, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opts[0].step()                                                 # its momentum exists from here on
    torch.cuda.current_stream().wait_stream(side)
    opts[1].step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        opts[0].step()
    for turn in range(4):
        g = update((40, 90), "low", 91 + turn).cuda()
        p.grad.copy_(g)
        q.grad.copy_(g)
        graph.replay()
        opts[1].step()
        torch.cuda.synchronize()
        assert torch.equal(p, q) and torch.equal(opts[0].state[p]["momentum_buffer"], opts[1].state[q]["momentum_buffer"])


@gpu
def test_optimizer():
    from fc3d import ops, optim
    torch.manual_seed(0)
    make = lambda: [torch.nn.Parameter(update(s, "gauss", 70 + i, dt).cuda()) for i, (s, dt) in  # noqa: E731
                    enumerate((((16, 8, 3, 3), F32), ((32, 20), BF16), ((5, 6), F32)))]
    ps, qs = make(), make()
    opt = optim.Muon([{"params": ps[:2], "lr": 0.1}, {"params": ps[2:], "nesterov": False}], lr=0.05, weight_decay=0.1)
    mom = [torch.zeros_like(q, dtype=F32) for q in qs]
    for turn in range(3):
        gs = [update(tuple(p.shape), "gauss", 80 + 3 * turn + i, p.dtype).cuda() for i, p in enumerate(ps)]
        for p, g in zip(ps, gs):
            p.grad = g.clone()
        if turn == 1:
            ps[2].grad = None                                          # stays as it is
        assert opt.step(lambda: 7.0) == 7.0
        with torch.no_grad():
            ops.muon_step(qs[:2], gs[:2], mom[:2], lr=0.1, weight_decay=0.1)
            if turn != 1:
                ops.muon_step(qs[2:], gs[2:], mom[2:], lr=0.05, nesterov=False, weight_decay=0.1)
        for p, q in zip(ps, qs):
            assert torch.equal(p, q)
    # saved and loaded: the momenta come back bit for bit, those of 16-bit weights in 32 bits
    again = optim.Muon([{"params": [torch.nn.Parameter(p.detach().clone()) for p in ps[:2]]},
                        {"params": [torch.nn.Parameter(ps[2].detach().clone())]}])
    again.load_state_dict(opt.state_dict())
    for g, h in zip(again.param_groups, opt.param_groups):
        assert g["lr"] == h["lr"] and g["nesterov"] == h["nesterov"]
        for p, q in zip(g["params"], h["params"]):
            a, b = again.state[p]["momentum_buffer"], opt.state[q]["momentum_buffer"]
            assert a.dtype == F32 and torch.equal(a, b) and a.data_ptr() != b.data_ptr()
            p.grad = torch.ones_like(p)
            q.grad = torch.ones_like(q)
    again.step()
    opt.step()
    for g, h in zip(again.param_groups, opt.param_groups):
        for p, q in zip(g["params"], h["params"]):
            assert torch.equal(p, q)


@gpu
def test_steps_in_graphs_and_on_streams():
    """Two captured steps replayed on new gradients, with eager steps of others in between; two streams at once."""
    from fc3d import ops

    def capture(shapes, seed):
        w = [update(s, "gauss", seed + i).cuda() for i, s in enumerate(shapes)]
        g = [torch.zeros_like(t) for t in w]
        m = [torch.zeros_like(t) for t in w]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.muon_step([t.clone() for t in w], g, [t.clone() for t in m])
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            ops.muon_step(w, g, m)
        return graph, w, g, m
    shapes = ([(40, 90), (64, 64)], [(30, 200), (9, 9), (70, 70)])
    graphs = [capture(s, 300 + 10 * i) for i, s in enumerate(shapes)]
    eager = [([t.clone() for t in w], [t.clone() for t in m]) for _, w, _, m in graphs]
    for turn in range(4):
        for (_, w, g, m), s in zip(graphs, shapes):
            for i, t in enumerate(g):
                t.copy_(update(s[i], "low", 400 + 10 * turn + i).cuda())
        for graph, _, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, w, g, m), (ew, em) in zip(graphs, eager):
            ops.muon_step(ew, g, em)
            torch.cuda.synchronize()
            for a, b in zip(w + m, ew + em):
                assert torch.equal(a, b)
    gs = [update((200, 300), "gauss", 500 + i).cuda() for i in range(2)]
    alone = [ops.orthogonalize(g) for g in gs]
    streams = [torch.cuda.Stream() for _ in gs]
    got = []
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(gs, streams):
            with torch.cuda.stream(s):
                got.append(ops.orthogonalize(g))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, alone[i % 2])


@gpu
def test_small_matrices_beside_large_ones():
    """What a matrix is listed with does not cost it: next to a large one, results of a few rows are as exact as alone.
    Bound: they are worked on in 64 bits, so their rounding to fp32 alone, half a step of each value, doubled."""
    from fc3d import ops
    shapes = [(2, 3), (3, 2), (16, 5), (5, 40), (1, 30), (16, 16), (40, 12), (7, 1000)]
    gs = [update(s, "gauss", 600 + i) for i, s in enumerate(shapes * 7)]           # more than a group of them
    large = update((100, 150), "gauss", 599)
    out = ops.orthogonalize([g.cuda() for g in gs[:20]] + [large.cuda()] + [g.cuda() for g in gs[20:]])
    near(out.pop(20), large, "the large one")
    for x, g in zip(out, gs):
        ref = ns(g, torch.float64)
        assert float((x.cpu().double() - ref).norm()) <= 2 * 2.0 ** -24 * float(ref.norm()), g.shape


def second_segment_slope():
    """The most that three default steps make of a relative error of A, in result: |P(l) - P(k)| / |l - k| s over the
    squares l, k of singular values up to the polynomial's maximum, 1.21, and s = sqrt(k)."""
    a, b, c = COEFFS

    def p(lam):
        out = torch.ones_like(lam)
        for _ in range(3):
            q = a + b * lam + c * lam * lam
            out, lam = out * q, lam * q * q
        return out
    s = torch.linspace(0, 1.21, 1500, dtype=torch.float64)
    lam = s * s
    d = lam[:, None] - lam[None, :]
    dd = (p(lam)[:, None] - p(lam)[None, :]) / d.masked_fill(d == 0, 1.0)
    dd.diagonal().copy_((p(lam + 1e-7) - p(lam - 1e-7)) / 2e-7)
    return float((dd.abs() * s[None, :]).max())


@gpu
@pytest.mark.parametrize("noise", [0.3, 0.1, 0.03])
@pytest.mark.parametrize("m,n", [(128, 128), (128, 300), (256, 512), (512, 700)])
def test_half_precision_results_lose_no_more_than_their_rounding(m, n, noise):
    """Strong directions over a noise floor in fp16.  Rounding the exact result leaves r; in front of the rounding the
    result may be off by e: four times what fp32 products are, 2^-20, and the Gram matrix of the segment of three steps,
    whose values are off by 2 * 2^-23 of themselves.  The rounding does not know of e, so the squares add; of N values, the
    sum of squares of a rounding scatters by 0.9 / sqrt(N) and the mixed term by less: 8 / sqrt(N) is four times both."""
    from fc3d import ops
    gen = torch.Generator().manual_seed(m + n)
    g = (1e-3 * (torch.randn(m, 4, generator=gen) @ torch.randn(4, n, generator=gen) +
                 noise * torch.randn(m, n, generator=gen))).half()
    ref = ns(g, torch.float64)
    norm = float(ref.norm())
    x2 = ns(g, torch.float64, 2)
    r = float((ref.half().double() - ref).norm()) / norm
    e = 4 * float((ns(g, F32).double() - ref).norm()) / norm + 2.0 ** -20
    e += second_segment_slope() * 2.0 ** -22 * float((x2 @ x2.t()).norm()) / norm
    tol = math.sqrt((r * r + e * e) * (1 + 8 / math.sqrt(m * n)))
    off = float((ops.orthogonalize(g.cuda()).cpu().double() - ref).norm()) / norm
    assert off <= tol, (off, tol, r)


@gpu
@pytest.mark.parametrize("dt", [BF16, F16], ids=lambda t: str(t).replace("torch.", ""))
def test_small_matrices_beside_large_ones_in_16_bits(dt):
    """Rows that nearly depend on each other, next to a large matrix.  Worked on in 64 bits and rounded twice, to fp32 and to
    the result's type: beside the rounding of the exact result 2 * 2^-24 of each value, where the first rounding moves it
    across the second one's middle."""
    from fc3d import ops
    gs = []
    for m in (1, 2, 3, 5, 8, 16):
        for n in (m, m + 1, m + 40):
            for noise in (0.1, 0.01, 0.001):
                gen = torch.Generator().manual_seed(1000 * m + n)
                x = torch.randn(m, 1, generator=gen) @ torch.randn(1, n, generator=gen) + noise * torch.randn(m, n, generator=gen)
                gs.append((x.t() if n % 2 else x).contiguous().to(dt))
    out = ops.orthogonalize([g.cuda() for g in gs] + [update((100, 150), "gauss", 598, dt).cuda()])
    for x, g in zip(out, gs):
        ref = ns(g, torch.float64)
        norm, r = float(ref.norm()), float((ref.to(dt).double() - ref).norm())
        assert float((x.cpu().double() - ref).norm()) <= r + 2 * 2.0 ** -24 * norm, tuple(g.shape)


def test_tracing_is_refused():
    """A tracer would record the results' allocation alone."""
    from fc3d import ops
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: ops.orthogonalize(t), (torch.zeros(4, 4),), check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: ops.muon_step([t], [t], [t]), (torch.zeros(4, 4),), check_trace=False)


def test_shared_parameters_that_are_left_under_a_later_name():
    from fc3d import optim

    class Net(torch.nn.Module):
        def __init__(self, shared=None):
            super().__init__()
            self.embed = torch.nn.Embedding(10, 4)
            self.hidden = torch.nn.Linear(4, 4)
            self.head = torch.nn.Linear(4, 10, bias=False)
            self.head.weight = self.embed.weight
            if shared is not None:
                self.hidden.weight = shared
    a = Net()
    matrices, others = optim.split_parameters(a, leave=("head",))
    assert [id(p) for p in matrices] == [id(a.hidden.weight)]
    assert [id(p) for p in others] == [id(a.embed.weight), id(a.hidden.bias)]
    b = Net(shared=a.hidden.weight)
    b.last = b.hidden                                                  # one more name of a module in both
    matrices, others = optim.split_parameters([a, b], leave=("head", "last"))
    assert matrices == []
    assert [id(p) for p in others] == [id(p) for p in (a.embed.weight, a.hidden.weight, a.hidden.bias, b.embed.weight, b.hidden.bias)]
    assert len(optim.split_parameters([a, b])[0]) == 3


@gpu
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("steps", [5, 8])
def test_eps_far_above_the_norm(dt, steps):
    """X starts at norm / eps of its usual size and grows by a step after step; what it loses stays a share of itself.  (In
    fp16 only as far as the results are normal numbers.)"""
    from fc3d import ops
    for shape in ((100, 130), (96, 300), (300, 70)):
        g = update(shape, "gauss", 700 + shape[0], dt)
        norm = float(g.double().norm())
        for ratio in ((1.0, 3.0, 40.0) if dt == F16 else (1.0, 3.0, 40.0, 1e3, 1e5, 1e8, 1e12, 1e20)):
            near(ops.orthogonalize(g.cuda(), steps=steps, eps=ratio * norm), g, f"{shape} {ratio} {steps}", steps, eps=ratio * norm)
        # beside a matrix that eps does not reach: no other bits than without eps
        big = (g.float() * 2.0 ** 60).to(dt) if dt != F16 else g
        pair = ops.orthogonalize([big.cuda(), g.cuda()], steps=steps, eps=norm * (1e5 if dt != F16 else 1.0))
        near(pair[1], g, f"{shape} beside another", steps, eps=norm * (1e5 if dt != F16 else 1.0))
        if dt != F16:
            near(pair[0], big, f"{shape} large", steps)


@gpu
def test_step_with_eps_far_above_the_norm():
    from fc3d import ops
    w, g = (torch.randn(90, 200, generator=torch.Generator().manual_seed(710)) / 8), update((90, 200), "gauss", 711)
    for ratio in (1e3, 1e7):
        wd, md = w.cuda(), torch.zeros(90, 200, device="cuda")
        u = 0.05 * g.double() + 0.95 * 0.05 * g.double()               # Nesterov's from a momentum of zero
        eps = ratio * float(u.norm())
        ops.muon_step([wd], [g.cuda()], [md], lr=ratio, eps=eps)
        o = ns(u, torch.float64, eps=eps)
        ref = w.double() - ratio * o
        # as in test_step_against_definition
        tol = ratio * float(o.norm()) * (bound(u.float(), o, eps=eps) + 2.0 ** -20)
        tol += 5 * 2.0 ** -24 * float(ref.norm() + (w.double() - ref).norm())
        assert float((wd.cpu().double() - ref).norm()) <= tol, ratio


def workspace(shapes):
    import ctypes
    from fc3d import _native
    n, I64 = len(shapes), ctypes.c_int64
    return _native.load().fc3d_orthogonalize_workspace(n, (I64 * n)(*[s[0] for s in shapes]), (I64 * n)(*[s[1] for s in shapes]))


def test_workspace_of_long_lists_is_bounded():
    """Matrices go through the workspace group after group: a GiB and the sums of shared depth (256 tiles of 128 x 128 at
    most), or what one matrix alone needs."""
    most = 2 ** 30 + 2 ** 25
    for shape, count in (((4096, 4096), 48), ((1024, 1024), 200), ((4096, 1024), 48), ((64, 40000), 48), ((9, 50), 1000)):
        assert workspace([shape]) <= workspace([shape] * count) <= max(most, workspace([shape]))
    assert workspace([(8192, 8192)] * 48) == workspace([(8192, 8192)])
    assert workspace([(8192, 8192), (5, 7), (64, 288)]) <= workspace([(8192, 8192)]) + 2 ** 25
    # as ever: lists that fit go in one group
    assert workspace([(1024, 1024)] * 20) > 19 * workspace([(1024, 1024)])


@gpu
def test_lists_beyond_one_group_of_a_gib():
    """2048 x 4096 takes 176 MiB: groups of five.  The same bits as the groups by themselves, nothing written behind the
    workspace."""
    import ctypes
    from fc3d import _native
    lib, I64, VP = _native.load(), ctypes.c_int64, ctypes.c_void_p
    gen = torch.Generator(device="cuda").manual_seed(720)
    gs = [torch.randn(2048, 4096, generator=gen, device="cuda").bfloat16() for _ in range(7)]

    def call(gs):
        n = len(gs)
        size = workspace([tuple(g.shape) for g in gs])
        ws = torch.full((size + 512,), 77, dtype=torch.uint8, device="cuda")
        out = [torch.empty_like(g) for g in gs]
        at = lambda ts: (VP * n)(*[t.data_ptr() for t in ts])  # noqa: E731
        sizes = lambda d: (I64 * n)(*[g.shape[d] for g in gs])  # noqa: E731
        assert (ws.data_ptr() + 256) % 256 == 0
        assert lib.fc3d_orthogonalize(torch.cuda.current_stream().cuda_stream, n, at(gs), at(out), sizes(0), sizes(1), 1, 5, *COEFFS, 1e-7,
                                      ws.data_ptr() + 256) == 0
        torch.cuda.synchronize()
        assert bool((ws[:256] == 77).all()) and bool((ws[256 + size:] == 77).all())
        return out
    together = call(gs)
    for x, y in zip(together, call(gs[:5]) + call(gs[5:])):
        assert torch.equal(x, y) and bool(torch.isfinite(x).all())
    # singular values of a square Gaussian half: 0.67 to 1.21 of the polynomial, and a bf16 rounding
    s = torch.linalg.svdvals(together[6].float())
    assert 0.65 <= float(s[-1]) and float(s[0]) <= 1.22


def ns_device(g, dt, eps=1e-7):
    """The definition on the GPU, for sizes that take the CPU too long."""
    a, b, c = COEFFS
    x = g.to(dt)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t().contiguous()
    x = x / (torch.linalg.vector_norm(x) + eps)
    for _ in range(5):
        s = torch.mm(x, x.t().contiguous())
        x = a * x + torch.mm(b * s + c * torch.mm(s, s), x)
    return x.t() if tall else x


RAGGED = [(2003, 2153), (513, 113), (888, 929)]
DEEP_128 = [(424, 2304), (71, 451), (437, 271), (2334, 2092), (64, 3595)]
DEEP_96 = [(2933, 1964), (74, 11861), (1024, 148), (70, 4139), (312, 133)]


@gpu
@pytest.mark.parametrize("op,dt,shapes,kernels", [
    ("orthogonalize", BF16, [(2370, 2019)], {"ns_product_96_1x1", "ns_product_96_2x2", "ns_product_128_2x1"}),
    ("orthogonalize", BF16, [(135, 10871), (403, 172), (245, 130)], {"ns_product_64_1x1", "ns_gram_sum_64", "ns_product_96_2x1"}),
    ("orthogonalize", BF16, RAGGED, {"ns_product_128_1x1", "ns_product_128_2x2", "ns_product_64_2x2"}),
    ("orthogonalize", F16, RAGGED, {"ns_product_128_1x1", "ns_product_128_2x2", "ns_product_64_2x2", "ns_product_128_2x1"}),
    ("orthogonalize", BF16, [(90, 150)], {"ns_product_64_2x1"}),
    ("orthogonalize", F32, DEEP_96, {"ns_product_96_2x2", "ns_gram_sum_96", "ns_product_128_2x2"}),
    ("step", BF16, [(129, 7250), (545, 258), (343, 1711)], {"ns_product_64_2x2", "ns_product_96_2x2"}),
    ("step", BF16, DEEP_128, {"ns_product_128_2x2", "ns_gram_sum_128", "ns_product_64_2x2"}),
    ("step", BF16, DEEP_96, {"ns_product_96_2x2", "ns_gram_sum_96"}),
    ("step", F32, RAGGED, set()),
], ids=lambda v: str(v).replace("torch.", "") if not isinstance(v, (list, set)) else str(len(v)))
def test_every_product_kernel(op, dt, shapes, kernels):
    """Every kernel that the rules pick, at sizes that are no multiples of its tile: the names in the profile say that it
    ran, the definition what it should give, and guards that nothing beyond the tensors and the workspace is written."""
    import ctypes
    from fc3d import _native, ops, profiler
    lib, n = _native.load(), len(shapes)
    I64, VP, FL = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
    pad, code = 64, {F32: 0, BF16: 1, F16: 2}[dt]
    gen = torch.Generator(device="cuda").manual_seed(730 + n)

    def guarded(values):
        buf = torch.full((values.numel() + 2 * pad,), 512.0, dtype=values.dtype, device="cuda")
        buf[pad:-pad] = values.reshape(-1)
        return buf

    def inside(buf, shape):
        assert bool((buf[:pad] == 512.0).all()) and bool((buf[-pad:] == 512.0).all())
        return buf[pad:-pad].view(shape)
    at = lambda bufs: (VP * n)(*[b.data_ptr() + pad * b.element_size() for b in bufs])  # noqa: E731
    rows, cols = (I64 * n)(*[s[0] for s in shapes]), (I64 * n)(*[s[1] for s in shapes])
    size = lib.fc3d_orthogonalize_workspace(n, rows, cols)
    ws = torch.full((size + 512,), 77, dtype=torch.uint8, device="cuda")
    base, stream = ws.data_ptr() + 256, torch.cuda.current_stream().cuda_stream
    assert base % 256 == 0
    gs = [(1e-3 * torch.randn(s, generator=gen, device="cuda")).to(dt) for s in shapes]
    gb = [guarded(g) for g in gs]
    out = [guarded((torch.randn(s, generator=gen, device="cuda") / 16).to(dt)) for s in shapes]
    old = [inside(o, s).double().clone() for o, s in zip(out, shapes)]
    mom = [guarded(1e-3 * torch.randn(s, generator=gen, device="cuda")) for s in shapes]
    before = [inside(m, s).double().clone() for m, s in zip(mom, shapes)]
    lr, beta, decay = 0.02, 0.9, 0.998
    profiler.report()
    profiler.enable()
    try:
        if op == "step":
            status = lib.fc3d_muon_step(stream, n, at(out), at(gb), at(mom), rows, cols, (FL * n)(*[lr] * n), code, code, beta, 1, decay, 5,
                                        *COEFFS, 1e-7, base)
        else:
            status = lib.fc3d_orthogonalize(stream, n, at(gb), at(out), rows, cols, code, 5, *COEFFS, 1e-7, base)
        ran = set(profiler.report())
    finally:
        profiler.enable(False)
    torch.cuda.synchronize()
    assert status == 0 and kernels <= ran, (status, ran)
    assert bool((ws[:256] == 77).all()) and bool((ws[256 + size:] == 77).all())
    for i, s in enumerate(shapes):
        g, got = gs[i].double(), inside(out[i], s).double()
        assert torch.equal(inside(gb[i], s), gs[i])
        u, half = g, torch.finfo(dt).eps / 2
        if op == "step":
            m = beta * before[i] + (1 - beta) * g
            # as in test_step_against_definition
            off = (inside(mom[i], s).double() - m).abs()
            assert bool((off <= 4 * 2.0 ** -24 * (beta * before[i].abs() + (1 - beta) * g.abs()) + 2.0 ** -149).all()), s
            u = (1 - beta) * g + beta * m
        ref = ns_device(u, torch.float64)
        norm = float(ref.norm())
        tol = 4 * float((ns_device(u, F32).double() - ref).norm()) / norm + 2.0 ** -20 + \
            (0.0 if dt == F32 else half + 6e-3 / math.sqrt(min(s)))
        if op == "step":
            want = decay * old[i] - lr * ref
            tol = lr * norm * (tol + 2.0 ** -20) + (half + 4 * 2.0 ** -24) * float(want.norm() + (old[i] - want).norm())
        else:
            want, tol = ref, tol * norm
        assert float((got - want).norm()) <= tol, (s, float((got - want).norm()), tol)


def ns_gram32(g, steps, segment):
    """The definition's Gram form in fp32, `segment` steps to a Gram matrix."""
    a, b, c = COEFFS
    x = g.float()
    x = x / (x.norm() + 1e-7)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    eye = torch.eye(x.shape[0])
    for start in range(0, steps, segment):
        s, p = x @ x.t(), eye
        for _ in range(min(segment, steps - start)):
            q = a * eye + b * s + c * (s @ s)
            p, s = q @ p, q @ s @ q
        x = p @ x
    return x.t() if tall else x


@gpu
@pytest.mark.parametrize("dt", [BF16, F16], ids=lambda t: str(t).replace("torch.", ""))
@pytest.mark.parametrize("steps", [6, 8, 10, 16])
def test_many_steps_lose_no_more_than_their_rounding(dt, steps):
    """As test_half_precision_results_lose_no_more_than_their_rounding, with what may be lost in front of the rounding taken
    from fp32 again, four times: from fp32 products step by step and from the Gram form of two steps at a time in fp32."""
    from fc3d import ops
    for m, n in ((128, 300), (300, 77), (256, 1024)):
        gen = torch.Generator().manual_seed(m + n)
        g = (1e-3 * (torch.randn(m, 4, generator=gen) @ torch.randn(4, n, generator=gen) +
                     0.1 * torch.randn(m, n, generator=gen))).to(dt)
        ref = ns(g, torch.float64, steps)
        norm = float(ref.norm())
        r = float((ref.to(dt).double() - ref).norm()) / norm
        e = 4 * max(float((y.double() - ref).norm()) / norm for y in (ns(g, F32, steps), ns_gram32(g, steps, 2))) + 2.0 ** -20
        tol = math.sqrt((r * r + e * e) * (1 + 8 / math.sqrt(m * n)))
        off = float((ops.orthogonalize(g.cuda(), steps=steps).cpu().double() - ref).norm()) / norm
        assert off <= tol, (m, n, off, tol, r, e)


@gpu
@pytest.mark.parametrize("m", [17, 24, 40, 64, 100, 128])
def test_one_direction_over_little_noise_in_bf16(m):
    """Matrices of few rows beside a large one, the sum of squares over twenty of them; otherwise as
    test_half_precision_results_lose_no_more_than_their_rounding."""
    from fc3d import ops
    gs = []
    for i in range(20):
        n = (m, m + 1, m + 8, 2 * m, 200)[i % 5]
        gen = torch.Generator().manual_seed(800 + m + i)
        x = torch.randn(m, 1, generator=gen) @ torch.randn(1, n, generator=gen) + (0.003, 0.001)[i % 2] * torch.randn(m, n, generator=gen)
        gs.append((x.t() if i % 3 == 0 else x).contiguous().bfloat16())
    out = ops.orthogonalize([g.cuda() for g in gs] + [update((150, 200), "gauss", 799, BF16).cuda()])
    off = allowed = count = 0.0
    for x, g in zip(out, gs):
        ref = ns(g, torch.float64)
        x2 = ns(g, torch.float64, 2)
        x2 = x2.t() if x2.shape[0] > x2.shape[1] else x2
        r = float((ref.bfloat16().double() - ref).norm())
        e = 4 * float((ns(g, F32).double() - ref).norm()) + 2.0 ** -20 * float(ref.norm())
        e += second_segment_slope() * 2.0 ** -22 * float((x2 @ x2.t()).norm())
        off += float((x.cpu().double() - ref).norm()) ** 2
        allowed += r * r + e * e
        count += g.numel()
    assert off <= allowed * (1 + 8 / math.sqrt(count)), (math.sqrt(off / allowed), count)


@gpu
def test_plans_of_few_and_of_many_rows_side_by_side():
    """bf16 matrices of up to 128 rows and of more go through other sequences of products in the same launches."""
    from fc3d import ops
    gs = [update(s, "gauss", 820 + i, BF16) for i, s in enumerate([(128, 200), (129, 200), (70, 300), (300, 140), (20, 500), (500, 65)])]
    for g, x in zip(gs, ops.orthogonalize([g.cuda() for g in gs])):
        near(x, g, f"{tuple(g.shape)}")
    for steps in (1, 2, 3, 4):
        for g, x in zip(gs, ops.orthogonalize([g.cuda() for g in gs], steps=steps)):
            near(x, g, f"{tuple(g.shape)} {steps}", steps)
