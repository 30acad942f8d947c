"""The U-Nets with a layer norm, Muon over their hidden convolutions, and the training step that uses both
(fc3d.nets, fc3d.optim, fc3d.capture.TrainStep)."""
import os
import sys

import numpy as np
import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
from test_muon import F32, bound, ns  # noqa: E402

gpu = pytest.mark.gpu


# ---- on the CPU -------------------------------------------------------------------------------------------------

def test_layer_norm_networks_on_the_cpu():
    from fc3d import nets
    with pytest.raises(ValueError, match="norm"):
        nets.UNet_xy(norm="group")
    with pytest.raises(ValueError, match="norm"):
        nets.ConvBN(3, 4, norm="group")
    plain, net = nets.UNet_z(), nets.UNet_z(norm="layer")
    names, other = set(plain.state_dict()), set(net.state_dict())
    assert not [n for n in names if ".norm." in n] and not [n for n in other if ".bn." in n or "running" in n]
    assert {n for n in names if ".conv." in n} == {n for n in other if ".conv." in n}
    assert not [n for n in other if n.startswith("up1_3.norm")]             # the head has none
    torch.manual_seed(3)
    x = torch.rand(2, 32, 48, 1)
    y = net(x)
    assert y.shape == (2, 32, 48, 1)
    y.sum().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in net.parameters())
    # a sample's result does not depend on its batch: train and eval modes agree, and each sample alone
    net.eval()
    with torch.no_grad():
        assert torch.equal(net(x), y.detach())
        assert float((net(x[1:]) - y[1:]).abs().max()) <= 1e-4              # other convolution kernels for other batches


def test_channel_norm_formula():
    from fc3d import nets
    torch.manual_seed(4)
    m = nets.ChannelNorm(6, relu=True, eps=1e-3).double()
    with torch.no_grad():
        m.weight.normal_()
        m.bias.normal_()
    x = torch.randn(2, 6, 3, 4, dtype=torch.float64)
    mu, var = x.mean(1, keepdim=True), x.var(1, unbiased=False, keepdim=True)
    want = ((x - mu) / (var + 1e-3).sqrt() * m.weight.view(1, 6, 1, 1) + m.bias.view(1, 6, 1, 1)).clamp(min=0.0)
    assert float((m(x) - want).detach().abs().max()) <= 1e-12


def test_split_parameters():
    from fc3d import nets, optim
    a, b = nets.UNet_xy(norm="layer"), nets.UNet_z(norm="layer")
    matrices, others = optim.split_parameters([a, b], leave=nets.UNet.EDGES)
    everything = list(a.parameters()) + list(b.parameters())
    assert sorted(map(id, matrices + others)) == sorted(map(id, everything))
    assert len(matrices) == 2 * 21 and all(p.dim() == 4 for p in matrices)
    kept = {n for n, p in a.named_parameters() if p.dim() == 4 and any(p is q for q in others)}
    assert kept == {"down1_1.conv.weight", "up1_3.conv.weight"}
    shared = torch.nn.Linear(3, 4)
    matrices, others = optim.split_parameters(torch.nn.Sequential(shared, shared))
    assert len(matrices) == 1 and len(others) == 1                          # a shared weight once
    twins = torch.nn.ModuleDict({"a": torch.nn.Linear(2, 2), "ab": torch.nn.Linear(2, 2)})
    matrices, others = optim.split_parameters(twins, leave=("a",))
    assert matrices == [twins["ab"].weight]                                 # a name, not a prefix of names


def test_train_step_refusals():
    from fc3d import capture
    with pytest.raises(ValueError, match="optimizer"):
        capture.TrainStep("cpu", optimizer="sgd")
    with pytest.raises(ValueError, match="norm"):
        capture.TrainStep("cpu", norm="group")


# ---- on the GPU -------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("memory", [torch.contiguous_format, torch.channels_last])
def test_block_and_its_gradients(memory):
    """One convolution with norm and ReLU: result and gradients against the same block in 64 bits on the CPU.
    Bound: the convolution sums k = 9 c_in products in fp32 in some order, sqrt(k) half steps at the usual spread and
    k at most; the norm adds its own few.  16 (1 + sqrt(k)) half steps of the largest value."""
    from fc3d import nets
    torch.manual_seed(5)
    ref = nets.ConvBN(24, 40, norm="layer").double()
    with torch.no_grad():
        ref.norm.weight.normal_(1.0, 0.3)
        ref.norm.bias.normal_(0.0, 0.3)
        for p in ref.parameters():
            p.copy_(p.float())
    net = nets.ConvBN(24, 40, norm="layer")
    net.load_state_dict({k: v.float() for k, v in ref.state_dict().items()})
    net = net.cuda().to(memory_format=memory)
    x = torch.randn(3, 24, 17, 21)
    up = torch.randn(3, 40, 17, 21)
    xr = x.double().requires_grad_()
    xd = x.cuda().contiguous(memory_format=memory).requires_grad_()
    # values within rounding of the ReLU's edge may fall on either side: their gradient is taken out on both
    pre = nets.F.layer_norm(ref.conv(nets.F.pad(xr, (1,) * 4, mode="reflect")).movedim(1, -1), (40,), ref.norm.weight,
                            ref.norm.bias, ref.norm.eps).movedim(-1, 1).detach()
    up = up * (pre.abs() > 1e-4)
    y, yr = net(xd), ref(xr)
    y.backward(up.cuda())
    yr.backward(up.double())
    half = 2.0 ** -24
    tol = 16 * (1 + (9 * 24) ** 0.5) * half
    off = float((y.detach().cpu().double() - yr.detach()).abs().max())
    assert off <= tol * float(yr.detach().abs().max())
    for name, a, b, terms in [("x", xd.grad, xr.grad, 9 * 40)] + \
            [(n, p.grad, q.grad, 3 * 17 * 21) for (n, p), (_, q) in zip(net.named_parameters(), ref.named_parameters())]:
        off = float((a.cpu().double() - b).norm() / b.norm())
        # the values themselves carry the forward's relative error into every gradient
        if name == "conv.bias":                       # sums of 1071 terms that nearly cancel: relative to the terms' size
            off *= float(b.norm()) / float(xr.grad.norm())
        assert off <= tol + 16 * (1 + terms ** 0.5) * half, (name, off)


@gpu
@pytest.mark.timeout(300)
def test_train_step_with_layer_norm_and_muon(monkeypatch):
    """A step's weights follow from its gradients by the two optimisers' formulas."""
    monkeypatch.setenv("MIOPEN_FIND_MODE", "FAST")
    import optics_pytorch as O
    from fc3d import capture, nets, optim, ops, synth
    B, H, W = 2, 64, 64
    O.PSFs_np = synth.make_psfs(21, 5, "disc")
    sc = synth.make_scene(B, H, W, 93)
    d = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    torch.manual_seed(0)
    step = capture.TrainStep(torch.device("cuda"), intrinsics=(W / 2, H / 2), norm="layer", optimizer="muon")
    assert isinstance(step.muon, optim.Muon)
    matrices, others = optim.split_parameters([step.model_xy, step.model_z], leave=nets.UNet.EDGES)
    assert [id(p) for p in step.muon.param_groups[0]["params"]] == [id(p) for p in matrices]
    momenta = [torch.zeros(p.shape, dtype=torch.float64) for p in matrices]
    for k in range(2):
        w0 = [p.detach().clone() for p in matrices]
        o0 = [p.detach().clone() for p in others]
        loss = float(step(d(sc["z_p"]), d(sc["z_c"]), d(sc["pose_p2c"])))
        assert np.isfinite(loss)
        for i, (p, w) in enumerate(zip(matrices, w0)):
            g = p.grad.cpu().double()
            momenta[i] = 0.95 * momenta[i] + 0.05 * g
            u = 0.05 * g + 0.95 * momenta[i]
            o = ns(u, torch.float64)
            scale = 0.02 * ops.muon_scale(p.shape, "spectral")
            want = w.cpu().double() - scale * o
            tol = scale * float(o.norm()) * (bound(u.float(), o, dt=F32) + 2.0 ** -20) + 4 * 2.0 ** -24 * float(want.norm() + w.norm())
            assert float((p.detach().cpu().double() - want).norm()) <= tol, (k, i, tuple(p.shape))
        # Adam moves by at most lr (1 + a little) a step, and every gradient that is not zero moves its weight
        for p, w in zip(others, o0):
            move = (p.detach() - w).abs()
            assert float(move.max()) <= 2e-4
            assert not bool(((p.grad != 0) & (move == 0) & (p.grad.abs() > 1e-6)).any()) or k > 0


@gpu
def test_graph_of_a_block_and_its_step(monkeypatch):
    """Forward, backward and the Muon step of a block captured into one graph, replayed several times with the program's
    own work in between: every replay against the eager run."""
    monkeypatch.setenv("MIOPEN_FIND_MODE", "FAST")
    from fc3d import nets, ops
    torch.manual_seed(6)
    norm = nets.ChannelNorm(48, relu=True).cuda()
    w = torch.randn(48, 48, device="cuda") / 7
    x = torch.randn(4, 48, 9, 10, device="cuda")
    up = torch.randn(4, 48, 9, 10, device="cuda")

    def step(w, mom, x):
        leaves = [x.detach().requires_grad_(), norm.weight.detach().requires_grad_(), norm.bias.detach().requires_grad_()]
        y = ops.layer_norm(leaves[0], leaves[1], leaves[2], dim=1, relu=True)
        dx, dw, db = torch.autograd.grad(y, leaves, up)
        g = dx.movedim(1, 0).reshape(48, -1)[:, :48].contiguous()
        ops.muon_step([w], [g], [mom])
        return y.detach(), dx, dw, db

    we, me = w.clone(), torch.zeros_like(w)
    wg, mg, xg = w.clone(), torch.zeros_like(w), x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(wg.clone(), mg.clone(), xg)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(wg, mg, xg)
    for k in range(4):
        xk = x * (1 + 0.25 * k)
        want = step(we, me, xk)
        xg.copy_(xk)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(list(out) + [wg, mg], list(want) + [we, me]):
            assert torch.equal(a, b), k


@gpu
@pytest.mark.timeout(300)
def test_traced_network(monkeypatch):
    """A frozen network traced for serving gives what the network gives: the norms are recorded as calls.  Other convolution
    kernels may be picked in the traced one: sums of up to 9 * 512 products in another order, through 23 convolutions."""
    monkeypatch.setenv("MIOPEN_FIND_MODE", "FAST")
    from fc3d import nets
    torch.manual_seed(7)
    net = nets.UNet_z(norm="layer").cuda().eval().requires_grad_(False)
    x = torch.rand(2, 32, 48, 1, device="cuda")
    traced = torch.jit.trace(net, (torch.rand(2, 32, 48, 1, device="cuda"),), check_trace=False)
    assert str(traced.inlined_graph).count("^LayerNormFn") == sum(isinstance(m, nets.ChannelNorm) for m in net.modules())
    want = net(x)
    assert float((traced(x) - want).abs().max()) <= 23 * (9 * 512) ** 0.5 * 2.0 ** -24 * 16 * float(want.abs().max())
