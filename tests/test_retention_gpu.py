"""The retention layers (satflow_amd.models.layers.Retention): norms, projections and linear attention together, against the same mathematics in float64.

Tolerance, fixed before the first run: errors are 2-norms relative to the result's.  Every operator of the chain is fp32-accurate, within 2^-19 of its result (sums
of some hundreds of terms); a layer chains five of them, and its norms pass relative errors on unchanged: two layers are within 10 * 2^-19, below 2^-15.  The backward
pass chains the same operators' gradients behind the forward ones: twice that, 2^-14."""
import pytest
import torch

from satflow_amd.models.layers import Retention

pytestmark = pytest.mark.gpu

FWD, BWD = 2.0**-15, 2.0**-14


def _rel(a, b):
    b = b.double()
    n = float(b.norm())
    return float((a.double() - b).norm()) / n if n else float(a.double().norm())


def _rms(x, w, eps, groups=1):
    y = x.unflatten(-1, (groups, -1))
    return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)).flatten(-2) * w


def _plain(model, params, x, states=None):
    """The stack in float64, token by token; params: name -> float64 leaf."""
    last = []
    for i, m in enumerate(model.layers):
        p = {n: params[f"layers.{i}.{n}"] for n, _ in m.named_parameters()}
        n, d, e = m.heads, m.key_dim, m.value_dim
        B, T, _ = x.shape
        y = _rms(x, p["norm_in"], m.eps) @ p["to_qkvg.weight"].t()
        q, k, v, g = y.split((n * d, n * d, n * e, n * e), -1)
        q, k, v = q.view(B, T, n, d), k.view(B, T, n, d), v.view(B, T, n, e)
        lam = torch.exp(m.log_decay.double())[None, :, None, None]
        S = torch.zeros(B, n, d, e, dtype=torch.float64, device=x.device) if states is None else states[i].double()
        o = []
        for t in range(T):
            S = lam * S + k[:, t, :, :, None] * v[:, t, :, None, :]
            o.append((q[:, t, :, :, None] * S).sum(2) * d**-0.5)
        o = torch.stack(o, 1).flatten(-2)
        a = torch.nn.functional.silu(g) * _rms(o, p["norm_heads"], m.eps, n)
        x = x + p["scale"] * _rms(a @ p["to_out.weight"].t(), p["norm_out"], m.eps)
        last.append(S)
    return x, last


def _model(device, *args, seed=0, **kw):
    torch.manual_seed(seed)
    m = Retention(*args, **kw)
    for p in m.parameters():
        if p.dim() == 1:
            p.data.add_(0.25 * torch.randn_like(p))
    return m.to(device)


@pytest.mark.parametrize("dim,layers,kw,B,T", [
    (32, 1, dict(heads=2), 3, 24),
    (64, 2, dict(heads=4, key_dim=12, value_dim=20), 2, 133),
    (48, 2, dict(heads=1, key_dim=128, value_dim=112), 1, 65),
    (16, 1, dict(heads=1), 5, 1),
])
def test_forward_and_gradients(device, dim, layers, kw, B, T):
    model = _model(device, dim, layers, **kw)
    x = torch.randn(B, T, dim, device=device, requires_grad=True)
    gy = torch.randn(B, T, dim, device=device)
    s0 = [0.5 * torch.randn_like(s) for s in model.initial_state(B)]
    for s in s0:
        s.requires_grad_()
    y, last = model(x, s0, return_state=True)
    gs = [torch.randn_like(s) for s in last]
    torch.autograd.backward([y, *last], [gy, *gs])

    params = {n: p.detach().double().requires_grad_() for n, p in model.named_parameters()}
    xd, sd = x.detach().double().requires_grad_(), [s.detach().double().requires_grad_() for s in s0]
    yd, ld = _plain(model, params, xd, sd)
    torch.autograd.backward([yd, *ld], [gy.double(), *[g.double() for g in gs]])
    assert _rel(y.detach(), yd.detach()) < FWD
    for a, b in zip(last, ld):
        assert _rel(a.detach(), b.detach()) < FWD
    assert _rel(x.grad, xd.grad) < BWD
    for a, b in zip(s0, sd):
        assert _rel(a.grad, b.grad) < BWD
    for n, p in model.named_parameters():
        assert _rel(p.grad, params[n].grad) < BWD, n


def test_prompt_and_steps_equal_one_pass(device):
    model = _model(device, 64, 2, heads=4, key_dim=24, value_dim=16)
    x = torch.randn(3, 90, 64, device=device)
    with torch.no_grad():
        whole, _ = _plain(model, {n: p.double() for n, p in model.named_parameters()}, x.double())
        assert _rel(model(x), whole) < FWD
        y, state = model(x[:, :70], return_state=True)
        parts = [y] + [model.step(x[:, t], state)[:, None] for t in range(70, 90)]
        assert _rel(torch.cat(parts, 1), whole) < FWD
        fresh = model.initial_state(3)
        assert _rel(torch.stack([model.step(x[:, t], fresh) for t in range(40)], 1), whole[:, :40]) < FWD


def test_steps_in_a_graph(device):
    """One captured step, replayed for every frame, with eager work between the replays."""
    model = _model(device, 32, 2, heads=2)
    frames = torch.randn(12, 5, 32, device=device)
    with torch.no_grad():
        eager_state = model.initial_state(5)
        eager = [model.step(f, eager_state) for f in frames]
        state, x = model.initial_state(5), torch.zeros(5, 32, device=device)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model.step(x, model.initial_state(5))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model.step(x, state)
        for s in state:
            s.zero_()
        for f, want in zip(frames, eager):
            x.copy_(f)
            graph.replay()
            assert torch.equal(y, want)
            model(frames[:4].transpose(0, 1).contiguous())
            torch.cuda.synchronize()
        for a, b in zip(state, eager_state):
            assert torch.equal(a, b)


def test_frames_are_sequences_of_pixels(device):
    model = _model(device, 16, 1, heads=2)
    x = torch.randn(2, 6, 16, 3, 5, device=device, requires_grad=True)
    lengths = torch.tensor([6, 4], dtype=torch.int32, device=device)
    y, last = model(x, lengths=lengths, return_state=True)
    assert y.shape == x.shape and last[0].shape == (30, 2, 8, 8)
    y[:, :4].sum().backward()
    assert x.grad[1, 4:].abs().max() == 0
    with torch.no_grad():
        one = model(x[1, :4, :, 2, 3][None].contiguous())
        assert _rel(y[1, :4, :, 2, 3], one[0]) < FWD
        state = model.initial_state(30)
        steps = torch.stack([model.step(x[:, t], state) for t in range(4)], 1)
        assert _rel(y[:, :4], steps) < FWD


def test_gradient_against_differences(device):
    model = _model(device, 16, 1, heads=2)
    x = torch.randn(2, 9, 16, device=device)
    gy = torch.randn_like(x)
    dirs = {n: torch.randn_like(p) for n, p in model.named_parameters()}
    (model(x) * gy).sum().backward()
    slope = sum(float((p.grad.double() * dirs[n].double()).sum()) for n, p in model.named_parameters())
    step = 2.0**-7   # difference of the float32 forward: error of the slope step^2 (third derivatives of order the slope's) and 2^-19 |loss| / step
    out = []
    with torch.no_grad():
        for sign in (1, -1):
            for n, p in model.named_parameters():
                p.add_(dirs[n], alpha=sign * step)
            out.append(float((model(x).double() * gy.double()).sum()))
            for n, p in model.named_parameters():
                p.sub_(dirs[n], alpha=sign * step)
    size = sum(float(p.grad.double().norm() * dirs[n].double().norm()) for n, p in model.named_parameters())
    assert abs((out[0] - out[1]) / (2 * step) - slope) < 2.0**-6 * size
