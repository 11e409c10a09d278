"""Retention layers on padded batches: lengths reach every pixel of their own sequence, in the outputs, the states that leave and the gradients.

Tolerances as for the layers' other results: a layer chains five operators that are within 2^-19 of their results, two layers are within 2^-15, gradients 2^-14."""
import pytest
import torch

from satflow_amd.models.layers import Retention

pytestmark = pytest.mark.gpu

FWD, BWD = 2.0**-15, 2.0**-14


def _rel(a, b):
    b = b.double()
    n = float(b.norm())
    return float((a.double() - b).norm()) / n if n else float(a.double().norm())


def test_lengths_of_frames(device):
    torch.manual_seed(0)
    model = Retention(16, 1, heads=2).to(device)
    x = torch.randn(2, 6, 16, 3, 5, device=device, requires_grad=True)
    lengths = torch.tensor([6, 4], dtype=torch.int32, device=device)
    y, last = model(x, lengths=lengths, return_state=True)
    gs = torch.randn_like(last[0])
    (gx,) = torch.autograd.grad(last, x, [gs])
    for b, n in enumerate((6, 4)):
        alone = x[b, :n][None].detach().requires_grad_()
        yb, sb = model(alone, return_state=True)
        (gb,) = torch.autograd.grad(sb, alone, [gs[15 * b:15 * b + 15]])
        assert _rel(y[b, :n].detach(), yb[0].detach()) < FWD
        assert _rel(last[0][15 * b:15 * b + 15].detach(), sb[0].detach()) < FWD
        assert _rel(gx[b, :n], gb[0]) < BWD
    assert not gx[1, 4:].any() and gx[0, 4:].abs().amax(dim=(1, 2, 3)).min() > 0


@pytest.mark.parametrize("T", [24, 150])
def test_lengths_of_tokens_through_two_layers(device, T):
    torch.manual_seed(1)
    model = Retention(48, 2, heads=4).to(device)
    lengths = [T, 0, 1, T - 5]
    x = torch.randn(4, T, 48, device=device, requires_grad=True)
    s0 = [torch.randn_like(s) for s in model.initial_state(4)]
    y, last = model(x, s0, lengths=torch.tensor(lengths, dtype=torch.int32, device=device), return_state=True)
    gy, gs = torch.randn_like(y), [torch.randn_like(s) for s in last]
    for b, n in enumerate(lengths):
        gy[b, n:] = 0
    params = list(model.parameters())
    got = torch.autograd.grad([y, *last], [x, *params], [gy, *gs])
    sums = [torch.zeros_like(p, dtype=torch.float64) for p in params]
    for b, n in enumerate(lengths):
        if n == 0:
            assert all(torch.equal(a[b], s[b]) for a, s in zip(last, s0))
            assert not got[0][b].any()
            continue
        alone = x[b, :n][None].detach().requires_grad_()
        yb, sb = model(alone, [s[b][None] for s in s0], return_state=True)
        gb = torch.autograd.grad([yb, *sb], [alone, *params], [gy[b, :n][None], *[g[b][None] for g in gs]])
        assert _rel(y[b, :n].detach(), yb[0].detach()) < FWD
        for a, s in zip(last, sb):
            assert _rel(a[b].detach(), s[0].detach()) < FWD
        assert _rel(got[0][b, :n], gb[0][0]) < BWD and not got[0][b, n:].any()
        for t, g in zip(sums, gb[1:]):
            t += g.double()
    for g, t in zip(got[1:], sums):
        assert _rel(g, t) < BWD


def test_no_sequences_and_no_frames(device):
    model = Retention(32, 2, heads=2).to(device)
    with torch.no_grad():
        y, last = model(torch.zeros(0, 5, 32, device=device), return_state=True)
        assert y.shape == (0, 5, 32) and [tuple(s.shape) for s in last] == [(0, 2, 16, 16)] * 2
        s0 = [torch.randn_like(s) for s in model.initial_state(3)]
        y, last = model(torch.zeros(3, 0, 32, device=device), s0, return_state=True)
        assert y.shape == (3, 0, 32) and all(torch.equal(a, b) for a, b in zip(last, s0))
        assert model.step(torch.zeros(0, 32, device=device), model.initial_state(0)).shape == (0, 32)
