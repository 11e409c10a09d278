"""Linear attention (satflow_amd.functional_seq) on the paths that a call's sizes, types and alignment choose, and at the ends of their ranges: the kernels of 64-token
chunks (bfloat16, both widths above 32), of 32-token chunks, for tensors that cannot be moved 16 bytes at a time (widths that are not multiples of 8), for sequences of at
most 32 tokens, and the segments' states joined by every workgroup or by a kernel (more than 65536 floats of them for each sequence and head).

Tolerances, fixed before the first run, are those of the same results elsewhere: 2-norms relative to the result's, 2^-8 for bfloat16 outputs (one rounding, at most half a
step of 2^-8 of the value, and less than that in front of it), 2^-19 for float32 outputs and all states (products of 24-bit operands, some hundreds of terms of both
signs)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-19}


def _rel(a, b):
    b = b.double()
    n = float(b.norm())
    return float((a.double() - b).norm()) / n if n else float(a.double().norm())


def _recurrence(q, k, v, g, s0, n, do, ds):
    """Outputs, last state and gradients, token by token in float64; n: tokens of each sequence."""
    q, k, v, do = q.double() * q.shape[-1] ** -0.5, k.double(), v.double(), do.double()
    lam, S, R = torch.exp(g.double())[None, :, None, None], s0.double(), ds.double()
    o, dq, dk, dv = torch.zeros_like(v), torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(v)
    T = q.shape[1]
    for t in range(T):
        live = (t < n)[:, None, None, None]
        S = torch.where(live, lam * S + k[:, t, :, :, None] * v[:, t, :, None, :], S)
        o[:, t] = torch.where(live[..., 0], (q[:, t, :, :, None] * S).sum(2), o[:, t])
        dq[:, t] = torch.where(live[..., 0], (S * do[:, t, :, None, :]).sum(-1) * q.shape[-1] ** -0.5, dq[:, t])
    for t in reversed(range(T)):
        live = (t < n)[:, None, None, None]
        at = R + q[:, t, :, :, None] * do[:, t, :, None, :]
        dk[:, t] = torch.where(live[..., 0], (at * v[:, t, :, None, :]).sum(-1), dk[:, t])
        dv[:, t] = torch.where(live[..., 0], (at * k[:, t, :, :, None]).sum(2), dv[:, t])
        R = torch.where(live, lam * at, R)
    return o, S, dq, dk, dv, R


NAMES = ("o", "state", "dq", "dk", "dv", "dstate")
TYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
# 64-token chunks (equal and unequal classes of widths), 32-token chunks, widths that are not multiples of 8
WIDTHS = pytest.mark.parametrize("dk,dv", [(64, 64), (128, 64), (40, 72), (128, 128), (32, 128), (20, 12)])


def _inputs(device, B, T, H, dk, dv, dtype, seed, slow=1.0):
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen).to(device)

    q, k, v, do = (rand(B, T, H, d).to(dtype) for d in (dk, dk, dv, dv))
    g = -torch.rand(H, generator=gen).to(device) * torch.tensor([0.003, 0.05, 0.7], device=device).repeat(H)[:H] * slow
    return q, k, v, g, rand(B, H, dk, dv), do, rand(B, H, dk, dv)


def _ours(q, k, v, g, s0, do, ds, lengths=None):
    from satflow_amd import functional_seq as S

    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, s0)]
    o, last = S.linear_attention(*leaves[:3], g, initial_state=leaves[3], lengths=lengths, return_state=True)
    return (o.detach(), last.detach(), *torch.autograd.grad([o, last], leaves, [do, ds]))


@TYPES
@WIDTHS
@pytest.mark.parametrize("T,lengths", [(20, [0, 1, 20, 19, 7]), (300, [300, 0, 1, 128, 255]), (70, [64, 65, 63, 99, -3]), (1100, [1100, 1, 999, 0, 512])])
def test_lengths(device, dtype, dk, dv, T, lengths):
    """What lies behind a sequence's length is not read, its outputs and gradients are zero, the state passes by it."""
    x = _inputs(device, len(lengths), T, 2, dk, dv, dtype, T + dk)
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    want = _recurrence(*x[:5], n, *x[5:])
    behind = torch.arange(T, device=device) >= n.clamp(0, T)[:, None]
    q, k, v, do = (t.masked_fill(behind[:, :, None, None], float("nan")) for t in (*x[:3], x[5]))
    got = _ours(q, k, v, x[3], x[4], do, x[6], n)
    for name, a, b in zip(NAMES, got, want):
        assert torch.isfinite(a).all() and _rel(a, b) <= TOL[a.dtype], (name, _rel(a, b))
        if "state" not in name:
            assert not a[behind].any(), name
    empty = n.clamp(0, T) == 0
    assert torch.equal(got[1][empty], x[4][empty]) and torch.equal(got[5][empty], x[6][empty])


@TYPES
@WIDTHS
@pytest.mark.parametrize("T", [30, 50, 130, 700])
def test_values_that_are_not_finite(device, dtype, dk, dv, T):
    """A bad q, k, v or gradient reaches the tokens that depend on it and no other, bit for bit, in the outputs and in every gradient; in one value column only where it stands
    in v; never another head."""
    x = _inputs(device, 1, T, 2, dk, dv, dtype, 3)
    at = T // 2 + 5
    base = _ours(*x)
    # which tokens of (o, dq, dk, dv) may change: o and dq depend on k and v of earlier tokens, dk and dv on q and do of later ones
    after, before, own = slice(at, None), slice(None, at + 1), slice(at, at + 1)
    none = slice(0, 0)
    reach = {0: (own, none, before, before), 1: (after, after, none, own), 2: (after, after, own, none), 5: (none, own, before, before)}
    for bad in (float("nan"), float("inf"), float("-inf")):
        for which, slices in reach.items():
            y = [t.clone() for t in x]
            y[which][:, at, 1, 3] = bad
            got = _ours(*y)
            for name, a, b, s in zip(("o", "dq", "dk", "dv"), (got[0], *got[2:5]), (base[0], *base[2:5]), slices):
                keep = torch.ones(T, dtype=torch.bool, device=device)
                keep[s] = False
                assert torch.equal(a[:, keep, 1], b[:, keep, 1]), (bad, which, name)
                assert torch.equal(a[:, :, 0], b[:, :, 0]), "the other head"
                assert torch.isfinite(a[:, keep]).all()
            if which == 2:   # (the state and the outputs in one column, where it stays)
                cols = torch.arange(dv, device=device) != 3
                assert torch.equal(got[0][..., cols], base[0][..., cols]) and torch.equal(got[1][..., cols], base[1][..., cols])
                assert not torch.isfinite(got[0][:, at:, 1, 3]).any() and not torch.isfinite(got[1][0, 1, :, 3]).any()
            if which == 5:
                assert not torch.isfinite(got[4][:, :at + 1, 1, 3]).any()


@TYPES
@WIDTHS
@pytest.mark.parametrize("decay", [0.0, -1e-4, -3.0, -60.0, float("-inf")])
def test_extreme_decays(device, dtype, dk, dv, decay):
    x = _inputs(device, 2, 333, 1, dk, dv, dtype, 9)
    x = (*x[:3], torch.full((1,), decay, device=device), *x[4:])
    want = _recurrence(*x[:5], torch.full((2,), 333, device=device), *x[5:])
    for name, a, b in zip(NAMES, _ours(*x), want):
        assert _rel(a, b) <= TOL[a.dtype], (name, _rel(a, b))


@TYPES
@pytest.mark.parametrize("B,T,H,dk,dv", [(1, 3001, 1, 128, 128), (2, 2500, 2, 64, 128), (3, 1000, 2, 100, 96), (1, 2900, 2, 64, 120)])
@pytest.mark.parametrize("padded", [False, True])
def test_joined_segments(device, dtype, B, T, H, dk, dv, padded):
    """States of the segments joined by the kernel of their own, under decays so slow that a state of the first tokens is felt by the last ones (exp(-0.0003 * 3000) = 0.4)."""
    from satflow_amd import _hip

    if padded:
        B = 5
    floats = _hip.lib().sf_linear_attention_workspace_bytes(B, T, H, dk, dv, 0) // 4
    segments = floats // (B * H * dk * dv)
    assert segments * dk * dv > 65536, "sizes of this test: the states are joined by the kernel"
    chunks = (T + 63) // 64
    tokens = (chunks + segments - 1) // segments * 64   # of a segment
    lengths = torch.tensor([0, 1, tokens, tokens + 1, T], dtype=torch.int32, device=device) if padded else None
    x = _inputs(device, B, T, H, dk, dv, dtype, T + B, slow=0.1)
    want = _recurrence(*x[:5], torch.full((B,), T, device=device) if lengths is None else lengths, *x[5:])
    for name, a, b in zip(NAMES, _ours(*x, lengths), want):
        assert _rel(a, b) <= TOL[a.dtype], (name, _rel(a, b))


@pytest.mark.parametrize("T,dk,dv", [(24, 32, 32), (100, 32, 32), (300, 64, 64), (2000, 128, 128), (777, 40, 72), (300, 20, 12)])
def test_bfloat16_outputs_are_nearly_correctly_rounded(device, T, dk, dv):
    """What is added in front of a bfloat16 output's one rounding: scores and states enter their products with 16 bits, so an error e of at most 2 * 2^-17 of the result in
    the mean.  It changes the rounded value with probability e / step, by one step (at most 2^-7 of the value): in the 2-norm sqrt(2^-16 * 2^-7) = 2^-11.5 against the
    exact result rounded to bfloat16.  (8 bits in one of the two places: 2^-9 instead of 2^-17, 2^-8.)"""
    x = _inputs(device, 2, T, 2, dk, dv, torch.bfloat16, 17)
    want = _recurrence(*x[:5], torch.full((2,), T, device=device), *x[5:])
    for name, a, b in zip(NAMES, _ours(*x), want):
        if "state" not in name:
            assert _rel(a, b.to(torch.bfloat16)) <= 2.0**-11.5, (name, _rel(a, b.to(torch.bfloat16)))


def test_longest_sequence(device):
    """The longest sequence there is, 2^31 - 66 tokens: its 2048 segments of 2^20 tokens end behind 2^31.  Under a decay of 0.05 a token nothing is left after 4096 tokens
    (exp(-204) is below 2^-290), so the last tokens (the last segment forward) and the first ones (the last segment of the reverse sweeps) are those of a call on
    either end alone, within the rounding of both to bf16 (2^-8 each); the state, fp32 sums of 24-bit products, within 2^-19 of the exact one in both."""
    from satflow_amd import functional_seq as S

    if torch.cuda.mem_get_info()[1] < 120 * 2**30:
        pytest.skip("takes 60 GB of device memory")
    T, end, keep = 2**31 - 66, 8192, 3000
    gen = torch.Generator(device=device).manual_seed(3)
    x = torch.randn(2**20, generator=gen, device=device, dtype=torch.float32).to(torch.bfloat16)
    long = torch.cat([x.repeat(2047), x[: 2**20 - 66].flip(0)]).view(1, T, 1, 1)
    g = torch.full((1,), -0.05, device=device)

    def run(t):
        k = (t.detach() * 0.5).requires_grad_()
        q, v = (t.detach().view_as(t).requires_grad_() for _ in range(2))
        o, last = S.linear_attention(q, k, v, g, return_state=True)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), t)), last.detach()

    whole, last = run(long)
    head, _ = run(long[:, :end].clone())
    tail, left = run(long[:, -end:].clone())
    for name, a, b, c in zip(("o", "dq", "dk", "dv"), whole, head, tail):
        assert _rel(a[:, :keep], b[:, :keep]) <= 2 * TOL[torch.bfloat16], name
        assert _rel(a[:, -keep:], c[:, -keep:]) <= 2 * TOL[torch.bfloat16], name
    assert _rel(last, left) <= 2 * TOL[torch.float32]


@TYPES
@pytest.mark.parametrize("T", [20, 150])
def test_broadcast_and_far_apart_tokens(device, dtype, T):
    """Tokens of stride 0 (one q for all), heads of stride 0 (one k for all heads), batches of stride 0, and tokens 2^25 elements apart, all read in place; the gradients of what
    is shared are summed."""
    from satflow_amd import functional_seq as S

    B, H, dk, dv = 2, 3, 32, 40
    x = _inputs(device, B, T, H, dk, dv, dtype, 5)
    shared = [x[0][:, :1].clone(), x[1][:, :, :1].clone(), x[2][:1].clone()]
    leaves = [t.requires_grad_() for t in shared]
    q, k, v = (t.expand_as(f) for t, f in zip(leaves, x[:3]))
    o = S.linear_attention(q, k, v, x[3], initial_state=x[4])
    grads = torch.autograd.grad(o, leaves, x[5])
    want = _recurrence(q, k, v, *x[3:5], torch.full((B,), T, device=device), x[5], torch.zeros_like(x[6]))
    assert _rel(o.detach(), want[0]) <= TOL[dtype]
    for name, a, full, axis in zip(("dq", "dk", "dv"), grads, want[2:5], (1, 2, 0)):   # (every summand is rounded once, torch sums them in float32 and rounds again)
        assert _rel(a, full.sum(axis, keepdim=True)) <= 3 * TOL[dtype], (name, _rel(a, full.sum(axis, keepdim=True)))
    far = torch.zeros(min(T, 24), 2**25 + 8, dtype=dtype, device=device)
    n = far.shape[0]
    far[:, :dk] = x[0][0, :n, 0]
    one = S.linear_attention(far[None, :, None, :dk], x[1][:1, :n, :1], x[2][:1, :n, :1], x[3][:1])
    want = S.linear_attention(x[0][:1, :n, :1], x[1][:1, :n, :1], x[2][:1, :n, :1], x[3][:1])
    assert _rel(one, want) <= 2 * TOL[dtype]
