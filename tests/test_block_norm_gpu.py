"""Norms before and after a block fused with gate, residual scale and residual sum (satflow_amd.functional_seq.pre_norm / post_norm) against float64.

Tolerances, fixed before the first run, as 2-norms relative to the result's: a bf16 output is rounded once (at most 2^-9 of the value, half a step of 2^-8), the
fp32 arithmetic in front of it adds less than a tenth of that: 2^-8.  fp32 outputs: about ten roundings of 2^-24 and sums over up to 16384 terms in trees of
depth 14: 2^-19; parameter gradients are sums over the rows of such terms, relative to their own size (terms of both signs: sqrt(rows) of it): 2^-18."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-19}
NAMES = ("u", "w", "b", "gate", "scale", "residual", "nw", "nb")


def _rel(a, b):
    b = b.double()
    n = float(b.norm())
    return float((a.double() - b).norm()) / n if n else float(a.double().norm())


def _norm(x, kind, groups, eps):
    x = x.unflatten(-1, (groups, -1))
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return (x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)).flatten(-2)


def _reference(t, kind, groups, eps):
    """r and y in float64 from the float64 leaves of ``t``."""
    z = _norm(t["u"], kind, groups, eps)
    z = z * t["w"] if t["w"] is not None else z
    z = z + t["b"] if t["b"] is not None else z
    z = z * t["gate"] * torch.sigmoid(t["gate"]) if t["gate"] is not None else z
    z = z * t["scale"] if t["scale"] is not None else z
    r = z + t["residual"] if t["residual"] is not None else z
    y = None
    if t["nw"] is not None:
        y = _norm(r, kind, 1, eps) * t["nw"]
        y = y + t["nb"] if t["nb"] is not None else y
    return r, y


def _make(device, rows, C, dtype, res, parts, seed):
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape, mul=1.0, add=0.0, dt=torch.float32):
        return (torch.randn(*shape, generator=gen) * mul + add).to(device).to(dt)

    t = dict.fromkeys(NAMES)
    t["u"] = rand(rows, C, mul=1.5, add=0.3, dt=dtype)
    for n, (mul, add) in dict(w=(0.3, 1.0), b=(0.2, 0.0), scale=(0.2, 0.6), nw=(0.3, 1.0), nb=(0.2, 0.0)).items():
        if n in parts:
            t[n] = rand(C, mul=mul, add=add)
    if "gate" in parts:
        t["gate"] = rand(rows, C, mul=1.5, dt=dtype)
    if "residual" in parts:
        t["residual"] = rand(rows, C, mul=2.0, dt=res)
    return t, rand(rows, C, dt=res if "residual" in parts else dtype), rand(rows, C, dt=dtype)


def _call(t, kind, groups, eps):
    from satflow_amd import functional_seq as S

    out = S.post_norm(t["u"], t["w"], t["b"], gate=t["gate"], scale=t["scale"], residual=t["residual"], groups=groups, next_weight=t["nw"], next_bias=t["nb"],
                      kind=kind, eps=eps)
    return out if t["nw"] is not None else (out, None)


ALL = ("w", "b", "gate", "scale", "residual", "nw", "nb")
CASES = [  # rows, C, groups, parts
    (1, 1, 1, ("w", "b")), (3, 7, 1, ALL), (50, 16, 1, ALL), (129, 64, 1, ALL), (33, 100, 1, ("w", "residual", "nw")), (40, 256, 8, ("w", "gate")),
    (65, 96, 3, ("w", "b", "gate", "scale", "residual")), (20, 63, 7, ("w", "gate", "residual")), (5, 520, 1, ALL), (700, 512, 1, ALL), (9, 777, 1, ALL),
    (17, 2048, 1, ALL), (6, 4096, 1, ("w", "gate", "scale", "residual", "nw")), (3, 8192, 1, ALL), (4, 8200, 1, ALL), (2, 16384, 1, ALL), (3, 16383, 1, ("w", "nw")),
    (4000, 40, 1, ("w", "b")), (300, 256, 1, ()), (300, 256, 1, ("residual",)), (2, 32768, 2, ("w", "gate")),
]


@pytest.mark.parametrize("dtype,res", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)], ids=["f32", "bf16", "bf16_f32"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,C,groups,parts", CASES)
def test_outputs_and_gradients(device, rows, C, groups, parts, kind, dtype, res):
    t, dr, dy = _make(device, rows, C, dtype, res, parts, rows + C)
    eps = 1e-5
    ours = {n: x.clone().requires_grad_() if x is not None else None for n, x in t.items()}
    ref = {n: x.double().requires_grad_() if x is not None else None for n, x in t.items()}
    r, y = _call(ours, kind, groups, eps)
    rr, ry = _reference(ref, kind, groups, eps)
    assert r.dtype == (res if "residual" in parts else dtype) and _rel(r, rr.detach()) <= TOL[r.dtype], _rel(r, rr.detach())
    # a one-channel layer norm is the bias alone: its input gradient is zero up to the rounding of (u - mean)
    outs, seeds, routs = [r], [dr], [rr]
    if y is not None:
        assert y.dtype == dtype and _rel(y, ry.detach()) <= TOL[dtype], _rel(y, ry.detach())
        outs, seeds, routs = [r, y], [dr, dy], [rr, ry]
    leaves = [n for n in NAMES if ours[n] is not None]
    got = torch.autograd.grad(outs, [ours[n] for n in leaves], seeds)
    want = torch.autograd.grad(routs, [ref[n] for n in leaves], [s.double() for s in seeds])
    for n, a, b in zip(leaves, got, want):
        assert a.dtype == t[n].dtype and a.shape == t[n].shape
        if C == 1 and n in ("u", "w"):
            continue
        tol = TOL[a.dtype] if n in ("u", "gate", "residual") else 2.0**-18
        assert _rel(a, b) <= tol, (n, _rel(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_and_leading_axes(device, dtype):
    """Row slices of wider tensors (not aligned to 16 bytes), a broadcast gate, three leading axes, a transposed gradient."""
    from satflow_amd import functional_seq as S

    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(4, 6, 5, 131, generator=gen).to(device).to(dtype)
    u, x = wide[..., 3:67], wide[..., 66:130]
    gate = wide[:1, :1, :1, 2:66].expand(4, 6, 5, 64)
    w = torch.randn(64, generator=gen).to(device)
    cot = torch.randn(64, 4, 6, 5, generator=gen).to(device).to(dtype).permute(1, 2, 3, 0)
    leaves = [t.detach().requires_grad_() for t in (u, gate, x)]
    r, y = S.post_norm(leaves[0], w, gate=leaves[1], residual=leaves[2], next_weight=w)
    got = torch.autograd.grad([r, y], leaves, [cot, cot])
    ref = [t.detach().double().requires_grad_() for t in (u, gate, x)]
    t = dict(dict.fromkeys(NAMES), u=ref[0], w=w.double(), gate=ref[1], residual=ref[2], nw=w.double())
    rr, ry = _reference(t, "rms", 1, 1e-6)
    want = torch.autograd.grad([rr, ry], ref, [cot.double(), cot.double()])
    for a, b in zip((r, y, *got), (rr, ry, *want)):
        assert a.shape == b.shape and _rel(a.detach(), b.detach()) <= TOL[dtype]


def test_one_output_and_some_leaves(device):
    """Only y, only r, only a parameter: what is not asked for is not needed."""
    t, dr, dy = _make(device, 37, 96, torch.float32, torch.float32, ALL, 5)
    ref = {n: x.double().requires_grad_() for n, x in t.items()}
    rr, ry = _reference(ref, "layer", 1, 1e-6)
    for outs in ("r", "y"):
        for leaf in NAMES:
            ours = {n: x.clone().requires_grad_(n == leaf) for n, x in t.items()}
            r, y = _call(ours, "layer", 1, 1e-6)
            o, ro, s = (r, rr, dr) if outs == "r" else (y, ry, dy)
            if outs == "r" and leaf in ("nw", "nb"):
                continue
            (a,) = torch.autograd.grad(o, ours[leaf], s)
            (b,) = torch.autograd.grad(ro, ref[leaf], s.double(), retain_graph=True)
            assert _rel(a, b) <= 2.0**-18, (outs, leaf, _rel(a, b))


def test_rows_are_independent_and_empty_input(device):
    from satflow_amd import functional_seq as S

    t, _, _ = _make(device, 60, 200, torch.bfloat16, torch.bfloat16, ALL, 6)
    r, y = _call(t, "layer", 1, 1e-6)
    bad = dict(t, u=t["u"].clone(), gate=t["gate"].clone(), residual=t["residual"].clone())
    bad["u"][7], bad["gate"][8], bad["residual"][9] = float("nan"), float("inf"), float("-inf")
    r2, y2 = _call(bad, "layer", 1, 1e-6)
    keep = torch.tensor([i not in (7, 8, 9) for i in range(60)], device=device)
    assert torch.equal(r2[keep], r[keep]) and torch.equal(y2[keep], y[keep])
    assert r2[7].isnan().all() and y2[9].isnan().all()
    assert torch.equal(S.pre_norm(torch.zeros(3, 64, device=device), None), torch.zeros(3, 64, device=device))
    u = torch.zeros(0, 64, device=device, requires_grad=True)
    w = torch.ones(64, device=device, requires_grad=True)
    o = S.pre_norm(u, w)
    gu, gw = torch.autograd.grad(o.sum(), [u, w])
    assert o.shape == gu.shape == (0, 64) and not gw.any()


def test_gradients_against_differences(device):
    """Central differences, step 2^-10 along random directions: truncation of the order of step^2 = 10^-6 of the third derivative, rounding of the fp32
    outputs over the step 2^-14 of them, averaged over 3500 outputs: 2e-3 of the gradient's norm holds both."""
    t, dr, dy = _make(device, 37, 96, torch.float32, torch.float32, ALL, 11)
    ours = {n: x.clone().requires_grad_() for n, x in t.items()}
    got = torch.autograd.grad(_call(ours, "layer", 1, 1e-6), [ours[n] for n in NAMES], [dr, dy])

    def loss(x):
        r, y = _call(x, "layer", 1, 1e-6)
        return float((r.double() * dr.double()).sum() + (y.double() * dy.double()).sum())

    gen = torch.Generator().manual_seed(3)
    for n, a in zip(NAMES, got):
        d = torch.randn(t[n].shape, generator=gen).to(device)
        h = 2.0**-10
        num = (loss(dict(t, **{n: t[n] + h * d})) - loss(dict(t, **{n: t[n] - h * d}))) / (2 * h)
        exact = float((a.double() * d.double()).sum())
        assert abs(num - exact) <= 2e-3 * float(a.double().norm()), (n, num, exact)


def test_repeats_streams_and_graph(device):
    t, dr, dy = _make(device, 3001, 320, torch.bfloat16, torch.float32, ALL, 12)

    def step(t):
        x = {n: v.detach().requires_grad_() for n, v in t.items()}
        r, y = _call(x, "rms", 1, 1e-6)
        return (r.detach(), y.detach(), *torch.autograd.grad([r, y], [x[n] for n in NAMES], [dr, dy]))

    sets = [t, {n: v * 0.5 for n, v in t.items()}, {n: v.flip(0) for n, v in t.items()}]
    eager = [step(x) for x in sets]
    for a, b in zip(step(sets[0]), eager[0]):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, x in zip(streams, sets):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(x))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for a, b in zip(got, eager) for x, y in zip(a, b))
    held = {n: v.clone() for n, v in t.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for i in (1, 2, 0, 1):
        for n in NAMES:
            held[n].copy_(sets[i][n])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, eager[i]))
        assert all(torch.equal(x, y) for x, y in zip(step(sets[2]), eager[2]))


def test_offsets_past_32_bits(device):
    """More than 2^32 elements: every row is worked on alone, so the last rows equal those of a call on them alone, bit for bit."""
    from satflow_amd import functional_seq as S

    rows, C, last = 1_050_000, 4096, 1000
    if torch.cuda.mem_get_info()[1] < 150 * 2**30:
        pytest.skip("takes 70 GB of device memory")
    gen = torch.Generator(device=device).manual_seed(4)
    u = torch.randn(10_500, C, generator=gen, device=device, dtype=torch.bfloat16).repeat(100, 1)
    assert u.numel() > 2**32
    u[-last:] = torch.randn(last, C, generator=gen, device=device, dtype=torch.bfloat16)
    w = torch.randn(C, generator=gen, device=device)

    def run(t):
        t = t.detach().view_as(t).requires_grad_()
        r, y = S.post_norm(t, w, gate=t.detach(), residual=t.detach(), next_weight=w)
        (du,) = torch.autograd.grad((r, y), t, (t.detach(), t.detach()))
        return [z[-last:].detach().clone() for z in (r, y, du)]

    for a, b in zip(run(u), run(u[-last:].contiguous())):
        assert torch.equal(a, b)
