"""Linear attention with a decay for each head (satflow_amd.functional_seq): the prompt form, its gradients and the single-token form against the recurrence
evaluated token by token in float64.

Tolerances, fixed before the first run.  Errors are 2-norms relative to the result's: a bf16 output is rounded once, at most half a step of 2^-8 of the value
(2^-9 and less in the mean square), and what the kernel adds in front of that rounding is held below it: 2^-8 in all.  fp32 outputs and all states: products of
operands kept to 24 bits, summed in fp32 over up to some hundreds of effective terms of both signs: 2^-24 per rounding, sqrt(#terms) of them: 2^-19."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-19}


def _rel(a, b):
    b = b.double()
    n = float(b.norm())
    return float((a.double() - b).norm()) / n if n else float(a.double().norm())


def _recurrence(q, k, v, g, s0, lengths, scale, do=None, ds=None):
    """o, last state and - with do - the gradients, in float64 on the tensors' device."""
    q, k, v = q.double(), k.double(), v.double()
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    lam = torch.exp(g.double())[None, :, None, None]
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64, device=q.device) if s0 is None else s0.double()
    n = torch.full((B,), T, device=q.device) if lengths is None else lengths.clamp(0, T)
    o, dq, dk_, dv_ = torch.zeros_like(v), torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(v)
    for t in range(T):
        live = (t < n)[:, None, None, None]
        S = torch.where(live, lam * S + k[:, t, :, :, None] * v[:, t, :, None, :], S)
        o[:, t] = torch.where(live[..., 0], (q[:, t, :, :, None] * S).sum(2) * scale, o[:, t])
        if do is not None:
            dq[:, t] = torch.where(live[..., 0], (S * do[:, t, :, None, :].double()).sum(-1) * scale, dq[:, t])
    if do is None:
        return o, S
    R = torch.zeros_like(S) if ds is None else ds.double()
    for t in reversed(range(T)):
        live = (t < n)[:, None, None, None]
        at = R + scale * q[:, t, :, :, None] * do[:, t, :, None, :].double()
        dk_[:, t] = torch.where(live[..., 0], (at * v[:, t, :, None, :]).sum(-1), dk_[:, t])
        dv_[:, t] = torch.where(live[..., 0], (at * k[:, t, :, :, None]).sum(2), dv_[:, t])
        R = torch.where(live, lam * at, R)
    return o, S, dq, dk_, dv_, R


def _inputs(device, B, T, H, dk, dv, dtype, seed, state=True, layout="dense"):
    gen = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen).to(device)

    if layout == "packed":      # q | k | v of one projection
        x = rand(B, T, H, 2 * dk + dv).to(dtype)
        q, k, v = x[..., :dk], x[..., dk:2 * dk], x[..., 2 * dk:]
    elif layout == "time":      # time-major frames, heads outermost in memory
        q, k, v = (rand(H, T, B, d).to(dtype).permute(2, 1, 0, 3) for d in (dk, dk, dv))
    else:
        q, k, v = (rand(B, T, H, d).to(dtype) for d in (dk, dk, dv))
    g = -torch.rand(H, generator=gen).to(device) * torch.tensor([0.003, 0.05, 0.7], device=device).repeat(H)[:H]
    g[-1] = 0.0 if H > 1 else g[-1]
    return q, k, v, g, rand(B, H, dk, dv) if state else None, rand(B, T, H, dv).to(dtype), rand(B, H, dk, dv)


SHAPES = [  # B, T, H, dk, dv
    (1, 1, 1, 16, 16), (2, 2, 3, 32, 32), (3, 24, 4, 32, 32), (2, 32, 3, 100, 72), (5, 31, 3, 128, 40), (2, 7, 2, 6, 128), (2, 63, 2, 64, 64), (1, 64, 2, 64, 128), (2, 65, 2, 128, 64), (1, 127, 3, 40, 72),
    (2, 129, 1, 128, 128), (1, 257, 2, 1, 1), (1, 200, 2, 17, 33), (1, 1000, 2, 100, 96), (3, 33, 5, 5, 128), (1, 3001, 2, 64, 64),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,T,H,dk,dv", SHAPES)
def test_outputs_states_and_gradients(device, B, T, H, dk, dv, dtype):
    from satflow_amd import functional_seq as S

    q, k, v, g, s0, do, ds = _inputs(device, B, T, H, dk, dv, dtype, 7 * T + dk)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    o, last = S.linear_attention(*leaves[:3], g, initial_state=leaves[3], return_state=True)
    grads = torch.autograd.grad([o, last], leaves, [do, ds])
    want = _recurrence(q, k, v, g, s0, None, dk ** -0.5, do, ds)
    for name, a, b in zip(("o", "state", "dq", "dk", "dv", "dstate"), (o, last, *grads), want):
        assert a.dtype == (torch.float32 if "state" in name else dtype)
        assert _rel(a, b) <= TOL[a.dtype], (name, _rel(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["packed", "time"])
@pytest.mark.parametrize("dk,dv", [(32, 64), (20, 12), (7, 9)])
def test_strided_inputs_without_state(device, dtype, layout, dk, dv):
    from satflow_amd import functional_seq as S

    q, k, v, g, _, do, _ = _inputs(device, 2, 150, 3, dk, dv, dtype, 5, layout=layout)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = S.linear_attention(*leaves, g, scale=0.3)
    grads = torch.autograd.grad(o, leaves, do.transpose(0, 1).contiguous().transpose(0, 1))
    want = _recurrence(q, k, v, g, None, None, 0.3, do)
    for name, a, b in zip(("o", "dq", "dk", "dv"), (o, *grads), (want[0], *want[2:5])):
        assert _rel(a, b) <= TOL[dtype], (name, _rel(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,lengths", [(20, [0, 1, 20, 19, 7]), (40, [0, 1, 40, 39, 17]), (300, [300, 0, 1, 128, 255]), (70, [64, 65, 63, 99, -3]), (2500, [2500, 1, 1999, 0, 1024])])
def test_lengths(device, dtype, T, lengths):
    """Tokens behind a sequence's length may hold anything: they are not read, their outputs and gradients are zero, the state passes by them."""
    from satflow_amd import functional_seq as S

    B, H, dk, dv = len(lengths), 2, 32, 48
    q, k, v, g, s0, do, ds = _inputs(device, B, T, H, dk, dv, dtype, T)
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    want = _recurrence(q, k, v, g, s0, n, dk ** -0.5, do, ds)
    behind = (torch.arange(T, device=device) >= n.clamp(0, T)[:, None])
    for bad in (float("nan"), float("inf")):
        dirty = [t.masked_fill(behind[:, :, None, None], bad) for t in (q, k, v, do)]
        leaves = [t.requires_grad_() for t in (*dirty[:3], s0.clone())]
        o, last = S.linear_attention(*leaves[:3], g, initial_state=leaves[3], lengths=n, return_state=True)
        grads = torch.autograd.grad([o, last], leaves, [dirty[3], ds])
        for name, a, b in zip(("o", "state", "dq", "dk", "dv", "dstate"), (o, last, *grads), want):
            assert torch.isfinite(a).all(), name
            assert _rel(a, b) <= TOL[a.dtype], (name, _rel(a, b))
            if "state" not in name:
                assert not a[behind].any(), name
    empty = n.clamp(0, T) == 0
    assert torch.equal(last[empty], s0[empty]) and torch.equal(grads[3][empty], ds[empty])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T", [30, 50, 130, 700])
def test_non_finite_values_do_not_reach_earlier_tokens(device, dtype, T):
    """Causality holds for values that are not finite too: what comes before such a token is what it is without it (bit for bit), forward and - with a
    non-finite gradient - backward (where a token's gradient depends on later tokens only: what comes AFTER the bad one stays)."""
    from satflow_amd import functional_seq as S

    q, k, v, g, s0, do, ds = _inputs(device, 1, T, 2, 32, 64, dtype, 3)
    at = T // 2 + 5   # (30: inside the one chunk)
    clean = S.linear_attention(q, k, v, g, initial_state=s0)
    for bad in (float("nan"), float("inf"), float("-inf")):
        for which in range(3):
            x = [t.clone() for t in (q, k, v)]
            x[which][:, at, 1, 3] = bad
            got = S.linear_attention(*x, g, initial_state=s0)
            assert torch.equal(got[:, :at], clean[:, :at]), (bad, which)
            assert torch.equal(got[:, :, 0], clean[:, :, 0]), "the other head"
            if which == 0:
                assert torch.equal(got[:, at + 1:], clean[:, at + 1:])
            if which == 2:   # one value column only, and there every later token
                cols = torch.arange(64, device=device) != 3
                assert torch.equal(got[..., cols], clean[..., cols])
                assert not torch.isfinite(got[:, at:, 1, 3]).any()
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = S.linear_attention(*leaves, g, initial_state=s0)
    base = torch.autograd.grad(o, leaves, do, retain_graph=True)
    bad_do = do.clone()
    bad_do[:, at, 1, 3] = float("nan")
    got = torch.autograd.grad(o, leaves, bad_do)
    for name, a, b in zip(("dq", "dk", "dv"), got, base):
        assert torch.equal(a[:, at + 1:], b[:, at + 1:]), name
        assert torch.equal(a[:, :, 0], b[:, :, 0]), name
    assert torch.equal(got[0][:, :at], base[0][:, :at])


@pytest.mark.parametrize("decay", [0.0, -1e-4, -3.0, -60.0, float("-inf")])
def test_extreme_decays(device, decay):
    from satflow_amd import functional_seq as S

    q, k, v, _, s0, do, ds = _inputs(device, 2, 500, 1, 32, 32, torch.float32, 9)
    g = torch.full((1,), decay, device=device)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    o, last = S.linear_attention(*leaves[:3], g, initial_state=leaves[3], return_state=True)
    grads = torch.autograd.grad([o, last], leaves, [do, ds])
    want = _recurrence(q, k, v, g, s0, None, 32 ** -0.5, do, ds)
    for name, a, b in zip(("o", "state", "dq", "dk", "dv", "dstate"), (o, last, *grads), want):
        assert _rel(a, b) <= TOL[torch.float32], (name, _rel(a, b))


def test_slow_decay_over_a_long_sequence(device):
    """A horizon of 5000 tokens over 40000: the powers of the decay keep their fp32 accuracy over the whole distance."""
    from satflow_amd import functional_seq as S

    q, k, v, _, _, _, _ = _inputs(device, 1, 40000, 1, 8, 8, torch.float32, 2)
    k, v = k.abs(), v.abs()   # sums of one sign: an error of the powers does not average out
    g = torch.full((1,), -1.0 / 5000, device=device)
    o, last = S.linear_attention(q.abs(), k, v, g, return_state=True)
    far = torch.arange(39999, -1, -1, device=device, dtype=torch.float64)
    want = torch.einsum("td,te->de", k[0, :, 0].double() * torch.exp(g.double() * far[:, None]), v[0, :, 0].double())
    assert _rel(last[0, 0], want) <= TOL[torch.float32], _rel(last[0, 0], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (1, 8, 64, 64), (3, 2, 128, 128), (2, 3, 40, 72), (5, 1, 33, 17), (70, 16, 16, 128), (2, 2, 128, 6)])
def test_single_token_form(device, dtype, B, H, dk, dv):
    from satflow_amd import functional_seq as S

    q, k, v, g, s0, _, _ = _inputs(device, B, 1, H, dk, dv, dtype, dk)
    want, last = _recurrence(q, k, v, g, s0, None, dk ** -0.5)
    o, new = S.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s0)
    assert o.dtype == dtype and new.dtype == torch.float32
    assert _rel(o, want[:, 0]) <= TOL[dtype] and _rel(new, last) <= 2.0**-23
    state = s0.clone()
    o2, same = S.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state, out_state=state)
    assert same is state and torch.equal(state, new) and torch.equal(o2, o)
    # strides: the state of every other sequence of a pool, packed tokens
    x = torch.cat([q, k, v], -1)[:, 0]
    pool = torch.zeros(2 * B, H, dk, dv, device=device)
    pool[::2] = s0
    o3, new3 = S.linear_attention_step(x[..., :dk], x[..., dk:2 * dk], x[..., 2 * dk:], g, pool[::2])
    assert torch.equal(o3, o) and torch.equal(new3, new)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_prompt_then_steps_equals_one_pass(device, dtype):
    """The forms together, as a program that streams frames uses them: a prompt, a continuation of two chunks, then token by token."""
    from satflow_amd import functional_seq as S

    q, k, v, g, _, _, _ = _inputs(device, 2, 180, 3, 48, 64, dtype, 21)
    whole, last = S.linear_attention(q, k, v, g, return_state=True)
    parts, state = [], None
    for lo, hi in ((0, 100), (100, 101), (101, 160)):
        o, state = S.linear_attention(q[:, lo:hi], k[:, lo:hi], v[:, lo:hi], g, initial_state=state, return_state=True)
        parts.append(o)
    for t in range(160, 180):
        o, state = S.linear_attention_step(q[:, t], k[:, t], v[:, t], g, state, out_state=state)
        parts.append(o[:, None])
    assert _rel(torch.cat(parts, 1), whole) <= 2 * TOL[dtype]
    assert _rel(state, last) <= 2 * TOL[torch.float32]


def test_gradients_against_differences(device):
    """Directional central differences of a float64-accumulated loss in fp32 inputs: the truncation error vanishes (the loss is linear in q, k and v each),
    what is left is the fp32 rounding of the outputs, 2^-24 / step = 2^-14 of them, averaged over 2000 outputs."""
    from satflow_amd import functional_seq as S

    q, k, v, g, s0, do, ds = _inputs(device, 2, 90, 2, 16, 24, torch.float32, 4)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    o, last = S.linear_attention(*leaves[:3], g, initial_state=leaves[3], return_state=True)
    grads = torch.autograd.grad([o, last], leaves, [do, ds])

    def loss(*x):
        o, last = S.linear_attention(*x[:3], g, initial_state=x[3], return_state=True)
        return float((o.double() * do.double()).sum() + (last.double() * ds.double()).sum())

    gen = torch.Generator().manual_seed(8)
    for i, name in enumerate(("q", "k", "v", "state")):
        d = torch.randn(leaves[i].shape, generator=gen).to(device)
        x = [t.detach() for t in leaves]
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + 2.0**-10 * d, x[i] - 2.0**-10 * d
        num = (loss(*up) - loss(*down)) / 2.0**-9
        got = float((grads[i].double() * d.double()).sum())
        assert abs(num - got) <= 2e-3 * float(grads[i].double().norm()), (name, num, got)


def test_no_rows_and_partial_gradients(device):
    from satflow_amd import functional_seq as S

    q, k, v, g, s0, do, ds = _inputs(device, 2, 10, 2, 16, 16, torch.float32, 4)
    o, last = S.linear_attention(q[:, :0], k[:, :0], v[:, :0], g, initial_state=s0, return_state=True)
    assert o.shape == (2, 0, 2, 16) and torch.equal(last, s0)
    o, last = S.linear_attention(q[:0], k[:0], v[:0], g, return_state=True)
    assert o.shape == (0, 10, 2, 16) and last.shape == (0, 2, 16, 16)
    x = [t.clone().requires_grad_() for t in (q[:, :0], k[:, :0], v[:, :0], s0)]
    _, last = S.linear_attention(*x[:3], g, initial_state=x[3], return_state=True)
    assert torch.equal(torch.autograd.grad(last, x[3], ds)[0], ds)
    # only the state, only the output, only one of the inputs
    x = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    want = _recurrence(q, k, v, g, s0, None, 0.25, torch.zeros_like(do), ds)
    _, last = S.linear_attention(*x[:3], g, initial_state=x[3], return_state=True)
    got = torch.autograd.grad(last, x[1:], ds)
    for a, b in zip(got, want[3:]):
        assert _rel(a, b) <= TOL[torch.float32]
    kk = k.clone().requires_grad_()
    (dk,) = torch.autograd.grad(S.linear_attention(q, kk, v, g, initial_state=s0), kk, do[:1, :1].expand_as(do))
    assert _rel(dk, _recurrence(q, k, v, g, s0, None, 0.25, do[:1, :1].expand_as(do))[3]) <= TOL[torch.float32]


def test_streams_and_repeated_graph(device):
    """A call on another stream than the tensors' own, two calls at once on two streams, and a captured training pass, replayed on new inputs with eager work
    between the replays: every result is the eager one, bit for bit."""
    from satflow_amd import functional_seq as S

    q, k, v, g, s0, do, ds = _inputs(device, 2, 600, 2, 64, 64, torch.bfloat16, 4)

    def step(q, k, v, s0):
        x = [t.detach().requires_grad_() for t in (q, k, v, s0)]
        o, last = S.linear_attention(*x[:3], g, initial_state=x[3], return_state=True)
        return (o.detach(), last.detach(), *torch.autograd.grad([o, last], x, [do, ds]))

    sets = [(q, k, v, s0), tuple(t * 0.5 for t in (q, k, v, s0)), tuple(t.flip(0) for t in (q, k, v, s0))]
    eager = [step(*x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, x in zip(streams, sets):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(*x))
    torch.cuda.synchronize()
    for a, b in zip(got, eager):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    held = [t.clone() for t in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for i in (1, 2, 0, 1):
        for h, t in zip(held, sets[i]):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, eager[i]))
        assert all(torch.equal(x, y) for x, y in zip(step(*sets[2]), eager[2]))


def test_result_does_not_depend_on_the_batch(device):
    """The same sequence alone and among others gives the same bits (the split of the work goes by sizes, never by values or neighbours)... for calls of the
    same number of tokens whose split is the same; across splits it is equal within the tolerance."""
    from satflow_amd import functional_seq as S

    q, k, v, g, s0, _, _ = _inputs(device, 4, 2000, 4, 64, 64, torch.bfloat16, 4)
    a, sa = S.linear_attention(q, k, v, g, initial_state=s0, return_state=True)
    b, sb = S.linear_attention(q, k, v, g, initial_state=s0, return_state=True)
    assert torch.equal(a, b) and torch.equal(sa, sb)
    c, sc = S.linear_attention(q[2:3], k[2:3], v[2:3], g, initial_state=s0[2:3], return_state=True)
    assert _rel(c, a[2:3]) <= TOL[torch.bfloat16] and _rel(sc, sa[2:3]) <= TOL[torch.float32]


def test_second_derivatives_are_refused(device):
    from satflow_amd import functional_seq as S

    q, k, v, g, _ = _inputs(device, 2, 40, 2, 8, 8, torch.float32, 5)[:5]
    q = q.detach().clone().requires_grad_()
    o = S.linear_attention(q, k, v, g)
    (dq,) = torch.autograd.grad(o.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dq.sum().backward()


def test_a_graph_notices_its_state_updated_in_place(device):
    from satflow_amd import functional_seq as S

    q, k, v, g, s0 = _inputs(device, 2, 40, 2, 8, 8, torch.float32, 6)[:5]
    q = q.detach().clone().requires_grad_()
    o = S.linear_attention(q, k, v, g, initial_state=s0)
    with torch.no_grad():
        S.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s0, out_state=s0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    with torch.inference_mode():
        s = torch.zeros_like(s0)
        S.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s, out_state=s)
    with pytest.raises(RuntimeError, match="cannot require a gradient"), torch.no_grad():
        S.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s0.clone(), out_state=s0.clone().requires_grad_())


def test_offsets_past_32_bits(device):
    """More than 2^32 elements: the last tokens against the same call on the sequence's tail alone, in front of which nothing is left of the state
    (exp(-0.05 * 3000) is below 2^-200).  Both are within 2^-8 of the exact result, so within 2^-7 of each other."""
    from satflow_amd import functional_seq as S

    T, H, d, tail, last = 4_300_000, 8, 128, 4096, 1000
    if torch.cuda.mem_get_info()[1] < 150 * 2**30:
        pytest.skip("takes 80 GB of device memory")
    gen = torch.Generator(device=device).manual_seed(3)
    block = torch.randn(1, 100_000, H, d, generator=gen, device=device, dtype=torch.bfloat16)
    x = block.repeat(1, T // 100_000, 1, 1)
    assert x.numel() > 2**32
    x[:, -tail:] = torch.randn(1, tail, H, d, generator=gen, device=device, dtype=torch.bfloat16)
    g = torch.full((H,), -0.05, device=device)

    def run(t):
        q, k, v = (t.detach().view_as(t).requires_grad_() for _ in range(3))
        o = S.linear_attention(q, k, v, g)
        grads = torch.autograd.grad(o, (q, k, v), t)
        return [y[:, -last:].detach().clone() for y in (o, *grads)]

    whole = run(x)
    for a, b in zip(whole, run(x[:, -tail:].contiguous())):
        assert _rel(a, b) < 2 * TOL[torch.bfloat16]
