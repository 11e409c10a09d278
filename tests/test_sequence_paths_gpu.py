"""Linear attention (satflow_amd.functional_seq) on the paths that a call's sizes, types and alignment choose, at the ends of their ranges."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-19}


def _rel(a, b):
    b = b.double()
    n = float(b.norm())
    return float((a.double() - b).norm()) / n if n else float(a.double().norm())


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
