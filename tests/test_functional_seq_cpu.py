"""CPU: what satflow_amd.functional_seq and the library entries behind it refuse, before anything is launched."""
import pytest
import torch

from satflow_amd import functional_seq as S


def _attn(**change):
    a = dict(q=torch.zeros(2, 5, 3, 8), k=torch.zeros(2, 5, 3, 8), v=torch.zeros(2, 5, 3, 4), log_decay=torch.zeros(3), initial_state=None, lengths=None)
    a.update(change)
    return S.linear_attention(a["q"], a["k"], a["v"], a["log_decay"], initial_state=a["initial_state"], lengths=a["lengths"])


@pytest.mark.parametrize("change,match", [
    (dict(), "HIP device"),
    (dict(k=torch.zeros(2, 5, 3, 9)), "same leading sizes"),
    (dict(v=torch.zeros(2, 6, 3, 4)), "same leading sizes"),
    (dict(q=torch.zeros(2, 5, 8)), "same leading sizes"),
    (dict(v=torch.zeros(2, 5, 3, 4, dtype=torch.bfloat16)), "one type"),
    (dict(q=torch.zeros(2, 5, 3, 8).half(), k=torch.zeros(2, 5, 3, 8).half(), v=torch.zeros(2, 5, 3, 4).half()), "one type"),
    (dict(q=torch.zeros(2, 5, 3, 129), k=torch.zeros(2, 5, 3, 129)), "1 to 128"),
    (dict(v=torch.zeros(2, 5, 3, 0)), "1 to 128"),
    (dict(log_decay=torch.zeros(4)), "3 values"),
    (dict(log_decay=torch.zeros(3, dtype=torch.float64)), "float32"),
    (dict(log_decay=torch.zeros(3, requires_grad=True)), "no gradient"),
    (dict(initial_state=torch.zeros(2, 3, 4, 8)), "initial_state"),
    (dict(initial_state=torch.zeros(2, 3, 8, 4, dtype=torch.bfloat16)), "initial_state"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(2, dtype=torch.int64)), "lengths"),
])
def test_linear_attention_refuses(change, match):
    with pytest.raises(RuntimeError, match=match):
        _attn(**change)


def test_linear_attention_step_refuses():
    q, k, v, g, s = torch.zeros(2, 3, 8), torch.zeros(2, 3, 8), torch.zeros(2, 3, 4), torch.zeros(3), torch.zeros(2, 3, 8, 4)
    for args, more, match in [
        ((q, k, v, g, s), {}, "HIP device"),
        ((q, k, v, g, s[:1]), {}, "`state`"),
        ((q, k, v, g, s.double()), {}, "`state`"),
        ((q[:, :, None], k, v, g, s), {}, "same leading sizes"),
        ((q, k, v, g, s), dict(out_state=torch.zeros(2, 3, 4, 8).transpose(2, 3)), "contiguous"),
        ((q.clone().requires_grad_(), k, v, g, s), {}, "no gradient"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            S.linear_attention_step(*args, **more)
    pool = torch.zeros(2 * 2 * 3 * 8 * 4)   # an output that overlaps the input without being it
    with pytest.raises(RuntimeError, match="memory of its own"):
        S.linear_attention_step(q, k, v, g, pool[:192].view(2, 3, 8, 4), out_state=pool[32:224].view(2, 3, 8, 4))


@pytest.mark.parametrize("change,match", [
    (dict(), "HIP device"),
    (dict(weight=torch.ones(7)), "`weight`"),
    (dict(weight=torch.ones(8, dtype=torch.bfloat16)), "`weight`"),
    (dict(scale=torch.ones(1)), "`scale`"),
    (dict(gate=torch.zeros(3, 1)), "`gate`"),
    (dict(gate=torch.zeros(3, 8).bfloat16()), "one type"),
    (dict(u=torch.zeros(3, 8).double()), "one type"),
    (dict(residual=torch.zeros(3, 8).bfloat16()), "residual"),
    (dict(residual=torch.zeros(8)), "`residual`"),
    (dict(groups=3), "equal groups"),
    (dict(groups=0), "equal groups"),
    (dict(groups=2, next_weight=torch.ones(8)), "groups=1"),
    (dict(next_bias=torch.ones(8)), "next_weight"),
    (dict(kind="batch"), "'rms' or 'layer'"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(u=torch.zeros(1, 16385), weight=None), "16384"),
    (dict(u=torch.zeros(3, 0), weight=None), "at least one channel"),
])
def test_post_norm_refuses(change, match):
    a = dict(u=torch.zeros(3, 8), weight=torch.ones(8))
    a.update(change)
    with pytest.raises(RuntimeError, match=match):
        S.post_norm(a.pop("u"), a.pop("weight"), **a)


def test_retention_layers_refuse():
    from satflow_amd.models.layers import Retention, RetentionLayer
    for kw, match in [(dict(dim=24), "multiples of 16"), (dict(dim=32, heads=3), "multiples of 16"), (dict(dim=32, heads=0), "0 heads"),
                      (dict(dim=32, heads=2, value_dim=20), "multiples of 16"), (dict(dim=32, heads=2, key_dim=129), "1 to 128"),
                      (dict(dim=512, heads=2), "1 to 128")]:
        with pytest.raises(ValueError, match=match):
            RetentionLayer(**kw)
    with pytest.raises(ValueError, match="0 layers"):
        Retention(32, 0)
    m = Retention(32, 2, heads=2)
    for x, match in [(torch.zeros(2, 3, 31), "got"), (torch.zeros(3, 32), "got"), (torch.zeros(2, 3, 32).bfloat16(), "got"), (torch.zeros(2, 3, 16, 4, 4), "got"),
                     (torch.zeros(2, 3, 32), "HIP device")]:
        with pytest.raises(RuntimeError, match=match):
            m(x)
    with pytest.raises(RuntimeError, match="1 states for 2"):
        m(torch.zeros(2, 3, 32), m.initial_state(2)[:1])
    with pytest.raises(RuntimeError, match="1 states for 2"):
        m.step(torch.zeros(2, 32), m.initial_state(2)[:1])
    assert sorted(n for n in m.state_dict() if n.startswith("layers.1.")) == [
        "layers.1.log_decay", "layers.1.norm_heads", "layers.1.norm_in", "layers.1.norm_out", "layers.1.scale", "layers.1.to_out.weight", "layers.1.to_qkvg.weight"]
    assert [tuple(s.shape) for s in m.initial_state(7)] == [(7, 2, 16, 16)] * 2


class _Stub:
    """The launches, replaced by zeros of the right shapes: what the public functions do with their arguments, without a device."""

    @staticmethod
    def install(monkeypatch):
        monkeypatch.setattr(S, "_same_device", lambda *a: None)
        monkeypatch.setattr(S, "_on", lambda t: S._HERE)
        monkeypatch.setattr(S.K, "linear_attention_fwd", lambda q, k, v, *a: (torch.zeros_like(v), torch.zeros(2, 3, 8, 4), None))
        monkeypatch.setattr(S.K, "linear_attention_step", lambda q, k, v, *a: torch.zeros_like(v))
        monkeypatch.setattr(S.K, "block_norm_fwd", lambda u, w, b, gate, scale, residual, next_w, *a: (torch.zeros_like(u), torch.zeros_like(u) if next_w is not None else None, None))


ATTENTION = dict(q=(2, 5, 3, 8), k=(2, 5, 3, 8), v=(2, 5, 3, 4), log_decay=(3,), initial_state=(2, 3, 8, 4))
STEP = dict(q=(2, 3, 8), k=(2, 3, 8), v=(2, 3, 4), log_decay=(3,), state=(2, 3, 8, 4), out_state=(2, 3, 8, 4))
NORM = dict(u=(3, 8), weight=(8,), bias=(8,), gate=(3, 8), scale=(8,), residual=(3, 8), next_weight=(8,), next_bias=(8,))


@pytest.mark.parametrize("call,shapes,dual", [(f, shapes, n) for f, shapes in (("linear_attention", ATTENTION), ("linear_attention_step", STEP), ("post_norm", NORM))
                                              for n in shapes] + [("pre_norm", dict(x=(3, 8), weight=(8,), bias=(8,)), n) for n in ("x", "weight", "bias")])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(monkeypatch, call, shapes, dual, grad):
    """A tangent is never dropped: a dual tensor in any place is an error, with and without grad mode; one that left its level is an ordinary tensor."""
    from torch.autograd import forward_ad

    _Stub.install(monkeypatch)
    args = {n: torch.zeros(shape) for n, shape in shapes.items()}
    with torch.set_grad_enabled(grad):
        getattr(S, call)(**args)
        with forward_ad.dual_level():
            getattr(S, call)(**args)
            args[dual] = forward_ad.make_dual(args[dual], torch.ones(shapes[dual]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                getattr(S, call)(**args)
        getattr(S, call)(**args)
