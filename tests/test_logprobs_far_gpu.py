"""GPU tests of the log probabilities' gradient for rows of logits far from zero, whose lse has few digits left for the sum."""
import pytest
import torch

from serving_ref import EPS32, HALF
from test_serving_gpu import grad_ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def dt(cuda):
    import dirktensor_b200

    return dirktensor_b200


def bound(x, g, h, dtype):
    """Half a step of the type, and the fp32 error of each term.  x is relative to the row's largest logit and so exact: a
    probability is off by the steps of its exponent (x, its difference, the base change: 8 + 4 |x - lse|), of the sum that divides it
    (V / 256 for a thread's share, 40 for the joins) and of the entropy, which the forward pass forms the same way."""
    lse = torch.logsumexp(x, -1, keepdim=True)
    lp = x - lse
    p = torch.exp(lp)
    ent = -(p * lp).sum(-1, keepdim=True)
    steps = 2 * (4 * lp.abs() + 8 + x.shape[-1] / 256 + 40)
    return EPS32 * steps * p * (g.abs()[:, None] + h.abs()[:, None] * (lp.abs() + ent + 1)) + 4 * EPS32 * g.abs()[:, None] * (p + 1e-30)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N, V", [(3, 2), (5, 57), (4, 1003), (3, 20011), (2, 100352)])
@pytest.mark.parametrize("at", [5e3, -7e4, 1e6, -3e9, 1e30, "lowest", "largest"])
def test_gradient_of_logits_far_from_zero(dt, cuda, dtype, N, V, at):
    g = torch.Generator(device=cuda).manual_seed(N + V)
    far = {"lowest": torch.finfo(dtype).min, "largest": torch.finfo(dtype).max}.get(at, at)
    x = (torch.randn((N, V + 1), generator=g, device=cuda) * 3 + (far if isinstance(at, float) else 0)).to(dtype)
    if not isinstance(at, float):
        x.fill_(far)                                    # a row masked whole
        x[-1, : V // 2] = far / 4 if at == "largest" else far
    x = x[:, 1:] if V % 2 else x[:, 1:].contiguous()    # rows at every offset from a 16-byte boundary
    t = torch.randint(0, V, (N,), generator=g, device=cuda)
    t[0] = -100
    up, ue = (torch.randn((N,), generator=g, device=cuda) for _ in range(2))
    r = dt.token_log_probs(x, t)
    got = dt.token_log_probs_backward(x, t, r.lse, r.entropy, up, ue)
    dt.check_device_error()
    near = (x.double() - x.double().amax(-1, keepdim=True)).clamp_min(-1e4)   # (what is farther has no weight)
    want = grad_ref(near, t, up, ue)
    tol = HALF[dtype] * want.abs() * 1.01 + bound(near, up * (t >= 0), ue, dtype) + 2.0 ** -126
    tol += 4 * EPS32 * torch.zeros_like(want).scatter_(1, t.clamp(0)[:, None], up.double().abs()[:, None])
    assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() - tol).max())
    y = x.clone()
    dt.token_log_probs_backward(y, t, r.lse, r.entropy, up, ue, out=y)  # (a row's share of the work is the same in place)
    assert torch.equal(y, got)
    only = dt.token_log_probs_backward(x, t, r.lse, None, up)
    assert bool(torch.isfinite(only).all()) and bool((only[0] == 0).all())
