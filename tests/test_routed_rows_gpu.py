"""Row steps and router gradients on the device: calls that the permutation's
own output does not lead to, and sizes that single branches wait for."""
import pytest

torch = pytest.importorskip("torch")

import routed_cases as rc  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("KK", [2, 8, 33, 64])
def test_a_position_named_twice(moe, KK):
    """Slots of a token that share a position each count: every place of the
    sorted list holds a position of the token's own."""
    T, D, cap = 40, 96, 50
    g = torch.Generator(device="cuda").manual_seed(KK)
    pos = torch.randint(-2, cap + 2, (T, KK), generator=g, device="cuda", dtype=torch.int32)
    pos[0], pos[1, :2] = 7, 49  # all slots the same; a pair
    pos[2] = -1
    y, rw = torch.randn(cap, D, generator=g, device="cuda"), torch.rand(cap, device="cuda")
    live = dict(tok_pos=torch.where(pos < cap, pos, -1))
    for weights in (rw, None):
        out = torch.empty(T, D, device="cuda")
        if weights is None:
            moe.dispatch_grad_dev(y, pos, out)
        else:
            moe.combine_dev(y, rw, pos, out)
        want, size = rc.combine(y, weights, live, T)
        assert ((out.double() - want).abs() <= (KK + 2) * U * size).all()
