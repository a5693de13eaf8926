"""The policy loss where a row is decided."""
import pytest

import memory64 as m

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 40, 1000, 2000, 50257])
@pytest.mark.parametrize("type_name", ["float32", "bfloat16"])
def test_entropy_of_a_row_that_is_decided(cuda, n, type_name):
    """One legal action: its probability is 1, the entropy 0, the gradient 0, all exactly (2^x at the largest logit is 1,
    its logarithm 0). A nearly decided row's entropy is not negative. It is log S - sum e t / S with S = sum e: a thread adds
    k = n / 512 values (at least 16) to each of its partial sums in fp32, each addition 2^-24 of the sum, in S and in sum e t;
    a term is off by 2^x's 2^-22 and by its argument's and its product's roundings, 2^-24 |t| and 2 2^-24. Relative to 1 + sum
    p |log p| that is (2 k + 8 + 2 max |log p|) 2^-24 at most."""
    import torch
    from t8b import ops
    T = getattr(torch, type_name)
    g = torch.Generator(device="cuda").manual_seed(n)
    rows = 24
    z = torch.randn(rows, n, device="cuda", generator=g).to(T)
    actions = torch.randint(n, (rows,), device="cuda", generator=g)
    at = torch.arange(rows, device="cuda")
    legal = torch.zeros(rows, n, dtype=torch.bool, device="cuda")
    legal[at, actions] = True
    old, advantages = torch.zeros(rows, device="cuda"), torch.randn(rows, device="cuda", generator=g)
    loss, lp, h, _, grad = ops.policy_loss(z, actions, old, advantages, mask=legal, entropy=0.5)
    assert not lp.any() and not h.any() and not grad.any()
    assert torch.equal(loss, -advantages)
    if n == 1:
        return
    z[at, actions] += torch.linspace(8, 50, rows, device="cuda").to(T)
    ones = torch.ones(rows, device="cuda")
    want = m.loss64(z, actions, old, advantages, None, entropy=0.5, weights=ones)
    h, _, grad = ops.policy_loss(z, actions, old, advantages, entropy=0.5, weights=ones)[2:]
    assert float(h.min()) >= 0
    bound = (2 * max(16, n // 512) + 8 + 2 * want["logp"].abs().amax(1)) * 2 ** -24 * (1 + (want["p"] * want["logp"].abs()).sum(1))
    assert bool(((h.double() - want["entropies"]).abs() <= bound).all())
