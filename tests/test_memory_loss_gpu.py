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


@pytest.mark.parametrize("n", [40, 368, 2000, 4099])
@pytest.mark.parametrize("kind", ["bits", "bytes"])
def test_masked_logits_of_a_row_that_is_not_finite(cuda, n, kind):
    """An infinite divergence, an advantage, an old log-probability or a weight that is infinite or NaN, a legal NaN: the
    gradient is 0 at masked logits all the same, and other rows are what they are alone."""
    import torch
    from test_memory_gpu import packed_bits
    from t8b import ops
    inf, nan = float("inf"), float("nan")
    for T in (torch.float32, torch.bfloat16):
        g = torch.Generator(device="cuda").manual_seed(n)
        rows = 8
        z, q = (torch.randn(rows, n, device="cuda", generator=g).to(T) for _ in range(2))
        legal = torch.rand(rows, n, device="cuda", generator=g) < 0.5
        actions, at = torch.randint(n, (rows,), device="cuda", generator=g), torch.arange(rows, device="cuda")
        legal[at, actions] = True
        legal[:, 5], actions[actions == 5] = True, 6
        legal[at, actions] = True
        old, advantages, weights = torch.full((rows,), -3.0, device="cuda"), torch.ones(rows, device="cuda"), torch.ones(rows, device="cuda")
        clean = ops.policy_loss(z, actions, old, advantages, mask=legal, reference=q, weights=weights, kl=0.5, entropy=0.1)
        q[0, 5], advantages[1], advantages[2], weights[4], z[5, 5] = -inf, nan, inf, inf, nan
        old[3], advantages[3] = -inf, -1  # an infinite ratio, which nothing clips on this side
        given = packed_bits(legal) if kind == "bits" else legal
        grad = ops.policy_loss(z, actions, old, advantages, mask=given, reference=q, weights=weights, kl=0.5, entropy=0.1)[4]
        assert not grad[~legal].any()
        for row in range(6):
            assert not bool(grad[row].isfinite().all()), row
        assert torch.equal(grad[6:], clean[4][6:])
        # without a reference, and its sampled form
        grad = ops.policy_loss(z, actions, old, advantages, mask=given, weights=weights, entropy=0.1)[4]
        assert not grad[~legal].any()
        sampled = torch.full((rows,), -3.0, device="cuda")
        sampled[6] = inf
        assert not ops.policy_loss(z, actions, old, advantages, mask=given, reference=sampled, weights=weights, kl=0.5)[4][~legal].any()
