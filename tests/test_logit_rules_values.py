"""Values of the logit rules where the penalty's power is very small or very large."""
import pytest
import torch

from air_rs import ops

DEV = "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("V", [64, 67])              # four entries at a time, one by one
def test_repetition_powers_near_the_ends_of_the_range(V):
    """x / rho^c and x * rho^c where rho^c is denormal, near the largest number, or past either end: quotients and
    products that fit are right, the others 0 or infinite."""
    rho = torch.tensor([0.05, 0.06, 17.0, 30.0, 0.9, 1.2])
    B = rho.numel()
    x = torch.randn(B, V, generator=torch.Generator().manual_seed(V)) * 1e-3
    counts = (torch.arange(V)[None] + torch.arange(B)[:, None] * 5).remainder(40).to(torch.uint8)
    got = ops.logit_rules(x.to(DEV), counts=counts.to(DEV), repetition=rho.to(DEV)).cpu().double()
    f = rho.double()[:, None] ** counts.double()
    want = torch.where(counts > 0, torch.where(x > 0, x.double() / f, x.double() * f), x.double())
    fits = want.abs() < 3.4e38
    # powf is good to 4 ulp (2^-21), and to 2^-147 where it is denormal, relatively 2^-147 / f; the quotient rounds once
    tol = want.abs() * (2.0 ** -20 + torch.minimum(2.0 ** -147 / f, torch.ones(()).double())) + 2.0 ** -148
    usable = fits & (f > 2.0 ** -140) & (f < 3.4e38)
    assert bool((got - want)[usable].abs().le(tol[usable]).all())
    assert int((usable & (f < 2.0 ** -128) & (x > 0)).sum()) > 0    # reciprocals that overflow are among them
    assert not torch.isnan(got).any()
    over = (f > 3.5e38)
    assert not got[over & (x > 0)].any() and bool(torch.isinf(got[over & (x < 0)]).all())


@pytest.mark.gpu
def test_penalties_over_different_counts_are_two_calls():
    B, V = 3, 500
    r = torch.Generator().manual_seed(0)
    x = torch.randn(B, V, generator=r)
    out = torch.randint(0, 3, (B, V), generator=r).to(torch.uint8)
    seen = out + torch.randint(0, 3, (B, V), generator=r).to(torch.uint8)
    rho, fr, pr = 1.1 + torch.rand(B, generator=r), torch.rand(B, generator=r), torch.rand(B, generator=r)
    d = lambda t: t.to(DEV)
    got = ops.logit_rules(ops.logit_rules(d(x), counts=d(seen), repetition=d(rho)), counts=d(out), frequency=d(fr), presence=d(pr))
    f = rho.double()[:, None] ** seen.double()
    want = torch.where(x > 0, x.double() / f, x.double() * f)
    mag = want.abs() + 4
    want = want - fr.double()[:, None] * out - pr.double()[:, None] * (out > 0)
    # powf 4 ulp (2^-21), the product or quotient, two differences of numbers up to mag
    assert bool(((got.cpu().double() - want).abs() <= 2.0 ** -20 * mag).all())
