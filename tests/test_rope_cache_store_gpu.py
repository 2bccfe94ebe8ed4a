"""What zentorch_rope_cache stores in an e4m3 cache is the quotient by the scale, rounded to nearest even."""
import pytest
import torch

from test_rope_cache_gpu import BF16, E4M3, F32, ops  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def store(ops, x, scale, page=4):  # noqa: F811
    """[tokens, heads, d] as keys (no rotated part) and as values; both come back as fp32."""
    t, h, d = x.shape
    kc, vc = (torch.zeros(-(-t // page), page, h, d, device="cuda").to(E4M3) for _ in range(2))
    i = torch.arange(t, device="cuda")
    ops.zentorch_rope_cache(torch.zeros_like(x), x, x, i, torch.zeros(0, device="cuda"), kc, vc, i, scale, scale)
    return [c.float().view(-1, h, d)[:t].cpu() for c in (kc, vc)]


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_ties_go_to_even(ops, dtype):  # noqa: F811
    """Elements that are exactly halfway between two e4m3 numbers times the scale, for scales without an exact reciprocal."""
    scale = torch.tensor([3.0, 5.0, 7.0, 3.0, 5.0, 7.0]) * torch.tensor([2.0 ** -9] * 3 + [2.0 ** 7] * 3)
    half = torch.arange(17, 32, 2).float() / 16                             # between 1, 9/8, .., 2
    target = torch.cat([half * 2.0 ** e for e in range(-4, 5)] + [half[:0]])
    target = torch.cat([target, -target])
    d = target.numel()                                                      # 144
    x = (target * scale[:, None])[None]
    assert torch.equal(x.to(dtype).float(), x) and d % 8 == 0
    want = target.to(E4M3).float().expand(6, d)
    for got in store(ops, x.to(dtype).cuda(), scale.cuda()):
        assert torch.equal(got[0], want)


def test_scales_whose_reciprocal_is_not_finite(ops):  # noqa: F811
    scale = torch.tensor([2.0 ** -140, -(2.0 ** -133), 2.0 ** -126, 2.0 ** 127])
    target = torch.tensor([0.0, 1.0, -2.5, 13.0, 448.0, -0.0, 0.875, 1.0625])
    x = (target.double() * scale.double()[:, None]).float()[None]
    exact = (x.double() / scale.double()[:, None])[0].clamp(-448, 448).float().to(E4M3).float()      # 2.5 * 2^127 is infinite: saturates
    for got in store(ops, x.cuda(), scale.cuda()):
        assert torch.equal(got[0], exact)
