"""GPU tests of the gated block quantiser where exp(g) is below the normal numbers of fp32 and the other half so large that the product is an ordinary one again."""

import pytest
import torch

from flydsl_amd import quant_device

pytestmark = pytest.mark.gpu
U = 2.0**-24
GATES = [-82.9, -83.1, -84.0, -87.0, -88.0, -90.0, -95.0, -100.0, -104.0, -110.0, -120.0, -131.0, -140.0, -150.0, -160.0, -170.0]


@pytest.mark.parametrize("dt,top", [(torch.float32, 2.0**127), (torch.float32, 2.0**110), (torch.float32, -1.7e38), (torch.bfloat16, 2.0**127), (torch.bfloat16, 2.0**110), (torch.float16, 60000.0)])
@pytest.mark.parametrize("dim", [128, 130])
def test_blocks_of_one_far_gate(dt, top, dim):
    """Every block has one gate and one other half, so its scale is what was made of the two: exp(-|g|) off by 3 u, the products of it by u each, the division by 448 by one (u = 2^-24; sigmoid is
    exp(-|g|) itself there), or by half of 2^-149 where it is a subnormal number.  Codes are +-448."""
    g = torch.tensor([v for v in GATES if abs(v) * 2.718281828**v * abs(top) >= 1e-36]).to(dt).unsqueeze(1).expand(-1, dim)
    u = torch.full(g.shape, top).to(dt)
    print(f"gate {dt} {top} {dim} {g.shape[0]} rows", flush=True)
    q, s = quant_device.per_1x128_f8_quant(torch.cat([g, u], 1).cuda(), gated=True)
    y = g.double() / (1 + torch.exp(-g.double())) * u.double()
    want = y[:, :1].abs().t() / 448
    assert ((s.double().cpu() - want).abs() <= 11.5 * U * want + 2.0**-150).all()
    assert (q.cpu().float() == 448 * torch.sign(y)).all()


def test_gates_from_near_to_far_in_one_block():
    """The nearest gate makes the scale; the others' codes are their own values', as far as 8 bits hold them."""
    g = torch.linspace(-84, -95, 128).repeat(3, 1)
    u = torch.full((3, 128), 2.0**110)
    u[1] = torch.exp(-g[1].double() - 84).float() * 2.0**100  # (so that all are of one size)
    u[2, ::2] = -u[2, ::2]
    q, s = quant_device.per_1x128_f8_quant(torch.cat([g, u], 1).cuda(), gated=True)
    y = g.double() * torch.exp(g.double()) * u.double()
    want = y.abs().amax(1) / 448
    assert ((s[0].double().cpu() - want).abs() <= 11.5 * U * want).all()
    v = y / want.unsqueeze(1)
    assert ((q.double().cpu() - v).abs() <= torch.clamp(2.0**-4 * v.abs(), min=2.0**-10) * (1 + 24 * U) + 24 * U * v.abs()).all()


def test_nothing_left_and_infinities():
    inf = float("inf")
    g = torch.tensor([-inf, -1000.0, -300.0, -250.0, -150.0, -150.0, 150.0, 300.0, inf, -100.0])
    u = torch.tensor([5.0, 2.0**127, 2.0**100, 1.0, 2.0**-149, inf, 2.0**-120, 1.0, 2.0, -inf])
    # -inf * 0 is NaN; what is below the smallest number is 0; silu(-150) * inf = -inf; inf; silu(-100) * -inf = inf
    y = torch.tensor([0.0, 0, 0, 0, 0, -448, 150 * 2.0**-120, 300, 448, 448])
    q, s = quant_device.per_1x128_f8_quant(torch.cat([g, u]).unsqueeze(0).cuda(), gated=True)
    assert s.item() == 1.0
    assert torch.equal(q.cpu().float().view(-1), y.to(torch.float8_e4m3fn).float())
