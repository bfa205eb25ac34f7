"""Calls on the AdamW operators at the edges of what their documentation allows, on the GPU."""
import pytest
import torch

from oracle import adamw_oracle as orc
from test_gpu_adamw import _place

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mb():
    import muon_b200
    return muon_b200


# ------------------------------------------------------------------------------------ conversion
@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "odd"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_signed_zeros_of_second_moments(mb, dtype, offset):
    """-0.0 is not negative: it gets the code of 0, the smallest. So do values under 0 that the rounding of an
    earlier run may have left; a block whose largest magnitude counts as zero has codes 0 and scale 0."""
    gen = torch.Generator().manual_seed(30)
    x = [torch.rand(n, generator=gen) for n in (256, 600, 1, 257)]
    x[0][::3] = -0.0
    x[1][1::2] = -0.0
    x[2][0] = -0.0
    x[3][256] = -0.0
    for k, y in enumerate((-1e-38, -1e-12, -2.0 ** -31, -1e-7, -1e-3, -0.5)):
        x[0][10 + k] = y
        x[1][300 + k] = y
    tiny = torch.full((300,), 2.0 ** -125) * torch.where(torch.arange(300) % 2 == 0, 1.0, -1.0)
    tiny[5], tiny[299] = -0.0, -0.0
    x = [y.to(dtype) for y in x + [tiny]]
    codes, scales = mb.quantize_state(_place(x, dtype, offset), "exp_avg_sq")
    for y, c, s in zip(x, codes, scales):
        want_c, want_s = orc.quantize(y, "exp_avg_sq")
        assert torch.equal(c.cpu(), want_c) and torch.equal(s.cpu(), want_s)
        assert (c.cpu()[torch.signbit(y)] == 0).all()
    assert (codes[4] == 0).all() and (scales[4] == 0).all()
