"""What the inverse of a rotation gives back (GPU)."""
import math

import pytest
import torch

from sage_testutil import have_gfx950

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not have_gfx950(), reason="needs a gfx950 GPU")]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scaling,size", [(None, 1.0), ("yarn", 0.1 * math.log(4.0) + 1.0)])
def test_the_inverse_gives_back_the_tables_size_squared(scaling, size, interleaved):
    from sageattention import apply_rotary, rotary_table
    gen = torch.Generator().manual_seed(1)
    table = rotary_table(300, 64, scaling=scaling, factor=4.0 if scaling else 1.0, original_length=100)
    pos = torch.randint(0, 300, (2, 33), generator=gen).int().cuda()
    x = torch.randn(2, 3, 33, 128, generator=gen).half().cuda()
    y = apply_rotary(x, table, pos, interleaved=interleaved)
    back = apply_rotary(y, table, pos, interleaved=interleaved, inverse=True).double().cpu()
    x = x.double().cpu()
    assert torch.equal(back[..., 64:], x[..., 64:])
    back, x = back[..., :64], x[..., :64]
    # a pair's two values of up to size * r, r its length, are off by 2^-11 of that, turned and scaled by
    # size once more, then by the result's own half step; three fp32 roundings of each add under 2^-20
    a, b = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    r = torch.empty_like(x)
    r[..., a] = r[..., b] = (x[..., a] ** 2 + x[..., b] ** 2).sqrt()
    bound = size ** 2 * r * (2 ** 0.5 * 2.0 ** -11 + 2.0 ** -11 * (1 + 2.0 ** -10) + 2.0 ** -19) + 2.0 ** -24
    assert ((back - size ** 2 * x).abs() <= bound).all()
