"""Block-scaled products whose rows fill an odd number of 128-row blocks: the CTA pair's second half has no rows, and no scales."""
import pytest
import torch

from chronicals_b200.ops import _ext, ref
from chronicals_b200.utils import fp8_utils as F8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 96, 128, 300, 384, 1300])
@pytest.mark.parametrize("N,K", [(192, 96), (392, 1056)])
def test_scales_end_with_the_last_block_of_rows(M, N, K):
    g = torch.Generator(device="cuda").manual_seed(M + N)
    a = torch.randn(M, K, device="cuda", generator=g).to(torch.float8_e4m3fn)
    b = torch.randn(N, K, device="cuda", generator=g).to(torch.float8_e4m3fn)
    sa = torch.randint(120, 134, (M, K // 32), device="cuda", generator=g, dtype=torch.uint8)
    sb = torch.randint(120, 134, (N, K // 32), device="cuda", generator=g, dtype=torch.uint8)
    packed = F8.pack_mx_scales(sa)
    assert packed.numel() == -(-M // 128) * -(-K // 128) * 512
    behind = torch.cat((packed, torch.full((8192,), 255, dtype=torch.uint8, device="cuda")))      # a scale of NaN
    want = ref.mxfp8_dequantize(a, sa) @ ref.mxfp8_dequantize(b, sb).t()
    for sf in (packed, behind[:packed.numel()]):
        y = F8.mxfp8_block_scaled_matmul(a.view(torch.uint8), sf, b.view(torch.uint8), F8.pack_mx_scales(sb, F8.PAIR_TILE_ROWS),
                                         b_tile_rows=F8.PAIR_TILE_ROWS).float()
        _ext.check_status()
        # products of fp8 numbers are exact, their sum is in 32 bits: one rounding to bf16
        assert ((y - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * want.abs().max()).all()
