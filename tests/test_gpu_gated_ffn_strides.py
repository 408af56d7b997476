"""gated_ffn on weights whose rows lie far apart, the last ones past 2^32 bytes: the
same bits as from contiguous copies, for few rows and for tiles of them."""

import pytest
import torch

from encoder_plain import ROUNDOFF, gated_ffn64, off
from late_interaction_kernels.encoder import gated_ffn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [3, 33, 130])
def test_weights_past_32_bits(rows):
    print("[case]", rows, flush=True)
    d, f, apart = 1088, 544, 2**21  # 1088 rows of 4 MB
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, d, generator=g).to(torch.bfloat16)
    wi = (torch.randn(2 * f, d, generator=g) * d**-0.5).to(torch.bfloat16)
    wo = (torch.randn(d, f, generator=g) * f**-0.5).to(torch.bfloat16)
    far = torch.empty(2 * f, apart, dtype=torch.bfloat16, device="cuda")
    assert far.numel() * 2 > 2**32
    far_in, far_out = far[:, :d], far[:, 2048 : 2048 + f]
    far_in.copy_(wi)
    far_out.copy_(wo)
    got = gated_ffn(x.cuda(), far_in, far_out)
    assert torch.equal(got, gated_ffn(x.cuda(), wi.cuda(), wo.cuda()))
    # h and the output are rounded: sqrt(2 / 3) of the roundoff in the 2-norm, 1.25 for small outputs
    assert off(got, gated_ffn64(x.double(), wi.double(), wo.double(), None, "gelu")) <= 1.25 * ROUNDOFF[torch.bfloat16]
