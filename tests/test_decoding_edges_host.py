"""Host side of the cached-decoding operators, edges, without a GPU."""

import pytest
import torch

from voyager_b200 import fp8block


def test_quantize_weight_of_a_block_whose_scale_underflows():
    """A block whose largest magnitude over 448 is 0 in float32 counts as a
    block of zeros (scale 1, codes 0), as quantize takes it; the least scale
    that is not 0 is used."""
    w = torch.zeros(130, 260)
    w[0, 0] = 2.0 ** -142      # / 448 is below half of the least float32, 2^-149
    w[3, 130] = 2.0 ** -140    # / 448 = 1.14 * 2^-149
    w[129, 259] = -1.0
    codes, scale = fp8block.quantize_weight(w)
    f = codes.float()
    assert not bool(f.isnan().any())
    assert scale[0, 0] == 1 and not bool(f[:128, :128].any())
    assert scale[0, 1] == 2.0 ** -149 and f[3, 130] == 448  # 2^9 saturates
    assert scale[1, 2] == 1 / 448 and f[129, 259] == -448
    assert scale[0, 2] == 1 and scale[1, 0] == 1 and scale[1, 1] == 1


def test_a_norm_needs_its_weight():
    """Without a weight there is no norm to compute: None is refused, not taken
    as `quantize`."""
    for residual in (None, torch.ones(2, 128)):
        with pytest.raises(TypeError, match="weight"):
            fp8block.rmsnorm_quantize(torch.ones(2, 128), None, 1e-5, residual)
