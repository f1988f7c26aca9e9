"""The 8-bit feed-forward operators at the ends of their ranges, and calls that
their documentation allows but ordinary tests do not make.

References, helpers and the way tolerances are counted are those of
test_feedforward.py; 8-bit values have to be the nearest whole numbers of the
exact quotient.
"""

import pytest
import torch

import flow2surf_b200 as f2s

# fp32 streams and weights s, w of 24 bits with 254 s1 w1 - c s0 w0 = r for c odd:
# 127 p / m is r / (2 m) off the half c / 2, less than 64-bit products tell (they
# have 56 bits). (s0, w0, s1, w1, c, r), s0 w0 the larger product.
NEXT_TO_HALVES = [
    (16374893, 16219904, 15165803, 16203002, 235, 4),
    (16101769, 16130341, 14068111, 16499603, 227, -1),
    (16679204, 16069049, 14716702, 14698572, 205, -4),
    (16637806, 15750364, 16438509, 13242591, 211, 2),
    (16301801, 16312208, 16179395, 16112083, 249, -2),
    (16719859, 16164048, 15467849, 16440575, 239, 2),
    (16646973, 15920774, 13441091, 16535252, 213, 2),
    (16442797, 16735767, 16560288, 15243182, 233, -3),
    (16373941, 16552341, 15664237, 14373156, 211, -3),
    (16622725, 16199528, 16492751, 15362987, 239, -2),
    (15860984, 15875619, 15848809, 13448347, 215, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, -20, 38])
@pytest.mark.parametrize("width", [2, 8, 200, 5000])
def test_norm_int8_of_products_next_to_halves(cuda, width, shift):
    """The exact quotient decides, whatever power of two the products carry."""
    for s0, w0, s1, w1, c, r in NEXT_TO_HALVES:
        assert 254 * s1 * w1 - c * s0 * w0 == r and c % 2 and 0 < s1 * w1 <= s0 * w0
        x, w = torch.zeros(3, width), torch.ones(width)
        x[1, :2] = torch.tensor([s0, s1]) * 2.0**shift
        x[2, :2] = torch.tensor([s0, -s1]) * 2.0**shift
        w[:2] = torch.tensor([w0, w1]) * 2.0**shift
        values = f2s.add_rms_norm_int8(x.to(cuda), w.to(cuda))[0].values
        q = (c + 1) // 2 if r > 0 else c // 2
        assert values[1:, :2].tolist() == [[127, q], [127, -q]]
