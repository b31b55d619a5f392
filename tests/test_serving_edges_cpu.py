"""CPU: what the serving operators refuse at the edges of their arguments' ranges, before anything touches a device."""
import pytest

from tests.test_serving_refusals_cpu import _attend, _prompt


@pytest.mark.parametrize("scale", [3e38, -3e38, 1e300])
def test_scales_whose_product_with_log2_e_is_not_finite(scale):
    for call in (_attend, _prompt):
        with pytest.raises(ValueError, match="scale"):
            call(scale=scale)
