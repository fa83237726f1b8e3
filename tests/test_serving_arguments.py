"""Arguments at the ends of their ranges, at the C ABI: refused before a device is touched."""
import ctypes as C

import pytest

from test_serving_refusals import attend, cache, prompt, refused


@pytest.mark.parametrize("scale", [3e38, 2.4e38])
def test_a_scale_whose_product_with_log2_e_overflows(scale):
    refused("scale", *attend(cache(), scale=scale))
    refused("scale", "bgtq_prompt_attend", C.byref(prompt(scale=scale)), None)
