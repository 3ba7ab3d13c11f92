"""Sizes at which the serving operators' indexes would pass 32 bits are
refused for their size, before the GPU is asked for anything."""
import pytest

from test_serve_cpu import pages


@pytest.mark.parametrize("max_tokens", [(1 << 30) + 1, (1 << 31) - 512, (1 << 31) - 1])
def test_plan_refuses_maps_past_32_bit_rows(ptlib, capfd, max_tokens):
    assert ptlib.ptc_plan_pages(pages(max_tokens=max_tokens), None) == -1
    err = capfd.readouterr().err
    assert "ptc_plan_pages: bad size" in err and f"max_tokens {max_tokens}" in err
