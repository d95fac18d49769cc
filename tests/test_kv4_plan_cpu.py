"""The launches of attention over the 4-bit cache: limits."""
import pytest

from kv4_plan import raw_plan

SHAPE = -2


@pytest.mark.parametrize("type", ["bf16", "f32"])
def test_limits_of_a_launch(type):
    """refused is what a launch cannot take (2^32 threads), not less"""
    assert raw_plan(type, 8, 8, 64, 1 << 17, 1, 100, 1 << 17) == (16, 1, 1, 1 << 20)
    assert raw_plan(type, 8, 8, 64, (1 << 20) - 1, 1, 100, (1 << 20) - 1, floats=1 << 24) == (16, 1, 1, (1 << 23) - 8)
    assert raw_plan(type, 8, 8, 64, 1 << 20, 1, 100, 1 << 20) == SHAPE
    assert raw_plan(type, 32, 1, 64, 1 << 22, 1, 100, 1 << 22) == (32, 1, 1, 1 << 22)
    assert raw_plan(type, 8, 8, 64, (1 << 21) - 1, 128, 100, 100 << 21) == (128, 1, 1, (1 << 24) - 8)
    assert raw_plan(type, 8, 8, 64, 1 << 21, 128, 100, 100 << 21) == SHAPE
    assert raw_plan(type, 8, 8, 64, 0, 1, 100, 0) == (0, 0, 0, 0)
