"""The launches of attention over the 4-bit cache: limits, scratch, which kernel the prompts of the device tests take."""
import ctypes as C
import random

import pytest

import test_gpu_kv4_borders as borders
import test_gpu_kv4_prompts as prompts
from kv4_plan import plan, raw_plan
from prima_cpp_amd import lib as L

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


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
def test_scratch_is_what_splits_want(d, type):
    """ops.kv4_work's size changes no plan that unlimited scratch would make, and some call uses all of it"""
    r, most = random.Random(d), 0
    floats = L.declare("pm355_attn_kv4_work_floats", C.c_size_t, [C.c_int] * 3)
    for _ in range(6000):
        G, R, n_tiles = r.choice([1, 2, 3, 4, 5, 7, 8, 16, 32]), r.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 28, 64, 128]), r.choice([1, 2, 3, 4, 7, 8, 16, 31, 32, 64, 100, r.randint(1, 600)])
        tile, keys = r.choice([1, max(1, 16 // R), max(1, 128 // R), r.randint(1, max(1, 128 // R))]), r.choice([0, 1, 300, 4000, 131100, r.randint(1, 1 << 20)])
        tokens, window = r.choice([n_tiles, n_tiles * tile, r.randint(1, n_tiles * tile)]), r.choice([0, 0, 500, 40000])
        n = floats(G * R, G, d)
        got = raw_plan(type, G * R, G, d, n_tiles, tile, keys, tokens, window, 4, n)
        assert got == raw_plan(type, G * R, G, d, n_tiles, tile, keys, tokens, window, 4, 1 << 40), (G, R, n_tiles, tile, keys, tokens, window)
        cols, _, splits, _ = got
        passes = -(-R * tile // cols) if cols < 128 else 1
        used = n_tiles * G * passes * splits * cols * (d + 2) if splits > 1 else 0
        assert used <= n
        most = max(most, used)
    assert most == floats(8, 8, d) == (512 if d <= 128 else 256) * 128 * (d + 2)


@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
def test_prompts_of_the_device_tests_are_prompts(d, type):
    """tests/test_gpu_kv4_prompts.py's cases go to the kernel of 128 columns with any window, some of them with split keys and some without"""
    splits = {plan(type, *prompts.CASES[c][:2], d, prompts.CASES[c][2], w, f, work) for c in prompts.CASES for w, f in prompts.WINDOWS + [(300, 9), (40, 6), (100, 5), (30, 6)] for work in (True, False)}
    assert {p[0] for p in splits} == {128} and {p[2] > 1 for p in splits} == {True, False}
    assert plan(type, 16, 16, d, borders.BATCHES["prompt"])[0] == 128 and all(plan(type, 16, 16, d, e)[0] < 128 for b, e in borders.BATCHES.items() if b != "prompt")
    assert plan(type, 16, 16, d, borders.BATCHES["far"])[2] > 1
