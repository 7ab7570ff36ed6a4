"""The choice of kernel and tile for products of the 8-bit floating tier (csrc/kxw4_f8_route.hpp), on the CPU: each shape
takes what was measured ahead on it, and no choice asks for what a launch cannot hold."""
import ctypes as C
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "knivesysl_xe_amd", "csrc")
CUS = 256
TILES = {0: (256, 256, 1), 1: (256, 128, 1), 2: (128, 128, 1), 3: (64, 128, 2), 4: (128, 128, 2), 5: (64, 128, 2)}


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("f8_route")
    src, out = d / "route.cpp", d / "route.so"
    src.write_text('#include "kxw4_f8_route.hpp"\n'
                   'using namespace kxw4;\n'
                   'static F8Sizes sizes(int rows, int K, int count, int M, int groups, int bf16) {\n'
                   f'    return F8Sizes{{{CUS}, rows, (K + 127) / 128, count, {{M, M, M, M}}, groups, bf16 != 0}};\n'
                   '}\n'
                   'extern "C" int stream(int rows, int K, int count, int M, int groups) { return f8_stream_rows(sizes(rows, K, count, M, groups, 1)); }\n'
                   'extern "C" int fused(int rows, int K, int count, int M, int groups) { return f8_stream_quantizes(sizes(rows, K, count, M, groups, 1)); }\n'
                   'extern "C" int fused32(int rows, int K, int M, int groups, int bytes) { return f8_stream32_quantizes(sizes(rows, K, 1, M, groups, 1), bytes); }\n'
                   'extern "C" int longer(int rows, int groups) { return f8_long_groups(sizes(rows, 128, 1, 128, groups, 1)); }\n'
                   'extern "C" int choose(int rows, int K, int count, int M, int bf16, int *splits) {\n'
                   '    const F8Choice c = f8_choose(sizes(rows, K, count, M, 0, bf16));\n'
                   '    *splits = c.splits;\n'
                   '    return c.id;\n'
                   '}\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(out)],
                   check=True)
    return C.CDLL(str(out))


def choose(rules, *a):
    s = C.c_int()
    return rules.choose(*a, C.byref(s)), s.value


def test_few_rows_take_the_stream(rules):
    # rows, K, weights, M, groups -> rows of a stream tile
    for case, want in (((1, 4096, 1, 4096, 0), 16), ((16, 17408, 1, 5120, 0), 16), ((17, 17408, 1, 5120, 0), 0),
                       ((32, 5120, 1, 5120, 0), 32), ((33, 5120, 1, 5120, 0), 0), ((128, 1456, 1, 2064, 0), 32),
                       ((97, 1456, 1, 2064, 0), 32), ((512, 1456, 1, 2064, 0), 0), ((128, 5120, 2, 1024, 64), 16),
                       ((1600, 5120, 1, 1024, 64), 0), ((450, 336, 1, 208, 5), 32)):
        assert rules.stream(*case) == want, case


def test_small_weights_are_streamed_by_one_launch(rules):
    assert rules.fused(1, 4096, 1, 4096, 0) and rules.fused(4, 1024, 1, 5120, 32)
    assert not rules.fused(1, 17408, 1, 5120, 0) and not rules.fused(8, 5120, 2, 17408, 0)
    assert not rules.fused(128, 5120, 2, 1024, 64)


def test_short_launches_of_32_rows_quantize_by_themselves(rules):
    # rows, K, M, groups
    for case, f32, bf16 in (((256, 1024, 1024, 0), 1, 1), ((200, 768, 1024, 0), 1, 1), ((450, 208, 336, 5), 1, 1),
                            ((64, 2048, 2048, 0), 0, 1), ((97, 1456, 2064, 0), 0, 1), ((256, 1024, 1024, 8), 0, 1),
                            ((32, 4096, 4096, 0), 0, 0), ((32, 5120, 5120, 0), 0, 0)):
        assert (rules.fused32(*case, 4), rules.fused32(*case, 2)) == (f32, bf16), case


def test_dense_tiles(rules):
    # BF16: rows, K, weights, M -> (tile, parts)
    assert choose(rules, 3965, 5120, 2, 17408, 1) == (0, 1)
    assert choose(rules, 2048, 5120, 1, 5120, 1) == (0, 1)
    assert choose(rules, 1024, 5120, 1, 5120, 1) == (1, 1)
    assert choose(rules, 512, 5120, 1, 5120, 1) == (2, 1)
    assert choose(rules, 512, 17408, 1, 5120, 1) == (1, 3)
    assert choose(rules, 64, 17408, 1, 5120, 1) == (3, 6)
    # FP32
    assert choose(rules, 97, 17408, 1, 5120, 0)[1] > 1
    assert choose(rules, 2048, 5120, 1, 5120, 0)[1] == 1


def test_every_choice_fits(rules):
    rng = random.Random(5)
    for _ in range(3000):
        rows, K, M = (int(2 ** rng.uniform(a, b)) for a, b in ((0, 17), (4, 15), (4, 16)))
        K, M, count = K // 16 * 16, M // 16 * 16, rng.choice([1, 2, 4])
        for bf16 in (0, 1):
            tile, parts = choose(rules, rows, K, count, M, bf16)
            bt, br, per_cu = TILES[tile]
            assert (tile < 4) == bool(bf16)
            kb = (K + 127) // 128
            assert 1 <= parts <= 8 and (parts == 1 or (kb // parts >= 4 and
                                                       -(-rows // bt) * -(-M // br) * count * parts <= CUS * per_cu))


def test_long_groups(rules):
    assert rules.longer(128 * 64, 64) and not rules.longer(128 * 64 - 1, 64)
