"""The shapes of the GPU tests of the 8-bit floating tier's products take the kernel that they stand for, and leave no kernel
out, by the rules that the library itself goes by (csrc/kxw4_f8_route.hpp; no GPU needed)."""
import ctypes as C
import os
import subprocess

import pytest

import f8_shapes as shapes

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "knivesysl_xe_amd", "csrc")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("f8_coverage")
    src, out = d / "route.cpp", d / "route.so"
    src.write_text('#include "kxw4_f8_route.hpp"\n'
                   'using namespace kxw4;\n'
                   'extern "C" void route(int rows, int K, int count, const int *M, int groups, int bf16, int *stream, int *is_long, int *id, int *parts) {\n'
                   f'    F8Sizes s{{{shapes.CUS}, rows, (K + 127) / 128, count, {{}}, groups, bf16 != 0}};\n'
                   '    for (int i = 0; i < count; ++i) s.M[i] = M[i];\n'
                   '    *stream = f8_stream_rows(s);\n'
                   '    *is_long = groups ? f8_long_groups(s) : 0;\n'
                   '    const F8Choice c = f8_choose(s);\n'
                   '    *id = c.id;\n'
                   '    *parts = c.splits;\n'
                   '}\n'
                   'extern "C" int stream(int rows, int K, int count, const int *M, int groups, int x_bytes, int *row_groups, int *waves) {\n'
                   f'    F8Sizes s{{{shapes.CUS}, rows, (K + 127) / 128, count, {{}}, groups, false}};\n'
                   '    for (int i = 0; i < count; ++i) s.M[i] = M[i];\n'
                   '    const int tile = f8_stream_rows(s);\n'
                   '    const F8StreamShape shape = f8_stream_shape(s, tile);\n'
                   '    *row_groups = shape.row_groups;\n'
                   '    *waves = shape.waves;\n'
                   '    return tile * (x_bytes && (tile == 16 ? f8_stream_quantizes(s) : f8_stream32_quantizes(s, x_bytes)) ? -1 : 1);\n'
                   '}\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(out)],
                   check=True)
    return C.CDLL(str(out))


@pytest.fixture(scope="module")
def route(lib):
    """route(rows, K, Ms, groups, bf16) -> ("stream", rows of a tile), ("groups", long) or (tile id, parts)"""
    def run(rows, K, Ms, groups=0, bf16=1):
        stream, is_long, tile, parts = C.c_int(), C.c_int(), C.c_int(), C.c_int()
        lib.route(rows, K, len(Ms), (C.c_int * 4)(*Ms), groups, bf16, C.byref(stream), C.byref(is_long), C.byref(tile),
                  C.byref(parts))
        if stream.value:
            return "stream", stream.value
        return ("groups", bool(is_long.value)) if groups else (tile.value, parts.value)

    return run


@pytest.mark.parametrize("bf16,table,tiles", [(1, shapes.DENSE_BF16, shapes.BF16_TILES), (0, shapes.DENSE_F32, shapes.F32_TILES)])
def test_dense_shapes_take_their_tile(route, bf16, table, tiles):
    for kernel, T, K, Ms in shapes.cases(table):
        tile, parts = route(T, K, Ms, 0, bf16)
        assert (tile, parts > 1) == (tiles[kernel.split()[0]], "parts" in kernel), (kernel, T, K, Ms)
    # every tile, with whole sums and with split ones
    assert set(table) == {name + end for name in tiles for end in ("", " parts")}


def test_every_tile_of_the_rules_is_named(route):
    text = open(os.path.join(CSRC, "kxw4_f8_gemm.hip")).read()
    built = sum(f"case {i}:" in text for i in range(16)) + text.count("default: return f8_dense")
    assert sorted([*shapes.BF16_TILES.values(), *shapes.F32_TILES.values()]) == list(range(built))


def test_grouped_shapes_take_their_tile(route):
    for kernel, T, k, E, K, Ms in shapes.cases(shapes.GROUPED):
        for bf16 in (0, 1):
            assert route(T * k, K, Ms, E, bf16) == ("groups", kernel == "long"), (kernel, T, k, E, K, Ms)
    assert set(shapes.GROUPED) == {"short", "long"}
    E, K, M, rows = shapes.PAST_32
    for kernel, T in rows.items():
        assert route(T, K, (M,), E, 0) == route(T, K, (M,), E, 1) == ("groups", kernel == "long"), kernel


def test_few_rows_take_their_kernel(lib):
    reached = set()
    for want, shapes_of in shapes.STREAM.items():
        for T, k, E, K, Ms in shapes_of:
            for x, size in (("codes", 0), ("bf16", 2), ("f32", 4)):
                rgs, waves = C.c_int(), C.c_int()
                tile = lib.stream(T * k, K, len(Ms), (C.c_int * 4)(*Ms), E, size, C.byref(rgs), C.byref(waves))
                assert (abs(tile), rgs.value, waves.value) == want, (T, k, E, K, Ms)
                reached.add((want[:2], E > 0, x if tile < 0 else "codes"))
    # every instance: rows of a tile, row-groups, by group or not, what the rows come as
    assert reached == {((rows, rgs), grouped, x) for rows in (16, 32) for rgs in (1, 2) for grouped in (False, True)
                       for x in ("codes", "bf16", "f32")}
