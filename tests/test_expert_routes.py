"""The tiles of the experts' projections (csrc/kxw4_route.hpp), on the CPU: each
shape goes to the kernel that was measured ahead on it (launches of a graph
replay with the weights from HBM on an MI355X; us beside the case)."""
import ctypes as C
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "knivesysl_xe_amd", "csrc")
CUS = 256


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("expert_route")
    src, out = d / "route.cpp", d / "route.so"
    src.write_text('#include "kxw4_route.hpp"\n'
                   'extern "C" int experts(long long N, int groups, int group, int r128, int r256, int blocks, int w8) {\n'
                   f'    return kxw4::expert_route({{{CUS}, N, groups, group, r128, r256, blocks != 0, w8 != 0}});\n'
                   '}\n'
                   'extern "C" int expert_splits(long long strips, int ktiles) { return kxw4::expert_splits(strips, ktiles); }\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(out)],
                   check=True)
    lib = C.CDLL(str(out))
    lib.experts.argtypes = [C.c_longlong] + [C.c_int] * 6
    lib.expert_splits.argtypes = [C.c_longlong, C.c_int]
    return lib


@pytest.mark.parametrize("mode,group,N,experts,rows,want", [
    # (us of the kernel named and of the one beside it)
    ("token", 128, 8, 64, [1024, 1024], 2),              # strips of 2 11.8, of 8 12.4
    ("token", 128, 64, 64, [1024, 1024], 8),             # 32.4, of 2 35.1
    ("token", 128, 128, 64, [1024, 1024], 8),            # 46.7, of 16 50.4
    ("token", 128, 176, 16, [576], 16),                  # 9.8, tiles of 32 15.8
    ("token", 128, 160, 8, [320, 320], 16),              # 8.7, tiles of 32 12.5
    ("token", 128, 544, 32, [640], 16),                  # 160 tiles for 256 CUs
    ("token", 128, 1152, 64, [704, 704], 132),           # 17.4, strips 17.9
    ("token", 128, 2400, 64, [1024, 1024], 164),         # 90, strips 111
    ("token", 128, 2144, 16, [320, 320], 132),           # 13.4, tiles of 64 18.5
    ("token", 128, 16384, 64, [1024, 1024], 228),        # 227, tiles of 64 258
    ("token", 128, 5920, 16, [1216, 1216], 164),         # 45.0, tiles of 128 51.5
    ("token", 64, 16384, 64, [1024, 1024], 164),         # 310, strips 434
    ("token", 64, 784, 64, [1088], 132),                 # 11.1, strips 11.6
    ("block", 32, 6, 128, [1216, 1216], 2),              # 8.0, of 8 9.2
    ("block", 64, 44, 32, [832, 832], 8),                # 11.0
    ("block", 32, 72, 16, [1472, 1472], 16),             # 8.9, of 8 10.0
    ("block", 32, 768, 32, [512, 512], 16),              # 14.6, of 32 15.1
    ("block", 32, 1067, 32, [832, 832], 32),             # 21.2, of 16 21.8
    ("w8", 32, 840, 64, [256, 256], 16),                 # 9.8, of 32 11.4
    ("w8", 32, 2168, 128, [768, 768], 32),               # 93, of 16 99
    ("token", 128, 1, 1, [16], 8),
    ("block", 64, 16384, 64, [1024], 264),               # 311, strips 399
    ("block", 32, 12000, 64, [512], 264),                # 71, strips 75
    ("block", 32, 4000, 32, [1024], 32),                 # 512 tiles: 119, tiles 117
    ("block", 32, 1800, 40, [1408], 32),                 # 44, tiles 51
    ("w8", 32, 16384, 64, [1024], 32),
])
def test_expert_tiles(rules, mode, group, N, experts, rows, want):
    r128, r256 = (sum((m + w - 1) // w for m in rows) for w in (128, 256))
    assert rules.experts(N, experts, group, r128, r256, mode != "token", mode == "w8") == want


def test_expert_splits(rules):
    for strips in (1, 64, 100, 1024, 2047, 2048, 10 ** 9):
        for ktiles in (1, 2, 3, 4, 7, 8, 40):
            S = rules.expert_splits(strips, ktiles)
            assert S in (1, 2, 4, 8) and S <= ktiles
            # no more than the strips ask for, no fewer than K has room for
            assert S == 1 or strips * (S // 2) < 2048
            assert S == 8 or strips * S >= 2048 or 2 * S > ktiles
