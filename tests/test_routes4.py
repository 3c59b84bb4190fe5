"""The rule that picks the tile of a 4-bit product (gemm4_pair in kiln_b200/csrc/routes.h) against measured times."""
import ctypes
import os
import subprocess
import tempfile

import pytest

from util_routes import CSRC, SMS

EPI = {"f32": 0, "f16": 1, "gelu16": 2, "resid": 3, "gelu4": 5}
# Device time (us) of one call on a B200 inside a CUDA graph, NV4: single CTAs, pairs
MEASURED = [  # M, N, K, epilogue
    (77, 2048, 1024, "f16", 3.84, 5.16),
    (200, 2048, 2048, "f16", 4.78, 6.60),
    (512, 2048, 2048, "f16", 4.88, 6.76),
    (1000, 2048, 2048, "f32", 6.17, 8.54),
    (1536, 2048, 2048, "f16", 7.51, 7.54),
    (2048, 2048, 2048, "f16", 8.24, 8.05),
    (3456, 2048, 2048, "f16", 11.23, 11.21),
    (4096, 2048, 2048, "f16", 13.02, 11.47),
    (4096, 2048, 2048, "f32", 15.16, 13.49),
    (4096, 2048, 2048, "resid", 21.37, 21.01),
    (512, 8192, 2048, "gelu4", 9.13, 9.74),
    (1024, 8192, 2048, "gelu4", 14.68, 14.02),
    (1536, 8192, 2048, "gelu4", 20.03, 18.30),
    (2304, 8192, 2048, "gelu4", 25.64, 23.07),
    (3456, 8192, 2048, "gelu4", 36.74, 35.55),
    (4096, 8192, 2048, "gelu4", 42.28, 36.95),
    (512, 8192, 2048, "gelu16", 9.77, 10.00),
    (1024, 8192, 2048, "gelu16", 15.18, 14.11),
    (1536, 8192, 2048, "gelu16", 20.04, 18.28),
    (3456, 8192, 2048, "gelu16", 36.87, 34.48),
    (4096, 8192, 2048, "gelu16", 42.83, 36.94),
    (512, 8192, 2048, "f16", 9.05, 8.63),
    (1024, 8192, 2048, "f16", 14.10, 12.15),
    (1536, 8192, 2048, "f16", 19.02, 15.74),
    (2304, 8192, 2048, "f16", 24.20, 20.19),
    (4096, 8192, 2048, "f16", 40.35, 32.44),
    (4096, 8192, 2048, "f32", 49.67, 42.23),
    (512, 2048, 8192, "f16", 11.53, 14.57),
    (1024, 2048, 8192, "f16", 11.96, 14.92),
    (1536, 2048, 8192, "f16", 18.53, 15.54),
    (2304, 2048, 8192, "f16", 20.37, 16.22),
    (4096, 2048, 8192, "f16", 35.96, 28.02),
    (4096, 2048, 8192, "f32", 38.45, 30.42),
    (1536, 2048, 8192, "resid", 21.79, 18.55),
    (4096, 2048, 8192, "resid", 43.90, 34.40),
    (4096, 8192, 256, "f16", 16.37, 14.94),
    (4096, 8192, 512, "f16", 19.34, 16.67),
    (4096, 8192, 512, "f32", 27.42, 25.32),
    (1100, 1000, 512, "f16", 3.95, 5.52),
    (700, 5000, 700, "f16", 5.65, 6.50),
    (8192, 8192, 8192, "f16", 256.34, 197.77),
]


@pytest.fixture(scope="module")
def pair():
    with tempfile.TemporaryDirectory() as d:
        src, out = os.path.join(d, "r.cpp"), os.path.join(d, "r.so")
        with open(src, "w") as f:
            f.write('#include "routes.h"\nextern "C" int pair(int M, int N, int ks, int epi, int sms) { return kb::gemm4_pair(M, N, ks, epi, sms); }\n')
        subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I" + CSRC, "-o", out, src], check=True)
        yield ctypes.CDLL(out).pair


def test_tile_against_measured_times(pair):
    taken = []
    for M, N, K, epi, single, two in MEASURED:
        p = pair(M, N, (K + 255) // 256, EPI[epi], SMS)
        taken.append(p)
        assert (two if p else single) <= 1.03 * min(single, two), f"{M} x {N} x {K} {epi}: {'pair' if p else 'single'}, {single} / {two} us"
    assert 0 < sum(taken) < len(taken)


def test_few_rows_take_single_tiles(pair):
    for M in (1, 2, 77, 128):
        for K in (64, 2048, 65536):
            assert not pair(M, 8192, (K + 255) // 256, 1, SMS)
    assert pair(1 << 20, 1 << 20, 1 << 16, 1, SMS)       # no overflow at the largest sizes
