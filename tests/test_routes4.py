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
    (77, 2048, 1024, "f16", 3.82, 5.38),
    (200, 2048, 2048, "f16", 4.79, 6.91),
    (512, 2048, 2048, "f16", 4.86, 7.44),
    (1000, 2048, 2048, "f32", 6.25, 8.96),
    (1536, 2048, 2048, "f16", 7.50, 8.12),
    (2048, 2048, 2048, "f16", 8.24, 8.74),
    (3456, 2048, 2048, "f16", 11.50, 12.66),
    (4096, 2048, 2048, "f16", 13.65, 12.91),
    (4096, 2048, 2048, "f32", 15.72, 15.38),
    (4096, 2048, 2048, "resid", 20.14, 21.29),
    (512, 8192, 2048, "gelu4", 9.48, 11.01),
    (1024, 8192, 2048, "gelu4", 15.06, 16.18),
    (1536, 8192, 2048, "gelu4", 20.42, 21.81),
    (2304, 8192, 2048, "gelu4", 26.24, 27.48),
    (3456, 8192, 2048, "gelu4", 37.85, 42.66),
    (4096, 8192, 2048, "gelu4", 43.59, 43.96),
    (512, 8192, 2048, "gelu16", 9.72, 11.12),
    (1024, 8192, 2048, "gelu16", 15.29, 15.47),
    (1536, 8192, 2048, "gelu16", 20.74, 19.63),
    (3456, 8192, 2048, "gelu16", 37.66, 37.16),
    (4096, 8192, 2048, "gelu16", 43.43, 38.91),
    (512, 8192, 2048, "f16", 9.47, 9.50),
    (1024, 8192, 2048, "f16", 15.00, 13.51),
    (1536, 8192, 2048, "f16", 20.14, 17.70),
    (2304, 8192, 2048, "f16", 25.49, 22.36),
    (4096, 8192, 2048, "f16", 41.33, 35.50),
    (4096, 8192, 2048, "f32", 51.92, 45.93),
    (512, 2048, 8192, "f16", 11.85, 15.19),
    (1024, 2048, 8192, "f16", 12.28, 15.59),
    (1536, 2048, 8192, "f16", 19.19, 16.29),
    (2304, 2048, 8192, "f16", 20.49, 16.86),
    (4096, 2048, 8192, "f16", 36.44, 28.95),
    (4096, 2048, 8192, "f32", 39.59, 31.46),
    (1536, 2048, 8192, "resid", 21.72, 18.35),
    (4096, 2048, 8192, "resid", 42.24, 34.01),
    (4096, 8192, 256, "f16", 16.28, 20.02),
    (4096, 8192, 512, "f16", 19.51, 21.83),
    (4096, 8192, 512, "f32", 28.43, 30.15),
    (1100, 1000, 512, "f16", 4.18, 5.98),
    (700, 5000, 700, "f16", 5.82, 6.92),
    (8192, 8192, 8192, "f16", 257.34, 203.12),
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
