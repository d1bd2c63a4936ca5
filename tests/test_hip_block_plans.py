"""The gated feed-forward block at sizes that take every way its products are cut into tiles (csrc/block/ffn_plan.h).

A form is written as the tile of the main launch ("256" 256 x 256, "192" 256 x 192, "128" 128 x 128, "128d" the same with four buffers, "64"
64 x 64), "*" where the k loop is split into shares, and behind "+" the tile of the second launch that takes the rows behind the last whole
256, if there is one.  256 x 192 is a weight gradient's tile alone.
"""
import ctypes
import os
import subprocess

import pytest
import torch

from tests.test_hip_block import check_mlp, make_mlp

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

ROWS = ["256", "256*", "256+128d*", "256+64", "256+64*", "128", "128*", "128d", "128d*", "64", "64*"]
WEIGHTS = ["256", "256*", "192", "192*", "128", "128*", "128d", "128d*", "64", "64*"]
FORMS = {"gate": ["256", "256+128d", "256+64", "128", "128d", "64"], "y": ROWS, "dh": ["256", "256+128d", "128", "128d", "64"], "dx": ROWS,
         "dw12": WEIGHTS, "dw3": WEIGHTS}
FORMS_FP32 = {**FORMS, "y": [*ROWS, "256+128*"], "dx": [*ROWS, "256+128*"]}

# M, D, H, O
SIZES_16 = [(63, 9, 8, 12), (1241, 8, 1932, 11), (16728, 96, 200, 208), (460, 439, 3049, 718), (17509, 139, 8, 1529), (6853, 83, 4554, 129),
            (3218, 543, 5138, 993), (277, 1064, 4320, 2864), (64, 2310, 2459, 1652), (8669, 2747, 67, 55), (8317, 2034, 636, 1946),
            (63, 16, 3664, 2280), (16519, 920, 136, 40), (1986, 330, 4179, 62), (7252, 56, 1151, 2268), (5448, 56, 2272, 2976), (5519, 2984, 1200, 360)]
SIZES_32 = [(87, 8, 8, 8), (4768, 8, 397, 11), (6200, 72, 696, 112), (10914, 128, 744, 168), (3681, 1122, 284, 1828), (140, 475, 3215, 1645),
            (8230, 1600, 72, 288), (8759, 277, 215, 1562), (64, 647, 2870, 843), (67, 852, 4865, 1758), (69, 1440, 4168, 2936), (18942, 232, 56, 1760),
            (3062, 56, 5672, 96), (5386, 2855, 268, 3000), (5961, 2767, 17, 81), (6600, 2424, 368, 2528), (7299, 2248, 1176, 608), (6596, 32, 2808, 2520)]

SHIM = '''
#include "ffn_plan.h"
static void put(const Plan& p, int64_t M, int64_t* o) {
    const bool two = p.main_rows < M;
    o[0] = p.shape; o[1] = p.splits; o[2] = two ? p.rest_shape : -1; o[3] = two ? p.rest_splits : 1;
}
extern "C" void plans(int64_t M, int64_t D, int64_t H, int64_t O, int es, int64_t* o) {
    const int pairs = es == 4 ? 6 : 1;
    const int64_t HP = pad8(H);
    put(gate_plan(M, HP, D, es, pairs, true), M, o);
    put(rows_plan(M, O, H, es, pairs), M, o + 4);
    put(dh_plan(M, HP, O, es, pairs), M, o + 8);
    put(rows_plan(M, D, 2 * HP, es, pairs), M, o + 12);
    put(weight_plan(2 * HP, D, M, es, pairs), 2 * HP, o + 16);
    put(weight_plan(O, H, M, es, pairs), O, o + 20);
}
'''


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    """plans(M, D, H, O, bytes of the type) -> {product: form}: the header that the launches go by, compiled by the host's compiler."""
    d = tmp_path_factory.mktemp("plans")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "iffnerf_amd", "csrc", "block"), "-o", str(d / "shim.so"),
                    str(d / "shim.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))

    def ask(M, D, H, O, es):
        out = (ctypes.c_int64 * 24)()
        lib.plans(*(ctypes.c_int64(v) for v in (M, D, H, O)), ctypes.c_int(es), out)
        tile = ["256", "192", "128", "128d", "64"]
        forms = {}
        for i, name in enumerate(FORMS):
            shape, splits, rest, rest_splits = out[4 * i:4 * i + 4]
            forms[name] = tile[shape] + "*" * (splits > 1) + ("" if rest < 0 else "+" + tile[rest] + "*" * (rest_splits > 1))
        return forms
    return ask


@pytest.mark.parametrize("sizes,es,forms", [(SIZES_16, 2, FORMS), (SIZES_32, 4, FORMS_FP32)], ids=["16 bits", "fp32"])
def test_the_sizes_take_every_form(plans, sizes, es, forms):
    taken = {name: set() for name in forms}
    for s in sizes:
        for name, form in plans(*s, es).items():
            taken[name].add(form)
    assert taken == {name: set(f) for name, f in forms.items()}


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("size", SIZES_16, ids=str)
def test_every_form_in_16_bits(size, dtype):
    check_mlp(*make_mlp(*size, dtype, True, seed=size[0]), "gelu" if size[0] % 2 else "silu")


@gpu
@pytest.mark.parametrize("size", SIZES_32, ids=str)
def test_every_form_in_fp32(size):
    check_mlp(*make_mlp(*size, torch.float32, True, seed=size[0]), "gelu" if size[0] % 2 else "silu")
