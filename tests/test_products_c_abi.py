"""Products grouped by expert and microscaled numbers at the C functions: sizes of workspaces and rows, and bad arguments,
which are refused before any device is touched."""
import os
import re

import pytest

from h2o4gpu_amd.libs import experts_hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "h2o4gpu_experts.h")
REFUSED = -2
P = 4096  # an address that nothing reads


def call(name, *args):
    return getattr(experts_hip.lib(), "h2o4gpu_" + name)(*args, None)


def test_side_matches_the_header():
    assert re.search(r"#define H2O4GPU_EXPERTS_MAX_SIDE \(1 << 20\)", open(HEADER).read())
    assert experts_hip.MAX_SIDE == 1 << 20


@pytest.mark.parametrize("cols,codes,scales", [(1, 128, 16), (256, 128, 16), (257, 256, 16), (512, 256, 16), (513, 384, 32),
                                               (8190, 4096, 256), (0, 0, 0), ((1 << 30) + 1, 0, 0)])
def test_pitches(cols, codes, scales):
    lib = experts_hip.lib()
    assert lib.h2o4gpu_microscale4_codes_pitch(cols) == codes
    assert lib.h2o4gpu_microscale4_scales_pitch(cols) == scales


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspace(dtype):
    """Whole matrices of floats, none for few rows, none where a matrix has tiles enough; 0 for bad arguments."""
    need = experts_hip.lib().h2o4gpu_experts_product_dweights_workspace
    assert need(dtype, 0, 4, 64, 64) == 0 and need(dtype, 512, 4, 64, 64) == 0
    for rows, experts, out, cols in ((513, 4, 64, 64), (100000, 2, 101, 77), (1 << 30, 600, 128, 128), (300000, 1000, 77, 101),
                                     ((1 << 31) - 65537, 1, 1, 1)):
        assert need(dtype, rows, experts, out, cols) % (4 * out * cols) == 0
        assert 0 < need(dtype, rows, experts, out, cols) <= min(4 * out * cols * 2 * 1025, 151 * 10 ** 6)
    assert need(dtype, 1 << 20, 4, 2048, 1024) == 0
    assert need(9, 100000, 2, 101, 77) == 0 and need(dtype, 100000, 0, 101, 77) == 0
    assert need(dtype, 1 << 31, 2, 101, 77) == 0 and need(dtype, 100000, 2, 0, 77) == 0


# each function's arguments that would be accepted, and what is wrong with one of them
PRODUCT = dict(dtype=1, rows=40, experts=4, out=24, cols=32, a=P, a_stride=32, w=P, apart=768, w_stride=32, offsets=P, y=P,
               y_stride=24)
WRONG = [("dtype", 3), ("dtype", -1), ("experts", 0), ("experts", 16385), ("out", 0), ("cols", 0), ("rows", 1 << 31),
         ("out", (1 << 30) + 1), ("cols", (1 << 30) + 1), ("a", None), ("w", None), ("y", None), ("offsets", None),
         ("a_stride", 23), ("w_stride", 31), ("w_stride", (1 << 23) + 1), ("y_stride", 23), ("a", P + 1), ("w", P + 1),
         ("y", P + 1)]


@pytest.mark.parametrize("what,value", WRONG, ids=["%s_%s" % w for w in WRONG])
@pytest.mark.parametrize("name", ["product", "product_drows"])
def test_products_refuse(name, what, value):
    assert call("experts_" + name, *dict(PRODUCT, **{what: value}).values()) == REFUSED


def test_nothing_to_do():
    for name in ("product", "product_drows"):
        assert call("experts_" + name, *dict(PRODUCT, rows=0, a=None, w=None, offsets=None, y=None).values()) == 0
    assert call("microscale4_quantize", 0, 0, 64, None, 64, None, None) == 0
    assert call("microscale4_dequantize", 0, 0, 64, None, None, None, 64) == 0
    assert call("microscale4_layout", 0, 64, None, 32, None, None, None) == 0
    assert call("microscale4_product", 0, 0, 8, 64, None, None, None, None, None, 8) == 0
    assert call("microscale4_experts_product", 0, 0, 2, 4, 8, 64, None, None, None, None, None, None, None, 8) == 0
    assert call("experts_align_rows", 1, 0, 5, 3, None, 0, 3, None) == 0


DWEIGHTS = dict(dtype=1, rows=1000, experts=4, out=24, cols=32, dy=P, dy_stride=24, x=P, x_stride=32, offsets=P, dw=P,
                work=P, bytes=1 << 20)
SIDE = (1 << 20) + 1
WRONG_DWEIGHTS = [("dtype", 3), ("experts", 0), ("out", 0), ("cols", 0), ("out", SIDE), ("cols", SIDE), ("rows", 1 << 31),
                  ("dy", None), ("x", None), ("dw", None), ("offsets", None), ("work", None), ("work", P + 8), ("bytes", 24 * 32 * 4),
                  ("dy_stride", 23), ("x_stride", 31), ("dy_stride", SIDE), ("x_stride", SIDE), ("dy", P + 1), ("x", P + 1),
                  ("dw", P + 1)]


@pytest.mark.parametrize("what,value", WRONG_DWEIGHTS, ids=["%s_%s" % w for w in WRONG_DWEIGHTS])
def test_gradients_of_matrices_refuse(what, value):
    assert call("experts_product_dweights", *dict(DWEIGHTS, **{what: value}).values()) == REFUSED


QUANTIZE = dict(dtype=1, rows=3, cols=64, x=P, stride=64, codes=P, scales=P)
DEQUANTIZE = dict(dtype=1, rows=3, cols=64, codes=P, scales=P, x=P, stride=64)
LAYOUT = dict(rows=3, cols=64, codes=P, stride=32, scales=P, laid=P, laid_scales=P)
ALIGN = dict(dtype=1, matrices=2, rows=3, cols=7, x=P, matrix=21, stride=7, out=P)


@pytest.mark.parametrize("name,args,what,value", [
    (name, args, what, value) for name, args, wrong in (
        ("microscale4_quantize", QUANTIZE, [("dtype", 3), ("cols", 0), ("cols", (1 << 30) + 1), ("rows", 1 << 50), ("x", None),
                                            ("stride", 63), ("codes", P + 8), ("scales", P + 8), ("scales", None), ("x", P + 1)]),
        ("microscale4_dequantize", DEQUANTIZE, [("dtype", 3), ("cols", 0), ("rows", 1 << 50), ("codes", None), ("codes", P + 4),
                                                ("stride", 63), ("x", P + 1), ("x", None)]),
        ("microscale4_layout", LAYOUT, [("cols", 0), ("rows", 1 << 50), ("stride", 31), ("codes", None), ("laid", P + 4),
                                        ("laid_scales", P + 4), ("laid", None)]),
        ("experts_align_rows", ALIGN, [("dtype", 3), ("cols", 0), ("matrices", 1 << 31), ("rows", 1 << 31), ("x", None),
                                       ("out", P + 8), ("x", P + 1), ("out", None)]))
    for what, value in wrong])
def test_numbers_refuse(name, args, what, value):
    assert call(name, *dict(args, **{what: value}).values()) == REFUSED


FOUR = dict(dtype=1, rows=5, out=8, cols=64, x=P, xs=P, w=P, ws=P, y=P, y_stride=8)
FOURS = dict(dtype=1, tokens=5, top_k=2, experts=4, out=8, cols=64, x=P, xs=P, w=P, ws=P, order=P, offsets=P, y=P, y_stride=8)
SHARED = [("dtype", 3), ("out", 0), ("cols", 0), ("x", None), ("xs", None), ("w", None), ("ws", None), ("y", None),
          ("y_stride", 7), ("x", P + 8), ("xs", P + 8), ("w", P + 8), ("ws", P + 8), ("y", P + 1)]


@pytest.mark.parametrize("what,value", SHARED + [("rows", 1 << 31)])
def test_microscaled_product_refuses(what, value):
    assert call("microscale4_product", *dict(FOUR, **{what: value}).values()) == REFUSED


@pytest.mark.parametrize("what,value", SHARED + [("tokens", 1 << 30), ("tokens", 1 << 40), ("top_k", 0), ("top_k", 65),
                                                 ("experts", 0), ("experts", 16385), ("offsets", None)])
def test_microscaled_products_of_experts_refuse(what, value):
    assert call("microscale4_experts_product", *dict(FOURS, **{what: value}).values()) == REFUSED
