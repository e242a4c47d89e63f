"""Which kernel takes a product (csrc/product_rules.h), on the CPU: the sizes named beside the rules go where these say
that they are fast."""
import pytest

from product_rules import Rules


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    return Rules(str(tmp_path_factory.mktemp("product_rules")))


@pytest.mark.parametrize("kind,dtype,rows,experts,out,cols,way", [
    ("forward", "bfloat16", 16, 8, 7168, 4096, "few rows"), ("forward", "bfloat16", 27 * 24, 27, 5184, 2504, "128"),
    ("forward", "float32", 27 * 40, 27, 5184, 2504, "few rows"), ("forward", "float16", 200, 1, 2048, 8192, "few rows"),
    ("forward", "float16", 400, 1, 2048, 8192, "128"), ("forward", "bfloat16", 65536, 64, 2048, 2048, "256"),
    ("forward", "bfloat16", 8000, 4, 512, 1024, "128"), ("forward", "float32", 64000, 16, 64, 2048, "any rows"),
    ("forward", "bfloat16", 64000, 64, 16, 640, "128"), ("forward", "bfloat16", 28800, 300, 777, 1001, "any rows"),
    ("drows", "bfloat16", 8 * 24, 8, 4096, 4096, "128"), ("drows", "float32", 8 * 48, 8, 4096, 4096, "few rows"),
    ("drows", "bfloat16", 65536, 64, 2048, 2048, "256"), ("dweights", "bfloat16", 65536, 64, 2048, 2048, "256"),
    ("dweights", "float32", 8 * 24, 8, 4096, 4096, "any rows"), ("dweights", "float32", 8 * 48, 8, 4096, 4096, "256"),
    ("dweights", "float32", 300000, 1000, 77, 101, "any rows"), ("dweights", "bfloat16", 16, 8, 4096, 4096, "256"),
])
def test_way(rules, kind, dtype, rows, experts, out, cols, way):
    assert rules.way(kind, dtype, rows, experts, out, cols) == way


@pytest.mark.parametrize("rows,out,cols,experts,gathered,way", [
    (1, 4096, 4096, 0, 0, "few rows"), (33, 11003, 8190, 0, 0, "kept"), (64, 2048, 4096, 0, 0, "kept"),
    (17, 16, 512, 0, 0, "kept"), (16, 4096, 4096, 0, 0, "few rows"), (65, 2048, 4096, 0, 0, "few rows"),
    (33, 4096, 8193, 0, 0, "few rows"), (33, 2048, 4096, 4, 33, "few rows"),
    (800, 2048, 8192, 0, 0, "128"), (8192, 8192, 8192, 0, 0, "256"), (256, 2048, 4096, 64, 64, "few rows"),
    (65536, 4096, 2048, 64, 16384, "256"), (1 << 23, 4096, 2048, 64, 1 << 23, "few rows"),
])
def test_way_of_four(rules, rows, out, cols, experts, gathered, way):
    assert rules.way_four(rows, out, cols, experts, gathered) == way


def test_parts(rules):
    assert rules.part("bfloat16", 100000, 2, 102, 102) == 512 and rules.part("bfloat16", 96000, 16, 256, 256) == 1152
    assert rules.part("bfloat16", 3200, 32, 1024, 1024) == 4096 and rules.part("float32", 3200, 32, 1024, 1024) == 2048
    assert rules.part("float32", 64000, 16, 2048, 64) == 1024 and rules.part("bfloat16", 1 << 20, 1, 2048, 1024) == 2 ** 31 - 1


@pytest.mark.parametrize("kind,rows,experts,out,cols,way", [
    ("forward", 4096, 4, 2048, 2048, "128"), ("drows", 4096, 4, 2048, 2048, "128"), ("forward", 8192, 16, 1024, 1024, "128"),
    ("forward", 6000, 8, 1536, 768, "128"), ("forward", 20000, 4, 640, 640, "256"), ("drows", 20000, 4, 640, 640, "256"),
    ("forward", 20000, 32, 768, 1536, "128"), ("dweights", 16384, 8, 512, 2048, "128"), ("dweights", 8192, 16, 1024, 1024, "128"),
    ("dweights", 4096, 1, 4096, 4096, "256"), ("dweights", 65536, 64, 1024, 1024, "128"),
])
def test_tiles_of_float32(rules, kind, rows, experts, out, cols, way):
    """A tile of float32 takes its operations' time, whether a CU has another or not."""
    assert rules.way(kind, "float32", rows, experts, out, cols) == way


@pytest.mark.parametrize("kind", ["forward", "drows", "dweights"])
def test_float32_always_begins_at_words(rules, kind):
    """Matrices of an odd number of elements go where even ones do: 4 bytes are a word."""
    for experts, rows in ((4, 4 * 64), (4, 4000), (300, 300 * 100)):
        assert rules.way(kind, "float32", rows, experts, 2049, 2047) == rules.way(kind, "float32", rows, experts, 2049, 2048)
        assert rules.way(kind, "bfloat16", rows, experts, 2049, 2047) == "any rows"


@pytest.mark.parametrize("kind", ["forward", "drows"])
def test_distance_of_one_matrix_is_nothing(rules, kind):
    """How far the next matrix would be is asked where there is one."""
    far = 2050 * 2048 + 1
    assert rules.way(kind, "bfloat16", 4000, 1, 2050, 2048, apart=far) == rules.way(kind, "bfloat16", 4000, 1, 2050, 2048)
    assert rules.way(kind, "bfloat16", 4000, 2, 2050, 2048, apart=far) == "any rows"


def test_one_matrix_is_not_copied_for_its_distance():
    import torch
    from h2o4gpu_amd import experts
    one = torch.zeros(200 * 128 + 1, dtype=torch.bfloat16).as_strided((1, 200, 128), (200 * 128 + 1, 128, 1))
    two = torch.zeros(2 * 200 * 128 + 1, dtype=torch.bfloat16).as_strided((2, 200, 128), (200 * 128 + 1, 128, 1))
    assert experts._at_words(one) and not experts._at_words(two)
    assert experts._at_words(torch.zeros(2, 3, 5)) and not experts._at_words(torch.zeros(2, 3, 5, dtype=torch.float16))


@pytest.mark.parametrize("rows,experts,out,cols", [(16384, 8, 1025, 1023), (16384, 8, 512, 2048), (8192, 16, 1024, 1024),
                                                   (65536, 64, 1024, 1024), (20000, 4, 640, 640)])
def test_parts_of_float32_are_taken_in_small_tiles(rules, rows, experts, out, cols):
    assert rules.part("float32", rows, experts, out, cols) < rows
    assert rules.way("dweights", "float32", rows, experts, out, cols) == "128"
