"""The cases of test_gpu_experts.py: plain values, so that the collecting process needs no torch.
experts_device_check.py runs them."""

TYPES = ("float32", "bfloat16", "float16")


def _route():
    out = []
    # (rows, experts, top_k): one of everything, powers of two and their neighbours, more experts than a
    # wavefront's lanes can hold in registers, top_k of all experts
    for rows, experts, top_k in ((1, 1, 1), (1, 8, 2), (3, 7, 7), (65, 64, 1), (64, 65, 4), (130, 16, 16), (33, 100, 3),
                                 (257, 129, 8), (100, 256, 8), (19, 257, 9), (17, 1000, 2), (9, 1025, 64),
                                 (5, 4099, 5), (2, 16384, 33), (1000, 8, 2), (77, 33, 17), (5000, 12, 4)):
        for dtype in TYPES:
            for largest in (True, False):
                for over_all in (False, True):
                    # strided: 0 contiguous rows, 1 one expert's scores side by side, 2 gaps in both directions
                    strided = (rows + experts + largest + 2 * over_all) % 3
                    out.append(dict(op="route", rows=rows, experts=experts, top_k=top_k, dtype=dtype,
                                    largest=largest, over_all=over_all, strided=strided, data="normal"))
    for data in ("ties", "masked", "all_masked", "lowest", "nan", "best_infinity", "wide", "scale0"):
        for dtype in TYPES:
            for over_all in (False, True):
                for rows, experts, top_k, strided in ((40, 9, 4, 0), (70, 64, 8, 1), (21, 300, 5, 0), (300, 10, 2, 1),
                                                      (11, 2000, 6, 2)):
                    out.append(dict(op="route", rows=rows, experts=experts, top_k=top_k, dtype=dtype,
                                    largest=(rows + over_all) % 2 == 0, over_all=over_all, strided=strided, data=data))
    return out


def _rows():
    out = []
    for op in ("dispatch", "combine"):
        for tokens, top_k, experts, cols in ((1, 1, 1, 1), (1, 2, 8, 64), (2, 3, 5, 7), (16, 2, 8, 4096), (33, 5, 3, 101),
                                             (64, 8, 64, 129), (100, 1, 1000, 33), (257, 4, 16, 515), (500, 7, 40, 24),
                                             (31, 64, 100, 66), (1200, 9, 6, 8), (70, 3, 12, 2056), (40, 17, 30, 1030)):
            for dtype in TYPES:
                for layout in ("plain", "strided", "unaligned"):
                    out.append(dict(op=op, tokens=tokens, top_k=top_k, experts=experts, cols=cols, dtype=dtype,
                                    layout=layout, dropped=(0.0, 0.2, 1.0)[(tokens + cols + len(layout)) % 3]))
    return out


def _sort():
    out = []
    for tokens, top_k, experts in ((0, 2, 3), (1, 1, 1), (5, 2, 1), (63, 1, 4), (64, 1, 64), (65, 2, 65), (1000, 8, 256),
                                   (4096, 2, 7), (8193, 1, 50), (3001, 3, 2047), (3000, 2, 2048), (9000, 4, 5000),
                                   (700, 2, 16384), (100_003, 3, 1000), (70_000, 1, 1), (300_000, 2, 64),
                                   (12_000, 8, 16384), (1_000_001, 2, 64)):
        for data in ("uniform", "skewed", "dropped", "none", "one"):
            out.append(dict(op="sort", tokens=tokens, top_k=top_k, experts=experts, data=data))
    return out


def _product():
    out = []
    for rows, n, cols, group in ((0, 5, 40, 32), (1, 1, 1, 32), (1, 16, 32, 32), (1, 17, 33, 32), (1, 100, 130, 64),
                                 (1, 256, 4096, 128), (2, 48, 127, 96), (3, 33, 4097, 128), (4, 64, 1000, 32),
                                 (5, 70, 513, 256), (8, 130, 96, 32), (15, 31, 2048, 64), (16, 64, 640, 160),
                                 (17, 65, 300, 128), (33, 200, 777, 64), (64, 96, 1024, 1024), (65, 40, 2176, 128),
                                 (130, 24, 520, 32), (1, 8, 9000, 4096), (200, 130, 260, 128), (31, 1000, 64, 64)):
        for dtype in TYPES:
            out.append(dict(op="product", rows=rows, out=n, cols=cols, group=group, dtype=dtype,
                            scale_dtype=TYPES[(rows + cols + n) % 3] if n % 2 else dtype,
                            layout=("plain", "strided", "unaligned")[(rows + n) % 3]))
    return out


def _experts_product():
    out = []
    for tokens, top_k, experts, n, cols, group in ((1, 1, 1, 5, 33, 32), (1, 2, 16, 100, 256, 32), (1, 4, 4, 17, 1000, 128),
                                                   (7, 2, 5, 40, 130, 64), (40, 3, 8, 64, 512, 128),
                                                   (64, 4, 3, 33, 96, 32), (3, 8, 300, 16, 64, 32),
                                                   (200, 2, 6, 48, 160, 64), (33, 6, 64, 20, 2050, 96),
                                                   (300, 1, 2, 70, 128, 128)):
        for dtype in TYPES:
            for dropped in (0.0, 0.3, 1.0):
                out.append(dict(op="experts_product", tokens=tokens, top_k=top_k, experts=experts, out=n, cols=cols,
                                group=group, dtype=dtype, dropped=dropped, books=(tokens + n) % 2 == 0,
                                layout=("plain", "strided", "unaligned")[(tokens + top_k) % 3]))
    return out


def _quantize():
    return [dict(op="quantize", out=n, cols=cols, group=group, dtype=dtype, scale_dtype=sdt, data=data)
            for n, cols, group in ((1, 1, 32), (5, 33, 32), (40, 200, 64), (9, 1000, 128))
            for dtype, sdt in (("float32", "float32"), ("bfloat16", "float16"), ("float16", "bfloat16"))
            for data in ("normal", "zeros", "huge", "nan")]


# (rows, out, cols, group): together every shape that a product's tiles take, with teams of one to eight wavefronts.
PRODUCTS = (
    (10, 259, 258, 128), (5, 268, 517, 128), (15, 258, 518, 64), (6, 264, 525, 32), (336, 1548, 37, 128),
    (401, 625, 155, 128), (230, 276, 513, 128), (373, 1309, 55, 64), (379, 321, 259, 64),
    (243, 261, 518, 64), (472, 1039, 37, 32), (293, 419, 270, 32), (211, 303, 517, 32),
    (463, 2115, 83, 128), (401, 1183, 130, 128), (369, 333, 515, 128), (474, 2110, 46, 64),
    (475, 544, 277, 64), (305, 390, 524, 64), (405, 2320, 42, 32), (453, 515, 336, 32), (470, 264, 517, 32),
    (401, 2590, 38, 128), (455, 527, 279, 128), (425, 2331, 36, 64), (465, 1028, 171, 64),
    (353, 1418, 131, 32), (456, 3276, 40, 128), (398, 1924, 139, 128), (405, 439, 787, 128),
    (451, 3171, 34, 64), (468, 780, 409, 64), (411, 449, 780, 64), (313, 6155, 43, 128),
    (338, 1424, 284, 128), (408, 596, 518, 128), (473, 4173, 41, 64), (452, 2084, 206, 64),
    (469, 517, 536, 64), (451, 3081, 64, 32), (414, 1846, 142, 32), (382, 665, 519, 32),
    (436, 4609, 34, 128), (408, 2554, 134, 128), (413, 615, 561, 128), (327, 6305, 35, 64),
    (500, 1049, 261, 64), (370, 677, 547, 64), (400, 7545, 47, 128), (404, 1957, 284, 128),
    (393, 949, 680, 128), (331, 9143, 130, 128), (178, 8083, 158, 128), (428, 871, 747, 128),
    (419, 6915, 359, 64), (367, 2038, 281, 64), (417, 867, 730, 64),
)

# (tokens, top_k, experts, out, cols, group): the same, and the last ones with more tiles than are counted.
EXPERTS_PRODUCTS = (
    (8, 1, 2, 266, 533, 128), (9, 1, 2, 259, 298, 32), (270, 1, 2, 277, 527, 128), (301, 2, 3, 815, 33, 64),
    (129, 3, 2, 318, 281, 32), (437, 1, 3, 270, 713, 128), (280, 3, 2, 1033, 49, 64),
    (225, 3, 2, 340, 331, 32), (196, 3, 2, 270, 530, 128), (193, 3, 2, 403, 283, 32),
    (162, 3, 2, 409, 806, 128), (412, 2, 2, 1575, 38, 64), (425, 2, 2, 280, 578, 128),
    (358, 3, 2, 1627, 67, 64), (280, 3, 2, 428, 419, 32), (251, 3, 2, 381, 564, 128),
    (424, 3, 3, 1671, 50, 64), (458, 3, 3, 260, 535, 128), (399, 2, 3, 447, 765, 128),
    (485, 2, 3, 3000, 47, 64), (300, 3, 100, 700, 130, 128), (310, 2, 200, 350, 300, 64),
    (500, 2, 25, 2640, 200, 64), (400, 2, 40, 1700, 260, 64), (600, 3, 70, 1000, 130, 128),
    (600, 3, 70, 1000, 264, 32), (700, 1, 100, 690, 33, 32), (300, 2, 300, 230, 70, 64),
)


def _shapes():
    out = []
    for rows, n, cols, group in PRODUCTS:
        for dtype in TYPES:
            out.append(dict(op="product", rows=rows, out=n, cols=cols, group=group, dtype=dtype,
                            scale_dtype=TYPES[(rows + cols + n) % 3] if n % 2 else dtype,
                            layout=("plain", "strided", "unaligned")[(rows + n) % 3]))
    for i, (tokens, top_k, experts, n, cols, group) in enumerate(EXPERTS_PRODUCTS):
        for dtype in TYPES:
            out.append(dict(op="experts_product", tokens=tokens, top_k=top_k, experts=experts, out=n, cols=cols,
                            group=group, dtype=dtype, dropped=(0.0, 0.3)[i % 2], books=(tokens + n) % 2 == 0,
                            layout=("plain", "strided", "unaligned")[(tokens + top_k) % 3]))
    return out


def all_cases():
    cases = _sort() + _route() + _rows() + _product() + _experts_product() + _quantize()
    cases += [dict(op=name) for name in ("differences_route", "differences_rows", "refusals", "graph", "other_stream",
                                         "broadcast_gradients", "unwanted_places", "fitted_codebook", "far_rows",
                                         "repeats", "long_cache", "c_refusals", "example")]
    cases += _shapes()
    for i, c in enumerate(cases):
        c["name"] = "%03d_%s" % (i, "_".join(str(v) for v in c.values()))
    return cases
