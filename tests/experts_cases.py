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


def all_cases():
    cases = _sort() + _route() + _rows() + _product() + _experts_product() + _quantize()
    cases += [dict(op=name) for name in ("differences_route", "differences_rows", "refusals", "graph", "other_stream",
                                         "broadcast_gradients", "unwanted_places", "fitted_codebook", "far_rows",
                                         "repeats", "long_cache", "c_refusals", "example")]
    for i, c in enumerate(cases):
        c["name"] = "%03d_%s" % (i, "_".join(str(v) for v in c.values()))
    return cases
