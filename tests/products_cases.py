"""The cases of test_gpu_products.py: plain values, so that the collecting process needs no torch.
products_device_check.py runs them."""

TYPES = ("float32", "bfloat16", "float16")
LAYOUTS = ("plain", "strided", "unaligned")

# (tokens, top_k, experts, out, cols): one of everything, odd sizes, sizes around a tile's, more experts than rows,
# rows that are no whole piece of 16 bytes, long sums, many rows of few experts
RAGGED = (
    (1, 1, 1, 1, 1), (1, 2, 16, 100, 256), (3, 2, 5, 7, 5), (17, 1, 3, 33, 31), (1, 4, 4, 17, 1000), (64, 4, 3, 33, 96),
    (40, 3, 8, 64, 512), (3, 8, 300, 16, 64), (200, 2, 6, 48, 160), (33, 6, 64, 20, 2050), (300, 1, 2, 130, 129),
    (257, 2, 2, 255, 257), (500, 2, 7, 129, 65), (1000, 1, 3, 257, 200), (128, 1, 1, 128, 64), (2000, 1, 1, 300, 72),
    (900, 3, 4, 96, 384), (31, 2, 2, 520, 4104), (5000, 1, 5, 24, 40), (20, 1, 4100, 8, 33), (140000, 1, 1030, 136, 72),
    # more rows than a gradient's part, parts that end inside tiles, large tiles that end inside matrices and stages
    (3001, 2, 3, 136, 264), (1500, 2, 2, 520, 1032), (700, 4, 5, 256, 512), (1100, 2, 7, 384, 136), (2500, 2, 1, 128, 128),
    (9000, 1, 2300, 16, 24), (90, 1, 3, 1100, 300), (40, 2, 4, 513, 129), (7, 1, 2, 65, 1000), (100, 4, 20, 128, 40), (2600, 2, 4, 200, 128), (900, 1, 3, 1000, 72), (300, 1, 1, 264, 2056),
)

# rows that begin at words and no more (cols % 8 = 2), narrow matrices, an expert of many parts, more experts than a table
# in LDS holds, few rows with large matrices
WORDS = ((701, 1, 3, 2002, 330), (702, 1, 3, 2002, 330), (21000, 1, 2, 18, 34), (30000, 1, 2, 30, 22), (170, 1, 3, 40, 50),
         (21, 1, 4, 264, 130), (3000, 1, 1030, 136, 130))


def _words():
    out = [dict(op="product", tokens=tokens, top_k=top_k, experts=experts, out=n, cols=cols, dtype=dtype, dropped=0.1,
                layout=LAYOUTS[(tokens + n) % 3], data="normal") for tokens, top_k, experts, n, cols in WORDS for dtype in TYPES]
    return out + [dict(op="product", tokens=9000, top_k=1, experts=520, out=20, cols=30, dtype=dtype, dropped=0.0,
                       layout="plain", data="one_expert") for dtype in TYPES]


def _products():
    out = []
    for i, (tokens, top_k, experts, n, cols) in enumerate(RAGGED):
        for dtype in TYPES:
            out.append(dict(op="product", tokens=tokens, top_k=top_k, experts=experts, out=n, cols=cols, dtype=dtype,
                            dropped=(0.0, 0.3)[i % 2], layout=LAYOUTS[(tokens + n) % 3], data="normal"))
    for data in ("nothing", "one_expert", "infinity", "nan_behind"):
        for dtype in TYPES:
            for tokens, top_k, experts, n, cols in ((40, 2, 5, 24, 40), (300, 2, 4, 136, 200), (2100, 1, 3, 130, 40),
                                                    (1300, 2, 3, 128, 192)):
                out.append(dict(op="product", tokens=tokens, top_k=top_k, experts=experts, out=n, cols=cols, dtype=dtype,
                                dropped=0.4 if data == "nan_behind" else 0.0, layout="plain", data=data))
    return out


def _quantize():
    return [dict(op="quantize", rows=rows, cols=cols, dtype=dtype, layout=LAYOUTS[(rows + cols) % 3], data=data)
            for rows, cols in ((1, 1), (3, 31), (5, 33), (2, 256), (7, 257), (40, 512), (9, 1000), (130, 520))
            for dtype in TYPES for data in ("normal", "wide", "ties", "tiny", "zeros", "not_finite")]


def _fours():
    out = []
    for i, (rows, n, cols) in enumerate(((1, 1, 1), (1, 40, 33), (1, 300, 4096), (2, 17, 100), (5, 64, 256), (16, 128, 512), (17, 33, 513),
                                         (33, 200, 777), (64, 96, 1024), (65, 40, 2176), (130, 24, 520), (128, 128, 768),
                                         (200, 130, 260), (300, 520, 96), (260, 257, 1300), (1, 8, 9000), (600, 700, 288),
                                         (513, 384, 1536), (1030, 129, 2560), (128, 4000, 128),
                                         (33, 4100, 777), (64, 4096, 8192), (20, 5000, 500), (47, 4099, 2100), (17, 4097, 7700),
                                         (60, 9000, 33))):
        for dtype in TYPES:
            out.append(dict(op="four", rows=rows, out=n, cols=cols, dtype=dtype, made=("quantize", "codes")[i % 2]))
    return out


def _fours_of_experts():
    out = []
    for i, (tokens, top_k, experts, n, cols) in enumerate(RAGGED):
        for dtype in (TYPES[i % 3], TYPES[(i + 1) % 3]):
            for in_order in (False, True):
                out.append(dict(op="four_experts", tokens=tokens, top_k=top_k, experts=experts, out=n, cols=cols,
                                dtype=dtype, dropped=(0.0, 0.3, 1.0)[(i + in_order) % 3], in_order=in_order))
    return out


CHECKS = ("differences", "broadcast", "graph", "graph_of_training", "other_stream", "repeats", "two_layers", "codes_back",
          "far_rows", "refusals", "c_refusals", "second_derivatives", "one_gradient", "empty", "not_finite_products",
          "labels", "example")


def all_cases():
    cases = _products() + _quantize() + _fours() + _fours_of_experts()
    cases += [dict(op=name) for name in CHECKS] + _words() + [dict(op="broadcast_between_words"), dict(op="two_at_once")]
    for i, c in enumerate(cases):
        c["name"] = "%03d_%s" % (i, "_".join(str(v) for v in c.values()))
    return cases
