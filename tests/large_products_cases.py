"""The cases of test_gpu_large_products.py: products that the rules send to pipe_kernel's tiles, and which of these each
pass takes (forward, rows' gradient, matrices' gradient); and numbers into 4 bits. Plain values, so that the collecting process needs no torch."""

HALVES = ("bfloat16", "float16")

# (tokens, top_k, experts, out, cols, most rows to one expert, the passes' tiles); five stages and more, ends inside tiles,
# stages and pieces, an expert without rows and slots without an expert, more tiles than workgroups
_SIXTEEN = (
    (4500, 2, 7, 1500, 2010, False, ("256", "256", "256")),
    (10000, 2, 5, 1500, 1002, False, ("256", "256", "128")),
    (9000, 1, 16, 1000, 1000, True, ("256", "256", "256")),  # parts of a gradient, in large tiles
    (50000, 4, 1030, 512, 512, False, ("256", "256", "256")),  # more experts than the table in LDS holds
    (1500, 1, 3, 700, 520, False, ("128", "128", "128")),
    (1500, 1, 3, 1500, 1600, False, ("128", "128", "128")),
    (1100, 2, 5, 392, 650, True, ("128", "128", "128")),
)
_FLOAT32 = (
    (4500, 2, 7, 1500, 1501, False, ("256", "256", "256")),
    (9000, 1, 16, 1000, 1000, True, ("128", "128", "128")),
    (2048, 2, 4, 2049, 2047, False, ("128", "128", "128")),
    (3000, 1, 3, 701, 520, False, ("128", "128", "128")),
    (25000, 4, 1030, 513, 333, False, ("128", "128", "128")),
)

# (rows, out, cols, tiles): one 4-bit matrix; a stage is 256 columns: odd and even numbers of them
_FOUR = (
    (1000, 2000, 1100, "128"), (1000, 2000, 1500, "128"), (900, 2501, 3900, "128"), (1111, 1777, 1024, "128"),
    (4000, 4000, 1100, "256"), (4000, 4000, 1500, "256"), (8200, 4100, 1300, "256"), (8200, 4099, 1100, "256"),
    (8200, 4100, 200, "256"), (8200, 4100, 700, "256"),
)
# (tokens, top_k, experts, out, cols, tiles)
_FOURS = (
    (300, 3, 7, 2000, 1100, "128"), (300, 3, 7, 2001, 1500, "128"), (4000, 3, 7, 2000, 1100, "256"),
    (4000, 3, 7, 2001, 1500, "256"), (4000, 3, 7, 2000, 700, "256"), (50000, 4, 1030, 512, 600, "256"),
    (140000, 1, 1030, 136, 72, "256"),
)
DROPPED = 0.07


def all_cases():
    cases = []
    for sizes, types in ((_SIXTEEN, HALVES), (_FLOAT32, ("float32",))):
        for tokens, top_k, experts, out, cols, most, ways in sizes:
            for dtype in types:
                cases.append(dict(op="large", tokens=tokens, top_k=top_k, experts=experts, out=out, cols=cols, dtype=dtype,
                                  most=most, ways=list(ways)))
    for i, (rows, out, cols, way) in enumerate(_FOUR):
        cases.append(dict(op="large_four", rows=rows, out=out, cols=cols, dtype=(HALVES + ("float32",))[i % 3], ways=[way]))
    for i, (tokens, top_k, experts, out, cols, way) in enumerate(_FOURS):
        for in_order in (False, True):
            cases.append(dict(op="large_fours", tokens=tokens, top_k=top_k, experts=experts, out=out, cols=cols, most=False,
                              dtype=(HALVES + ("float32",))[(i + in_order) % 3], in_order=in_order, ways=[way]))
    cases.append(dict(op="rows_of_any_stride", ways=[]))
    for i, c in enumerate(cases):
        c["name"] = "%02d_%s" % (i, "_".join(str(v) for k, v in c.items() if k != "ways"))
    return cases
