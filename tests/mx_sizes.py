"""Sizes of the product with MXFP4 weights, by the kernel that they reach: (tokens, rows, cols), each over several steps
of a row (128 values) with a row's end inside one, and tokens and rows that no tile divides."""

SMALL, FEW, TILES = "small", "few", "tiles"


def few(tokens):
    return (FEW, tokens)


def tile(rows, ct, rg, kg):
    """Rows of a wavefront, 32-token columns, groups of rows, groups that share the length of the rows."""
    return (TILES, rows, ct, rg, kg)


_SIXTEEN = {  # bf16, f16, and e4m3 where it has no kernel of its own
    (100, 131, 352): (SMALL,),
    (1, 131, 1184): few(1),
    (1, 9001, 1184): tile(32, 1, 1, 4),
    (13, 9001, 2208): tile(32, 1, 1, 4),
    (20, 131, 2208): tile(32, 1, 1, 8),
    (70, 131, 3232): tile(32, 1, 1, 8),
    (40, 5001, 2208): tile(64, 1, 1, 8),
    (200, 5001, 1184): tile(64, 1, 1, 4),
    (30, 16500, 1184): tile(64, 1, 1, 4),
    (301, 1001, 224): tile(32, 1, 1, 1),
    (700, 3001, 256): tile(64, 1, 1, 1),
    (640, 4099, 672): tile(64, 2, 4, 1),
    (1290, 4110, 416): tile(64, 4, 4, 1),
}

SIZES = {
    "bf16": _SIXTEEN,
    "f16": {**_SIXTEEN, (1290, 4110, 416): tile(64, 2, 4, 1)},
    "e4m3": {**_SIXTEEN, (200, 5001, 1184): tile(64, 2, 1, 4)},
    "f32": {
        (100, 131, 352): (SMALL,),
        (1, 9001, 1184): few(1),
        (2, 131, 1184): few(2),
        (3, 131, 1184): few(4),
        (20, 131, 2208): tile(32, 1, 1, 4),
        (40, 5001, 1184): tile(64, 1, 1, 4),
        (70, 9001, 672): tile(64, 1, 1, 4),
        (640, 4099, 416): tile(64, 1, 4, 1),
    },
}


# A product whose operands may lie as far apart as a tile's 32-bit offsets reach: the rows of each that one tile takes.
FAR = (20, 40, 2208)
FAR_COUNTS = {"x": 20, "x_scales": 20, "weight": 32, "scales": 32}


def far_stride(operand, size):
    """The largest stride, in elements of `size` bytes, with which a tile's rows and 512 bytes more lie within 2^32."""
    return (2**32 - 1 - 512) // size // (FAR_COUNTS[operand] - 1)
