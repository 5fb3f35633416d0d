"""Sizes of the mixture-of-experts layer by the way in which its products are made: (tokens, experts, top_k, cols, inner,
type of x) with rows of whole steps of 256 values and not."""

INNER = ("16 rows", "64 rows", "stream 2", "stream 4")
OUTER = ("sums of 1", "sums of 2", "64 rows", "chunks")

SIZES = {  # inner products, outer products, whether the choice is a launch of its own
    (1, 6, 2, 2080, 352, "bf16"): ("16 rows", "sums of 1", False),
    (1, 40, 3, 96, 2016, "f32"): ("16 rows", "sums of 1", False),
    (2, 5, 2, 512, 480, "f16"): ("16 rows", "sums of 2", False),
    (2, 6, 4, 320, 2528, "bf16"): ("16 rows", "chunks", False),
    (1, 8, 3, 480, 6048, "bf16"): ("64 rows", "chunks", False),
    (1, 64, 32, 64, 512, "bf16"): ("64 rows", "sums of 1", False),
    (2, 20, 20, 2048, 96, "f32"): ("64 rows", "sums of 2", True),
    (2, 4, 2, 2336, 736, "bf16"): ("stream 2", "sums of 2", False),
    (2, 4, 2, 4128, 736, "f16"): ("stream 4", "sums of 2", False),
    (3, 9, 2, 352, 1056, "bf16"): ("16 rows", "64 rows", False),
    (4, 3, 3, 416, 4128, "bf16"): ("16 rows", "chunks", False),
    (7, 11, 3, 1120, 1504, "f16"): ("64 rows", "64 rows", False),
    (9, 7, 2, 1056, 544, "f32"): ("64 rows", "64 rows", True),
    (33, 5, 2, 640, 1248, "bf16"): ("64 rows", "64 rows", True),
    (33, 3, 2, 640, 1248, "bf16"): ("64 rows", "chunks", True),
    (20, 40, 4, 1184, 1312, "bf16"): ("64 rows", "chunks", True),
    (5, 6, 3, 2112, 1120, "f32"): ("stream 2", "64 rows", False),
    (30, 4, 2, 3008, 992, "bf16"): ("stream 2", "64 rows", True),
    (64, 3, 2, 1120, 832, "bf16"): ("stream 2", "chunks", True),
    (21, 6, 2, 2144, 3232, "f32"): ("stream 2", "chunks", True),
    (6, 4, 2, 4320, 2336, "bf16"): ("stream 4", "chunks", False),
    (17, 6, 2, 8160, 608, "f16"): ("stream 4", "64 rows", True),
    (40, 3, 2, 5056, 2400, "bf16"): ("stream 4", "chunks", True),
    (64, 2, 1, 96, 14336, "bf16"): ("64 rows", "chunks", True),
    (10, 2, 1, 96, 32800, "bf16"): ("64 rows", "64 rows", True),
    (10, 2, 1, 8224, 96, "bf16"): ("64 rows", "64 rows", True),
}
