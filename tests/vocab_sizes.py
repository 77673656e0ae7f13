"""Sizes of calls of the losses over many classes that between them reach every tile of the logits, of the gradient and of the sums
(test_vocab_plan_host.py asks the library whether they do, test_gpu_vocab_tiles.py runs them): (kind, rows, features, classes, places)."""

TILES = ("large", "middle", "small", "short", "few", "quad", "small_apart", "few_apart")

SIZES = [
    # 256 x 256: several tiles in turn to a workgroup, partial ones at both edges; 8, 33 and 64 places, which no tile writes itself
    ("entropy", 4099, 1040, 7201, 1), ("distill", 4099, 1040, 7201, 40), ("distill", 2053, 1040, 13001, 33),
    # its sums: copied operands and a cut reduction; two pieces of the classes, the logits of six tiles in turn
    ("entropy", 1003, 997, 20011, 1), ("distill", 1003, 997, 20011, 64), ("entropy", 4099, 2048, 24001, 1), ("distill", 4099, 2048, 24001, 8),
    # 128 x 128 in a ring of two; lists that the tile writes and longer ones
    ("entropy", 256, 1024, 10001, 1), ("distill", 256, 1024, 10001, 32), ("distill", 300, 600, 7003, 33), ("entropy", 300, 600, 7003, 1),
    # 128 x 128 in one buffer
    ("entropy", 520, 1040, 33000, 1), ("distill", 513, 72, 33000, 33), ("entropy", 8200, 128, 4090, 1),
    # 64 x 64, and with stages of their own
    ("distill", 600, 2000, 1111, 12), ("entropy", 128, 1024, 10000, 1), ("distill", 100, 4096, 504, 40), ("entropy", 64, 2000, 300, 1),
    # up to 32 rows
    ("entropy", 16, 64, 5000, 1), ("distill", 30, 1024, 5000, 129), ("entropy", 31, 1024, 40000, 1), ("distill", 32, 96, 40000, 128),
]
