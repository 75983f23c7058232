"""Calls of the 8-bit floating-point products by the kernel that takes them: tests/test_fp8_forms.py holds the rules to these on the
CPU, tests/test_gpu_fp8_forms.py runs them, so that a rule that changes cannot leave a kernel untested unnoticed.

A form is (tile, parts) of the tiles and (rows, strips, waves) of the few-rows kernel; tiles of 256 are for bf16 outputs, others take
128 there."""

# (m, n, k) -> form. The last column tile is cut between its waves' columns.
CUT_TILES = [((300, 3000, 384), (64, 1)), ((1500, 4168, 136), (128, 1)), ((3000, 8376, 136), (256, 1))]

# (m, n, k) -> form: as many rows, strips and waves as there are.
ROWS = [((20, 200, 640), (16, 1, 2)), ((16, 256, 4096), (16, 1, 4)), ((6, 2000, 5000), (16, 1, 8)), ((3, 1000, 12288), (16, 1, 16)),
        ((1, 40, 8192), (16, 1, 8)), ((1, 70000, 128), (16, 2, 4)), ((12, 66000, 200), (16, 2, 4)), ((17, 5000, 384), (32, 2, 8)),
        ((32, 9000, 300), (32, 2, 4))]

# (m, n, k) -> form: the inner axis in parts
PARTS = [((64, 1024, 8192), (64, 8)), ((70, 1001, 6000), (64, 8)), ((130, 2000, 3000), (64, 4))]

# (rows of each expert, n, k) -> form, with AROUND rows of d more that no expert has
AROUND = 42
GROUPED = [([1, 2, 0, 3] * 32, 1100, 384, (16, 2, 4)), ([9, 20, 30, 1] * 8, 600, 384, (32, 2, 4)), ([33, 0, 70, 1] * 16, 1000, 384, (64, 1)),
           ([600, 0, 1200, 513] * 2 + [257, 1, 300], 4100, 136, (128, 1)), ([600, 1200, 0, 900, 257, 700] * 4, 4200, 136, (256, 1))]

# a rank's quarter of the experts: (tokens, active, routed, experts, n, k) -> form, by the rows that there may be
SHARES = [(600, 4, 64, 16, 1000, 384, (64, 1)), (3000, 4, 32, 8, 4200, 136, (256, 1))]
