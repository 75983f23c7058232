"""Calls of the 8-bit floating-point products by the kernel that takes them: tests/test_fp8_forms.py holds the rules to these on the
CPU, tests/test_gpu_fp8_forms.py runs them, so that a rule that changes cannot leave a kernel untested unnoticed.

A form is (tile, parts) of the tiles and (rows, strips, waves) of the few-rows kernel."""

# (m, n, k) -> form for bf16 outputs. The last column tile is cut between its waves' columns.
CUT_TILES = [((300, 3000, 384), (64, 1)), ((1500, 4168, 136), (128, 1)), ((3000, 8376, 136), (256, 1))]
