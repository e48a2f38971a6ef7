"""Workspace queries of the class distributions at the ends of what their arguments hold: answered, with 0 where the call is refused
(by name: callers ask for the workspace first)."""
import pytest

from multimae_amd import _lib

MOST = 2 ** 31 - 1
LIMIT = 2 ** 31 - 64  # positions of a call


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("outer,classes,inner", [(MOST, 1, 1), (LIMIT + 1, 9000, 1), (1, MOST, 1), (1, (1 << 30) + 1, 1), (1, (1 << 30) + 1, 64),
                                                 (1, 5, MOST), (1 << 16, 700, 1 << 16), (MOST, MOST, MOST), (LIMIT + 1, 3, 1)])
def test_sizes_that_are_refused_have_no_workspace(outer, classes, inner, dtype):
    lib = _lib.load()
    for k in (0, 1, 64):
        assert lib.mmae_class_log_probs_workspace_bytes(dtype, outer, classes, inner, k) == 0
        assert lib.mmae_distill_workspace_bytes(dtype, outer, classes, inner, k) == 0
    ld = classes * inner
    if ld >= 2 ** 63:
        return
    P = 4096  # never read
    for rc in (lib.mmae_class_log_probs(P, dtype, outer, classes, inner, ld, P, 1, 1.0, P, P, P, P, P, P, None, 0, None),
               lib.mmae_distill(P, dtype, outer, classes, inner, ld, P, 8, P, 0, 1, 0, 1.0, None, 1, 1, None, 0, 0, P, P, P, 0, None)):
        assert rc == -2 and b"workspace" not in lib.mmae_last_error()


@pytest.mark.parametrize("rows", [1, 2047, 2048, 2049, LIMIT - 2048, LIMIT - 100, LIMIT])
@pytest.mark.parametrize("classes", [1, 9000, 1 << 30])
def test_the_largest_sizes_have_a_workspace(rows, classes):
    lib = _lib.load()
    want = (8 * 256 + rows - 1) // rows  # workgroups a row, none without a tile of 4096 or 8192
    for bytes_, tile in ((lib.mmae_class_log_probs_workspace_bytes(0, rows, classes, 1, 3), 4096), (lib.mmae_distill_workspace_bytes(0, rows, classes, 1, 3), 8192)):
        tiles = -(-classes // tile)
        slices = -(-tiles // -(-tiles // min(want, tiles, 64)))
        if tile == 8192:
            assert bytes_ >= rows * (8 + 16 * slices)
        else:
            assert bytes_ == (rows * slices * (16 + 3 * 8) if slices > 1 else 0)
    for bad in (-1, 65):
        assert lib.mmae_class_log_probs_workspace_bytes(0, 4, 9000, 1, bad) == 0 and lib.mmae_distill_workspace_bytes(0, 4, 9000, 1, bad) == 0
