"""Which kernels of the normalisation over channels the GPU tests' shapes reach (no GPU): the rule by which rows are laid on threads,
written out again."""
from test_rms_norm_gpu import SHAPES
from test_rms_norm_walks_gpu import WALKS, WIDTHS

ALL = range(8, 16384 + 8, 8)


def _cover(C, two):
    """(lanes, vectors, threads) of rows of C channels; 0 lanes: a block for a row. `two`: backward, or forward with a residual."""
    cg = C // 8
    if cg > 128:
        v = 2 if cg <= 1024 else 3 if cg <= 1536 else 4
        return 0, v, (-(-cg // v) + 31) // 32 * 32
    best = None
    for lanes in (32, 16, 8, 4):
        v = -(-cg // lanes)
        if (v == 1 or lanes == 32 or v == 3 and not (two and cg <= 32)) and v <= 4 and (best is None or lanes * v < best[0] * best[1]):
            best = lanes, v, 256
    return best


def test_every_width_is_held():
    for C in ALL:
        for two in (False, True):
            lanes, v, threads = _cover(C, two)
            assert (lanes or threads) * v * 8 >= C and threads <= 512
            assert (lanes, v) in [(4, 1), (4, 3), (8, 1), (8, 3), (16, 1), (16, 3), (32, 1), (32, 2), (32, 3), (32, 4), (0, 2), (0, 3), (0, 4)]


def test_shapes_reach_every_kernel():
    for two in (False, True):
        built = {_cover(C, two)[:2] for C in ALL}
        assert built == {_cover(C, two)[:2] for _, C, _ in SHAPES + WIDTHS}
        # ... and walk in each: an SM holds 2048 threads at most
        walk = set()
        for rows, C, _ in WALKS:
            lanes, v, threads = _cover(C, two)
            group = 256 // lanes if lanes else 1
            if rows > 148 * (2048 // threads) * group and (rows % group or not lanes):
                walk.add((lanes, v))
        assert walk == built, built - walk


def test_shapes_end_inside_of_a_vector_and_of_a_lane():
    assert {valid % 8 for _, C, valid in SHAPES + WIDTHS + WALKS if valid < C} == set(range(8))
