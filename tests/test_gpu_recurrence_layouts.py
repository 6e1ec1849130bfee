"""Recurrences on each side of every border between layouts: how many lanes lie side by side, and
whether time is split."""
import pytest
from test_gpu_policy import DTYPES, _check_recurrence, _scan_case

pytestmark = pytest.mark.gpu

# few channels: 8, 16 and 32 lanes; groups and blocks for splits and not
NARROW = [(350, 70, 8), (400, 70, 8), (760, 70, 8), (780, 70, 8), (1600, 40, 8), (100, 1300, 8),
          (100, 1600, 8), (190, 2113, 8), (193, 2113, 8), (250, 1700, 8), (510, 1650, 3)]
# one channel, along time
LINE = [(143, 20500, 1), (144, 20500, 1), (3, 10241, 1), (3, 12289, 1), (5, 24580, 1)]
# many channels: 64 lanes in splits, 32 lanes, 64 lanes whole
WIDE = [(55, 1000, 64), (56, 700, 64), (128, 300, 64), (129, 300, 64), (60, 300, 129),
        (2, 640, 65), (2, 900, 65)]


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", NARROW + LINE + WIDE)
def test_recurrence_borders_of_layouts(ws, device, shape, dtype, reverse):
    b, t, c = shape
    if dtype != "float32" and 1 < c:  # as many lanes, two channels each
        c *= 2
    _check_recurrence(ws, *_scan_case((b, t, c), dtype), reverse)
