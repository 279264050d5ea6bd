"""The gated-delta example: it learns, clips and streams (GPU)."""

import importlib.util
import math
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "gated_delta_stream.py"


def test_example_trains_and_streams():
    spec = importlib.util.spec_from_file_location("gated_delta_stream", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    losses, norms, difference = module.main(["--steps", "25", "--time", "2560"])
    assert all(math.isfinite(x) for x in losses.tolist() + norms.tolist())
    assert float(losses[-1]) < 0.7 * float(losses[0])
    # the same products in another order, through two layers and a head: each is a sum of at
    # most 128 terms whose additions lose 2^-23 at most (torch's matrix products are 32-bit here)
    assert difference <= 8 * 128 * 2.0 ** -23
