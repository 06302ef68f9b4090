"""The serving example: both forms of the layer agree at every stage.

The two forms round different things: the expanded form its keys and values to the type, the absorbed form its queries and its
outputs.  One rounding is 2^-8 of a value; scores are sums of 192 products whose rounding errors add like a random walk, to about
2^-9 of a score of standard deviation 1, and outputs carry a handful of roundings: the largest of some 10^5 differences, in units of
the outputs' RMS, stays below 16 roundings, 2^-4.  Moved pages change nothing at all."""
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_latent_serving():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import latent_serving
    found = latent_serving.main()
    assert found["prompt"] < 2 ** -4 and found["step"] < 2 ** -4 and found["prefix"] < 2 ** -4
    assert found["dropped"] < 2 ** -4 and found["compacted"] == 0.0
