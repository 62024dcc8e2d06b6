"""The step entries' Q1.17 table with every scaling of its frequencies."""
import numpy as np
import pytest

from test_gpu_rotary import SCALINGS, frequencies, make_scaling

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scaling", list(SCALINGS))
@pytest.mark.parametrize("magnitude", [1.0, 1.25, -0.5, 1.9999999])
def test_scaled_table(skv, ctx, oracle, scaling, magnitude):
    """RNE(2^17 m cos|sin), within the 19 bits of a word.  A 64-bit angle of up to 20000 is off by 2^-38 at most, and a
    frequency by as much relatively, so a word differs only where 2^17 m cos is that near to a half."""
    sc, positions = SCALINGS[scaling], 20000
    lut = skv.RopeLut.generate_scaled(ctx, make_scaling(skv, magnitude, **sc), positions)
    got = oracle.rope_unpack(np.frombuffer(lut.export(), np.uint8))
    angle = np.arange(positions)[:, None] * frequencies(skv, 128, **sc)
    for words, turn in zip(got, (np.cos, np.sin)):
        exact = 2.0 ** 17 * magnitude * turn(angle)
        want = np.clip(np.rint(exact), -2 ** 18, 2 ** 18 - 1)
        off = np.abs(np.asarray(words).reshape(want.shape) - want)
        near = np.abs(np.abs(exact - np.trunc(exact)) - 0.5) < 2.0 ** -16
        assert off[~near].max() == 0 and off.max() <= 1
