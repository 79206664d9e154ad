"""rotary_frequencies at the ends of its range, on the host."""
import math

import pytest

import bmb


def plan(dims):
    p = bmb.Rotary(head_size=256, dims=dims, layout=bmb.ROTARY_HALF, amplitude=1.0)
    p.freq[:] = [7.0] * 128
    return p


@pytest.mark.parametrize("dims,base,scaling,factor", [
    (4, 1e300, bmb.ROTARY_BASE, 1e10), (256, 1e308, bmb.ROTARY_BASE, 2.0),
    (128, 10000.0, bmb.ROTARY_BASE, 1e306), (256, 5e-324, bmb.ROTARY_UNSCALED, 1.0),
    (256, 5e-324, bmb.ROTARY_LINEAR, 2.0)])
def test_not_finite(capfd, dims, base, scaling, factor):
    """A base past 64 bits would leave every frequency but the first at 0."""
    p = plan(dims)
    with pytest.raises(ValueError):
        bmb.rotary_frequencies(p, base, scaling, factor)
    assert "finite" in capfd.readouterr().err
    assert list(p.freq) == [7.0] * 128


@pytest.mark.parametrize("dims,base,scaling,factor", [
    (2, 1e308, bmb.ROTARY_BASE, 1e308), (2, 5e-324, bmb.ROTARY_UNSCALED, 1.0),
    (4, 1e300, bmb.ROTARY_BASE, 10.0), (256, 1e-300, bmb.ROTARY_UNSCALED, 1.0),
    (256, 1e308, bmb.ROTARY_LINEAR, 1e3), (64, 1.0, bmb.ROTARY_BASE, 1.0)])
def test_ends(dims, base, scaling, factor):
    """What 64 bits hold is as accurate as anywhere (a step or two of pow, through logarithms)."""
    p = plan(dims)
    bmb.rotary_frequencies(p, base, scaling, factor)
    for i in range(dims // 2):
        log = -2.0 * i / dims * math.log(base)
        if scaling == bmb.ROTARY_BASE and dims > 2:
            log -= 2.0 * i / (dims - 2) * math.log(factor)
        if scaling == bmb.ROTARY_LINEAR:
            log -= math.log(factor)
        # a logarithm below 1024 is off by 2^-44 at most, three of them
        assert math.log(p.freq[i]) == pytest.approx(log, rel=0, abs=2.0 ** -42)
    assert list(p.freq)[dims // 2:] == [7.0] * (128 - dims // 2)
