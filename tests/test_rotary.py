"""Rotations as tuples: three fields, as before they had axes, and the axes beside them."""

from __future__ import annotations

import copy
import pickle

import pytest
import torch

from cachebridge_amd.online.queries import Rotary
from cachebridge_amd.rope import rope_frequencies


@pytest.mark.parametrize("sections", [None, (8, 4, 4)])
def test_a_rotation_unpacks_into_three(sections):
    spin = Rotary.build(32, 1e4, interleaved=True, sections=sections, device="cpu")
    inv, magnitude, interleaved = spin
    assert len(spin) == 3 and torch.equal(inv, rope_frequencies(32, 1e4, None)[0]) and magnitude == 1.0 and interleaved is True
    assert spin[0] is spin.inv_freq and spin._fields == ("inv_freq", "magnitude", "interleaved")
    again = Rotary(*spin)
    assert again.axes is None and (again == spin) == (sections is None)


def test_axes_stay_with_a_rotation():
    spin = Rotary.build(32, 1e4, sections=(8, 4, 4), device="cpu")
    axes = bytes([0] * 8 + [1] * 4 + [2] * 4)
    assert spin.axes == axes and Rotary(spin.inv_freq, axes=axes) == spin and Rotary(spin.inv_freq, 1.0, False, axes) == spin
    for other in (spin._replace(magnitude=0.5), copy.copy(spin), copy.deepcopy(spin), pickle.loads(pickle.dumps(spin))):
        assert type(other) is Rotary and other.axes == axes and torch.equal(other.inv_freq, spin.inv_freq)
    plain = spin._replace(axes=None)
    assert plain.axes is None and spin.axes == axes and plain != spin and plain == Rotary(spin.inv_freq)
    assert hash(plain) != hash(spin) and "axes=None" in repr(plain)
    with pytest.raises(ValueError):
        spin._replace(sections=(16,))
    with pytest.raises(TypeError):
        Rotary()
