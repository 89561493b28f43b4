"""Scaling dictionaries whose fields would change the rotation are not taken without them."""

from __future__ import annotations

import pytest
import torch

from cachebridge_amd.rope import rope_frequencies

YARN = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=8192)


@pytest.mark.parametrize("field,value", [("attention_factor", 1.2), ("mscale", 0.707), ("mscale_all_dim", 1.0), ("truncate", False)])
def test_yarn_fields_that_are_not_computed_are_refused(field, value):
    with pytest.raises(ValueError, match=field):
        rope_frequencies(128, 1e6, dict(YARN, **{field: value}))


def test_fields_that_say_what_is_computed_anyway_are_taken():
    plain = rope_frequencies(128, 1e6, YARN)
    more = rope_frequencies(128, 1e6, dict(YARN, attention_factor=None, truncate=True, beta_fast=32, beta_slow=1))
    assert torch.equal(plain[0], more[0]) and plain[1] == more[1]
