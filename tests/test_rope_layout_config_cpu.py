"""A configuration whose heads are rotated in part says which layout it means, or the loader says which it takes."""
import pytest

from skyrl_b200.models import decoder
from skyrl_b200.models.decoder import ModelArgs


@pytest.mark.parametrize("extra,warned,interleaved", [
    ({}, 0, False),
    ({"partial_rotary_factor": 1.0}, 0, False),
    ({"partial_rotary_factor": 0.5}, 1, False),
    ({"rope_parameters": {"rope_type": "default", "rope_theta": 1e4, "partial_rotary_factor": 0.5}}, 1, False),
    ({"partial_rotary_factor": 0.5, "rope_interleaved": False}, 0, False),
    ({"partial_rotary_factor": 0.5, "rope_interleaved": True}, 0, True),
    ({"rope_interleaved": True}, 0, True),
])
def test_layout_of_partly_rotated_heads(monkeypatch, extra, warned, interleaved):
    said = []
    monkeypatch.setattr(decoder.logger, "warning", lambda *a, **kw: said.append(a[0] % a[1:]))
    a = ModelArgs.from_hf_config({**ModelArgs().to_hf_config(), **extra})
    assert a.rope_interleaved == interleaved and len(said) == warned
    assert all("rope_interleaved" in m and "0.5" in m for m in said)
    # what the framework writes it also reads without a question
    b = ModelArgs.from_hf_config(a.to_hf_config())
    assert len(said) == warned
    assert (b.rope_interleaved, b.partial_rotary_factor) == (a.rope_interleaved, a.partial_rotary_factor)
