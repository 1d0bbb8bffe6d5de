"""The 8-bit cache in the models, at the ends of what they decode."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from test_decode_scores_gpu import _vae, _z  # noqa: E402

pytestmark = pytest.mark.gpu


def test_cache_error_of_no_tokens_is_zero(monkeypatch):
    "latents of predicted length 0 have no keys and values to be wrong about; beside others they change nothing"
    vae = _vae()
    z = _z(4)
    whole = vae.kv_cache_error(z[:2])
    length = vae.model.encoder.predict_mask_length
    monkeypatch.setattr(vae.model.encoder, "predict_mask_length", lambda m: torch.zeros_like(length(m)))
    e = vae.kv_cache_error(z)
    assert e.shape == whole.shape and torch.equal(e, torch.zeros_like(e))
    monkeypatch.setattr(vae.model.encoder, "predict_mask_length", lambda m: torch.cat([length(m[:2]), torch.zeros_like(length(m[2:]))]))
    assert torch.allclose(vae.kv_cache_error(z), whole, rtol=2.0 ** -18, atol=0)
