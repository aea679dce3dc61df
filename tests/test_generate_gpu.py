"""The generation example: MonarchAttention encoder, caches, one-token attention
together, against the same decoder computed densely in fp32 over all tokens."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu

# Relative to the largest logit: activations are rounded to bf16 (2^-8) about ten
# times a layer, two layers, each error passed on by random weights of norm about 1,
# so 2^-8 * sqrt(20) = 0.02 and three times that for the largest of thousands of
# logits; codes of the keys and values add half a step of 3 bits (2^-4) or 2^-8 of
# the largest for int8, averaged over the tokens attended to.
TOL = {"bf16": 0.06, "f16": 0.06, "int8": 0.08, "e4m3": 0.15}


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("generate", os.path.join(ROOT, "examples", "generate.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("cache", ["bf16", "f16", "int8", "e4m3"])
def test_generation_matches_the_dense_decoder(cache, example, cuda_device):
    dtype = torch.float16 if cache == "f16" else torch.bfloat16
    r = example.generate(batch=3, source_len=200, tokens=70, layers=2, heads=4, dim=64, vocab=200,
                         block=16, cache=cache, dtype=dtype)
    want = example.dense_logits(r)
    got = r["logits"].float()
    assert torch.isfinite(got).all()
    assert (got - want).abs().max() <= TOL[cache] * want.abs().max()
    for c in r["own"]:
        assert c.lengths.tolist() == [70] * 3
    # the cached context, read back, is what MonarchAttention takes
    k, v, mask = r["own"][0].read()
    z = r["model"].attention(k, k, v, mask)
    assert mask.all() and z.shape == (3, 4, 70, 64) and torch.isfinite(z).all()
