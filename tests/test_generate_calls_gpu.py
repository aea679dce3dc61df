"""Every attention call of the generation example, on what the example puts into its caches,
against the formula in 64 bits."""
import importlib.util
import math
import os
import sys

import pytest
import torch

import monarch_attention_b200 as mab
from conftest import ROOT

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # of a result's unit, one flipped bit


@pytest.fixture
def example():
    spec = importlib.util.spec_from_file_location("generate", os.path.join(ROOT, "examples", "generate.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("cache", ["bf16", "f16", "int8", "e4m3"])
def test_the_example_runs_as_a_program(cache, example, cuda_device, monkeypatch, capsys):
    """Every choice of its command line."""
    monkeypatch.setattr(sys, "argv", ["generate.py", "--cache", cache, "--tokens", "3", "--batch", "2",
                                      "--source-len", "128"])
    example.main()
    assert f"2 x 3 tokens from 128 with a {cache} cache" in capsys.readouterr().out


@pytest.mark.parametrize("cache", ["bf16", "f16", "int8", "e4m3"])
def test_calls_of_the_example(cache, example, cuda_device, monkeypatch):
    """Scores are right to (D + 8) u of their size, weights to 2^-16 of theirs, sums of n to
    (n / 4 + 64) u, each result to half a unit of its type (fp16: of its smallest one too)."""
    kernel, calls = mab.kv_cache.decode_attention, []

    def both(q, k_pages, v_pages, table, lengths, mask=None, *, scales=None, **kw):
        out = kernel(q, k_pages, v_pages, table, lengths, mask, scales=scales, **kw)
        E, H, _, D = q.shape
        at = table.long().clamp(min=0)

        def rows(pages, scale):
            x = pages.float().double()[at]
            x = x if scale is None else x * scale.double()[at][..., None]
            return x.permute(0, 2, 1, 3, 4).reshape(E, pages.shape[1], -1, D)

        k, v = (rows(p, None if scales is None else scales[i]) for i, p in enumerate((k_pages, v_pages)))
        n = k.shape[2]
        ok = torch.arange(n, device=q.device)[None] < lengths[:, None]
        if mask is not None:
            ok &= torch.nn.functional.pad(mask, (0, max(0, n - mask.shape[1])))[:, :n]
        k, v = (torch.where(ok[:, None, :, None], x, 0.0) for x in (k, v))
        s = q.double() @ k.transpose(2, 3) / math.sqrt(D)
        w = torch.softmax(s.masked_fill(~ok[:, None, None], -math.inf), -1)
        want = w @ v
        mag = (q.double().abs() @ k.abs().transpose(2, 3)).amax(-1) / math.sqrt(D)
        rel = 2 * (2 * (D + 8) * U * mag + 2.0 ** -16 + (n / 4 + 64) * U)[..., None]
        tol = rel * (w @ v.abs()) + HALF[q.dtype] * want.abs() + 2.0 ** -25 * (q.dtype == torch.float16)
        over = (out.double() - want).abs() - tol
        calls.append((float(over.max()), bool(torch.isfinite(out).all())))
        return out

    monkeypatch.setattr(mab.kv_cache, "decode_attention", both)
    dtype = torch.float16 if cache == "f16" else torch.bfloat16
    example.generate(batch=3, source_len=200, tokens=70, layers=2, heads=4, dim=64, vocab=200, block=16,
                     cache=cache, dtype=dtype)
    assert len(calls) == 70 * 2 * 2
    assert all(fine and over <= 0 for over, fine in calls), max(calls)
