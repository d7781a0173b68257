"""The Llama-architecture driver with its keys and values in pages."""
import argparse
import importlib.util
import os

import pytest
import torch

from tests.gpu_util import DEV, assert_clean_device, set_config

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _driver():
    spec = importlib.util.spec_from_file_location("llama_infer", os.path.join(ROOT, "examples", "llama_infer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_driver_with_a_paged_cache():
    """Prompt and decode run, captured and not, to the same tokens; a prompt read in two parts leaves the logits of one read at once: the linear
    layers see the same rows, attention's sums come in another order."""
    L = _driver()
    set_config(64, torch.bfloat16)
    a = argparse.Namespace(layers=2, hidden=256, heads=4, head_dim=64, ffn=704, vocab=512, batch=2, prompt=24, decode=6, block=64, cache="paged")
    captured = L.run(a, rank=0, world=1, dev=torch.device(DEV), eager=False)
    eager = L.run(a, rank=0, world=1, dev=torch.device(DEV), eager=True)
    assert captured["tokens"] == eager["tokens"] and len(eager["tokens"][0]) == a.decode
    model = L.Llama(a, torch.device(DEV), rank=0, world=1)
    ids = torch.randint(0, a.vocab, (a.batch, a.prompt), generator=torch.Generator().manual_seed(4000)).to(DEV)
    whole = model(ids, 0, 32)
    for layer in model.layers:
        for t in layer.cache:
            t.fill_(float("nan"))
    model(ids[:, :17], 0, 32)
    parts = model(ids[:, 17:], 17, 32)
    assert torch.isfinite(whole).all() and torch.isfinite(parts).all()
    # a step of bf16 here and there in two layers: far below the logits' own size
    assert (whole.float() - parts.float()).abs().max() <= 2.0 ** -4 * whole.float().abs().max()
    assert_clean_device()
