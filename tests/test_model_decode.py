"""The prefill harness on this package's attention kernels and its decoding through the paged cache, on a reduced model.

Tolerance.  Both sides round activations to bf16 about ten times a layer (norm, projections, rotation, attention, MLP), each
time by a relative u = 2^-8 of a value at most, u / sqrt(3) on average with independent signs: over 6 layers sqrt(60) u /
sqrt(3) = 1.7 % of the logits' norm, and the two sides' errors are independent: 2.5 %.  Asserted: twice that."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture()
def reduced(monkeypatch):
    m = importlib.import_module("bench_lucid_model")
    for key, value in dict(layers=6, hidden=512, mlp=1024, vocab=4096, window=96).items():
        monkeypatch.setitem(m.CFG, key, value)
    return m, m.Model(torch.device("cuda", 0))


def off(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("lucid", [False, True])
def test_kernels_and_torch_attention_agree(reduced, lucid):
    m, model = reduced
    ids = torch.randint(0, 4096, (1, 768), device="cuda")
    # torch's form of the window layers takes whole windows: 768 = 8 * 96
    assert off(model.prefill(ids, lucid, attention="kernels"), model.prefill(ids, lucid)) < 0.05


@pytest.mark.parametrize("lucid", [False, True])
def test_prompt_and_decoding_equal_a_longer_prompt(reduced, lucid):
    m, model = reduced
    B, P, N = 2, 384, 512
    ids = torch.randint(0, 4096, (B, N), device="cuda")
    cache = m.KVCache(B, N, torch.device("cuda", 0), page=32)
    first = model.prefill_cached(ids[:, :P], lucid, cache)
    assert off(first, model.prefill(ids[:, :P], lucid, attention="kernels")) < 0.05
    for n in range(P, N):
        last = model.decode(ids[:, n], lucid, cache)
    assert int(cache.lens[0]) == N
    whole = m.KVCache(B, N, torch.device("cuda", 0), page=32)
    assert off(last, model.prefill_cached(ids, lucid, whole)) < 0.05


def test_decode_probe_runs(reduced):
    m, model = reduced
    r = m.decode_probe(model, torch.randint(0, 4096, (1, 256), device="cuda"), 8)
    assert r["softmax"]["finite"] and r["lucid"]["finite"] and r["lucid"]["ms_per_token"] > 0
