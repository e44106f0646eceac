"""llmk_process_logits and llmk_logprobs on the GPU where their documentation
makes a promise that ordinary inputs do not reach.  Tolerances as derived in
test_gpu_logits.py."""
import numpy as np
import pytest
import torch

import llmk
from test_gpu_logits import Case, dev, rows_on_device, sampler  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_greedy_rows_are_sampled_from_processed_logits_at_temperature_0(sampler, dtype):  # noqa: F811
    """Rows at and about the greedy limit beside sampled ones: the processed
    logits give the fused call's tokens if the greedy rows keep a temperature of
    0, or if the division is left to the sampling call.  At temperature 1 the
    greedy rows would be drawn."""
    B, V = 48, 20003
    rng = np.random.default_rng(22)
    case = Case(rng, B, V, hist=300, bias=0, mask=False)
    T = np.resize(np.float32([0.0, 0.9, 1e-5, 1.4, -1.0, 0.6, 1.00001e-5, 1.0]), B).astype(np.float32)
    _, view, _ = rows_on_device(case.lg * 0.2, dtype, pad=5)  # flat rows: a draw is rarely the likeliest
    lb = case.batch(view)
    lb.temperature = dev(T, torch.float32)
    common = dict(uniforms=dev(rng.random(B), torch.float32), vocab=V)
    fused = sampler.sample_batch(llmk.DeviceBatch(
        logits=view, temperature=lb.temperature, repetition_penalty=lb.repetition_penalty,
        presence_penalty=lb.presence_penalty, frequency_penalty=lb.frequency_penalty,
        hist_offsets=lb.hist_offsets, hist_tokens=lb.hist_tokens, **common), out_cap=8)
    greedy = lb.temperature <= 1e-5
    x = sampler.process_logits(lb)
    ones = torch.ones(B, device="cuda:0")
    kept = sampler.sample_batch(llmk.DeviceBatch(
        logits=x, temperature=torch.where(greedy, 0.0, ones), **common), out_cap=8)
    lb.temperature = None
    late = sampler.sample_batch(llmk.DeviceBatch(
        logits=sampler.process_logits(lb), temperature=dev(T, torch.float32), **common), out_cap=8)
    for y in (kept, late):
        assert torch.equal(fused.tokens, y.tokens) and torch.equal(fused.count, y.count)
        for b in range(B):
            n = min(8, int(fused.count[b]))
            assert torch.equal(fused.ids[b, :n], y.ids[b, :n])
            assert torch.equal(fused.probs[b, :n], y.probs[b, :n])
    g = greedy.cpu().numpy()
    assert g.sum() == 3 * B // 8
    best = sampler.logprobs(x, top_n=1).top_ids[:, 0]
    assert torch.equal(fused.tokens[greedy], best[greedy])
    drawn = sampler.sample_batch(llmk.DeviceBatch(logits=x, **common)).tokens
    assert torch.equal(drawn[~greedy], fused.tokens[~greedy])
    assert not torch.equal(drawn[greedy], best[greedy])
    assert sampler.status() == 0
