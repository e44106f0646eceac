"""llmk_process_logits and llmk_logprobs on the GPU where their documentation
makes a promise that ordinary inputs do not reach.  Tolerances as derived in
test_gpu_logits.py."""
import numpy as np
import pytest
import torch

import llmk
from test_gpu_logits import Case, dev, expect_logprobs, rows_on_device, sampler  # noqa: F401

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


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("bf16", "same"), ("f16", "same")])
def test_infinite_logits_under_a_softcap(sampler, dtype, out):  # noqa: F811
    """process_logits takes them to +-softcap, as the sampling call does, and a
    mask or a bias of -inf bans behind it; logprobs keeps -inf; for logits
    without it the two agree."""
    B, V, cap = 2, 5000, 30.0
    lg = np.random.default_rng(50).normal(0, 20, (B, V)).astype(np.float32)
    lg[:, [0, 700]], lg[:, [1, 4999]], lg[:, [2, 3]] = np.inf, -np.inf, -np.inf
    _, view, vals = rows_on_device(lg, dtype)
    mask = np.full((B, (V + 31) // 32), -1, np.int32)
    mask[:, 0] = ~np.int32(1 << 2)
    lb = llmk.LogitsBatch(logits=view, softcap=cap, allow_mask=dev(mask), bias_offsets=dev([0, 1, 2]),
                          bias_tokens=dev([3, 3]), bias_values=dev([-np.inf, -np.inf], torch.float32))
    odt = torch.float32 if out == "f32" else view.dtype
    x = torch.empty(B, V, dtype=odt, device="cuda:0")
    sampler.process_logits(lb, out=x)
    assert (x[:, [0, 700]] == cap).all() and (x[:, [1, 4999]] == -cap).all()
    assert (x[:, [2, 3]] == -np.inf).all() and torch.isfinite(x[:, 4:]).all()
    # the sampling call's probability of a token at -inf is that of -softcap
    u = dev([0.5, 0.5], torch.float32)
    d = sampler.sample_batch(llmk.DeviceBatch(logits=view, softcap=cap, uniforms=u), out_cap=V)
    for b in range(B):
        n = int(d.count[b])
        assert n == V and 1 in d.ids[b, n - 4:].tolist() and d.probs[b, n - 1].item() > 0
    # tokens 0 and 700 lie at +inf, the lowest ones at -inf
    r = sampler.logprobs(view, dev([0, 1]), top_n=4, softcap=cap)
    assert r.top_ids[:, :2].tolist() == [[0, 700]] * 2 and torch.isfinite(r.top_logprobs).all()
    assert r.logprobs[0].item() == r.top_logprobs[0, 0].item() and r.logprobs[1].item() == -np.inf
    view[:, [1, 2, 3, 4999]] = -50.0
    tok = dev([17, 700])
    one = sampler.logprobs(view, tok, top_n=8, softcap=cap)
    y = sampler.process_logits(llmk.LogitsBatch(logits=view, softcap=cap))
    two = sampler.logprobs(y, tok)
    # both from the same capped values, in sums of another order where the types
    # differ: each is within the bound for those values, so 2 of them apart
    yv = y.double().cpu().numpy()
    _, _, _, tol = expect_logprobs(yv, None, 0, 0.0)
    off = (one.logprobs.double() - two.logprobs.double()).abs().cpu().numpy()
    assert (off <= 2 * tol[[0, 1], [17, 700]]).all()


@pytest.mark.parametrize("B,V,dtype", [(1, 100, "f32"), (3, 5003, "bf16"), (2, 40000, "f32"), (260, 17000, "f16")])
def test_biases_listed_more_than_once_are_summed_in_listing_order(sampler, B, V, dtype):  # noqa: F811
    """Bit for bit the f32 sums in the list's order, on logits of zero: tokens
    listed once, twice on both sides of a multiple of 256 and hundreds of times,
    ids past the vocabulary, whole lists repeated, lists without a repetition."""
    rng = np.random.default_rng(V)
    lists = []
    for b in range(B):
        m = int(rng.integers(1, 600))
        t = rng.choice(V + 50, min(m, V))
        kind = b % 4
        if kind == 0:
            t = np.concatenate([t, t])
        elif kind == 1:
            t = np.concatenate([t, np.full(300, t[0]), t[:2]])
        elif kind == 2 and m > 3:
            t = np.concatenate([[t[0]], np.arange(V, V + 255), [t[0]], t, [t[1]]])
        lists.append((t, (rng.normal(0, 1, len(t)) * 10.0 ** rng.integers(-6, 7, len(t))).astype(np.float32)))
    want = np.zeros((B, V), np.float32)
    for b, (t, v) in enumerate(lists):
        seen = set()
        for i, x in zip(t, v):
            if i < V:
                want[b, i] = want[b, i] + x if i in seen else x
                seen.add(i)
    off = np.concatenate([[0], np.cumsum([len(t) for t, _ in lists])])
    lg = torch.zeros(B, V, dtype={"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype],
                     device="cuda:0")
    lb = llmk.LogitsBatch(logits=lg, bias_offsets=dev(off), bias_tokens=dev(np.concatenate([t for t, _ in lists])),
                          bias_values=dev(np.concatenate([v for _, v in lists]), torch.float32))
    got = sampler.process_logits(lb).cpu().numpy()
    assert np.array_equal(got, want)


def test_nan_biases_of_any_kind_on_a_token_listed_twice(sampler):  # noqa: F811
    """The NaN whose bits are all ones among them, first and last in a list."""
    bits = np.array([0xFFFFFFFF, 0x7FFFFFFF, 0x7F800001, 0xFFFFFFFF], np.uint32).view(np.float32)
    vals = np.array([bits[0], 1.0, 2.0, bits[1], bits[2], 3.0, bits[3], bits[3], 4.0, 5.0], np.float32)
    lb = llmk.LogitsBatch(logits=torch.ones(1, 3000, device="cuda:0"), bias_offsets=dev([0, 10]),
                          bias_tokens=dev([5, 5, 8, 8, 2100, 2100, 2900, 2900, 40, 40]),
                          bias_values=torch.as_tensor(vals).cuda())
    g = sampler.process_logits(lb)[0].cpu()
    assert torch.isnan(g[[5, 8, 2100, 2900]]).all() and int(torch.isnan(g).sum()) == 4
    assert g[40] == 10.0 and g[0] == 1.0 and g[2999] == 1.0


@pytest.mark.parametrize("B", [1, 64])
def test_a_repeated_bias_costs_in_proportion_to_the_list(sampler, B):  # noqa: F811
    """20000 pairs with one token listed twice, or half of them, against the
    same number of distinct ones."""
    V, n = 151936, 20000
    rng = np.random.default_rng(0)
    lg, out = torch.randn(B, V, device="cuda:0"), torch.empty(B, V, device="cuda:0")

    def time(repeated):
        tok = np.stack([rng.choice(V, n, replace=False) for _ in range(B)])
        tok[:, n - repeated:] = tok[:, :repeated]
        lb = llmk.LogitsBatch(logits=lg, bias_offsets=dev(np.arange(B + 1) * n), bias_tokens=dev(tok.reshape(-1)),
                              bias_values=torch.randn(B * n, device="cuda:0"))
        best = float("inf")
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            sampler.process_logits(lb, out=out)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    once = time(0)
    # walking the list anew for every listed token takes several hundred times as long
    assert time(1) < 40 * once and time(n // 2) < 40 * once


def test_as_many_rows_as_a_grid_holds(sampler):  # noqa: F811
    """2^24 - 1 rows, a workgroup each: every row is served."""
    B = 2**24 - 1
    lg = torch.randn(B, 2, device="cuda:0")
    x = sampler.process_logits(llmk.LogitsBatch(logits=lg, temperature=torch.full((B,), 2.0, device="cuda:0")))
    assert torch.equal(x, lg / 2)
    r = sampler.logprobs(lg, torch.ones(B, dtype=torch.int32, device="cuda:0"))
    assert torch.equal(r.ranks, (lg[:, 0] >= lg[:, 1]).int())
    # two terms, a difference, a logarithm below 1 and a last difference
    want = lg[:, 1].double() - torch.logsumexp(lg.double(), 1)
    tol = 2.0 ** -24 * (32 + 4 * (lg[:, 0] - lg[:, 1]).abs().double())
    assert bool(((r.logprobs.double() - want).abs() <= tol).all())
    more = torch.empty(B + 1, 2, device="cuda:0")
    with pytest.raises(llmk.SamplerError, match="too large"):
        sampler.process_logits(llmk.LogitsBatch(logits=more))
    with pytest.raises(llmk.SamplerError, match="too large"):
        sampler.logprobs(more, top_n=1)


def test_the_smallest_softcap(sampler):  # noqa: F811
    """2^-126: a logit of 0 stays 0, the others become +-softcap."""
    cap = 2.0 ** -126
    lg = dev([[0.0, -0.0, 3.0, -1e30, cap * 32, -np.inf]], torch.float32)
    x = sampler.process_logits(llmk.LogitsBatch(logits=lg, softcap=cap))
    assert x[0].tolist() == [0.0, 0.0, cap, -cap, cap, -cap]
    r = sampler.logprobs(lg, dev([0]), top_n=5, softcap=cap)
    assert torch.isfinite(r.logprobs).all() and torch.isfinite(r.top_logprobs).all()


@pytest.mark.parametrize("V", [262144, 262145, 524289, 900001, 2**20])
@pytest.mark.parametrize("B,n", [(1, 1), (3, 20), (70, 32), (300, 5)])
def test_logprobs_of_vocabularies_whose_tiles_are_selected_in_groups(sampler, V, B, n):  # noqa: F811
    """More than 256 tiles of 1024 logits: in groups of two to four, with ties
    within a group and across groups, rows that hold nothing and little."""
    if B * V > 10**8:
        V = V // 8 * 3 + 1  # (as few groups as a row of many needs)
        V = max(V, 262145)
    rng = np.random.default_rng(V + B)
    rows = min(B, 6)
    lg = rng.normal(0, 3, (rows, V)).astype(np.float32)
    if rows > 1:
        lg[1] = np.round(lg[1])
    if rows > 2:
        lg[2] = -np.inf
        lg[2, [V - 1, 5, 2048, 2049, 300000 % V]] = [1.0, 1.0, 0.0, 0.0, 2.0]
    if rows > 3:
        lg[3] = np.arange(V) // 1024 % 7
        lg[4] = np.nan
        lg[4, V - 3] = -1.0
        lg[5, ::7] = lg[5].max()
    many = np.resize(np.arange(rows), B)
    x = dev(lg, torch.float32)[dev(many).long()]
    tok = rng.integers(0, V, B)
    tok[::3] = [np.nanargmax(lg[r]) for r in many[::3]]
    lp, rank, order, tol = expect_logprobs(lg.astype(np.float64), None, n, 0.0)
    r = sampler.logprobs(x, dev(tok), top_n=n)
    assert np.array_equal(r.ranks.cpu().numpy(), rank[many, tok])
    assert np.array_equal(r.top_ids.cpu().numpy(), order[many])
    for got, want, t in ((r.logprobs, lp[many, tok], tol[many, tok]),
                         (r.top_logprobs, np.take_along_axis(lp, order, 1)[many],
                          np.take_along_axis(tol, order, 1)[many])):
        got = got.double().cpu().numpy()
        fin = np.isfinite(want)
        assert np.array_equal(got[~fin], want[~fin])
        assert (np.abs(got[fin] - want[fin]) <= t[fin]).all()
