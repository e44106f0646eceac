"""llmk_process_logits and llmk_logprobs on the GPU against the same formulas in
64 bits (numpy), at odd sizes, strides and types, with rows whose mask leaves
nothing, infinities and NaN, tokens listed twice; chained into the sampling
call; captured into a graph; on another stream; past 32-bit offsets.

Tolerances, with u = 2^-24 (half a unit in the last place of f32):

* process: every step is one f32 operation, so its error is at most u times
  its result.  With A = |logit| (or the cap) + |bias| and R = max(r, 1/r), no
  intermediate is above M = A R + |presence| + n |frequency|; there are at most
  six operations before the division and one for it, and each error before it
  is carried on with a factor of at most R (the penalty) and 1/T: 7 R u M / T.
  A softcap adds 7 u relative to the capped value (the scale 1/cap, the
  product, two units of tanh, the last product).  Rounding to 16 bits adds half
  a unit, finfo.eps / 2 relative to the value, or half the smallest step.
* logprobs: a lane sums at most n = 16 ceil(tiles / 4) + 2 terms in sequence
  and then 10 more partial sums, each adding u relative; a term's exponent
  carries two roundings of a difference d (2 u |d|, whose mean under the
  softmax is at most log V) and the exponential's own 2 u.  With x - M, the
  logarithm and the last difference, the error is at most
  u (n + 20 + 2 log V + 2 |x - M| + 2 |log S| + |log p|), plus 8 u cap with
  a softcap (tanh by one exponential and a reciprocal, each of 2 u, of terms of
  at most 2 cap).
"""
import math

import numpy as np
import pytest
import torch

import llmk
from llmk import _lib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def sampler():
    s = llmk.HipSampler(max_batch=64, max_vocab=160000)
    yield s
    s.close()


def dev(a, dt=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dt).to("cuda:0")


def rows_on_device(lg, dtype, pad=0, offset=0):
    """[B, V] logits in rows of V + pad elements from element `offset` of a
    buffer that is NaN elsewhere, and their values as the type holds them."""
    B, V = lg.shape
    buf = torch.full((offset + B * (V + pad) + 16,), float("nan"), dtype=DT[dtype], device="cuda:0")
    view = buf.as_strided((B, V), (V + pad, 1), offset)
    view.copy_(torch.as_tensor(lg, dtype=torch.float32))
    return buf, view, view.double().cpu().numpy()


def csr(lists):
    off = np.zeros(len(lists) + 1, np.int64)
    off[1:] = np.cumsum([len(x) for x in lists])
    flat = np.concatenate([np.asarray(x, np.int64) for x in lists]) if off[-1] else np.zeros(1, np.int64)
    return off, flat


class Case:
    """Inputs of one call, and what it should return in 64 bits."""

    def __init__(self, rng, B, V, chain=1, hist=0, form="csr", bias=0, mask=False, T=True, rep=True,
                 pres=True, freq=True, softcap=0.0, twice=False):
        S = (B + chain - 1) // chain
        self.B, self.V, self.S, self.chain, self.softcap = B, V, S, chain, softcap
        self.lg = rng.normal(0, 4, (B, V)).astype(np.float32)
        f = lambda lo, hi: rng.uniform(lo, hi, S).astype(np.float32)  # noqa: E731
        self.T = f(0.5, 1.5) if T else None
        if T and S > 2:
            self.T[1], self.T[2] = 0.0, 1.0  # greedy, off
        self.rep, self.pres, self.freq = f(0.8, 1.5) if rep else None, f(-1, 1) if pres else None, \
            f(-0.5, 0.5) if freq else None
        # histories, some of them empty, with ids past the vocabulary
        self.hists = [list(rng.integers(0, V + V // 8 + 1, rng.integers(0, hist + 1))) if hist else []
                      for _ in range(S)]
        if hist:
            self.hists[0] = [int(rng.integers(0, V))] * hist
        self.form = form
        self.extra = [[list(rng.integers(0, V, i)) for i in range(chain)] for _ in range(S)] \
            if chain > 1 else None
        self.bias = [[] for _ in range(S)]
        if bias:
            for q in range(S):
                toks = rng.choice(V + 3, min(bias, V), replace=False)
                if twice:
                    toks = np.concatenate([toks, toks[: len(toks) // 2], toks[:1]])
                    rng.shuffle(toks)
                self.bias[q] = [(int(t), np.float32(rng.uniform(-5, 5))) for t in toks]
            self.bias[-1] = []  # a sequence without any
        self.has_bias = bias > 0
        self.mask = self.mask_index = None
        if mask:
            bits = rng.random((3, V)) < 0.3
            bits[1] = False  # leaves nothing
            words = (V + 31) // 32 + 1
            w = np.zeros((3, words), np.uint32)
            for v in range(V):
                w[:, v >> 5] |= bits[:, v].astype(np.uint32) << np.uint32(v & 31)
            w[:, V >> 5] |= np.uint32(0) if V % 32 == 0 else ~np.uint32((1 << (V % 32)) - 1)  # past V
            self.mask, self.bits = w, bits
            self.mask_index = rng.integers(-1, 3, B)

    def batch(self, view):
        kw = {}
        for n, x in (("temperature", self.T), ("repetition_penalty", self.rep),
                     ("presence_penalty", self.pres), ("frequency_penalty", self.freq)):
            if x is not None:
                kw[n] = dev(x, torch.float32)
        if self.chain > 1:
            kw["row_seq"] = dev(np.arange(self.B) // self.chain)
            lists = [self.extra[b // self.chain][b % self.chain] for b in range(self.B)]
            off, flat = csr(lists)
            kw.update(extra_begin=dev(off[:-1]), extra_count=dev(np.diff(off)), extra_tokens=dev(flat))
        if any(self.hists):
            if self.form == "csr":
                off, flat = csr(self.hists)
                kw.update(hist_offsets=dev(off), hist_tokens=dev(flat))
            elif self.form == "buffers":
                cap = max(len(h) for h in self.hists) + 3
                buf = np.zeros((self.S, cap), np.int64)  # token 0 past each history
                for q, h in enumerate(self.hists):
                    buf[q, :len(h)] = h
                kw.update(hist_offsets=dev(np.arange(self.S) * cap), hist_tokens=dev(buf.reshape(-1)),
                          hist_lengths=dev([len(h) for h in self.hists]))
            else:  # count tables, one token split over two entries
                tok, cnt = [], []
                for h in self.hists:
                    t, n = np.unique(np.asarray(h, np.int64), return_counts=True)
                    t, n = list(t), list(n)
                    if n and n[0] > 2:
                        t.append(t[0])
                        n.append(n[0] - 1)
                        n[0] = 1
                    tok.append(t)
                    cnt.append(n)
                off, flat = csr(tok)
                kw.update(hist_offsets=dev(off), hist_tokens=dev(flat), hist_counts=dev(csr(cnt)[1]))
        if self.has_bias:
            off, flat = csr([[t for t, _ in x] for x in self.bias])
            vals = [v for x in self.bias for _, v in x] or [0.0]
            kw.update(bias_offsets=dev(off), bias_tokens=dev(flat), bias_values=dev(vals, torch.float32))
        if self.mask is not None:
            kw.update(allow_mask=dev(self.mask.view(np.int32)), mask_index=dev(self.mask_index))
        return llmk.LogitsBatch(logits=view, softcap=self.softcap, **kw)

    def expect(self, vals):
        """The results in 64 bits, and how far f32 may be off."""
        out, tol = np.empty((self.B, self.V)), np.empty((self.B, self.V))
        one = lambda x, q, d: float(x[q]) if x is not None else d  # noqa: E731
        for b in range(self.B):
            q = b // self.chain
            x = vals[b].copy()
            e = np.zeros(self.V)
            if self.softcap:
                x = self.softcap * np.tanh(x / self.softcap)
                e += 7 * U * np.abs(x)
            add = np.zeros(self.V)
            size = np.abs(x)
            for t, v in self.bias[q]:
                if t < self.V:
                    add[t] += float(v)
                    size[t] += abs(float(v))
                    e[t] += U * 4 * abs(float(v))  # the sum of several biases
            x = x + add
            toks = self.hists[q] + (self.extra[q][b % self.chain] if self.extra else [])
            n = np.bincount([t for t in toks if t < self.V], minlength=self.V).astype(float)
            r, p, f = one(self.rep, q, 1.0), one(self.pres, q, 0.0), one(self.freq, q, 0.0)
            y = np.where(x > 0, x / r, x * r) - (p + n * f)
            x = np.where(n > 0, y, x)
            R = max(r, 1 / r)
            M = size * R + abs(p) + n * abs(f)
            if self.mask is not None and self.mask_index[b] >= 0:
                x = np.where(self.bits[self.mask_index[b]], x, -np.inf)
            T = one(self.T, q, 1.0)
            T = T if T > 1e-5 else 1.0
            out[b], tol[b] = x / T, (7 * U * M + e) * R / T
        return out, tol


def check_process(sampler, case, dtype, out="f32", pad=0, offset=0, inplace=False):
    buf, view, vals = rows_on_device(case.lg, dtype, pad, offset)
    if inplace:
        obuf, oview = buf, view
    else:
        odt = DT[dtype] if out == "same" else torch.float32
        obuf = torch.full((offset + case.B * (case.V + pad) + 16,), 77.0, dtype=odt, device="cuda:0")
        oview = obuf.as_strided((case.B, case.V), (case.V + pad, 1), offset)
    before = obuf.clone()
    got = sampler.process_logits(case.batch(view), out=oview)
    torch.cuda.synchronize()
    assert sampler.status() == 0
    want, tol = case.expect(vals)
    if got.dtype != torch.float32:
        fi = torch.finfo(got.dtype)
        tol = tol * (1 + fi.eps) + np.abs(want) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
    g = got.double().cpu().numpy()
    inf = np.isinf(want)
    assert np.array_equal(g[inf], want[inf])
    off, tol = np.abs(g[~inf] - want[~inf]), tol[~inf]
    bad = off > tol
    assert not bad.any(), (off[bad][:5], tol[bad][:5])
    # nothing outside the rows is written
    mark = torch.ones(obuf.numel(), dtype=torch.bool, device="cuda:0")
    mark.as_strided((case.B, case.V), (case.V + pad, 1), offset).fill_(False)
    as_int = {4: torch.int32, 2: torch.int16}[obuf.element_size()]
    assert torch.equal(obuf.view(as_int)[mark], before.view(as_int)[mark])
    return got


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("bf16", "same"),
                                       ("f16", "f32"), ("f16", "same")])
@pytest.mark.parametrize("B,V,pad,offset", [(1, 1, 0, 0), (3, 7, 1, 1), (5, 2048, 0, 0), (4, 2049, 3, 1),
                                            (70, 8193, 1, 3), (8, 50257, 0, 2)])
def test_process_every_step(sampler, dtype, out, B, V, pad, offset):
    case = Case(np.random.default_rng(B * V), B, V, hist=min(3 * V, 900), bias=min(V, 40), mask=V > 8)
    check_process(sampler, case, dtype, out, pad, offset)


@pytest.mark.parametrize("form", ["csr", "buffers", "counts"])
@pytest.mark.parametrize("chain,inplace", [(1, False), (4, False), (3, True)])
def test_process_histories_and_chains(sampler, form, chain, inplace):
    case = Case(np.random.default_rng(chain), 12, 5003, chain=chain, hist=3000, form=form, T=not inplace)
    check_process(sampler, case, "f32", inplace=inplace, pad=5)


@pytest.mark.parametrize("which", ["rep", "pres", "freq", "T", "bias", "mask", "softcap", "nothing"])
@pytest.mark.parametrize("inplace", [False, True])
def test_process_one_step_alone(sampler, which, inplace):
    on = {k: k == which for k in ("T", "rep", "pres", "freq")}
    case = Case(np.random.default_rng(5), 6, 10007, hist=500, bias=30 if which == "bias" else 0,
                mask=which == "mask", softcap=20.0 if which == "softcap" else 0.0, **on)
    check_process(sampler, case, "bf16" if inplace else "f32", out="same", inplace=inplace, offset=1)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_process_softcap_and_everything(sampler, dtype):
    case = Case(np.random.default_rng(9), 9, 4099, chain=3, hist=200, bias=20, mask=True, softcap=30.0)
    check_process(sampler, case, dtype, "f32", pad=1)


def test_process_a_bias_listed_more_than_once(sampler):
    """The sum in listing order, whatever order the threads run in: two runs
    are the same bits."""
    case = Case(np.random.default_rng(11), 4, 30011, bias=3000, twice=True, hist=50)
    a = check_process(sampler, case, "f32")
    b = check_process(sampler, case, "f32")
    assert torch.equal(a, b)
    # one token listed 2000 times, sums exact in f32
    lg = torch.zeros(1, 100, device="cuda:0")
    n = 2000
    lb = llmk.LogitsBatch(logits=lg, bias_offsets=dev([0, n]), bias_tokens=dev(np.full(n, 42)),
                          bias_values=dev(np.arange(n), torch.float32))
    got = sampler.process_logits(lb)
    assert got[0, 42].item() == n * (n - 1) / 2 and got.sum().item() == n * (n - 1) / 2


def test_process_infinities_and_nan(sampler):
    V = 300
    lg = np.zeros((2, V), np.float32)
    lg[:, :4] = [np.inf, -np.inf, np.nan, np.finfo(np.float32).min]
    lg[:, 10:14] = lg[:, :4]  # the same ones without a history
    lg[:, 20:24] = lg[:, :4]  # and masked
    mask = np.full((2, 10), -1, np.int32)
    mask[:, 0] = ~np.int32(0b1111 << 20)
    lb = llmk.LogitsBatch(logits=dev(lg, torch.float32), hist_offsets=dev([0, 4, 8]),
                          hist_tokens=dev([0, 1, 2, 3, 3, 2, 1, 0]), allow_mask=dev(mask),
                          repetition_penalty=dev([1.5, 1.5], torch.float32),
                          presence_penalty=dev([0.5, 0.5], torch.float32))
    g = sampler.process_logits(lb).cpu().numpy()
    for base in (0, 10):
        assert g[0, base] == np.inf and g[0, base + 1] == -np.inf and np.isnan(g[0, base + 2])
    assert g[0, 3] == -np.inf  # the lowest number, times 1.5
    assert g[0, 13] == np.finfo(np.float32).min
    assert (g[:, 20:24] == -np.inf).all()
    assert np.array_equal(g[0], g[1], equal_nan=True)
    assert sampler.status() == 0


def test_process_rows_that_are_refused(sampler):
    """A sequence past the end, a mask row past the end, a parameter that is not
    finite: those rows are NaN, the others as ever."""
    B, V = 5, 9001
    case = Case(np.random.default_rng(2), B, V, hist=100)
    case.T[:] = 0.9
    _, view, vals = rows_on_device(case.lg, "f32")
    lb = case.batch(view)
    lb.row_seq = dev([0, 1, 5, 2**31 - 1, 4])
    lb.temperature[4] = float("nan")
    lb.allow_mask = dev(np.full((2, (V + 31) // 32), -1))
    lb.mask_index = dev([-1, 2, 0, 1, 1])
    g = sampler.process_logits(lb).double().cpu().numpy()
    assert np.isnan(g[1:]).all()
    want, tol = case.expect(vals)
    assert (np.abs(g[0] - want[0]) <= tol[0]).all()
    assert sampler.status() == _lib.LLMK_STATUS_INVALID_PARAMS
    assert sampler.status() == 0


def test_process_interleaved_rows(sampler):
    """Logits and results as the two halves of one buffer's rows."""
    case = Case(np.random.default_rng(8), 6, 1000, hist=100)
    buf = torch.zeros(6, 2000, device="cuda:0")
    buf[:, :1000] = torch.as_tensor(case.lg)
    want, tol = case.expect(case.lg.astype(np.float64))
    sampler.process_logits(case.batch(buf[:, :1000]), out=buf[:, 1000:])
    assert (np.abs(buf[:, 1000:].double().cpu().numpy() - want) <= tol).all()
    assert torch.equal(buf[:, :1000].cpu(), torch.as_tensor(case.lg))
    with pytest.raises(llmk.SamplerError, match="overlaps"):
        sampler.process_logits(case.batch(buf[:, :1000]), out=buf[:, 999:1999])


def test_process_then_sample_is_the_fused_call(sampler):
    """Sampling the processed logits at temperature 1 gives the tokens, counts
    and probabilities of sampling the logits with every parameter (the same f32
    operations in the same order)."""
    B, V = 48, 32003
    rng = np.random.default_rng(21)
    case = Case(rng, B, V, hist=600)
    _, view, _ = rows_on_device(case.lg, "bf16", pad=5)
    lb = case.batch(view)
    mask = dev(rng.integers(-2**31, 2**31, (B, (V + 31) // 32)).astype(np.int32))
    lb.allow_mask, lb.mask_index = mask, dev(np.arange(B))
    lb.temperature.clamp_(min=0.5)
    common = dict(uniforms=dev(rng.random(B), torch.float32), vocab=V,
                  top_k=dev(np.full(B, 40)), top_p=dev(np.full(B, 0.9), torch.float32))
    fused = sampler.sample_batch(llmk.DeviceBatch(
        logits=view, temperature=lb.temperature, repetition_penalty=lb.repetition_penalty,
        presence_penalty=lb.presence_penalty, frequency_penalty=lb.frequency_penalty,
        hist_offsets=lb.hist_offsets, hist_tokens=lb.hist_tokens, allow_mask=mask, **common), out_cap=40)
    split = sampler.sample_batch(llmk.DeviceBatch(logits=sampler.process_logits(lb), **common), out_cap=40)
    for x, y in ((fused.tokens, split.tokens), (fused.count, split.count)):
        assert torch.equal(x, y)
    for b in range(B):
        n = int(fused.count[b])
        assert torch.equal(fused.ids[b, :n], split.ids[b, :n])
        assert torch.equal(fused.probs[b, :n], split.probs[b, :n])


# ---- logprobs ----------------------------------------------------------------

def expect_logprobs(vals, tokens, n, softcap):
    """numpy, 64 bits; the order on the raw logits, NaN read as -inf."""
    B, V = vals.shape
    v = np.where(np.isnan(vals), -np.inf, vals)
    x = np.where(v == -np.inf, v, softcap * np.tanh(v / softcap)) if softcap else v
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        d = x - np.where(m == -np.inf, 0.0, m)
        logS = np.log(np.exp(d).sum(1, keepdims=True))
        lp = np.where(v == -np.inf, -np.inf, d - logS)
    order = np.argsort(-(v + 0.0), axis=1, kind="stable")
    rank = np.empty_like(order)
    np.put_along_axis(rank, order, np.arange(V)[None, :], 1)
    tiles = -(-V // 1024)
    tol = U * (16 * -(-tiles // 4) + 22 + 2 * math.log(V) + 2 * np.abs(d) + 2 * np.abs(logS) +
               np.abs(lp) + 8 * softcap)
    return lp, rank, order[:, :n], tol


def check_logprobs(sampler, lg, dtype, n, pad=0, offset=0, softcap=0.0, tokens=None, seed=0):
    B, V = lg.shape
    _, view, vals = rows_on_device(lg, dtype, pad, offset)
    if tokens is None:
        tokens = np.random.default_rng(seed).integers(0, V, B)
        tokens[::3] = np.where(np.isnan(vals), -np.inf, vals).argmax(1)[::3]
    r = sampler.logprobs(view, dev(tokens), top_n=n, softcap=softcap)
    torch.cuda.synchronize()
    lp, rank, order, tol = expect_logprobs(vals, tokens, n, softcap)
    at = np.arange(B)
    assert np.array_equal(r.ranks.cpu().numpy(), rank[at, tokens])

    def close(got, want, t):
        same = (got == want) | (np.isnan(got) & np.isnan(want))
        with np.errstate(invalid="ignore"):
            assert (same | (np.abs(got - want) <= t)).all(), np.abs(got - want)[~same].max()

    close(r.logprobs.double().cpu().numpy(), lp[at, tokens], tol[at, tokens])
    if n:
        ids, top = r.top_ids.cpu().numpy(), r.top_logprobs.double().cpu().numpy()
        k = min(n, V)
        assert np.array_equal(ids[:, :k], order[:, :k])
        assert (ids[:, k:] == -1).all() and (top[:, k:] == -np.inf).all()
        close(top[:, :k], np.take_along_axis(lp, order[:, :k], 1), np.take_along_axis(tol, order[:, :k], 1))
    return r


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,V,n,pad,offset", [
    (1, 1, 1, 0, 0), (3, 5, 20, 1, 1), (2, 64, 32, 0, 0), (4, 1023, 8, 0, 0), (3, 1025, 5, 2, 1),
    (70, 4097, 1, 1, 0), (65, 5000, 0, 0, 3), (2, 50257, 20, 0, 0), (1, 151936, 32, 0, 0),
    (64, 32000, 20, 0, 0), (2000, 3001, 3, 0, 1)])
def test_logprobs(sampler, dtype, B, V, n, pad, offset):
    lg = np.random.default_rng(V).normal(0, 3, (B, V)).astype(np.float32)
    check_logprobs(sampler, lg, dtype, n, pad, offset, seed=B)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("V", [33, 20000])
def test_logprobs_softcap(sampler, dtype, V):
    lg = np.random.default_rng(V).normal(0, 30, (5, V)).astype(np.float32)
    lg[:, 3] = -np.inf
    check_logprobs(sampler, lg, dtype, 8, softcap=30.0)


@pytest.mark.parametrize("V,n", [(100, 32), (5000, 20), (151936, 8)])
def test_logprobs_rows_of_ties(sampler, V, n):
    """Equal logits everywhere, two values, zeros of both signs, rising and
    falling rows: the lower id comes first."""
    lg = np.zeros((7, V), np.float32)
    lg[1, 1::2] = 1.0
    lg[2, ::2] = -0.0
    lg[3] = np.arange(V) / 16.0 % 4096
    lg[4] = -np.arange(V) / 16.0
    lg[5] = np.round(np.random.default_rng(0).normal(0, 2, V))
    lg[6, V // 2:] = -1.0
    check_logprobs(sampler, lg, "f32", n)


@pytest.mark.parametrize("V", [70, 9000])
def test_logprobs_masked_rows(sampler, V):
    """Nothing allowed; one token allowed; fewer than the list; NaN among the
    masked; the type's lowest value as a mask; +inf."""
    n = 8
    lg = np.full((7, V), -np.inf, np.float32)
    lg[1, V - 1] = 3.0
    lg[2, [5, 40, 60]] = [1.0, 2.0, 2.0]
    lg[3, ::2] = np.nan
    lg[3, 7] = 0.5
    lg[4] = np.finfo(np.float32).min
    lg[4, 11] = 4.0
    lg[5] = np.finfo(np.float32).min
    lg[6, :30] = 0.0
    lg[6, 20] = np.inf
    r = check_logprobs(sampler, lg, "f32", n, tokens=np.array([3, V - 1, 40, 7, 11, 69, 20]))
    assert r.logprobs[0].item() == -np.inf and r.logprobs[1].item() == 0.0
    r = check_logprobs(sampler, lg, "f32", n, tokens=np.array([0, 0, 0, 2, 0, 0, 5]))
    assert torch.isnan(r.logprobs[6]) and r.logprobs[2].item() == -np.inf


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_logprobs_nan_of_any_kind(sampler, dtype, softcap):
    """Quiet and signalling NaN of both signs: single ones, whole tiles of
    them, and rows with little else, read as -inf wherever they stand."""
    B, V = 9, 9001
    lg = np.random.default_rng(12).normal(0, 3, (B, V)).astype(np.float32)
    x = dev(lg, torch.float32).to(DT[dtype])
    bits = x.view(torch.int32 if dtype == "f32" else torch.int16)
    kinds = {"f32": [0x7F800001, 0x7FC00000, -0x7FFFFF, -1], "bf16": [0x7F81, 0x7FC0, -0x7F, -1],
             "f16": [0x7C01, 0x7E00, -0x3FF, -1]}[dtype]
    for i, k in enumerate(kinds):
        bits[0, 5 + 977 * i] = k
        bits[1, 1000 + i:4000:4] = k
        bits[2, 17 + i::5] = k  # every fifth token is left
        bits[3, i::4] = k
    bits[3, 4242] = bits[4, 4242]  # one token is left
    bits[4, 8990:] = kinds[0]
    x[5, :4096] = float("-inf")
    bits[5, 100:200] = kinds[0]
    vals = x.double().cpu().numpy()
    assert np.isnan(vals[3]).sum() == V - 1
    tokens = np.array([5, 2000, 17, 4242, 8999, 150, 3, 9000, 0])
    lp, rank, order, tol = expect_logprobs(vals, tokens, 6, softcap)
    r = sampler.logprobs(x, dev(tokens), top_n=6, softcap=softcap)
    torch.cuda.synchronize()
    at = np.arange(B)
    assert np.array_equal(r.ranks.cpu().numpy(), rank[at, tokens])
    assert np.array_equal(r.top_ids.cpu().numpy(), order)
    for got, want, t in ((r.logprobs, lp[at, tokens], tol[at, tokens]),
                         (r.top_logprobs, np.take_along_axis(lp, order, 1), np.take_along_axis(tol, order, 1))):
        got = got.double().cpu().numpy()
        inf = np.isinf(want)
        assert np.array_equal(got[inf], want[inf])
        assert (np.abs(got[~inf] - want[~inf]) <= t[~inf]).all()


def test_logprobs_tokens_past_the_vocabulary(sampler):
    lg = torch.zeros(3, 100, device="cuda:0")
    r = sampler.logprobs(lg, dev([100, -1, 5]), vocab=100)
    assert torch.isnan(r.logprobs[:2]).all() and (r.ranks[:2] == -1).all()
    assert r.ranks[2].item() == 5 and abs(r.logprobs[2].item() + math.log(100)) < 1e-5
    # the top list alone
    r = sampler.logprobs(lg, top_n=2)
    assert r.logprobs is None and r.top_ids.tolist() == [[0, 1]] * 3


def test_logprobs_more_rows_than_the_handle_holds():
    s = llmk.HipSampler(max_batch=2, max_vocab=1024)
    lg = np.random.default_rng(1).normal(0, 3, (40, 9000)).astype(np.float32)
    check_logprobs(s, lg, "f32", 5)
    check_logprobs(s, lg[:2], "f32", 5)
    s.close()


def test_process_then_logprobs_then_sample(sampler):
    """A step that answers with log-probabilities: the processed logits, their
    log-probabilities, a draw from them; the drawn token's log-probability is
    that of the probability the sampler reports (no top-k, no top-p)."""
    B, V = 16, 20011
    rng = np.random.default_rng(4)
    case = Case(rng, B, V, hist=300, mask=True)
    case.mask_index[case.mask_index == 1] = 0
    case.T[1] = 0.8
    _, view, _ = rows_on_device(case.lg, "bf16")
    x = sampler.process_logits(case.batch(view))
    d = sampler.sample_batch(llmk.DeviceBatch(logits=x, uniforms=dev(rng.random(B), torch.float32)),
                             out_cap=V)
    r = sampler.logprobs(x, d.tokens, top_n=20)
    check_logprobs(sampler, x.cpu().numpy(), "f32", 20, tokens=d.tokens.cpu().numpy())
    for b in range(B):
        at = int((d.ids[b, :int(d.count[b])] == d.tokens[b]).nonzero()[0])
        assert at == r.ranks[b].item()
        p = d.probs[b, at].item()
        # the sampler's sum is the sequential f32 one: V u at the very worst
        assert abs(math.log(p) - r.logprobs[b].item()) < V * U + 1e-5


# ---- streams, graphs, long offsets -------------------------------------------

def test_graph_replays(sampler):
    """Both calls captured into one graph (with two segments per row and the
    arrival counters that go with them), replayed on new inputs with eager calls
    and synchronizations in between."""
    B, V = 6, 9001
    rng = np.random.default_rng(3)
    case = Case(rng, B, V, hist=400, bias=20, mask=True)
    _, view, _ = rows_on_device(case.lg, "bf16")
    lb = case.batch(view)
    out = torch.empty(B, V, device="cuda:0")
    tok = dev(rng.integers(0, V, B))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        sampler.process_logits(lb, out=out)
        sampler.logprobs(out, tok, top_n=5)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sampler.process_logits(lb, out=out)
        r = sampler.logprobs(out, tok, top_n=5)
    for i in range(4):
        view.copy_(torch.randn(B, V, device="cuda:0") * (i + 1))
        tok.copy_(torch.randint(0, V, (B,), device="cuda:0"))
        g.replay()
        got = [t.clone() for t in (out, r.logprobs, r.ranks, r.top_ids, r.top_logprobs)]
        torch.cuda.synchronize()
        e = sampler.process_logits(lb)
        q = sampler.logprobs(e, tok, top_n=5)
        for x, y in zip(got, (e, q.logprobs, q.ranks, q.top_ids, q.top_logprobs)):
            assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


def test_another_stream(sampler):
    case = Case(np.random.default_rng(6), 8, 30000, hist=100)
    _, view, _ = rows_on_device(case.lg, "f32")
    lb, tok = case.batch(view), dev(np.arange(8))
    a = sampler.process_logits(lb)
    ra = sampler.logprobs(a, tok, top_n=4)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    out = torch.empty_like(a)
    sampler.process_logits(lb, out=out, stream=s)
    rb = sampler.logprobs(out, tok, top_n=4, stream=s)
    s.synchronize()
    assert torch.equal(a, out) and torch.equal(ra.logprobs, rb.logprobs) and torch.equal(ra.top_ids, rb.top_ids)


def test_outputs_of_another_stream_take_no_block_in_use(sampler):
    """A block freed on the current stream while work that reads it waits there
    is not what a call on another stream writes its results to."""
    B, V = 64, 50001
    lg, tok = torch.randn(B, V, device="cuda:0"), torch.zeros(B, dtype=torch.int32, device="cuda:0")
    cache = llmk.PageCache(sampler, B, 4, 16, 50001)
    grown = torch.ones(B, dtype=torch.int32, device="cuda:0")
    s = torch.cuda.Stream()
    calls = ((B * V, lambda: sampler.process_logits(llmk.LogitsBatch(logits=lg), stream=s)),
             (B * 20, lambda: sampler.logprobs(lg, tok, top_n=20, stream=s)),
             (B, lambda: cache.update(new_lengths=grown, stream=s)),
             (50001, lambda: cache.compact(stream=s)))
    for n, call in calls:
        x = torch.full((n,), 5.0, device="cuda:0")
        torch.cuda.synchronize()
        torch.cuda._sleep(20_000_000)
        y = x.clone()
        del x
        r = call()
        torch.cuda.synchronize()
        assert bool((y == 5.0).all())
        del r


def test_rows_past_32_bit_offsets(sampler):
    """A row stride of more than 2^31 elements (bf16: 4 GiB from row to row)."""
    V, stride = 3001, 2**31 + 8
    case = Case(np.random.default_rng(7), 2, V, hist=50)
    buf = torch.empty(stride + V + 8, dtype=torch.bfloat16, device="cuda:0")
    view = buf.as_strided((2, V), (stride, 1), 0)
    view.copy_(torch.as_tensor(case.lg))
    want, tol = case.expect(view.double().cpu().numpy())
    got = sampler.process_logits(case.batch(view))
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    _, _, order, _ = expect_logprobs(view.double().cpu().numpy(), np.array([5, 6]), 4, 0.0)
    r = sampler.logprobs(view, dev([5, 6]), top_n=4)
    assert np.array_equal(r.top_ids.cpu().numpy(), order)
    # and rows written that far apart, in place
    case.T = None
    want, tol = case.expect(view.double().cpu().numpy())
    sampler.process_logits(case.batch(view), out=view)
    half = torch.finfo(torch.bfloat16).eps / 2
    assert (np.abs(view.double().cpu().numpy() - want) <= tol * (1 + half) + np.abs(want) * half).all()


def test_tensors_of_another_device_are_refused(sampler):
    with pytest.raises(llmk.SamplerError, match="logits on|on cuda|the logits on"):
        sampler.process_logits(llmk.LogitsBatch(logits=torch.zeros(2, 8, device="cuda:0"),
                                                temperature=torch.ones(2)))
    with pytest.raises(llmk.SamplerError, match="tokens is on cpu"):
        sampler.logprobs(torch.zeros(2, 8, device="cuda:0"), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(llmk.SamplerError, match="entries"):
        sampler.logprobs(torch.zeros(2, 8, device="cuda:0"), dev([1]))
    with pytest.raises(llmk.SamplerError, match="rows, the logits have 2"):
        sampler.process_logits(llmk.LogitsBatch(logits=torch.zeros(2, 8, device="cuda:0"),
                                                temperature=dev([1.0], torch.float32)))


@pytest.mark.parametrize("T", [0.7, 1.2, 0.0313, 1.9999999, 3.0, 2e-5, 4.9e5, 1e7])
def test_division_by_the_temperature_is_the_division(sampler, T):
    """Bit for bit IEEE's quotient, from the smallest numbers to the largest:
    every exponent, random significands, zeros of both signs, infinities."""
    g = torch.Generator(device="cuda:0")
    g.manual_seed(int(T * 1000))
    n = 1 << 20
    bits = torch.randint(-2**31, 2**31 - 1, (n,), generator=g, device="cuda:0").int()
    x = bits.view(torch.float32)
    x = torch.where(torch.isnan(x), torch.randn(n, generator=g, device="cuda:0"), x)
    x[:n // 2] = torch.randn(n // 2, generator=g, device="cuda:0") * 8
    x[5], x[9], x[77], x[81] = 0.0, -0.0, float("inf"), float("-inf")
    x = x.view(4, n // 4)
    t = torch.full((4,), T, device="cuda:0")
    got = sampler.process_logits(llmk.LogitsBatch(logits=x, temperature=t))
    assert torch.equal(got.view(torch.int32), (x / t[:, None]).view(torch.int32))


@pytest.mark.parametrize("inplace", [False, True])
def test_process_a_segment_with_thousands_of_history_tokens(sampler, inplace):
    """Nearly every token of the row is in the history, some many times, with
    biases: more than a segment lists."""
    case = Case(np.random.default_rng(31), 3, 20000, hist=60000, bias=5000, T=not inplace, twice=True)
    check_process(sampler, case, "f32", inplace=inplace)
    case = Case(np.random.default_rng(32), 80, 9000, hist=30000, T=not inplace)
    check_process(sampler, case, "bf16", "same", inplace=inplace)


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("bf16", "same"),
                                       ("f16", "f32"), ("f16", "same")])
@pytest.mark.parametrize("B,softcap", [(1041, 0.0), (528, 25.0)])
def test_process_many_rows(sampler, dtype, out, B, softcap):
    """Enough rows for long segments, with rows in eights and not."""
    case = Case(np.random.default_rng(B), B, 5003, chain=1 if softcap else 3, hist=600, bias=40, mask=True,
                softcap=softcap)
    check_process(sampler, case, dtype, out, 1, 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_process_many_rows_in_place_with_full_lists(sampler, dtype):
    case = Case(np.random.default_rng(33), 520, 4500, hist=12000, T=False)
    check_process(sampler, case, dtype, "same", inplace=True)


def test_empty_lists_and_batches(sampler):
    """Histories, extra tokens and biases that hold nothing at all; no rows."""
    lg = torch.randn(3, 1000, device="cuda:0")
    none = torch.empty(0, dtype=torch.int32, device="cuda:0")
    zeros = torch.zeros(4, dtype=torch.int32, device="cuda:0")
    lb = llmk.LogitsBatch(logits=lg, hist_offsets=zeros, hist_tokens=none, hist_counts=none,
                          extra_begin=zeros, extra_count=zeros, extra_tokens=none, bias_offsets=zeros,
                          bias_tokens=none, bias_values=none.float(),
                          repetition_penalty=torch.full((3,), 1.5, device="cuda:0"))
    assert torch.equal(sampler.process_logits(lb), lg)
    assert sampler.process_logits(llmk.LogitsBatch(logits=lg[:0])).shape == (0, 1000)
    r = sampler.logprobs(lg[:0], none, top_n=3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)
    with pytest.raises(llmk.SamplerError, match="Empty"):
        sampler.process_logits(llmk.LogitsBatch(logits=lg[:, :0]))
    with pytest.raises(llmk.SamplerError, match="Empty"):
        sampler.logprobs(lg[:, :0], zeros[:3])


def test_a_bias_of_minus_infinity_bans_a_token(sampler):
    """-inf as a bias, on a token of the history and off it; +inf and -inf on one
    token are NaN; a NaN bias."""
    lg = torch.ones(1, 50, device="cuda:0")
    inf = float("inf")
    lb = llmk.LogitsBatch(logits=lg, hist_offsets=dev([0, 2]), hist_tokens=dev([4, 5]),
                          presence_penalty=dev([0.5], torch.float32), bias_offsets=dev([0, 5]),
                          bias_tokens=dev([4, 9, 11, 11, 12]),
                          bias_values=dev([-inf, -inf, inf, -inf, float("nan")], torch.float32))
    g = sampler.process_logits(lb)[0].cpu()
    assert g[4] == -inf and g[9] == -inf and g[5] == 0.5 and g[0] == 1
    assert torch.isnan(g[[11, 12]]).all() and int(torch.isnan(g).sum()) == 2


def test_two_calls_at_once(sampler):
    """process_logits keeps nothing between the workgroups of a call: calls that
    overlap on two streams do not disturb each other."""
    cases = [Case(np.random.default_rng(40 + i), 64, 50000, hist=800, bias=30) for i in range(2)]
    lbs = [c.batch(rows_on_device(c.lg, "f32")[1]) for c in cases]
    alone = [sampler.process_logits(lb) for lb in lbs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(a) for a in alone]
    for _ in range(5):
        for lb, o, s in zip(lbs, outs, streams):
            sampler.process_logits(lb, out=o, stream=s)
    torch.cuda.synchronize()
    for a, o in zip(alone, outs):
        assert torch.equal(a, o)


def test_two_graphs_of_one_handle(sampler):
    """Two captured calls that share the handle's workspace, replayed in turn."""
    lg = [torch.randn(5, 30000, device="cuda:0"), torch.randn(7, 50000, device="cuda:0").bfloat16()]
    tok = [dev(np.arange(5)), dev(np.arange(7))]
    graphs, outs = [], []
    for x, t in zip(lg, tok):
        sampler.logprobs(x, t, top_n=6)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sampler.logprobs(x, t, top_n=6))
        graphs.append(g)
    for i in range(4):
        for x in lg:
            x.copy_(torch.randn(x.shape, device="cuda:0") * (i + 1))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, t, r in zip(lg, tok, outs):
            e = sampler.logprobs(x, t, top_n=6)
            assert torch.equal(r.logprobs, e.logprobs) and torch.equal(r.ranks, e.ranks)
            assert torch.equal(r.top_ids, e.top_ids) and torch.equal(r.top_logprobs, e.top_logprobs)
