"""The operators around a sampling step, as measurable cases.

Three kinds of work that a serving loop does next to HipSampler.sample_batch:

  "process"   HipSampler.process_logits: softcap, logit bias, penalties over the
              token histories, grammar masks and temperature, into new logits
  "logprobs"  HipSampler.logprobs: log-probability and rank of one token per
              row, and the likeliest tokens
  "update", "compact", "copy"
              the pages of a cache (llmk.PageCache): rows fork, grow, shrink
              and end; live pages move to the front; pages are copied

With `own` false, run() computes them with elementary torch operations; with
it true, through the framework.  Cases are dicts of plain values:

  process    B rows of V logits of dtype, `out` "f32" or "same"; `chain` rows
             per sequence (a speculative chain's positions share a history,
             and each has the drafts before it as extra tokens); `hist` tokens
             as "csr", per-row "buffers" or (token, count) tables "counts";
             rep/pres/freq/T (None: not given); `bias` pairs per sequence;
             `mask` grammar states shared by the rows; softcap; `pad` elements
             between rows past V; `inplace`: on a copy of the logits
  logprobs   B, V, dtype, `top` likeliest tokens, softcap, pad
  update     `rows` of the table, `page` tokens per page, rows of `low` to
             `high` tokens; `forks` children per forked row (0: no forks); a
             few rows end and a few begin; `tight`: too few pages for all of
             them; pools of `bytes` per page
  compact    rows, page, low, high, the share `live` of rows that remain
  copy       `n` of `pages` pages, pools of `bytes` per page
"""
import math
import os
import sys

import torch

own = False

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-rs_amd"))

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one user decoding: the smallest call, all latency
        dict(name="process_1", kind="process", B=1, V=151936, dtype="f32", out="f32", chain=1,
             hist=64, form="csr", rep=1.1, pres=None, freq=None, T=0.8, bias=0, mask=0,
             softcap=0.0, pad=0, inplace=False),
        # speculative verification of structured output: 64 sequences, five
        # positions each, bf16 logits of an odd vocabulary and stride, a
        # logit_bias map per request, a grammar state per position
        dict(name="process_chain_320", kind="process", B=320, V=50257, dtype="bf16", out="f32",
             chain=5, hist=700, form="buffers", rep=1.1, pres=0.2, freq=0.1, T=None, bias=40,
             mask=48, softcap=0.0, pad=0, inplace=False),
        # a full decode batch, every penalty on
        dict(name="process_256", kind="process", B=256, V=151936, dtype="f32", out="f32", chain=1,
             hist=2048, form="csr", rep=1.1, pres=0.5, freq=0.3, T=0.7, bias=0, mask=0,
             softcap=0.0, pad=0, inplace=False),
        # one user's token with the twenty alternatives an API returns
        dict(name="logprobs_1", kind="logprobs", B=1, V=128256, dtype="bf16", top=20, softcap=0.0, pad=0),
        # every request of a decode batch asks for alternatives
        dict(name="logprobs_256", kind="logprobs", B=256, V=151936, dtype="f32", top=8, softcap=0.0, pad=0),
        # scoring a prompt: the log-probability of each of its tokens
        dict(name="logprobs_prompt", kind="logprobs", B=2047, V=32000, dtype="f16", top=1, softcap=0.0, pad=0),
        # a decode step: every row grows by a token, a few end, a few begin
        dict(name="pages_step", kind="update", rows=256, page=16, low=100, high=8000, forks=0,
             bytes=4096, pools=2, tight=False),
        # several samples per prompt: long rows fork, and each copy of a
        # partial last page comes with its first token
        dict(name="pages_fork", kind="update", rows=320, page=32, low=2000, high=30000, forks=4,
             bytes=8192, pools=4, tight=False),
        # a small cache after most of its rows ended
        dict(name="compact_small", kind="compact", rows=64, page=16, low=50, high=1000, live=0.4,
             bytes=2048, pools=2),
        # a large one, moved whole in one go
        dict(name="compact_large", kind="compact", rows=384, page=64, low=500, high=6000, live=0.5,
             bytes=32768, pools=2),
        # a few shared pages made private
        dict(name="copy_few", kind="copy", n=24, pages=1024, bytes=8192, pools=8),
        # a long prefix duplicated
        dict(name="copy_many", kind="copy", n=4000, pages=9001, bytes=32768, pools=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any batch and vocabulary up to 39 million logits, any
    mix of penalties, masks, biases and layouts; caches of any page size."""
    kind = rng.choice(["process"] * 3 + ["logprobs"] * 2 + ["update", "compact", "copy"])
    if kind in ("process", "logprobs"):
        v = _log(rng, 2000, 256000)
        b = _log(rng, 1, min(2048, 38_000_000 // v))
        d = rng.choice(["f32", "bf16", "f16"])
        sc, pad = rng.choice([0.0, 0.0, 0.0, 30.0]), rng.choice([0, 0, 1, 7, 64])
        if kind == "logprobs":
            return dict(kind=kind, B=b, V=v, dtype=d, top=rng.choice([0, 1, 5, 8, 20]), softcap=sc, pad=pad)
        chain = rng.choice([1, 1, 2, 5])
        b = max(chain, b // chain * chain)
        h = rng.choice([0, 1, 130, 700, 2048, 4096])
        inplace = rng.random() < 0.3
        return dict(kind=kind, B=b, V=v, dtype=d, out="same" if inplace else rng.choice(["f32", "same"]),
                    chain=chain, hist=h, form=rng.choice(["csr", "buffers", "counts"]),
                    rep=rng.choice([None, 1.1, 1.3]), pres=rng.choice([None, 0.5]),
                    freq=rng.choice([None, 0.3]), T=rng.choice([None, 0.7, 1.2]),
                    bias=rng.choice([0, 0, 10, 300]), mask=rng.choice([0, 0, 1, 40]),
                    softcap=sc, pad=pad, inplace=inplace)
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if kind == "update":
        forks = rng.choice([0, 0, 1, 3, 4])
        low = _log(rng, 1, 2000)
        c = dict(kind=kind, rows=_log(rng, 4, 512), page=page, low=low, high=low + _log(rng, 10, 10000),
                 forks=forks, bytes=rng.choice([64, 1000, 2048, 4096]), pools=rng.choice([1, 2, 3]),
                 tight=rng.random() < 0.25)
    if kind == "compact":
        low = _log(rng, 1, 500)
        c = dict(kind=kind, rows=_log(rng, 2, 400), page=page, low=low, high=low + _log(rng, 10, 4000),
                 live=rng.choice([0.1, 0.5, 0.9]), bytes=rng.choice([60, 1024, 4096, 8192]),
                 pools=rng.choice([1, 2, 4]))
    if kind in ("update", "compact"):  # a cache of a gigabyte at most
        most = 500_000_000 // (c["bytes"] * c["pools"] + 8)
        c["rows"] = max(4, min(c["rows"], most // (c["high"] // page + 1)))
        return c
    n = _log(rng, 1, 4000)
    return dict(kind=kind, n=n, pages=2 * n + rng.randrange(1, 1000), bytes=rng.choice([12, 2048, 8192, 20480]),
                pools=rng.choice([1, 2, 4]))


# ---- inputs, made on the GPU from the seed alone -----------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randint(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _logits(c, g):
    """A bulk of normal logits and, per row, a falling series of likely tokens,
    in rows of V + pad elements."""
    B, V = c["B"], c["V"]
    lg = torch.randn(B, V + c["pad"], generator=g, device="cuda").mul_(2.5)
    k = 64
    step = V // k
    at = _randint(g, 0, step, B, k) + torch.arange(k, device="cuda") * step
    order = _rand(g, B, k).argsort(1).float()
    lg.scatter_(1, at, _rand(g, B, 1) * 8 + 10 - order * (_rand(g, B, 1) * 0.35 + 0.05))
    return lg.to(_DT[c["dtype"]])[:, :V]


def _zipf(g, rows, n, V):
    """[rows, n] token ids, Zipf(1) ranks of one permuted vocabulary."""
    u = torch.rand(rows, n, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(V + 1)).long() - 1).clamp_(0, V - 1)
    return torch.randperm(V, generator=g, device="cuda")[rank]


def _grammar(g, n, V):
    """int32 [n, words]: runs of 8..64 allowed tokens, a few per cent of the row."""
    runs = max(1, V * 3 // 100 // 36)
    s = _randint(g, 0, max(1, V - 64), n, runs)
    w = _randint(g, 8, 65, n, runs)
    words = (V + 31) // 32
    d = torch.zeros(n, words * 32 + 1, dtype=torch.int32, device="cuda")
    one = torch.ones(n, runs, dtype=torch.int32, device="cuda")
    d.scatter_add_(1, s, one)
    d.scatter_add_(1, (s + w).clamp_(max=V), -one)
    bits = (d.cumsum(1)[:, :-1] > 0).view(n, words, 32)
    out = torch.zeros(n, words, dtype=torch.int64, device="cuda")
    for i in range(32):
        out += bits[:, :, i].long() << i
    return torch.where(out >= 2**31, out - 2**32, out).int()


def _process_inputs(c, seed):
    g = _gen(seed)
    B, V, S = c["B"], c["V"], c["B"] // c["chain"]
    x = {"logits": _logits(c, g)}
    for key, name in (("rep", "repetition_penalty"), ("pres", "presence_penalty"),
                      ("freq", "frequency_penalty"), ("T", "temperature")):
        if c[key] is not None:  # requests differ a little from each other
            x[name] = c[key] * (1 + 0.1 * _rand(g, S))
    if c["hist"]:
        h = _zipf(g, S, c["hist"], V)
        n = _randint(g, max(1, c["hist"] // 2), c["hist"] + 1, S)  # tokens of each
        keep = torch.arange(c["hist"], device="cuda")[None, :] < n[:, None]
        row = torch.arange(S, device="cuda")[:, None].expand(S, c["hist"])
        x["hist_row"], x["hist_tok"] = row[keep], h[keep]  # occurrences in order, for exact()
        if c["form"] == "buffers":  # a buffer of hist tokens per sequence
            x["hist_offsets"] = (torch.arange(S, device="cuda") * c["hist"]).int()
            x["hist_lengths"] = n.int()
            x["hist_tokens"] = h.reshape(-1).int()
        elif c["form"] == "csr":
            x["hist_offsets"] = torch.cat([torch.zeros(1, device="cuda"), n.cumsum(0)]).int()
            x["hist_tokens"] = h[keep].int()
        else:
            key, cnt = torch.unique(x["hist_row"] * V + x["hist_tok"], return_counts=True)
            x["hist_offsets"] = torch.searchsorted(key, torch.arange(S + 1, device="cuda") * V).int()
            x["hist_tokens"], x["hist_counts"] = (key % V).int(), cnt.int()
    if c["chain"] > 1:
        k = c["chain"]
        x["row_seq"] = (torch.arange(B, device="cuda") // k).int()
        x["extra_tokens"] = _zipf(g, S, k - 1, V).reshape(-1).int()
        x["extra_begin"] = x["row_seq"] * (k - 1)
        x["extra_count"] = (torch.arange(B, device="cuda") % k).int()
    if c["bias"]:
        m = min(c["bias"], V // 4)
        step = V // m
        at = _randint(g, 0, step, S, m) + torch.arange(m, device="cuda") * step
        x["bias_offsets"] = (torch.arange(S + 1, device="cuda") * m).int()
        x["bias_tokens"] = at.reshape(-1).int()
        x["bias_values"] = (_rand(g, S, m) * 20 - 10).reshape(-1)
    if c["mask"]:
        x["allow_mask"] = _grammar(g, c["mask"], V)
        # one row in eight is free of a grammar
        i = _randint(g, 0, c["mask"], B)
        x["mask_index"] = torch.where(_rand(g, B) < 0.125, -1, i).int()
    return x


def _pools(g, c, pages):
    """Each pool [pages, bytes]: what a page holds is of no matter."""
    return [torch.randint(0, 256, (pages, c["bytes"]), generator=g, device="cuda", dtype=torch.uint8)
            for _ in range(c["pools"])]


def _lens(g, c, rows):
    """Row lengths, evenly spread from low to high, in an order of their own."""
    n = torch.linspace(c["low"], c["high"], rows, device="cuda").round().long()
    return n[torch.randperm(rows, generator=g, device="cuda")]


def _fill(g, c, lens, N, P):
    """A cache in the middle of its life: rows of `lens` tokens whose pages lie
    anywhere among the N pages."""
    need = (lens + c["page"] - 1) // c["page"]
    total = int(need.sum())
    perm = torch.randperm(N, generator=g, device="cuda")[:total]
    table = torch.full((lens.numel(), P), 7, dtype=torch.int64, device="cuda")
    table[torch.arange(P, device="cuda")[None, :] < need[:, None]] = perm
    refs = torch.zeros(N, dtype=torch.int64, device="cuda")
    refs[perm] = 1
    return table.int().contiguous(), lens.int(), refs.int()


def _update_inputs(c, seed):
    g = _gen(seed)
    R, ps = c["rows"], c["page"]
    row = torch.arange(R, device="cuda")
    # a quarter of the pages is free, or only about what a third of the rows ask for
    if c["forks"]:
        # the first rows hold prompts, the rest are their children to be
        k = max(1, R // (c["forks"] + 1))
        lens = torch.cat([_lens(g, c, k), torch.zeros(R - k, dtype=torch.int64, device="cuda")])
        parents = torch.where(row < k, -1, row % k)
        grown = lens[row % k] + 1
        total = int(((lens + ps - 1) // ps).sum())
        N = total + (R // 3 + 1 if c["tight"] else total // 4 + 2 * R)
    else:
        parents = torch.full((R,), -1, device="cuda")
        lens, prompt = _lens(g, c, R), _lens(g, c, R)
        total = int(((lens + ps - 1) // ps).sum())
        N = total + (R // 3 + 1 if c["tight"] else total // 4 + R)
        k = max(1, R // 25)  # rows of each kind
        order = torch.randperm(R, generator=g, device="cuda")
        grown = lens + 1
        lens[order[:k]] = 0  # begin
        grown[order[:k]] = c["high"] if c["tight"] else prompt[order[:k]]
        grown[order[k:2 * k]] = 0  # end
        grown[order[2 * k:3 * k]] = -1  # wait
    table, lens32, refs = _fill(g, c, lens, N, c["high"] // ps + 3)
    return dict(table=table, lengths=lens32, refs=refs, parents=parents.int(),
                grown=grown.int(), pools=_pools(g, c, N))


def _compact_inputs(c, seed):
    g = _gen(seed)
    R, ps = c["rows"], c["page"]
    lens = _lens(g, c, R)
    total = int(((lens + ps - 1) // ps).sum())
    P, N = c["high"] // ps + 2, total + total // 4 + 1
    table, lens32, refs = _fill(g, c, lens, N, P)
    gone = _rand(g, R) >= c["live"]  # the rows that ended
    gone[0] = False
    held = torch.arange(P, device="cuda")[None, :] < ((lens + ps - 1) // ps)[:, None]
    refs[table[held & gone[:, None]].long()] = 0
    lens32 = torch.where(gone, 0, lens32)
    # two rows share the first half of a prompt
    half = int(lens[0]) // 2 // ps
    refs[table[1, :(int(lens32[1]) + ps - 1) // ps].long()] = 0
    table[1, :half] = table[0, :half]
    refs[table[0, :half].long()] += 1
    lens32[1] = half * ps
    return dict(table=table, lengths=lens32, refs=refs, pools=_pools(g, c, N))


def prepare(case, seed):
    c = dict(case)
    s = {"case": c}
    if c["kind"] == "process":
        x = _process_inputs(c, seed)
        s.update(x)
        out = _DT[c["dtype"]] if c["out"] == "same" else torch.float32
        s["out"] = (torch.zeros(c["B"], c["V"] + c["pad"], dtype=out, device="cuda")[:, :c["V"]])
        if own:
            import llmk
            s["sampler"] = llmk.HipSampler(max_batch=c["B"], max_vocab=c["V"])
            names = ("repetition_penalty", "presence_penalty", "frequency_penalty", "temperature",
                     "hist_offsets", "hist_tokens", "hist_lengths", "hist_counts", "row_seq",
                     "extra_begin", "extra_count", "extra_tokens", "bias_offsets", "bias_tokens",
                     "bias_values", "allow_mask", "mask_index")
            s["batch"] = llmk.LogitsBatch(logits=s["out"] if c["inplace"] else s["logits"],
                                          softcap=c["softcap"], **{k: x.get(k) for k in names})
    elif c["kind"] == "logprobs":
        g = _gen(seed)
        s["logits"] = _logits(c, g)
        # the row's sampled token: among the likely ones as a rule
        noisy = s["logits"].float()
        noisy = noisy + torch.randn(noisy.shape, generator=g, device="cuda")
        s["tokens"] = noisy.argmax(1).int()
        if own:
            import llmk
            s["sampler"] = llmk.HipSampler(max_batch=c["B"], max_vocab=c["V"])
    elif c["kind"] == "copy":
        g = _gen(seed)
        s["pools"] = _pools(g, c, c["pages"])
        at = torch.randperm(c["pages"], generator=g, device="cuda")[:2 * c["n"]].int()
        s["src"], s["dst"] = at[:c["n"]].contiguous(), at[c["n"]:].contiguous()
        if own:
            import llmk
            s["sampler"] = llmk.HipSampler(max_batch=1, max_vocab=1024)
            s["pages"] = llmk.PagePools(s["pools"])
    else:
        s.update((_update_inputs if c["kind"] == "update" else _compact_inputs)(c, seed))
        N, (R, P) = s["refs"].numel(), s["table"].shape
        if own:
            import llmk
            s["sampler"] = llmk.HipSampler(max_batch=1, max_vocab=1024)
            s["cache"] = llmk.PageCache(s["sampler"], rows=R, max_pages=P, page_tokens=c["page"],
                                        num_pages=N, pools=s["pools"])
            s["cache"].load(s["table"], s["lengths"])
            s["before"] = s["cache"].state.clone()
        else:
            s["before"] = torch.cat([s["refs"], s["lengths"], s["table"].reshape(-1)])
            s["now"] = s["before"].clone()
    return s


# ---- the plain forms ---------------------------------------------------------

def _flat_rows(offsets, n):
    """The row of each of n CSR entries."""
    at = torch.arange(n, device="cuda")
    return torch.searchsorted(offsets.long(), at, right=True) - 1


def _process_plain(s):
    c = s["case"]
    B, V, S = c["B"], c["V"], c["B"] // c["chain"]
    get = s.get
    x = s["logits"].float()
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    seq = s["row_seq"].long() if "row_seq" in s else None
    per_row = (lambda t: t[:, None] if seq is None else t[seq][:, None])  # noqa: E731
    if c["bias"]:
        m = s["bias_tokens"].numel()
        b = torch.zeros(S * V, device="cuda")
        b.index_add_(0, _flat_rows(s["bias_offsets"], m) * V + s["bias_tokens"].long(), s["bias_values"])
        b = b.view(S, V)
        x = x + (b if seq is None else b[seq])
    if c["hist"] or seq is not None:
        n = torch.zeros(S * V, device="cuda")
        if c["hist"]:
            t = s["hist_tokens"].long()
            i = torch.arange(t.numel(), device="cuda")
            if c["form"] == "buffers":
                row = i // c["hist"]
                w = (i % c["hist"] < s["hist_lengths"][row]).float()
            else:
                row = _flat_rows(s["hist_offsets"], t.numel())
                w = s["hist_counts"].float() if c["form"] == "counts" else torch.ones(t.numel(), device="cuda")
            n.index_add_(0, row * V + t, w)
        n = n.view(S, V)
        if seq is not None:
            n = n[seq]
            k = c["chain"]
            e = torch.arange(k - 1, device="cuda")[None, :]
            tok = s["extra_tokens"].long()[s["extra_begin"].long()[:, None] + e]
            n.scatter_add_(1, tok, (e < s["extra_count"][:, None]).float())
        seen = n > 0
        y = x
        if get("repetition_penalty") is not None:
            r = per_row(s["repetition_penalty"])
            y = torch.where(y > 0, y / r, y * r)
        if get("presence_penalty") is not None or get("frequency_penalty") is not None:
            d = 0.0
            if get("frequency_penalty") is not None:
                d = n * per_row(s["frequency_penalty"])
            if get("presence_penalty") is not None:
                d = per_row(s["presence_penalty"]) + d
            y = y - d
        x = torch.where(seen, y, x)
    if c["mask"]:
        i = s["mask_index"].long()
        w = s["allow_mask"][i.clamp(min=0)]
        e = torch.arange(V, device="cuda")
        ok = (w[:, e >> 5] >> (e & 31).int()[None, :]) & 1
        x = torch.where((ok == 1) | (i < 0)[:, None], x, float("-inf"))
    if get("temperature") is not None:
        x = x / per_row(s["temperature"])
    s["out"].copy_(x)
    return s["out"]


def _order(lg):
    """Keys whose order is (logit descending, index ascending)."""
    b = (lg.float() + 0.0).view(torch.int32).long()  # -0 is 0
    k = torch.where(b < 0, -1 - (b & 0x7FFFFFFF), b)
    return (k << 20) + (lg.shape[1] - 1 - torch.arange(lg.shape[1], device="cuda"))


def _logprobs_plain(s):
    c = s["case"]
    lg, t = s["logits"], s["tokens"].long()[:, None]
    x = lg.float()
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    m = x.amax(1, keepdim=True)
    z = torch.log(torch.exp(x - m).sum(1, keepdim=True))
    lt = lg.gather(1, t)
    e = torch.arange(c["V"], device="cuda")
    out = {"logprobs": ((x.gather(1, t) - m) - z)[:, 0],
           "ranks": ((lg > lt).sum(1) + ((lg == lt) & (e < t)).sum(1)).int()}
    if c["top"]:
        ids = (c["V"] - 1) - (_order(lg).topk(c["top"], 1).values & 0xFFFFF)
        out["top_ids"], out["top_logprobs"] = ids.int(), (x.gather(1, ids) - m) - z
    return out


def _state(s):
    """The cache's arrays, as they were before the call."""
    s["now"].copy_(s["before"])
    N, R = s["refs"].numel(), s["lengths"].numel()
    refs, lengths, table = s["now"][:N], s["now"][N:N + R], s["now"][N + R:].view(R, -1)
    return refs, lengths, table


def _update_plain(s):
    c = s["case"]
    ps = c["page"]
    refs, lengths, table = _state(s)
    N, (R, P) = refs.numel(), table.shape
    col = torch.arange(P, device="cuda")[None, :]
    parent, new = s["parents"].long(), s["grown"].long()
    pages = lambda n: (n + ps - 1) // ps  # noqa: E731
    # forks: the child's table begins as the parent's
    par = parent.clamp(min=0)
    child = parent >= 0
    ln = lengths.long()
    flen = torch.where(new >= 0, torch.minimum(ln[par], new), ln[par])
    cur = torch.where(child, flen, ln)
    tab = table.long()
    held = child[:, None] & (col < pages(cur)[:, None])
    tab = torch.where(held, tab[par], tab)
    # entries past N of `ref` take what no page is meant by
    sink = N + torch.arange(R * P, device="cuda")
    sink_row = sink[:R]
    ref = torch.cat([refs.long(), torch.zeros(R * P, dtype=torch.int64, device="cuda")])
    ref.index_add_(0, torch.where(held.reshape(-1), tab.reshape(-1), sink), held.reshape(-1).long())
    # rows that shrink or end give their pages back
    less = (new >= 0) & (new < cur)
    drop = less[:, None] & (col >= pages(new)[:, None]) & (col < pages(cur)[:, None])
    ref.index_add_(0, torch.where(drop.reshape(-1), tab.reshape(-1), sink), -drop.reshape(-1).long())
    cur = torch.where(less, new, cur)
    ref[N:] = 1
    # rows that grow; one whose partial last page is shared gets a copy of it,
    # but for the last of its holders when all of them grow
    grow = new > cur
    last = tab.gather(1, torch.clamp(cur // ps, max=P - 1)[:, None])[:, 0]
    tied = grow & (cur % ps != 0)
    tied = tied & (ref[torch.where(tied, last, sink_row)] > 1)
    row = torch.arange(R, device="cuda")
    at = torch.where(tied, last, sink_row)
    who = torch.zeros(N + R, dtype=torch.int64, device="cuda").index_add_(0, at, tied.long())
    top = torch.full((N + R,), -1, dtype=torch.int64, device="cuda").scatter_reduce_(0, at, row, "amax")
    keeps = tied & (who[at] == ref[at]) & (top[at] == row)
    own_copy = tied & ~keeps
    need = torch.where(grow, pages(new) - pages(cur) + own_copy.long(), 0)
    free = ref[:N] == 0
    upto = need.cumsum(0)
    refused = grow & (upto > free.sum()) & ((need > 0) | keeps)
    go = grow & ~refused
    order = torch.zeros(2 * N, dtype=torch.int64, device="cuda")  # free pages, lowest first
    order.scatter_(0, torch.where(free, free.long().cumsum(0) - 1, N + torch.arange(N, device="cuda")),
                   torch.arange(N, device="cuda"))
    first = upto - need
    cp = go & own_copy
    dst = order[torch.where(cp, first, 0)]
    ref.index_add_(0, torch.where(cp, last, sink_row), -cp.long())
    more = go[:, None] & (col >= pages(cur)[:, None]) & (col < pages(new)[:, None])
    pick = first[:, None] + own_copy[:, None].long() + (col - pages(cur)[:, None])
    got = order[torch.where(more, pick, 0)]
    tab = torch.where(more, got, tab)
    tab = torch.where(cp[:, None] & (col == (cur // ps)[:, None]), dst[:, None], tab)
    ref.index_fill_(0, torch.where(more.reshape(-1), got.reshape(-1), sink), 1)
    ref.index_fill_(0, torch.where(cp, dst, sink_row), 1)
    refs.copy_(ref[:N])
    lengths.copy_(torch.where(go, new, cur))
    table.copy_(tab)
    # the copies: rows without one repeat the first of them, so that no page is
    # written in two ways (page 0 onto itself if no row has one)
    a, b = torch.where(cp, last, 0), torch.where(cp, dst, 0)
    k = cp.long().argmax(0, keepdim=True)
    a, b = torch.where(cp, a, a[k]), torch.where(cp, b, b[k])
    for p in s["pools"]:
        p.index_copy_(0, b, p[a])
    return {"granted": (~refused).int(), "lengths": lengths, "refs": refs, "table": table, "pools": s["pools"]}


def _compact_plain(s):
    c = s["case"]
    refs, lengths, table = _state(s)
    N, (R, P) = refs.numel(), table.shape
    col = torch.arange(P, device="cuda")[None, :]
    page = torch.arange(N, device="cuda")
    used = refs > 0
    live = used.sum()
    src, dst = used & (page >= live), ~used & (page < live)
    away = N + page
    hole = torch.zeros(2 * N, dtype=torch.int64, device="cuda")
    hole.scatter_(0, torch.where(dst, dst.long().cumsum(0) - 1, away), page)
    to = torch.where(src, hole[torch.where(src, src.long().cumsum(0) - 1, away)], page)
    now = torch.zeros(2 * N, dtype=refs.dtype, device="cuda")
    now.scatter_(0, torch.where(used, to, away), refs)
    refs.copy_(now[:N])
    held = col < ((lengths.long() + c["page"] - 1) // c["page"])[:, None]
    t = table.long()
    table.copy_(torch.where(held, to[torch.where(held, t, 0)], t))
    for p in s["pools"]:
        a = src.nonzero()[:, 0]
        p[to[a]] = p[a]
    return {"map": to.int(), "lengths": lengths, "refs": refs, "table": table, "pools": s["pools"]}


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        if kind == "copy":
            for p in s["pools"]:
                p[s["dst"].long()] = p[s["src"].long()]
            return s["pools"]
        return {"process": _process_plain, "logprobs": _logprobs_plain, "update": _update_plain,
                "compact": _compact_plain}[kind](s)
    if kind == "process":
        if c["inplace"]:
            s["out"].copy_(s["logits"])
        return s["sampler"].process_logits(s["batch"], out=s["out"])
    if kind == "logprobs":
        r = s["sampler"].logprobs(s["logits"], s["tokens"], top_n=c["top"], softcap=c["softcap"])
        out = {"logprobs": r.logprobs, "ranks": r.ranks}
        if c["top"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    if kind == "copy":
        s["sampler"].copy_pages(s["pages"], s["src"], s["dst"])
        return s["pools"]
    cache = s["cache"]
    cache.state.copy_(s["before"])
    if kind == "update":
        out = {"granted": cache.update(s["grown"], s["parents"])}
    else:
        out = {"map": cache.compact()}
    out.update(lengths=cache.lengths, refs=cache.refs, table=cache.table, pools=s["pools"])
    return out


def work(case):
    """Each input read once, each output written once."""
    c = dict(case)
    if c["kind"] == "process":
        B, V, S = c["B"], c["V"], c["B"] // c["chain"]
        n = B * V * (_SIZE[c["dtype"]] + (4 if c["out"] == "f32" else _SIZE[c["dtype"]]))
        n += S * c["hist"] * 3 + S * c["bias"] * 8 + 32 * B
        if c["mask"]:
            n += 4 * min(c["mask"], B) * ((V + 31) // 32)
        return {"bytes": n, "flops": B * V * (1 + (c["softcap"] > 0) * 20 + (c["T"] is not None))}
    if c["kind"] == "logprobs":
        return {"bytes": c["B"] * (c["V"] * _SIZE[c["dtype"]] + 12 + 8 * c["top"]),
                "flops": c["B"] * c["V"] * (4 + (c["softcap"] > 0) * 20)}
    if c["kind"] == "copy":
        return {"bytes": 2 * c["n"] * c["bytes"] * c["pools"] + 8 * c["n"], "flops": 0}
    mean = (c["low"] + c["high"]) // 2 // c["page"] + 1
    if c["kind"] == "update":
        n, copies = 24 * c["rows"], 0
        if c["forks"]:  # tables of the children, references, the last pages
            kids = c["rows"] - c["rows"] // (c["forks"] + 1)
            n += kids * mean * 16
            copies = kids
        else:  # about one row in twenty-five ends, one begins
            n += max(1, c["rows"] // 25) * 2 * mean * 8
        return {"bytes": n + 2 * copies * c["bytes"] * c["pools"], "flops": 0}
    pages = c["rows"] * mean
    moved = int(pages * c["live"] * (1 - c["live"] / 1.25))  # live pages past the live count
    return {"bytes": 2 * moved * c["bytes"] * c["pools"] + int(pages * c["live"]) * 8 + pages * 5, "flops": 0}


# ---- the same results in 64 bits ----------------------------------------------

def exact(case, seed):
    c = dict(case)
    if c["kind"] == "process":
        return _process_exact(c, seed)
    if c["kind"] == "logprobs":
        return _logprobs_exact(c, seed)
    return None  # pages are whole numbers


def _process_exact(c, seed):
    x = _process_inputs(c, seed)
    B, V, k = c["B"], c["V"], c["chain"]
    out = torch.empty(B, V, dtype=torch.float64, device="cuda")
    if c["hist"]:
        first = torch.searchsorted(x["hist_row"], torch.arange(B // k + 1, device="cuda")).tolist()
    value = lambda name, q, d: float(x[name][q]) if name in x else d  # noqa: E731
    for b in range(B):
        q = b // k
        v = x["logits"][b].double()
        if c["softcap"]:
            v = torch.tanh(v / c["softcap"]) * c["softcap"]
        if c["bias"]:
            m = x["bias_tokens"].numel() // (B // k)
            v[x["bias_tokens"][q * m:(q + 1) * m].long()] += x["bias_values"][q * m:(q + 1) * m].double()
        toks = x["hist_tok"][first[q]:first[q + 1]] if c["hist"] else torch.zeros(0, dtype=torch.int64, device="cuda")
        if k > 1:
            toks = torch.cat([toks, x["extra_tokens"][q * (k - 1):q * (k - 1) + b % k].long()])
        if toks.numel():
            n = torch.bincount(toks, minlength=V).double()
            r = value("repetition_penalty", q, 1.0)
            y = torch.where(v > 0, v / r, v * r)
            y = y - (value("presence_penalty", q, 0.0) + n * value("frequency_penalty", q, 0.0))
            v = torch.where(n > 0, y, v)
        if c["mask"] and int(x["mask_index"][b]) >= 0:
            w = x["allow_mask"][int(x["mask_index"][b])].long()
            bits = (w[:, None] >> torch.arange(32, device="cuda")[None, :]) & 1
            v[bits.reshape(-1)[:V] == 0] = float("-inf")
        out[b] = v / value("temperature", q, 1.0)
    return out


def _logprobs_exact(c, seed):
    s = prepare_plain_logprobs(c, seed)
    lp = torch.empty(c["B"], dtype=torch.float64, device="cuda")
    top = torch.empty(c["B"], c["top"], dtype=torch.float64, device="cuda")
    for at in range(0, c["B"], 64):
        v = s["logits"][at:at + 64].double()
        if c["softcap"]:
            v = torch.tanh(v / c["softcap"]) * c["softcap"]
        v = v - torch.logsumexp(v, 1, keepdim=True)
        lp[at:at + 64] = v.gather(1, s["tokens"][at:at + 64].long()[:, None])[:, 0]
        if c["top"]:
            top[at:at + 64] = v.sort(1, descending=True).values[:, :c["top"]]
    out = {"logprobs": lp, "ranks": None}
    if c["top"]:
        out["top_ids"], out["top_logprobs"] = None, top
    return out


def prepare_plain_logprobs(c, seed):
    """The logits and tokens of a "logprobs" case, and nothing of the framework."""
    g = _gen(seed)
    lg = _logits(c, g)
    noisy = lg.float()
    noisy = noisy + torch.randn(noisy.shape, generator=g, device="cuda")
    return {"logits": lg, "tokens": noisy.argmax(1).int()}
