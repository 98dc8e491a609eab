"""The sparse attention and the 8-bit key/value cache, case by case.

Two groups of operators next to the dense attention of this package:

* attention over blocks of keys that a cheap score selects for each block of
  queries: ``block_means`` (the mean row of each block), ``select_blocks``
  (the score of every pair of blocks, and the best of them) and
  ``sparse_attention`` over the selected blocks, as one provider call;
* a paged cache of keys and values in 8 bits: ``KVCache.write`` quantises new
  rows as they are stored, ``KVCache.read`` gives rows back in 16 bits.

``run`` computes a case in elementary torch operations, or with ``own`` set
through the package's entry points.  Sizes come from the video and image
models whose layers the package runs (12, 24 and 40 heads of 128; 4096, 4608,
32760 and 75600 tokens; the heads that one of several GPUs holds) and from
streaming generation, where each step appends three latent frames.
"""
import math

import torch

own = False

HEAD = 128
E4M3_MAX, INT8_MAX = 448.0, 127.0
AMAX_FLOOR = 2.0 ** -100  # the smallest magnitude a row's scale is made from

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ------------------------------------------------------------------ the cases
def attend(name, queries, keys, heads, keep, kv_heads=None, batch=1, dtype="bf16", query_block=256, key_block=128,
           ragged=False, causal=False, kept_means=False, kind="attend"):
    return {"name": name, "kind": kind, "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads or heads, "dtype": dtype, "query_block": query_block, "key_block": key_block,
            "keep": keep, "ragged": ragged, "causal": causal, "kept_means": kept_means}


def cache(name, kind, rows, heads, context, batch=1, page=64, dtype="bf16", stored="e4m3", ragged=False):
    return {"name": name, "kind": kind, "batch": batch, "rows": rows, "heads": heads, "context": context,
            "page": page, "dtype": dtype, "stored": stored, "ragged": ragged}


def listed():
    return [
        # One new query over a short cached context whose key means are kept: what counts is latency.
        attend("token", 1, 4096, 12, 8, kept_means=True),
        # One new query per sequence of a padded batch with shared key/value heads, long contexts, small key blocks.
        attend("tokens in a batch", 1, 32760, 40, 96, kv_heads=8, batch=4, dtype="fp16", key_block=64, ragged=True,
               kept_means=True),
        # A layer of the small video model on one GPU: a quarter of 4096 keys.
        attend("video 4096", 4096, 4096, 12, 8),
        # Joint text and image rows of an image model in fp16, 64-key blocks, half of them kept.
        attend("joint 4608", 4608, 4608, 24, 36, dtype="fp16", key_block=64),
        # The large video model's sequence on one of four GPUs (10 of 40 heads): a quarter of the keys.
        attend("video 32760", 32760, 32760, 10, 64),
        # The long clip on one of eight GPUs (5 of 40 heads): a tenth of the keys, in 64-key blocks.
        attend("video 75600", 75600, 75600, 5, 118, key_block=64),
        # A padded batch of odd lengths (one sequence empty) with shared heads, where a block sees the past only.
        attend("padded batch", 5003, 5003, 12, 20, kv_heads=4, batch=3, key_block=64, ragged=True, causal=True),
        # The selection alone for the long clip: a plan that several steps then share.
        attend("select 75600", 75600, 75600, 5, 118, key_block=64, kind="select"),
        # One new row for each of eight sequences.
        cache("write one row", "write", 1, 12, 4096, batch=8, page=16),
        # One step of streaming generation: three latent frames of 30 x 52 tokens, all 40 heads.
        cache("write 4680", "write", 4680, 40, 32760, page=128),
        # The whole context read back for one layer's attention.
        cache("read 32760", "read", 32760, 40, 32760, page=128),
        # Append and read back for a padded batch in int8 and fp16, odd lengths, pages that end inside everything.
        cache("step in int8", "step", 311, 10, 3001, batch=3, page=48, dtype="fp16", stored="int8", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "token", "select", "write", "read", "step"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind in ("write", "read", "step"):
        batch, heads = rng.choice([1, 1, 2, 3, 5]), rng.choice([1, 3, 5, 8, 10, 12, 24, 40])
        most = max(1, min(32760, 32760 * 40 // (batch * heads)))
        context = _log(rng, 1, most)
        rows = context if kind == "read" else min(context, _log(rng, 1, 4680))
        c = cache("", kind, rows, heads, context, batch, rng.choice([16, 48, 64, 100, 128, 256]), dtype,
                  rng.choice(["e4m3", "int8"]), rng.random() < 0.4)
    else:
        kv_heads, group, batch = rng.choice([1, 2, 3, 4, 5, 8, 10]), rng.choice([1, 1, 2, 3, 5]), rng.choice([1, 1, 2, 3])
        key_block = rng.choice([64, 64, 128, 128, 192, 256])
        query_block = rng.choice([256, 256, 512])
        # a selection is a choice: no fewer than eight blocks where it alone is asked for, and not all of them
        keys = _log(rng, 8 * key_block if kind == "select" else 1, 75600)
        blocks = -(-keys // key_block)
        queries = rng.randint(1, 8) if kind == "token" else keys if rng.random() < 0.7 else _log(rng, 1, 75600)
        keep = max(1, min(blocks, int(blocks * rng.choice([0.08, 0.15, 0.25, 0.4, 0.6, 0.75 if kind == "select" else 1.0]))))
        # no more scores, and no more pairs of blocks, than the largest listed cases have
        rows = lambda n: -(-n // query_block) * query_block  # noqa: E731
        while batch * kv_heads * group * rows(queries) * keep * key_block > 10 * 32768 * 64 * 128:
            if keep > 4 and rng.random() < 0.5:
                keep = keep * 2 // 3
            elif queries > 512:
                queries = queries * 2 // 3
            elif group * kv_heads * batch > 1:
                batch, group, kv_heads = max(1, batch - 1), max(1, group - 1), max(1, kv_heads - 1)
            else:
                keep = max(1, keep // 2)
        c = attend("", queries, keys, kv_heads * group, keep, kv_heads, batch, dtype, query_block, key_block,
                   rng.random() < 0.4, kind == "attend" and queries == keys > 2 * query_block and rng.random() < 0.3,
                   kind == "token",
                   "select" if kind == "select" else "attend")
    del c["name"]
    return c


# ------------------------------------------------------------------ what a case's sizes say
def _lengths(n, batch, ragged):
    """Rows in use of each sequence: all, or uneven ones with an empty sequence in batches of three or more."""
    if not ragged:
        return [n] * batch
    return [max(0, n - (i * n) // max(1, batch - 1)) if batch > 2 else max(1, n - i * (n // 3) - 1) for i in range(batch)]


def _sees(case):
    """allowed[i][j]: whether query block i may see key block j.  The past only, and nothing for the first block."""
    nq, nk = -(-case["queries"] // case["query_block"]), -(-case["keys"] // case["key_block"])
    i, j = torch.arange(nq)[:, None], torch.arange(nk)[None]
    return (j * case["key_block"] < i * case["query_block"]) if case["causal"] else torch.ones(nq, nk, dtype=torch.bool)


def work(case):
    b, d = case["batch"], HEAD
    if case["kind"] in ("write", "read", "step"):
        row = case["heads"] * d
        held, wide = row + 4 * case["heads"], 2 * row  # codes and scales; 16 bits
        new = sum(min(case["rows"], n) for n in _lengths(case["context"], b, case["ragged"]))
        old = sum(min(case["rows"], n) if case["kind"] == "read" else n for n in _lengths(case["context"], b, case["ragged"]))
        rows = {"write": new * (wide + held), "read": old * (wide + held),
                "step": new * (wide + held) + old * wide + (old - new) * held}[case["kind"]]
        return {"bytes": 2 * rows, "flops": 0}
    hq, hk, qb, kb = case["heads"], case["kv_heads"], case["query_block"], case["key_block"]
    sees = _sees(case)
    nbytes = flops = 0
    for lq, lk in zip(_lengths(case["queries"], b, case["ragged"]), _lengths(case["keys"], b, case["ragged"])):
        nq, nk = -(-lq // qb), -(-lk // kb)
        counts = sees[:nq, :nk].sum(1).clamp_max(case["keep"])
        rows = torch.tensor([min(qb, lq - i * qb) for i in range(nq)])
        seen = torch.clamp(counts * kb, max=lk)
        if case["kind"] == "select":
            nbytes += 2 * d * (lq * hq + lk * hk) + 4 * hq * nq * (case["keep"] + 1)
            flops += 2 * d * hq * int((sees[:nq, :nk].sum(1)).sum())
            continue
        flops += 4 * d * hq * int((rows * seen).sum()) if nq else 0
        # every query and output row; the keys and values that some query block must read: with kept means at least
        # the largest selection, without them every key (its mean is needed) and no fewer values than one selection
        most = int(seen.max()) if nq else 0
        nbytes += 2 * 2 * d * lq * hq + 2 * d * hk * (2 * most if case["kept_means"] else lk + most)
        nbytes += 4 * d * hk * nk if case["kept_means"] else 0
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ inputs
def _rows(g, b, n, h, dtype, drift):
    """Rows as a layer makes them: noise around a direction that holds for some tokens (a patch of the picture)."""
    x = torch.randn(b, n, h, HEAD, generator=g, device="cuda", dtype=torch.float32)
    if drift:
        c = torch.randn(b, -(-n // 96), h, HEAD, generator=g, device="cuda") * drift
        x += c.repeat_interleave(96, 1)[:, :n]
    return x.to(dtype)


def _after(lengths, n):
    return torch.arange(n, device="cuda")[None] >= lengths[:, None]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, dtype = case["batch"], TYPES[case["dtype"]]
    s = dict(case)
    if case["kind"] in ("write", "read", "step"):
        page, n, h = case["page"], case["context"], case["heads"]
        per = -(-n // page)
        total = b * per + 3
        s["table"] = torch.randperm(total, generator=g, device="cuda")[:b * per].view(b, per).to(torch.int32)
        lengths = torch.tensor(_lengths(n, b, case["ragged"]), device="cuda", dtype=torch.int32)
        s["lengths"] = lengths
        if case["kind"] != "read":  # the last rows of each sequence are new
            s["new"] = torch.clamp(lengths, max=case["rows"])
            s["start"] = lengths - s["new"]
            s["x_k"], s["x_v"] = (_rows(g, b, case["rows"], h, dtype, 0.7) for _ in range(2))
        for t in ("k", "v"):
            x = torch.randn(total, page, h, HEAD, generator=g, device="cuda")
            if case["stored"] == "int8":
                s[t] = (x * 40).round().clamp(-127, 127).to(torch.int8)
            else:
                s[t] = (x * 130).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            del x
            s[t + "_scale"] = torch.rand(total, page, h, generator=g, device="cuda") * 0.01 + 0.005
            if case["kind"] != "write":
                s[t + "_out"] = torch.zeros(b, case["rows"] if case["kind"] == "read" else n, h, HEAD, device="cuda", dtype=dtype)
        return s
    s["q"] = _rows(g, b, case["queries"], case["heads"], dtype, 0.7)
    s["k"] = _rows(g, b, case["keys"], case["kv_heads"], dtype, 0.7)
    s["v"] = _rows(g, b, case["keys"], case["kv_heads"], dtype, 0.0)
    s["allowed"] = _sees(case).cuda() if case["causal"] else None
    s["query_lengths"] = s["key_lengths"] = None
    if case["ragged"]:
        for name, tensors, n in (("query_lengths", "q", case["queries"]), ("key_lengths", "kv", case["keys"])):
            s[name] = torch.tensor(_lengths(n, b, True), device="cuda", dtype=torch.int32)
            for t in tensors:  # what lies behind a sequence is anything
                s[t].masked_fill_(_after(s[name], n)[..., None, None], float("nan"))
    if case["kept_means"]:
        s["key_means"] = _means(s["k"], case["key_block"], s["key_lengths"])
    return s


# ------------------------------------------------------------------ the plain form
def _means(x, block, lengths):
    """Mean row of each block, over the rows in use: [B, blocks, H, D] in 32 bits from sums in 64."""
    b, n, h, d = x.shape
    x = x.double()
    if lengths is not None:
        x = x.masked_fill(_after(lengths, n)[..., None, None], 0.0)
    nb = -(-n // block)
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nb * block - n)).view(b, nb, block, h, d).sum(2)
    used = torch.full((b,), n, device=x.device) if lengths is None else lengths
    rows = (used[:, None] - torch.arange(nb, device=x.device) * block).clamp(0, block)
    return (x / rows.clamp_min(1)[..., None, None]).float()


def _select(s, q_means, k_means):
    """The `keep` highest scores of each query block (ties: the lower index), in ascending order; -1 behind them."""
    b, nk, hk, _ = k_means.shape
    nq, h = q_means.shape[1:3]
    group = h // hk
    q = q_means.double().permute(0, 2, 1, 3).view(b, hk, group, nq, HEAD)
    score = (q @ k_means.double().permute(0, 2, 3, 1)[:, :, None]).view(b, h, nq, nk)
    may = torch.ones(b, h, nq, nk, dtype=torch.bool, device=score.device)
    if s["allowed"] is not None:
        may &= s["allowed"]
    if s["key_lengths"] is not None:
        may &= (torch.arange(nk, device=score.device) * s["key_block"] < s["key_lengths"][:, None])[:, None, None]
        may &= (torch.arange(nq, device=score.device) * s["query_block"] < s["query_lengths"][:, None])[:, None, :, None]
    score = score.masked_fill(~may, -math.inf)
    keep = min(s["keep"], nk)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    best = torch.where(may.gather(-1, best), best, nk).sort(-1).values
    counts = may.sum(-1).clamp_max(keep)
    return torch.where(best < nk, best, -1).to(torch.int32), counts.to(torch.int32)


def _attention(s, blocks):
    """Softmax attention of each query block over the keys of its listed blocks; a row that sees nothing is zero."""
    q, k, v, qb, kb = s["q"], s["k"], s["v"], s["query_block"], s["key_block"]
    b, nq, h, d = q.shape
    n, hk = k.shape[1:3]
    blocks_q = blocks.shape[2]
    q = torch.nn.functional.pad(q.float(), (0, 0, 0, 0, 0, blocks_q * qb - nq)).view(b, blocks_q, qb, h, d).permute(0, 3, 1, 2, 4)
    at = (blocks.long()[..., None] * kb + torch.arange(kb, device=q.device)).flatten(-2)  # [B, H, query blocks, keys]
    used = torch.full((b,), n, device=q.device) if s["key_lengths"] is None else s["key_lengths"]
    ok = ((blocks >= 0)[..., None].expand(*blocks.shape, kb).flatten(-2)) & (at < used[:, None, None, None])
    at = at.clamp(0, n - 1)
    i = torch.arange(b, device=q.device)[:, None, None, None]
    j = (torch.arange(h, device=q.device) // (h // hk))[None, :, None, None]
    score = q @ k[i, at, j].float().transpose(-1, -2)
    score = (score * d ** -0.5).masked_fill_(~ok[..., None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isinf(top), 0.0, top))
    del score
    total = p.sum(-1, keepdim=True)
    out = p @ v[i, at, j].float().masked_fill_(~ok[..., None], 0.0)
    out = out / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 2, 3, 1, 4).reshape(b, blocks_q * qb, h, d)[:, :nq]
    if s["query_lengths"] is not None:
        out = out.masked_fill(_after(s["query_lengths"], nq)[..., None, None], 0.0)
    return out.to(s["q"].dtype)


def _slots(s, at):
    """Row of the page pool that holds position `at[b, i]` of sequence b."""
    page = s["page"]
    return s["table"].long().gather(1, (at // page).clamp(max=s["table"].shape[1] - 1)) * page + at % page


def _write(s):
    i = torch.arange(s["rows"], device="cuda")[None]
    ok = i < s["new"][:, None]
    slots = _slots(s, s["start"][:, None].long() + i)[ok]
    most = INT8_MAX if s["stored"] == "int8" else E4M3_MAX
    for t in ("k", "v"):
        x = s["x_" + t].float()[ok]
        amax = x.abs().amax(-1).clamp_min(AMAX_FLOOR)
        codes = x * torch.div(torch.full_like(amax, most), amax)[..., None]
        codes = codes.round().clamp(-most, most) if s["stored"] == "int8" else codes.clamp(-most, most)
        s[t].view(torch.uint8).flatten(0, 1)[slots] = codes.to(TYPES[s["stored"]]).view(torch.uint8)
        s[t + "_scale"].flatten(0, 1)[slots] = amax * torch.tensor(1.0 / most, device="cuda")


def _read(s):
    n = s["k_out"].shape[1]
    i = torch.arange(n, device="cuda")[None]
    ok = i < s["lengths"][:, None]
    slots = _slots(s, i.expand(s["batch"], n))[ok]
    for t in ("k", "v"):
        codes = s[t].view(torch.uint8).flatten(0, 1)[slots].view(TYPES[s["stored"]])
        s[t + "_out"][ok] = (codes.float() * s[t + "_scale"].flatten(0, 1)[slots][..., None]).to(TYPES[s["dtype"]])


# ------------------------------------------------------------------ one pass
_package = {}


def _own():
    if not _package:
        import __graft_entry__
        __graft_entry__.load_package()
        from powershard_b200 import cache as caches, sparse
        _package.update(cache=caches, sparse=sparse)
    return _package


def run(s):
    if s["kind"] in ("write", "read", "step"):
        if own:
            held = _own()["cache"].KVCache.over(s["k"], s["v"], s["k_scale"], s["v_scale"])
            if s["kind"] != "read":
                held.write(s["x_k"], s["x_v"], s["table"], s["start"], s["new"])
            if s["kind"] != "write":
                held.read(s["table"], s["lengths"], s["k_out"], s["v_out"])
        else:
            if s["kind"] != "read":
                _write(s)
            if s["kind"] != "write":
                _read(s)
        names = ("k", "v", "k_scale", "v_scale") if s["kind"] == "write" else ("k_out", "v_out")
        return {t: s[t] for t in names}
    if own:
        sparse = _own()["sparse"]
        if s["kind"] == "select":
            means = (sparse.block_means(s["q"], s["query_block"], s["query_lengths"]),
                     sparse.block_means(s["k"], s["key_block"], s["key_lengths"]))
            blocks, counts = sparse.select_blocks(
                *means, s["keep"], allowed=s["allowed"], query_block=s["query_block"], key_block=s["key_block"],
                query_lengths=s["query_lengths"], key_lengths=s["key_lengths"])
            return {"blocks": blocks, "counts": counts}
        provider = _package.get(("provider", s["keep"], s["query_block"], s["key_block"]))
        if provider is None:
            provider = sparse.SparseProvider(s["keep"], query_block=s["query_block"], key_block=s["key_block"])
            _package["provider", s["keep"], s["query_block"], s["key_block"]] = provider
        return {"out": provider(s["q"], s["k"], s["v"], allowed=s["allowed"], key_means=s.get("key_means"),
                                query_lengths=s["query_lengths"], key_lengths=s["key_lengths"])}
    k_means = s["key_means"] if s["kept_means"] else _means(s["k"], s["key_block"], s["key_lengths"])
    blocks, counts = _select(s, _means(s["q"], s["query_block"], s["query_lengths"]), k_means)
    if s["kind"] == "select":
        return {"blocks": blocks, "counts": counts}
    return {"out": _attention(s, blocks)}


# ------------------------------------------------------------------ in 64 bits, from the definition
def exact(case, seed):
    """One sequence, head and block at a time, straight from the definition."""
    s = prepare(case, seed)
    if case["kind"] in ("write", "read", "step"):
        return _exact_cache(s)
    d, qb, kb, group = HEAD, case["query_block"], case["key_block"], case["heads"] // case["kv_heads"]
    b, nq, h, _ = s["q"].shape
    nk = -(-case["keys"] // kb)
    sees = _sees(case)
    keep = min(case["keep"], nk)
    blocks = torch.full((b, h, -(-nq // qb), keep), -1, dtype=torch.int32)
    counts = torch.zeros(b, h, -(-nq // qb), dtype=torch.int32)
    out = torch.zeros(b, nq, h, d, dtype=torch.float64, device="cuda")
    q_len, k_len = _lengths(nq, b, case["ragged"]), _lengths(case["keys"], b, case["ragged"])
    mean = lambda x: x.double().mean(0).float().double()  # noqa: E731  (a block's mean is held in 32 bits)
    for i in range(b):
        for j in range(h):
            k, v = s["k"][i, :k_len[i], j // group], s["v"][i, :k_len[i], j // group]
            if not k_len[i] or not q_len[i]:
                continue
            k_means = torch.stack([mean(x) for x in k.split(kb)]) if j % group == 0 else k_means
            for t, rows in enumerate(s["q"][i, :q_len[i], j].split(qb)):
                may = sees[t, :len(k_means)].cuda().nonzero()[:, 0]
                if not len(may):
                    continue
                order = (k_means[may] @ mean(rows)).sort(descending=True, stable=True).indices
                chosen = may[order[:keep]].sort().values
                counts[i, j, t] = len(chosen)
                blocks[i, j, t, :len(chosen)] = chosen.to("cpu", torch.int32)
                if case["kind"] == "select":
                    continue
                at = (chosen[:, None] * kb + torch.arange(kb, device="cuda")).flatten()
                at = at[at < k_len[i]]
                p = torch.softmax(rows.double() @ k[at].double().T / math.sqrt(d), -1)
                out[i, t * qb:t * qb + len(rows), j] = p @ v[at].double()
    return {"blocks": blocks, "counts": counts} if case["kind"] == "select" else {"out": out}


def _exact_cache(s):
    most = INT8_MAX if s["stored"] == "int8" else E4M3_MAX
    page = s["page"]
    got = {}
    for t in ("k", "v"):
        codes, scale = s[t].double(), s[t + "_scale"].double()
        if s["kind"] != "read":
            for i, (first, n) in enumerate(zip(s["start"].tolist(), s["new"].tolist())):
                at = torch.arange(first, first + n, device="cuda")
                pages, slots = s["table"][i].long()[at // page], at % page
                x = s["x_" + t][i, :n].double()
                sc = x.abs().amax(-1).clamp_min(AMAX_FLOOR) / most
                scale[pages, slots] = sc
                codes[pages, slots] = (x / sc[..., None]).clamp(-most, most).round() if s["stored"] == "int8" else \
                    (x / sc[..., None]).clamp(-most, most).to(torch.float8_e4m3fn).double()
        if s["kind"] == "write":
            got[t] = None if s["stored"] == "int8" else codes
            got[t + "_scale"] = scale
            continue
        out = s[t + "_out"].double()
        for i, n in enumerate(s["lengths"].tolist()):
            at = torch.arange(min(n, out.shape[1]), device="cuda")
            pages, slots = s["table"][i].long()[at // page], at % page
            out[i, :len(at)] = codes[pages, slots] * scale[pages, slots][..., None]
        got[t + "_out"] = out
    return got
