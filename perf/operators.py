"""The serving operators of a softmax-attention recommender, as they are measured: appending rotated keys to the paged
KV cache, attention over that cache (sliding window and sinks; a prefix shared by a group of requests) and drawing items
from scores.  ``own`` selects the framework's calls; otherwise ``run`` computes the plain forms."""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one user's next token: nothing but latency
        dict(name="append_one", op="append", tokens=1, requests=1, past=700, heads=8, kv_heads=8, dim=64, rotary=64, page=32,
             interleaved=False, dtype="bf16"),
        # prompts of a batch go into the cache: ragged, several pages each, part of each head rotated in neighbouring pairs
        dict(name="append_prompts", op="append", tokens=20011, requests=13, past=300, heads=32, kv_heads=8, dim=128, rotary=64,
             page=64, interleaved=True, dtype="fp16"),
        # the next token of four users with short histories
        dict(name="step_few", op="window", requests=4, new=1, mean_new=1, past=1024, heads=8, kv_heads=8, dim=64, page=32, window=512,
             sinks=4, dtype="bf16"),
        # the next token of a full batch with long, very uneven histories
        dict(name="step_many", op="window", requests=128, new=1, mean_new=1, past=16384, heads=32, kv_heads=8, dim=128, page=64,
             window=4096, sinks=4, dtype="bf16"),
        # new interactions appended to a cached history of about 2048 items (the serving benchmark's users)
        dict(name="delta_users", op="window", requests=64, new=128, mean_new=100, past=2048, heads=8, kv_heads=8, dim=64, page=64,
             window=1024, sinks=16, dtype="fp16"),
        # whole prompts up to the model's length, nothing cached
        dict(name="prompts", op="window", requests=5, new=4096, mean_new=2100, past=0, heads=32, kv_heads=8, dim=128, page=64,
             window=1024, sinks=4, dtype="bf16"),
        # eight beams of one user
        dict(name="beams_one_user", op="prefix", groups=1, per_group=8, prefix=2048, suffix=4, new=1, heads=8, kv_heads=8, dim=64,
             page=32, dtype="bf16"),
        # 32 candidates lists of 16 users, histories of uneven length
        dict(name="beams_users", op="prefix", groups=16, per_group=32, prefix=4096, suffix=64, new=2, heads=8, kv_heads=8, dim=64,
             page=64, dtype="fp16"),
        # one long instruction in front of every request of the batch
        dict(name="long_prefix", op="prefix", groups=1, per_group=96, prefix=30011, suffix=512, new=1, heads=32, kv_heads=8, dim=128,
             page=64, dtype="bf16"),
        # one row of item scores
        dict(name="sample_one", op="sample", rows=1, width=50021, ragged=False, dtype="fp32", temperature=0.8, top_k=50, top_p=0.9,
             min_p=0.0),
        # one item for each of 64 users out of their own candidates
        dict(name="sample_candidates", op="sample", rows=64, width=1024, ragged=True, dtype="fp32", temperature=0.7, top_k=0,
             top_p=0.95, min_p=0.0),
        # a batch over a whole catalogue
        dict(name="sample_catalogue", op="sample", rows=256, width=131071, ragged=False, dtype="bf16", temperature=1.0, top_k=0,
             top_p=0.9, min_p=0.002),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, wide):
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    while kv * group > (32 if wide else 16):
        group = max(1, group // 2)
    return dict(heads=kv * group, kv_heads=kv, dim=dim, page=rng.choice([16, 32, 48, 64, 128]), dtype=rng.choice(["bf16", "fp16"]))


def draw(rng):
    case = _draw(rng)
    while work(case)["flops"] > 2e11:                                # none above the largest listed case
        case = _draw(rng)
    return case


def _draw(rng):
    op = rng.choice(["append", "window", "window", "prefix", "sample"])
    if op == "append":
        c = _heads(rng, True)
        n = _log_int(rng, 1, 16000)
        return dict(op=op, tokens=n, requests=rng.randint(1, min(n, 64)), past=rng.randint(0, 2000), interleaved=rng.random() < 0.5,
                    rotary=rng.choice([16, 32, 48, 64] if c["dim"] == 64 else [16, 64, 96, 128]), **c)
    if op == "window":
        c = _heads(rng, True)
        win, sinks = rng.choice([0, _log_int(rng, 1, 4096)]), rng.choice([0, 1, 4, rng.randint(1, 200)])
        if rng.random() < 0.5:                                   # steps: one or a few new tokens over a cache
            b = _log_int(rng, 1, 128)
            new = rng.choice([1, 1, 2, 5])
            return dict(op=op, requests=b, new=new, mean_new=new, past=_log_int(rng, 1, min(16384, 400000 // b)), window=win,
                        sinks=sinks, **c)
        b = rng.randint(1, 8)
        new = _log_int(rng, 16, 3000)
        return dict(op=op, requests=b, new=new, mean_new=max(1, int(new * rng.uniform(0.3, 1.0))), past=rng.choice([0, rng.randint(1, 2000)]),
                    window=win, sinks=sinks, **c)
    if op == "prefix":
        c = _heads(rng, True)
        groups = _log_int(rng, 1, 16)
        return dict(op=op, groups=groups, per_group=_log_int(rng, 1, min(96, 512 // groups)), prefix=_log_int(rng, 1, 30000 // groups),
                    suffix=_log_int(rng, 1, 300), new=rng.choice([1, 1, 2, 4]), **c)
    ragged = rng.random() < 0.5
    rows = _log_int(rng, 1, 256)
    return dict(op=op, rows=rows, width=_log_int(rng, 2, 4096 if ragged else 130000), ragged=ragged,
                dtype=rng.choice(["fp32", "bf16", "fp16"]), temperature=rng.choice([0.0, 1.0, rng.uniform(0.2, 1.5)]),
                top_k=rng.choice([0, 1, _log_int(rng, 2, 2000)]), top_p=rng.choice([1.0, rng.uniform(0.3, 0.99)]),
                min_p=rng.choice([0.0, rng.uniform(0.001, 0.2)]))


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(n, most, mean, seed):
    """n whole numbers in [1, most] with about the given mean, the first of them ``most``.  They depend on the
    sizes alone, so the work of a case is known without its inputs."""
    g = torch.Generator().manual_seed(seed)
    if most <= 1:
        return [1] * n
    spread = min(1.0, 2.0 * mean / most)
    x = 1 + torch.floor(torch.rand(n, generator=g, dtype=torch.float64) * (most * spread - 1e-9)).long().clamp_(0, most - 1)
    x[0] = most
    return x.tolist()


def _shape(case):
    """-> (new tokens per request, keys per request, prefix keys per group)."""
    if case["op"] == "append":
        n, b = case["tokens"], case["requests"]
        cuts = sorted(torch.randperm(max(n - 1, 1), generator=torch.Generator().manual_seed(5))[: b - 1].add(1).tolist())
        new = [e - s for s, e in zip([0] + cuts, cuts + [n])]
        past = _lengths(len(new), case["past"] + 1, case["past"] / 2, 7)
        return new, [a + p - 1 for a, p in zip(new, past)], []
    if case["op"] == "window":
        b = case["requests"]
        new = _lengths(b, case["new"], case["mean_new"], 11) if case["mean_new"] < case["new"] else [case["new"]] * b
        past = [p - 1 for p in _lengths(b, case["past"] + 1, case["past"] / 2, 13)]
        return new, [a + p for a, p in zip(new, past)], []
    b = case["groups"] * case["per_group"]
    new = [case["new"]] * b
    own_keys = [max(a, s) for a, s in zip(new, _lengths(b, case["suffix"], case["suffix"] / 2, 17))]
    return new, own_keys, _lengths(case["groups"], case["prefix"], 0.75 * case["prefix"], 19)


def _offsets(lens, dev):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)


def _pages(lens, page, perm, used):
    counts = [(n + page - 1) // page for n in lens]
    return perm[used:used + sum(counts)], counts, used + sum(counts)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    if case["op"] == "sample":
        rows, width, dt = case["rows"], case["width"], DT[case["dtype"]]
        if case["ragged"]:
            lens = _lengths(rows, width, width / 2, 23)
            s["offsets"] = _offsets(lens, dev)
            s["longest"] = max(lens)
            x = torch.randn(sum(lens), generator=g, device=dev) * 2.0
        else:
            s["offsets"] = None
            # a model's scores over a catalogue: a broad bulk and a few items far above it
            x = torch.randn(rows, width, generator=g, device=dev) * 2.0
            hot = torch.randint(0, width, (rows, 8), generator=g, device=dev)
            x.scatter_add_(1, hot, 4.0 + 3.0 * torch.rand(rows, 8, generator=g, device=dev))
        s["scores"] = x.to(dt)
        s["uniform"] = torch.rand(rows, generator=g, device=dev)
        return s
    dt, dim, h, hk, page = DT[case["dtype"]], case["dim"], case["heads"], case["kv_heads"], case["page"]
    new, keys, prefix = _shape(case)
    total_pages = sum((n + page - 1) // page for n in keys + prefix) + 3
    perm = torch.randperm(total_pages, generator=g, device=dev).int()
    s["page_ids"], counts, used = _pages(keys, page, perm, 0)
    s["page_indptr"] = _offsets(counts, dev)
    s["q_offsets"], s["k_offsets"] = _offsets(new, dev), _offsets(keys, dev)
    s["max_q"], s["max_k"] = max(new), max(keys)
    # the pages hold what earlier requests left there, too
    cache = torch.empty(total_pages, 2, page, hk, dim, dtype=dt, device=dev)
    for a in range(0, total_pages, 1024):
        n = min(1024, total_pages - a)
        cache[a:a + n] = torch.randn(n, 2, page, hk, dim, generator=g, device=dev).to(dt)
    s["cache"] = cache
    t = sum(new)
    if case["op"] == "append":
        # q, k and v are slices of one fused projection's output
        qkv = torch.randn(t, (h + 2 * hk) * dim, generator=g, device=dev).to(dt)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, dim)) for x in qkv.split([h * dim, hk * dim, hk * dim], dim=1))
        batch = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
        first = torch.tensor([k - n for k, n in zip(keys, new)])
        start = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist()[:-1])
        s["batch_indices"] = batch.int().to(dev)
        s["positions"] = (torch.arange(t) - start[batch] + first[batch]).int().to(dev)
        half = case["rotary"] // 2
        ang = torch.arange(max(keys) + 1, dtype=torch.float64)[:, None] * torch.pow(
            torch.tensor(10000.0, dtype=torch.float64), -torch.arange(half, dtype=torch.float64) / half)[None, :]
        s["table"] = torch.cat([ang.cos(), ang.sin()], dim=1).float().to(dev)
        return s
    s["q"] = torch.randn(t, h, dim, generator=g, device=dev).to(dt)
    if case["op"] == "prefix":
        s["prefix_page_ids"], counts, used = _pages(prefix, page, perm, used)
        s["prefix_page_indptr"] = _offsets(counts, dev)
        s["prefix_offsets"] = _offsets(prefix, dev)
        s["group_offsets"] = torch.arange(0, len(new) + 1, case["per_group"], dtype=torch.int32, device=dev)
        s["max_prefix"] = max(prefix)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "window": _plain_window, "prefix": _plain_prefix, "sample": _plain_sample}[s["op"]](s)


def _own(s):
    from recsdk_b200.ops import sampling, softmax_attention

    if s["op"] == "append":
        q = softmax_attention.append_kv_rotary(s["q"], s["k"], s["v"], s["cache"], s["batch_indices"], s["positions"], s["page_ids"],
                                               s["page_indptr"], s["page"], s["table"], interleaved=s["interleaved"])
        return {"q": q, "cache": s["cache"]}
    if s["op"] == "window":
        return softmax_attention.softmax_attention_paged(s["q"], s["cache"], s["q_offsets"], s["k_offsets"], s["page_ids"],
                                                         s["page_indptr"], s["page"], window=s["window"], num_sinks=s["sinks"])
    if s["op"] == "prefix":
        return softmax_attention.softmax_attention_shared_prefix(
            s["q"], s["cache"], s["q_offsets"], s["k_offsets"], s["page_ids"], s["page_indptr"], s["prefix_offsets"],
            s["prefix_page_ids"], s["prefix_page_indptr"], s["page"], group_offsets=s["group_offsets"])
    ids, logprobs = sampling.sample_scores(s["scores"], s["uniform"], offsets=s["offsets"], temperature=s["temperature"],
                                           top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"ids": ids, "logprobs": logprobs}


# ------------------------------------------------------------------------------------------------ plain forms
def _rotate(x, cos, sin, interleaved):
    """x [t, heads, dim]; cos, sin [t, 1, rotary / 2]: the first ``rotary`` elements of every head turn, the rest stay."""
    half = cos.shape[-1]
    x = x.float()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _plain_append(s):
    pos, b, page = s["positions"].long(), s["batch_indices"].long(), s["page"]
    cos, sin = s["table"][pos][:, None, :].chunk(2, dim=-1)
    where = s["page_ids"].long()[s["page_indptr"].long()[b] + pos // page]
    s["cache"][where, 0, pos % page] = _rotate(s["k"], cos, sin, s["interleaved"]).to(s["cache"].dtype)
    s["cache"][where, 1, pos % page] = s["v"]
    return {"q": _rotate(s["q"], cos, sin, s["interleaved"]).to(s["q"].dtype), "cache": s["cache"]}


def _rows(q, offsets, longest):
    """Jagged rows, padded: ([B, longest, ...] in 32 bits, which of them are there [B, longest])."""
    o = offsets.long()
    t = torch.arange(longest, device=q.device)
    there = t[None, :] < (o[1:] - o[:-1])[:, None]
    return q[(o[:-1, None] + t).clamp(max=q.shape[0] - 1)].float(), there


def _keys(cache, offsets, page_ids, indptr, page, longest):
    """The pages of every sequence, padded: K and V [B, longest, heads, dim] in 32 bits, and which keys are there."""
    o = offsets.long()
    j = torch.arange(longest, device=cache.device)
    there = j[None, :] < (o[1:] - o[:-1])[:, None]
    pg = page_ids.long()[(indptr.long()[:-1, None] + j // page).clamp(max=page_ids.numel() - 1)]
    slot = (j % page)[None, :].expand_as(pg)
    return cache[pg, 0, slot].float(), cache[pg, 1, slot].float(), there


def _scores(q, k, scale):
    """q [B, rows, heads, dim], k [B, keys, kv heads, dim] -> [B, kv heads, heads per kv head, rows, keys]."""
    b, r, h, d = q.shape
    hk = k.shape[2]
    qq = q.view(b, r, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    return (qq @ k.permute(0, 2, 3, 1) * scale).view(b, hk, h // hk, r, k.shape[1])


def _values(p, v):
    b, hk, g, r, n = p.shape
    o = (p.reshape(b, hk, g * r, n) @ v.permute(0, 2, 1, 3)).view(b, hk, g, r, v.shape[3])
    return o.permute(0, 3, 1, 2, 4).reshape(b, r, hk * g, v.shape[3])


def _per_row(x):
    b, hk, g, r = x.shape
    return x.permute(0, 3, 1, 2).reshape(b, r, hk * g)


def _causal(s, there_k):
    o, k = s["q_offsets"].long(), s["k_offsets"].long()
    first = (k[1:] - k[:-1]) - (o[1:] - o[:-1])
    p = first[:, None, None] + torch.arange(s["max_q"], device=first.device)[None, :, None]
    j = torch.arange(s["max_k"], device=first.device)[None, None, :]
    return there_k[:, None, :] & (j <= p), j, p


def _plain_window(s):
    q, there_q = _rows(s["q"], s["q_offsets"], s["max_q"])
    k, v, there_k = _keys(s["cache"], s["k_offsets"], s["page_ids"], s["page_indptr"], s["page"], s["max_k"])
    sees, j, p = _causal(s, there_k)
    if s["window"]:
        sees = sees & ((j > p - s["window"]) | (j < s["sinks"]))
    x = _scores(q, k, 1.0 / math.sqrt(s["dim"])).masked_fill_(~sees[:, None, None], -math.inf)
    m = x.amax(dim=-1, keepdim=True)
    e = (x - m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = _per_row(e.sum(dim=-1)).unsqueeze(-1)
    o = _values(e, v) / total.masked_fill(total == 0, 1.0)
    return o[there_q].to(s["q"].dtype)


def _plain_prefix(s):
    scale = 1.0 / math.sqrt(s["dim"])
    q, there_q = _rows(s["q"], s["q_offsets"], s["max_q"])
    k, v, there_k = _keys(s["cache"], s["k_offsets"], s["page_ids"], s["page_indptr"], s["page"], s["max_k"])
    sees, _, _ = _causal(s, there_k)
    xs = _scores(q, k, scale).masked_fill(~sees[:, None, None], -math.inf)
    # every row of a group against the group's prefix
    groups, b, r, h, d = s["groups"], q.shape[0], q.shape[1], q.shape[2], q.shape[3]
    kp, vp, there_p = _keys(s["cache"], s["prefix_offsets"], s["prefix_page_ids"], s["prefix_page_indptr"], s["page"], s["max_prefix"])
    xp = _scores(q.view(groups, -1, h, d), kp, scale).masked_fill(~there_p[:, None, None, None, :], -math.inf)
    ms, mp = _per_row(xs.amax(dim=-1)), _per_row(xp.amax(dim=-1)).reshape(b, r, h)
    m = torch.maximum(ms, mp)
    m = m.masked_fill(m == -math.inf, 0.0)
    es = (xs - m.reshape(b, r, k.shape[2], -1).permute(0, 2, 3, 1).unsqueeze(-1)).exp()
    ep = (xp - m.reshape(groups, -1, k.shape[2], h // k.shape[2]).permute(0, 2, 3, 1).unsqueeze(-1)).exp()
    total = _per_row(es.sum(dim=-1)) + _per_row(ep.sum(dim=-1)).reshape(b, r, h)
    o = _values(es, v) + _values(ep, vp).reshape(b, r, h, d)
    o = o / total.masked_fill(total == 0, 1.0).unsqueeze(-1)
    return o[there_q].to(s["q"].dtype)


def _plain_sample(s):
    x = s["scores"].double()
    if s["offsets"] is not None:
        o = s["offsets"].long()
        t = torch.arange(s["longest"], device=x.device)
        there = t[None, :] < (o[1:] - o[:-1])[:, None]
        x = x[(o[:-1, None] + t).clamp(max=x.numel() - 1)].masked_fill(~there, -math.inf)
    n = x.shape[1]
    x = x.masked_fill(x.isnan(), -math.inf)
    best = x.amax(dim=1, keepdim=True)
    nothing = best == -math.inf
    # the scores' own border values: everything that is summed or compared here is in 64 bits
    f32 = lambda f: torch.tensor(f, dtype=torch.float32, device=x.device).double()  # noqa: E731
    if s["temperature"] == 0.0:
        ids = (x == best).int().argmax(dim=1)
        return {"ids": ids.masked_fill(nothing[:, 0], -1), "logprobs": torch.zeros(x.shape[0], device=x.device).masked_fill(nothing[:, 0], -math.inf)}
    ordered, at = x.sort(dim=1, descending=True, stable=True)
    w = ((ordered - best.masked_fill(nothing, 0.0)) / f32(s["temperature"])).exp()
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] > 0:
        keep &= torch.arange(n, device=x.device) < s["top_k"]
    if s["top_p"] < 1.0:
        wk = w * keep
        keep &= wk.cumsum(dim=1) - wk < f32(s["top_p"]) * wk.sum(dim=1, keepdim=True)
    if s["min_p"] > 0.0:
        keep &= w >= f32(s["min_p"])
    w = torch.zeros_like(w).scatter(1, at, w * keep)                 # back in the order of the items
    below = w.cumsum(dim=1)
    total = below[:, -1:]
    ids = (below <= s["uniform"].double()[:, None] * total).sum(dim=1, keepdim=True)
    last = n - 1 - (w.flip(1) > 0).int().argmax(dim=1, keepdim=True)
    ids = torch.minimum(ids, last)
    logprobs = (w.gather(1, ids) / total).log()
    return {"ids": ids.masked_fill(nothing, -1)[:, 0], "logprobs": logprobs.masked_fill(nothing, -math.inf)[:, 0].float()}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "sample":
        return _exact_sample(s)
    new, keys, prefix = _shape(case)
    hk, group, page, dim = case["kv_heads"], case["heads"] // case["kv_heads"], case["page"], case["dim"]
    out = torch.zeros(sum(new), case["heads"], dim, dtype=torch.float64, device="cuda")
    t0 = p0 = 0
    pp0, at = [0], 0
    for n in prefix:
        at += (n + page - 1) // page
        pp0.append(at)

    def fetch(ids, n):
        c = s["cache"][ids.long()].double()                          # [pages, 2, page, kv heads, dim]
        return [c[:, i].reshape(-1, hk, dim)[:n].transpose(0, 1) for i in (0, 1)]

    for b, (n, nk) in enumerate(zip(new, keys)):
        pages = (nk + page - 1) // page
        k, v = fetch(s["page_ids"][p0:p0 + pages], nk)
        i = torch.arange(nk - n, nk, device="cuda")[:, None]
        j = torch.arange(nk, device="cuda")[None, :]
        sees = j <= i
        if case.get("window"):
            sees = sees & ((i - j < case["window"]) | (j < case["sinks"]))
        if prefix:
            u = b // case["per_group"]
            kp, vp = fetch(s["prefix_page_ids"][pp0[u]:pp0[u + 1]], prefix[u])
            k, v = torch.cat([kp, k], dim=1), torch.cat([vp, v], dim=1)
            sees = torch.cat([torch.ones(n, prefix[u], dtype=torch.bool, device="cuda"), sees], dim=1)
        q = s["q"][t0:t0 + n].double().view(n, hk, group, dim)
        for a in range(hk):
            for u in range(group):
                x = (q[:, a, u] @ k[a].T / dim ** 0.5).masked_fill(~sees, -math.inf)
                out[t0:t0 + n, a * group + u] = torch.softmax(x, dim=1) @ v[a]
        t0, p0 = t0 + n, p0 + pages
    return out


def _exact_append(s):
    half = s["rotary"] // 2
    pos = s["positions"].long()
    z = torch.complex(s["table"][pos, :half].double(), s["table"][pos, half:].double())[:, None, :]

    def turn(x):
        x = x.double().clone()
        first = slice(0, 2 * half, 2) if s["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if s["interleaved"] else slice(half, 2 * half)
        r = torch.complex(x[..., first], x[..., second]) * z
        x[..., first], x[..., second] = r.real, r.imag
        return x

    cache = s["cache"].double()
    b = s["batch_indices"].long()
    for kind, x in ((0, turn(s["k"])), (1, s["v"].double())):
        flat = s["page_ids"].long()[s["page_indptr"].long()[b] + torch.div(pos, s["page"], rounding_mode="floor")] * 2 + kind
        cache.view(-1, *cache.shape[3:])[flat * s["page"] + pos.remainder(s["page"])] = x
    return {"q": turn(s["q"]), "cache": cache}


def _exact_sample(s):
    ids, logs = [], []
    off = None if s["offsets"] is None else s["offsets"].tolist()
    f32 = lambda f: float(torch.tensor(f, dtype=torch.float32))  # noqa: E731
    us = s["uniform"].double().tolist()
    for r in range(s["rows"]):
        x = (s["scores"][r] if off is None else s["scores"][off[r]:off[r + 1]]).double()
        order = torch.argsort(-x, stable=True)
        if s["temperature"] == 0.0:
            ids.append(int(order[0]))
            logs.append(0.0)
            continue
        p = torch.exp((x[order] - x[order[0]]) / f32(s["temperature"]))
        n = min(s["top_k"], p.numel()) if s["top_k"] > 0 else p.numel()
        order, p = order[:n], p[:n]
        if s["top_p"] < 1.0:
            c = torch.cumsum(p, 0)
            n = min(int((c < f32(s["top_p"]) * c[-1]).sum()) + 1, n)
            order, p = order[:n], p[:n]
        if s["min_p"] > 0.0:
            n = max(1, int((p >= f32(s["min_p"])).sum()))
            order, p = order[:n], p[:n]
        back = torch.argsort(order)
        order, p = order[back], p[back]
        c = torch.cumsum(p, 0)
        i = min(int(torch.searchsorted(c, us[r] * c[-1], right=True)), p.numel() - 1)
        ids.append(int(order[i]))
        logs.append(math.log(float(p[i] / c[-1])))
    return {"ids": torch.tensor(ids, device="cuda"), "logprobs": torch.tensor(logs, dtype=torch.float64, device="cuda")}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["width"]
        if case["ragged"]:
            n = sum(_lengths(case["rows"], case["width"], case["width"] / 2, 23))
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + 16 * case["rows"], "flops": 3 * n}
    new, keys, prefix = _shape(case)
    t, h, hk, d = sum(new), case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        return {"bytes": t * ((h + 2 * hk) * d * 2 * 2 + 4 * case["rotary"] + 8), "flops": 3 * t * (h + hk) * case["rotary"]}
    pairs, read = 0, sum(prefix)
    win, sinks = case.get("window", 0), case.get("sinks", 0)
    for b, (n, nk) in enumerate(zip(new, keys)):
        if prefix:
            pairs += n * prefix[b // case["per_group"]]
        if win:
            for i in range(nk - n, nk):
                lo = max(0, i - win + 1)
                pairs += i + 1 - lo + min(sinks, lo)
            lo = max(0, nk - n - win + 1)
            read += nk - lo + min(sinks, lo)
        else:
            pairs += n * nk - n * (n - 1) // 2
            read += nk
    return {"bytes": 2 * t * h * d * 2 + read * hk * d * 2 * 2, "flops": 4 * d * h * pairs}
