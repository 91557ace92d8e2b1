"""The paged cache, the attention of new tokens over it and the verification of drafted tokens: their cases, in
plain form and as a user calls the framework's operators.

A case is a dict with a "kind":
  store       the new tokens' keys and values go into the pages of a 16-bit cache
  store_load  the same into an int8 cache with a scale per token and head, and read back from it
  load        what the pages hold for each sequence, back into rows
  attention   each sequence's new tokens attend over its pages (a prompt, a chunk of one, drafted tokens, one token)
  step        store, then attention: what a layer does with its cache
  verify      drafted tokens against the target's logits, from given random numbers
"""
import math
import random
import sys

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "s8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "s8": 1}
INF = float("inf")


def mq():
    if "mojo-adreno_b200" not in sys.path:
        sys.path.insert(0, "mojo-adreno_b200")
    import mq as package

    return package


def _cache_case(kind, batch, new, longest, heads, kv_heads, dim, page, cache, x, mix, even=False, window=0, order="head"):
    """new: the most new tokens of a sequence (each has that many where even); longest: the most a sequence
    holds with them; order: whether a page's rows lie head by head or position by position."""
    return {"kind": kind, "batch": batch, "new": new, "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "cache": cache, "x": x, "mix": mix, "even": even, "window": window, "order": order}


def listed():
    return [
        # One token of one request into a layer's cache of Llama-3.2-1B: the smallest call, all latency.
        {"name": "store 1 token", **_cache_case("store", 1, 1, 333, 32, 8, 64, 16, "f16", "f16", 0, even=True)},
        # A batch of 13 prompts, 8192 tokens at most each: Qwen3-8B's keys and values.
        {"name": "store 13 prompts", **_cache_case("store", 13, 8192, 8192, 32, 8, 128, 64, "bf16", "bf16", 1)},
        # A prompt of 431 tokens (the benchmark's length) quantised into the cache and read back.
        {"name": "store_load 431 int8", **_cache_case("store_load", 1, 431, 431, 32, 8, 64, 16, "s8", "f16", 2, even=True)},
        # All that 64 requests hold in int8, back as rows: requests that move to another cache.
        {"name": "load 64 int8", **_cache_case("load", 64, 4001, 4001, 32, 8, 128, 32, "s8", "bf16", 3)},
        # One request decoding in Llama-3.2-1B, a thousand tokens in: the layer's whole work on its cache.
        {"name": "step 1 token, 1001", **_cache_case("step", 1, 1, 1001, 32, 8, 64, 16, "bf16", "bf16", 4, even=True)},
        # 64 requests of different lengths decoding in Qwen3-8B from an int8 cache: a stream of keys and values.
        {"name": "attention 64x1 int8", **_cache_case("attention", 64, 1, 8000, 32, 8, 128, 64, "s8", "bf16", 5)},
        # 16 requests, four drafted tokens and the one before them each: 32 heads on 4 (Qwen3-30B-A3B).
        {"name": "attention 16x5", **_cache_case("attention", 16, 5, 4100, 32, 4, 128, 32, "f16", "f16", 6, even=True,
                                                 order="position")},
        # A prompt of 431 tokens, Llama-3.2-1B.
        {"name": "attention 431", **_cache_case("attention", 1, 431, 431, 32, 8, 64, 16, "f16", "f16", 7, even=True)},
        # A chunk of 2048 tokens of a long prompt, 30000 tokens in, int8.
        {"name": "attention 2048 of 30000 int8", **_cache_case("attention", 1, 2048, 30001, 32, 8, 128, 64, "s8", "bf16", 8,
                                                               even=True)},
        # A long prompt at once: the largest call.
        {"name": "attention 8192", **_cache_case("attention", 1, 8192, 8192, 32, 8, 128, 128, "bf16", "bf16", 9, even=True)},
        # One request with four drafted tokens, Qwen3's vocabulary.
        {"name": "verify 1x4x151669", "kind": "verify", "batch": 1, "drafts": 4, "vocab": 151669, "x": "f32", "draft": True,
         "mix": 10},
        # A batch of 64, Llama's vocabulary.
        {"name": "verify 64x4x128256", "kind": "verify", "batch": 64, "drafts": 4, "vocab": 128256, "x": "f32",
         "draft": True, "mix": 11},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "store_load", "load", "step", "attention", "attention", "attention", "attention", "verify",
                       "verify"])
    mix = rng.randrange(1 << 20)
    if kind == "verify":
        case = {"kind": kind, "batch": _log(rng, 1, 64), "drafts": rng.randint(1, 8), "vocab": _log(rng, 1000, 151936),
                "x": rng.choice(["f32", "f16", "bf16"]), "draft": rng.random() < 0.7, "mix": mix}
        while case["batch"] * (case["drafts"] + 1) * case["vocab"] > 3e7:
            case["batch"] = max(1, case["batch"] // 2)
            case["vocab"] = case["vocab"] // 2 + 1
        return case
    kv_heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 128, 128, 96])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    page, cache = rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16", "s8"])
    x = rng.choice(["f16", "bf16"]) if cache == "s8" else cache
    if kind in ("store", "step") and cache == "s8":
        cache = x
    if kind == "store_load":
        cache, x = "s8", rng.choice(["f16", "bf16"])
    batch = _log(rng, 1, 64)
    longest = _log(rng, 1, 30000)
    new = longest if kind in ("store", "store_load", "load") else rng.choice([1, 1, rng.randint(2, 8), _log(rng, 1, longest)])
    case = _cache_case(kind, batch, min(new, longest), longest, heads, kv_heads, dim, page, cache, x, mix,
                       rng.random() < 0.5, rng.choice([0, 0, 0, _log(rng, 1, longest)]) if kind == "attention" else 0,
                       rng.choice(["head", "position"]))
    while work(case)["flops"] > 2e11 or work(case)["bytes"] > 2e8 or batch * longest * kv_heads * dim > 4e8:
        case["batch"] = batch = max(1, batch // 2)
        if batch == 1:
            case["longest"] = longest = longest // 2 + 1
            case["new"] = min(case["new"], longest)
    return case


def _sizes(c):
    """(new tokens, length with them) of each sequence."""
    rng = random.Random(c["mix"])
    sizes = []
    for _ in range(c["batch"]):
        new = c["new"] if c["even"] else rng.randint(1, c["new"])
        if c["kind"] in ("store_load", "load"):
            sizes.append((new, new))
        else:
            sizes.append((new, c["longest"] if c["batch"] == 1 else rng.randint(new, c["longest"])))
    return sizes


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _pool(g, c, pages, dtype):
    """Pages of earlier content, [pages, kv_heads, page, dim] whatever order their rows lie in."""
    shape = (c["kv_heads"], c["page"]) if c["order"] == "head" else (c["page"], c["kv_heads"])
    pool = torch.empty(pages, *shape, c["dim"], dtype=dtype, device="cuda")
    for i in range(0, pages, 1024):
        part = _normal(g, *pool[i:i + 1024].shape)
        pool[i:i + 1024] = (part * 33).round_().clamp_(-127, 127) if dtype == torch.int8 else part
    return pool if c["order"] == "head" else pool.transpose(1, 2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, {"case": case}
    if c["kind"] == "verify":
        b, n, v = c["batch"], c["drafts"], c["vocab"]
        target = _normal(g, b, n + 1, v) * 2.5
        target[torch.rand(target.shape, generator=g, device="cuda") < 0.02] = -INF  # tokens that are not allowed here
        draft = target[:, :n] * 0.9 + _normal(g, b, n, v)
        target, draft = target.to(DT[c["x"]]), draft.to(DT[c["x"]])
        mix = random.Random(c["mix"])
        s["temperature"] = torch.tensor([mix.choice([0.0, 0.7, 1.0, 1.0]) for _ in range(b)], device="cuda")
        hot = s["temperature"].view(b, 1, 1)
        noise = -torch.log(-torch.log(torch.rand(b, n, v, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)))
        s["drafted"] = (draft.float() + noise * hot).argmax(-1).int()  # the drafter's own samples
        s["target"], s["draft"] = target.view(b * (n + 1), v), draft.view(b * n, v) if c["draft"] else None
        s["uniform"] = torch.rand(b, n + 1, generator=g, device="cuda")
        s["tokens"] = torch.empty(b, n + 1, dtype=torch.int32, device="cuda")
        s["accepted"] = torch.empty(b, dtype=torch.int32, device="cuda")
        s["logprobs"] = torch.empty(b, n + 1, device="cuda")
        if own:
            s["workspace"] = torch.empty(mq().verify_workspace(b, n, v), dtype=torch.uint8, device="cuda")
        return s
    sizes = _sizes(c)
    tokens, page = sum(n for n, _ in sizes), c["page"]
    need = [-(-length // page) for _, length in sizes]
    pages = sum(need) + 3
    s["sizes"] = sizes
    s["k_pages"], s["v_pages"] = _pool(g, c, pages, DT[c["cache"]]), _pool(g, c, pages, DT[c["cache"]])
    if c["cache"] == "s8":
        s["k_scale"] = torch.rand(pages, c["kv_heads"], page, generator=g, device="cuda") * 0.04 + 0.01
        s["v_scale"] = torch.rand(pages, c["kv_heads"], page, generator=g, device="cuda") * 0.04 + 0.01
    order = torch.randperm(pages, generator=g, device="cuda").int()
    s["table"] = torch.zeros(c["batch"], max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        s["table"][b, :n] = order[at:at + n]
        at += n
    s["lengths"] = torch.tensor([length for _, length in sizes], dtype=torch.int32, device="cuda")
    ends = [0]
    for n, _ in sizes:
        ends.append(ends[-1] + n)
    s["starts"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    x = DT[c["x"]]
    if c["kind"] in ("store", "store_load", "step"):
        s["k"], s["v"] = (_normal(g, tokens, c["kv_heads"], c["dim"]).to(x) for _ in range(2))
    if c["kind"] in ("store_load", "load"):
        s["k_out"], s["v_out"] = (torch.empty(tokens, c["kv_heads"], c["dim"], dtype=x, device="cuda") for _ in range(2))
    if c["kind"] in ("attention", "step"):
        s["q"] = (_normal(g, tokens, c["heads"], c["dim"]) * 2).to(x)
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["cache"] = mq().PagedCache(s["k_pages"], s["v_pages"], s.get("k_scale"), s.get("v_scale"))
        if c["kind"] in ("attention", "step"):
            nbytes = mq().paged_attention_workspace(s["cache"], c["heads"], c["batch"], tokens, c["new"])
            s["workspace"] = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    return s


def _places(s):
    """(page, row within it) of each new token."""
    page, parts = s["case"]["page"], []
    for b, (n, length) in enumerate(s["sizes"]):
        at = torch.arange(length - n, length, device="cuda")
        parts.append((s["table"][b, at // page].long(), at % page))
    return torch.cat([p for p, _ in parts]), torch.cat([r for _, r in parts])


def _store(s):
    at, row = _places(s)
    for name in ("k", "v"):
        pages, x = s[name + "_pages"], s[name].float()
        if pages.dtype == torch.int8:
            most = x.abs().amax(-1, keepdim=True)
            s[name + "_scale"][at, :, row] = (most / 127)[..., 0]
            x = (x * (127 / most.clamp_min(1e-30))).round()
        pages[at, :, row] = x.to(pages.dtype)


def _load(s):
    at, row = _places(s)
    got = {}
    for name in ("k", "v"):
        x = s[name + "_pages"][at, :, row].float()
        if name + "_scale" in s:
            x = x * s[name + "_scale"][at, :, row][..., None]
        got[name] = x.to(DT[s["case"]["x"]])
    return got


def _rows(s, name, b, length, dtype):
    """What sequence b's pages hold: [kv_heads, length, dim]."""
    page = s["case"]["page"]
    at = s["table"][b, :-(-length // page)].long()
    x = s[name + "_pages"][at].to(dtype)
    if name + "_scale" in s:
        x = x * s[name + "_scale"][at][..., None].to(dtype)
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :length]


def _attend(s):
    c = s["case"]
    group, out, first = c["heads"] // c["kv_heads"], torch.empty_like(s["q"]), 0
    for b, (n, length) in enumerate(s["sizes"]):
        k, v = _rows(s, "k", b, length, torch.float32), _rows(s, "v", b, length, torch.float32)
        step = max(1, (1 << 28) // (c["heads"] * length))
        for t in range(0, n, step):
            m = min(step, n - t)
            q = s["q"][first + t:first + t + m].float().view(m, c["kv_heads"], group, -1).permute(1, 2, 0, 3)
            z = (q.reshape(c["kv_heads"], group * m, -1) @ k.transpose(1, 2)) * c["dim"] ** -0.5
            z = z.view(c["kv_heads"], group, m, length)
            at = torch.arange(length - n + t, length - n + t + m, device="cuda")[:, None]
            key = torch.arange(length, device="cuda")
            seen = key <= at if not c["window"] else (key <= at) & (key > at - c["window"])
            z = torch.where(seen, z, torch.full_like(z, -INF))
            p = (z - z.amax(-1, keepdim=True)).exp()
            o = (p.view(c["kv_heads"], group * m, length) @ v).view(c["kv_heads"], group, m, -1)
            o = o / p.sum(-1)[..., None]
            out[first + t:first + t + m] = o.permute(2, 0, 1, 3).reshape(m, c["heads"], -1).to(out.dtype)
        first += n
    return out


def _distribution(z, hot):
    """softmax(z / hot) in 64 bits; where hot is 0, all on the first of the largest."""
    z = z.double()
    top = z.amax(-1, keepdim=True)
    at = torch.arange(z.shape[-1], device=z.device)
    first = torch.where(z == top, at, z.shape[-1]).amin(-1, keepdim=True)
    p = ((z - top) / torch.where(hot > 0, hot, torch.ones_like(hot)).double()).exp()
    p = p / p.sum(-1, keepdim=True)
    return torch.where(hot > 0, p, (at == first).double())


def _verify(s):
    c = s["case"]
    b, n, v = c["batch"], c["drafts"], c["vocab"]
    hot, drafted, u = s["temperature"].view(b, 1, 1), s["drafted"].long(), s["uniform"].double()
    p = _distribution(s["target"].view(b, n + 1, v), hot)
    if c["draft"]:
        q = _distribution(s["draft"].view(b, n, v), hot)
    else:
        q = (torch.arange(v, device="cuda") == drafted[..., None]).double()
    p_of, q_of = p[:, :n].gather(2, drafted[..., None])[..., 0], q.gather(2, drafted[..., None])[..., 0]
    # At temperature 0 a drafted token is kept where it is the target's best, whatever the drafter thought of it.
    keep = torch.where(hot[..., 0] > 0, u[:, :n] * q_of < p_of, p_of > 0)
    accepted = keep.int().cumprod(1).sum(1)
    i = torch.arange(b, device="cuda")
    left = p[i, accepted]
    rest = (left - q[i, accepted.clamp_max(n - 1)]).clamp_min(0)
    rejected = (accepted < n) & (s["temperature"] > 0) & (rest.sum(-1) > 0)
    left = torch.where(rejected[:, None], rest, left)
    mass = left.cumsum(-1)
    drawn = (mass <= u[:, n:] * mass[:, -1:]).sum(-1).clamp_max(v - 1)
    at = torch.arange(n + 1, device="cuda")
    tokens = torch.cat([drafted, drafted[:, :1]], 1)
    tokens = torch.where(at < accepted[:, None], tokens, torch.where(at == accepted[:, None], drawn[:, None], -1))
    logprobs = p.gather(2, tokens.clamp_min(0)[..., None])[..., 0].log()
    return {"tokens": tokens.int(), "accepted": accepted.int(),
            "logprobs": torch.where(tokens < 0, torch.zeros_like(logprobs), logprobs).float()}


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        return _run_own(s, c, kind)
    if kind == "verify":
        return _verify(s)
    if kind in ("store", "store_load", "step"):
        _store(s)
    if kind in ("store_load", "load"):
        return _load(s)
    if kind == "store":
        return {"k": s["k_pages"], "v": s["v_pages"]}
    out = _attend(s)
    return {"out": out, "k": s["k_pages"], "v": s["v_pages"]} if kind == "step" else out


def _run_own(s, c, kind):
    m = mq()
    if kind == "verify":
        tokens, accepted, logprobs = m.verify_drafts(
            s["target"], s["drafted"], s["uniform"], draft=s["draft"], temperature=s["temperature"], tokens=s["tokens"],
            accepted=s["accepted"], logprobs=s["logprobs"], workspace=s["workspace"])
        return {"tokens": tokens, "accepted": accepted, "logprobs": logprobs}
    cache, where = s["cache"], (s["table"], s["lengths"], s["starts"])
    if kind in ("store", "store_load", "step"):
        m.kv_store(s["k"], s["v"], cache, *where)
    if kind in ("store_load", "load"):
        k, v = m.kv_load(cache, *where, k=s["k_out"], v=s["v_out"])
        return {"k": k, "v": v}
    if kind == "store":
        return {"k": s["k_pages"], "v": s["v_pages"]}
    out = m.paged_attention(s["q"], cache, *where, out=s["out"], window=c["window"], max_new=c["new"],
                            workspace=s["workspace"])
    return {"out": out, "k": s["k_pages"], "v": s["v_pages"]} if kind == "step" else out


def work(case):
    c = case
    if c["kind"] == "verify":
        rows = c["batch"] * (c["drafts"] + 1 + (c["drafts"] if c["draft"] else 0))
        return {"bytes": rows * c["vocab"] * SIZE[c["x"]] + c["batch"] * (20 * c["drafts"] + 20), "flops": 4 * rows * c["vocab"]}
    sizes = _sizes(c)
    tokens, row = sum(n for n, _ in sizes), c["dim"] * c["kv_heads"]
    kept = row * SIZE[c["cache"]] + (4 * c["kv_heads"] if c["cache"] == "s8" else 0)  # of a token's keys
    total, flops = 8 * c["batch"], 0
    if c["kind"] in ("store", "store_load", "step"):
        total += 2 * tokens * (row * SIZE[c["x"]] + kept)
        flops += 2 * tokens * row
    if c["kind"] in ("store_load", "load"):
        total += 2 * tokens * (row * SIZE[c["x"]] + kept)
        flops += 2 * tokens * row
    if c["kind"] in ("attention", "step"):
        total += 2 * tokens * c["heads"] * c["dim"] * SIZE[c["x"]]
        for n, length in sizes:
            window = c["window"] or length
            past, most = length - n, min(window, length)  # the row at position p sees min(p + 1, window) keys
            short = max(0, min(n, window - past))  # rows that see all before them
            pairs = short * past + short * (short + 1) // 2 + (n - short) * most
            total += 2 * kept * min(length, window + n - 1)
            flops += 4 * c["dim"] * c["heads"] * pairs
    return {"bytes": total, "flops": flops}


def exact(case, seed):
    c, f64 = case, torch.float64
    s = prepare(case, seed)
    if c["kind"] == "verify":  # by the definition, one request and one drafted token at a time
        n, logprobs = c["drafts"], torch.zeros(c["batch"], c["drafts"] + 1, dtype=f64, device="cuda")
        for b, hot in enumerate(s["temperature"].tolist()):
            for i in range(n + 1):
                z, u = s["target"][b * (n + 1) + i].to(f64), s["uniform"][b, i].item()
                if hot == 0:
                    if i == n or int(s["drafted"][b, i]) != int((z == z.max()).nonzero()[0]):
                        break
                    continue
                logp = torch.log_softmax(z / hot, -1)
                weight, token = logp.exp(), int(s["drafted"][b, i]) if i < n else -1
                if i < n:
                    q = torch.zeros_like(weight)
                    if c["draft"]:
                        q = torch.softmax(s["draft"][b * n + i].to(f64) / hot, -1)
                    else:
                        q[token] = 1
                    if u * q[token].item() < weight[token].item():
                        logprobs[b, i] = logp[token]
                        continue
                    weight = torch.relu(weight - q)
                mass = torch.cumsum(weight, 0)
                logprobs[b, i] = logp[torch.searchsorted(mass, s["uniform"][b, n].item() * mass[-1], right=True).clamp_max(c["vocab"] - 1)]
                break
        return {"tokens": None, "accepted": None, "logprobs": logprobs}
    where = [(b, i) for b, (n, length) in enumerate(s["sizes"]) for i in range(length - n, length)] \
        if c["kind"] != "attention" else []
    at = torch.tensor([b for b, _ in where], dtype=torch.long, device="cuda")
    position = torch.tensor([i for _, i in where], dtype=torch.long, device="cuda")
    page = s["table"].long()[at, torch.div(position, c["page"], rounding_mode="floor")] if where else None
    got = {}
    for name in ("k", "v"):
        if c["kind"] in ("store", "step"):
            full = s[name + "_pages"].to(f64).transpose(1, 2).contiguous()  # [pages, page, kv_heads, dim]
            full.view(-1, c["kv_heads"], c["dim"])[page * c["page"] + position % c["page"]] = s[name].to(f64)
            got[name] = full.transpose(1, 2)
        elif c["kind"] == "store_load":
            x = s[name].to(f64)
            step = x.abs().max(-1, keepdim=True).values / 127
            got[name] = torch.round(x / step) * step
        elif c["kind"] == "load":
            flat = page * c["page"] + position % c["page"]
            scale = s[name + "_scale"].to(f64) if name + "_scale" in s else torch.ones(s["k_pages"].shape[:3], dtype=f64, device="cuda")
            values = s[name + "_pages"].transpose(1, 2).reshape(-1, c["kv_heads"], c["dim"])[flat].to(f64)
            got[name] = values * scale.transpose(1, 2).reshape(-1, c["kv_heads"], 1)[flat]
    if c["kind"] not in ("attention", "step"):
        return got
    out = torch.empty(s["q"].shape, dtype=f64, device="cuda")
    first, group = 0, c["heads"] // c["kv_heads"]
    for b, (n, length) in enumerate(s["sizes"]):
        if c["kind"] == "step":  # the new tokens' rows are in the pages by then
            keys = [got[name][s["table"][b].long()].permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, c["dim"])[:, :length]
                    for name in ("k", "v")]
        else:
            keys = [_rows(s, name, b, length, f64) for name in ("k", "v")]
        position = torch.arange(length - n, length, device="cuda")
        back = position[:, None] - torch.arange(length, device="cuda")[None, :]
        hidden = back < 0
        if c["window"]:
            hidden |= back >= c["window"]
        for h in range(c["heads"]):  # one head at a time
            z = torch.einsum("td,ld->tl", s["q"][first:first + n, h].to(f64), keys[0][h // group]) / math.sqrt(c["dim"])
            out[first:first + n, h] = torch.softmax(z.masked_fill_(hidden, -INF), -1) @ keys[1][h // group]
        first += n
    return {"out": out, **got} if c["kind"] == "step" else out
