"""The int8 products, the norms around a block and the beam-search step: their cases, in plain form and
as a user calls the framework's operators.

A case is a dict with a "kind":
  product   y = xs * ws * (xq . wq^T) (+ bias): the int8 projection with a scale per token and channel
  gate_up   silu(gate) * up of one fused [2f][k] int8 matrix
  linear    the norm before a block, quantised per token, and the int8 projection that reads it
  pre_norm  the norm before a block
  post_norm residual + scale * gate * norm(block output), and the next block's norm of the sum
  select    the best beams over beams x vocabulary
  reorder   the key/value states follow their beams, in place
  step      select, then reorder
"""
import math
import sys

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
INF = float("inf")


def mq():
    if "mojo-adreno_b200" not in sys.path:
        sys.path.insert(0, "mojo-adreno_b200")
    import mq as package

    return package


def listed():
    return [
        # Llama-3.2-1B's attention output projection for one token: the smallest call, all latency.
        {"name": "product 1x2048x2048", "kind": "product", "m": 1, "n": 2048, "k": 2048, "bias": False, "out": "f16"},
        # Its vocabulary head for one token: a long stream of weights, fp32 logits.
        {"name": "product head 1x128256x2048", "kind": "product", "m": 1, "n": 128256, "k": 2048, "bias": False,
         "out": "f32"},
        # Its gate|up for a decode batch of 64.
        {"name": "gate_up 64x8192x2048", "kind": "gate_up", "m": 64, "n": 8192, "k": 2048, "out": "f16"},
        # A prompt of 431 tokens through the down projection (the benchmark's prompt length, ragged).
        {"name": "product 431x2048x8192", "kind": "product", "m": 431, "n": 2048, "k": 8192, "bias": True, "out": "f32"},
        # Qwen3-8B's gate|up for a long prefill: the largest call.
        {"name": "gate_up 8192x12288x4096", "kind": "gate_up", "m": 8192, "n": 12288, "k": 4096, "out": "bf16"},
        # A few sequences decoding together, an odd width: norm, quantisation and projection as one path.
        {"name": "linear 5x4099x2048", "kind": "linear", "m": 5, "n": 4099, "k": 2048, "x": "bf16", "out": "bf16"},
        # The norm before a block over a long prefill.
        {"name": "pre_norm 8192x4096", "kind": "pre_norm", "m": 8192, "k": 4096, "x": "bf16", "out": "bf16"},
        # Between two blocks while decoding one token: the post norm with a per-channel gate, and the next norm.
        {"name": "post_norm 1x4096", "kind": "post_norm", "m": 1, "k": 4096, "x": "f32", "out": "f16", "gates": 1},
        # The same between two blocks of a long batch of 13 sequences, each with a gate of its own.
        {"name": "post_norm 12337x4096", "kind": "post_norm", "m": 12337, "k": 4096, "x": "bf16", "out": "bf16",
         "gates": 13},
        # One request, four beams: selection over Qwen3's vocabulary and its states.
        {"name": "step 1x4x151669", "kind": "step", "batch": 1, "beams": 4, "vocab": 151669, "x": "f16", "tensors": 8,
         "heads": 8, "length": 333, "most": 512, "dim": 128},
        # A batch of 64 requests with 8 beams each over Llama's vocabulary, fp32 logits.
        {"name": "select 64x8x128256", "kind": "select", "batch": 64, "beams": 8, "vocab": 128256, "x": "f32"},
        # Their states after a thousand tokens: two of a layer's tensors, the cache longer than what is filled.
        {"name": "reorder 64x8 len 1001", "kind": "reorder", "batch": 64, "beams": 8, "moved": 5, "tensors": 2,
         "heads": 8, "length": 1001, "most": 1024, "dim": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["product", "product", "gate_up", "linear", "pre_norm", "post_norm", "select", "step", "reorder"])
    out, x = rng.choice(["f32", "f16", "bf16"]), rng.choice(["f32", "f16", "bf16"])
    if kind in ("product", "gate_up", "linear"):
        m, n, k = _log(rng, 1, 8192), _log(rng, 17, 24000), _log(rng, 31, 12300)
        while (2 if kind == "gate_up" else 1) * m * n * k > 5e11:
            m = max(1, m // 2)
        case = {"kind": kind, "m": m, "n": n, "k": k, "out": out}
        if kind == "product":
            case["bias"] = rng.random() < 0.5
        if kind == "linear":
            case["x"], case["out"] = x, rng.choice(["f16", "bf16"])
        return case
    if kind in ("pre_norm", "post_norm"):
        m, k = _log(rng, 1, 12000), _log(rng, 100, 8200)
        while m * k > 5e7:
            m = m // 2
        case = {"kind": kind, "m": m, "k": k, "x": x, "out": out}
        if kind == "post_norm":
            case["gates"] = rng.choice([0, 1, m])
        return case
    batch, beams = _log(rng, 1, 64), rng.randint(2, 8)
    if kind == "select":
        return {"kind": kind, "batch": batch, "beams": beams, "vocab": _log(rng, 1000, 128256), "x": x}
    length = _log(rng, 1, 1000)
    case = {"kind": kind, "batch": batch, "beams": beams, "tensors": rng.randint(1, 4), "heads": rng.choice([2, 4, 8]),
            "length": length, "most": length + rng.choice([0, 7, 64]), "dim": rng.choice([64, 128])}
    while case["batch"] * beams * case["tensors"] * case["heads"] * case["most"] * case["dim"] > 4e8:
        case["batch"] = max(1, case["batch"] // 2)
        case["tensors"] = max(1, case["tensors"] // 2)
    if kind == "reorder":
        case["moved"] = rng.randint(1, beams - 1)
    else:
        case["vocab"], case["x"] = _log(rng, 1000, 151936), x
        while case["batch"] * beams * case["vocab"] > 3e7:
            case["batch"] = max(1, case["batch"] // 2)
            case["vocab"] = case["vocab"] // 2 + 1
    return case


def _int8(g, rows, cols):
    """Quantised values as they come from normally distributed numbers: int8 rows, 16 bytes aligned."""
    q = torch.empty(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    step = max(1, (1 << 27) // cols)
    for r in range(0, rows, step):
        part = torch.randn(min(step, rows - r), cols, generator=g, device="cuda")
        q[r:r + step, :cols] = (part * 33).round_().clamp_(-127, 127).to(torch.int8)
    return q[:, :cols]


def _uniform(g, shape, lo, hi):
    return torch.rand(shape, generator=g, device="cuda") * (hi - lo) + lo


def _hidden(g, rows, cols, dtype):
    """Hidden states: rows of different sizes, a few channels far larger than the others."""
    x = torch.randn(rows, cols, generator=g, device="cuda") * _uniform(g, (rows, 1), 0.3, 3.0)
    x[:, :: max(1, cols // 5)] *= 12
    return x.to(DT[dtype])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, kind = case, case["kind"]
    s = {"case": case}
    if kind in ("product", "gate_up", "linear"):
        rows = 2 * c["n"] if kind == "gate_up" else c["n"]
        s["wq"], s["ws"] = _int8(g, rows, c["k"]), _uniform(g, rows, 2e-4, 1e-3)
        if kind == "linear":
            s["x"], s["w"] = _hidden(g, c["m"], c["k"], c["x"]), _uniform(g, c["k"], 0.5, 1.5).to(DT[c["x"]])
            s["q"] = torch.empty(c["m"], (c["k"] + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :c["k"]]
            s["s"] = torch.empty(c["m"], device="cuda")
        else:
            s["xq"], s["xs"] = _int8(g, c["m"], c["k"]), _uniform(g, c["m"], 5e-3, 5e-2)
        if c.get("bias"):
            s["bias"] = torch.randn(c["n"], generator=g, device="cuda")
        s["y"] = torch.empty(c["m"], c["n"], dtype=DT[c["out"]], device="cuda")
    elif kind in ("pre_norm", "post_norm"):
        s["x"], s["w"] = _hidden(g, c["m"], c["k"], c["x"]), _uniform(g, c["k"], 0.5, 1.5).to(DT[c["x"]])
        s["h"] = torch.empty(c["m"], c["k"], dtype=DT[c["out"]], device="cuda")
        if kind == "post_norm":
            s["residual"], s["next_w"] = _hidden(g, c["m"], c["k"], c["x"]), _uniform(g, c["k"], 0.5, 1.5).to(DT[c["x"]])
            s["gate"] = torch.randn(c["gates"], c["k"], generator=g, device="cuda").to(DT[c["x"]]) if c["gates"] else None
            s["r"] = torch.empty_like(s["residual"])
    if kind in ("select", "step"):
        b, i, v = c["batch"], c["beams"], c["vocab"]
        s["logits"] = torch.empty(b * i, v, dtype=DT[c["x"]], device="cuda")
        for r in range(0, b * i, 64):
            part = torch.randn(min(64, b * i - r), v, generator=g, device="cuda") * 2.5
            part[torch.rand(part.shape, generator=g, device="cuda") < 0.05] = -INF  # tokens that are not allowed here
            s["logits"][r:r + 64] = part.to(DT[c["x"]])
        s["scores"] = _uniform(g, (b, i), -30.0, -20.0).sort(-1, descending=True).values.contiguous()
        s["scores"][:: 5, 1:] = -INF  # a request at its first step: one beam counts
        s["finished"] = (torch.rand(b, i, generator=g, device="cuda") < 0.1).to(torch.uint8)
        s["eos"] = 2
        for name, t in (("next_scores", torch.float32), ("tokens", torch.int32), ("parents", torch.int32),
                        ("next_finished", torch.uint8)):
            s[name] = torch.empty(b, i, dtype=t, device="cuda")
    if kind in ("reorder", "step"):
        b, i = c["batch"], c["beams"]
        full = torch.randn(c["tensors"], b * i, c["heads"], c["most"], c["dim"], generator=g, device="cuda",
                           dtype=torch.float16)
        s["states"] = full[:, :, :, :c["length"]]
        s["each"] = list(s["states"])
        if kind == "reorder":  # some beams die; each takes over from one that lives on
            order = torch.rand(b, i, generator=g, device="cuda").argsort(-1)
            dead, alive = order[:, :c["moved"]], order[:, c["moved"]:]
            take = torch.arange(c["moved"], device="cuda") % alive.shape[1]
            s["parents"] = torch.arange(i, device="cuda").expand(b, i).contiguous().scatter_(1, dead, alive[:, take]).int()
    return s


def _norm(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()


def _product(xq, xs, wq, ws):
    return (xq.float() @ wq.float().T) * xs[:, None] * ws


def _select(s):
    b, i, v = s["case"]["batch"], s["case"]["beams"], s["case"]["vocab"]
    z = s["logits"].float().view(b, i, v)
    top = z.amax(-1, keepdim=True)
    z = s["scores"][..., None] + (z - (top + (z - top).exp().sum(-1, keepdim=True).log()))
    z = torch.where(z.isnan(), torch.full_like(z, -INF), z)
    done = s["finished"].bool()
    at_eos = torch.arange(v, device=z.device) == s["eos"]
    z = torch.where(done[..., None], torch.where(at_eos, s["scores"][..., None], torch.full_like(z[:, :, :1], -INF)), z)
    value, at = z.view(b, i * v).sort(dim=-1, descending=True, stable=True)
    value, at = value[:, :i].contiguous(), at[:, :i]
    parents, tokens = at // v, at % v
    after = done.gather(1, parents) | (tokens == s["eos"])
    return {"scores": value, "tokens": tokens.int(), "parents": parents.int(), "finished": after.to(torch.uint8)}


def _reorder(s, parents):
    c = s["case"]
    base = torch.arange(c["batch"], device="cuda")[:, None] * c["beams"]
    s["states"].copy_(s["states"].index_select(1, (base + parents).view(-1)))
    return s["states"]


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        return _run_own(s, c, kind)
    out = DT[c.get("out", "f32")]
    if kind == "product":
        y = _product(s["xq"], s["xs"], s["wq"], s["ws"])
        return (y + s["bias"] if c["bias"] else y).to(out)
    if kind == "gate_up":
        y = _product(s["xq"], s["xs"], s["wq"], s["ws"])
        g, u = y[:, :c["n"]], y[:, c["n"]:]
        return (g / (1 + torch.exp(-g)) * u).to(out)
    if kind == "linear":
        h = _norm(s["x"], s["w"])
        scale = h.abs().amax(-1) / 127
        q = (h / scale[:, None]).round()
        return _product(q, scale, s["wq"], s["ws"]).to(out)
    if kind == "pre_norm":
        return _norm(s["x"], s["w"]).to(out)
    if kind == "post_norm":
        h = _norm(s["x"], s["w"])
        if c["gates"]:
            h = (h.view(c["gates"], -1, c["k"]) * s["gate"].float()[:, None]).view(c["m"], c["k"])
        r = s["residual"].float() + 0.7 * h
        return {"residual": r.to(s["residual"].dtype), "h": _norm(r, s["next_w"]).to(out)}
    if kind == "reorder":
        return _reorder(s, s["parents"])
    got = _select(s)
    if kind == "step":
        got["states"] = _reorder(s, got["parents"])
    return got


def _run_own(s, c, kind):
    m = mq()
    if kind == "product":
        return m.gemm_w8a8(s["xq"], s["xs"], s["wq"], s["ws"], s["y"], bias=s.get("bias"))
    if kind == "gate_up":
        return m.gate_up_w8a8(s["xq"], s["xs"], s["wq"], s["ws"], s["y"])
    if kind == "linear":
        q, scale = m.pre_norm_s8(s["x"], s["w"], EPS, s["q"], s["s"])
        return m.gemm_w8a8(q, scale, s["wq"], s["ws"], s["y"])
    if kind == "pre_norm":
        return m.pre_norm(s["x"], s["w"], EPS, s["h"])
    if kind == "post_norm":
        r, h = m.post_norm(s["x"], s["w"], s["residual"], s["next_w"], gate=s["gate"], scale=0.7, eps=EPS, out=s["r"],
                           h=s["h"])
        return {"residual": r, "h": h}
    if kind == "reorder":
        m.beam_reorder(s["each"], s["parents"])
        return s["states"]
    scores, tokens, parents, finished = m.beam_select(
        s["logits"], s["scores"], finished=s["finished"], eos=s["eos"], next_scores=s["next_scores"], tokens=s["tokens"],
        parents=s["parents"], next_finished=s["next_finished"])
    got = {"scores": scores, "tokens": tokens, "parents": parents, "finished": finished}
    if kind == "step":
        m.beam_reorder(s["each"], parents)
        got["states"] = s["states"]
    return got


def work(case):
    c, kind = case, case["kind"]
    total, flops = 0, 0
    if kind in ("product", "gate_up", "linear"):
        rows = 2 * c["n"] if kind == "gate_up" else c["n"]
        total += rows * c["k"] + 4 * rows + c["m"] * c["n"] * SIZE[c["out"]] + (4 * c["n"] if c.get("bias") else 0)
        total += c["m"] * c["k"] * (SIZE[c["x"]] if kind == "linear" else 1) + (0 if kind == "linear" else 4 * c["m"])
        total += SIZE[c["x"]] * c["k"] if kind == "linear" else 0
        flops += 2 * c["m"] * rows * c["k"]
    elif kind == "pre_norm":
        total += (c["m"] + 1) * c["k"] * SIZE[c["x"]] + c["m"] * c["k"] * SIZE[c["out"]]
        flops += 4 * c["m"] * c["k"]
    elif kind == "post_norm":
        total += (3 * c["m"] + 2 + c["gates"]) * c["k"] * SIZE[c["x"]] + c["m"] * c["k"] * SIZE[c["out"]]
        flops += 10 * c["m"] * c["k"]
    if kind in ("select", "step"):
        rows = c["batch"] * c["beams"]
        total += rows * c["vocab"] * SIZE[c["x"]] + 18 * rows
        flops += 4 * rows * c["vocab"]
    if kind in ("reorder", "step"):
        row = c["tensors"] * c["heads"] * c["length"] * c["dim"] * 2
        moved = c["moved"] if kind == "reorder" else c["beams"] - 1  # of a step about all but one move
        sources = min(moved, c["beams"] - moved) if kind == "reorder" else 1
        total += c["batch"] * (moved + sources) * row
    return {"bytes": total, "flops": flops}


def exact(case, seed):
    s, c = prepare(case, seed), case
    kind, f64 = c["kind"], torch.float64

    def rms(x, w):
        return x / ((x * x).sum(-1, keepdim=True) / c["k"] + EPS).sqrt() * w.to(f64)

    if kind in ("product", "gate_up", "linear"):
        if kind == "linear":
            h = rms(s["x"].to(f64), s["w"])
            biggest = h.abs().max(-1).values
            xq, xs = torch.round(h * (127 / biggest)[:, None]), biggest / 127
        else:
            xq, xs = s["xq"].to(f64), s["xs"].to(f64)
        y = torch.einsum("tk,rk->tr", xq, s["wq"].to(f64)) * torch.outer(xs, s["ws"].to(f64))
        if c.get("bias"):
            y += s["bias"].to(f64)
        return y[:, :c["n"]] * torch.sigmoid(y[:, :c["n"]]) * y[:, c["n"]:] if kind == "gate_up" else y
    if kind == "pre_norm":
        return rms(s["x"].to(f64), s["w"])
    if kind == "post_norm":
        h = rms(s["x"].to(f64), s["w"])
        if c["gates"]:
            h *= s["gate"].to(f64).repeat_interleave(c["m"] // c["gates"], 0)
        r = s["residual"].to(f64) + 0.7 * h
        return {"residual": r, "h": rms(r, s["next_w"])}
    base = (torch.arange(c["batch"] * c["beams"], device="cuda") // c["beams"] * c["beams"])
    if kind == "reorder":
        return s["states"][:, base + s["parents"].view(-1).long()].to(f64)
    v, rows = c["vocab"], []
    for b in range(c["batch"]):  # by the definition, one request at a time
        z = s["logits"][b * c["beams"]:(b + 1) * c["beams"]].to(f64)
        z = torch.log_softmax(z, -1) + s["scores"][b].to(f64)[:, None]
        done = s["finished"][b].bool()
        z[done] = -INF
        z[done, s["eos"]] = s["scores"][b][done].to(f64)
        rows.append(z.view(-1).topk(c["beams"]))
    got = {"scores": torch.stack([r.values for r in rows]), "tokens": None, "parents": None, "finished": None}
    if kind == "step":
        parents = torch.stack([r.indices for r in rows]) // v
        got["states"] = s["states"][:, base + parents.view(-1)].to(f64)
    return got
