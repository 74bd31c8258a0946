"""Cases for the operators at the end of a decode step, with their plain forms in torch:

* ``moe``      the whole MoE feed-forward layer of a few tokens over Q4_0 experts: RMSNorm (optional), routing,
               SwiGLU experts, gate-weighted sum, gated shared expert and residual (optional);
* ``lora``     a projection over GGUF weights shared by all tokens, beside each token's own low-rank adapter;
* ``logprobs`` log probabilities of given tokens, entropy and the most likely alternatives, from logits.

``run`` takes the plain form where ``own`` is false and the framework's entry points where it is true.
"""
import math

import torch

own = False

DEV = "cuda"
NEG_INF = float("-inf")
ADAPTER_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LOGIT_TYPES = ADAPTER_TYPES
QTYPE = {"q8_0": 8, "q4_0": 2}
BLOCK_BYTES = {"q8_0": 34, "q4_0": 18}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _moe(name, T, d, f, E, k, shared, bias=False, norm=False, residual=False):
    return dict(name=name, op="moe", T=T, d=d, f=f, E=E, k=k, shared=shared, bias=bias, norm=norm, residual=residual)


def _lora(name, T, n_in, n_out, q, rank, adapters, dtype):
    return dict(name=name, op="lora", T=T, n_in=n_in, n_out=n_out, q=q, rank=rank, adapters=adapters, dtype=dtype)


def _logprobs(name, T, V, dtype, top, targets, masked=False, pad=0):
    return dict(name=name, op="logprobs", T=T, V=V, dtype=dtype, top=top, targets=targets, masked=masked, pad=pad)


def listed():
    return [
        # one request decoding: a stack layer with its norm and residual, where latency counts
        _moe("moe 1 token", 1, 2048, 512, 256, 8, True, norm=True, residual=True),
        # a handful of requests decoding together, skewed expert load
        _moe("moe 5 tokens", 5, 2048, 512, 256, 8, True, bias=True),
        # sixteen tokens of a small model without a shared expert
        _moe("moe 16 tokens 64 experts", 16, 1024, 256, 64, 4, False),
        # the largest batch of the path: most experts are touched
        _moe("moe 16 tokens 256 experts", 16, 2048, 512, 256, 8, True, norm=True, residual=True),
        # one request's adapter beside a square projection
        _lora("lora 1 token", 1, 2048, 2048, "q8_0", 16, 4, "f16"),
        # sixteen requests, eight adapters of rank up to 64, a wide 4-bit projection
        _lora("lora 16 tokens 4 bits", 16, 4096, 12288, "q4_0", 64, 8, "bf16"),
        # an odd batch and odd sizes, adapters kept in 32 bits
        _lora("lora 37 tokens ragged", 37, 1024, 3001, "q4_0", 12, 5, "f32"),
        # the LM head of a decode batch with sixteen adapters
        _lora("lora 64 tokens LM head", 64, 2048, 151936, "q8_0", 16, 16, "f16"),
        # the sampled token of one request with its twenty best alternatives
        _logprobs("logprobs 1 row", 1, 151936, "f32", 20, 1),
        # a masked vocabulary, several candidate tokens a row, rows at an odd stride
        _logprobs("logprobs 7 rows masked", 7, 50257, "f16", 20, 4, masked=True, pad=3),
        # a decode batch
        _logprobs("logprobs 64 rows", 64, 151936, "f32", 5, 1),
        # scoring a prompt
        _logprobs("logprobs 2048 rows", 2048, 32000, "bf16", 1, 1),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["moe", "lora", "logprobs"])
    if op == "moe":
        d, f = rng.choice([1024, 2048, 4096]), rng.choice([128, 256, 512, 1024])
        E = _log_int(rng, 8, min(512, 256 * 512 * 2048 // (d * f)))
        c = _moe(None, _log_int(rng, 1, 16), d, f, E, rng.randint(1, min(8, E)), rng.random() < 0.7,
                 rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5)
    elif op == "lora":
        n_in = 32 * _log_int(rng, 8, 256)
        T = _log_int(rng, 1, 256)
        n_out = _log_int(rng, 200, 151936)
        rank = _log_int(rng, 1, 128)
        while n_in * n_out > 2048 * 151936 or T * n_out * rank > 64 * 151936 * 16 or T * n_in * n_out > 64 * 2048 * 151936:
            n_out = max(1, n_out // 2)
        c = _lora(None, T, n_in, n_out, rng.choice(["q8_0", "q4_0"]), rank, _log_int(rng, 1, 32),
                  rng.choice(["f16", "bf16", "f32"]))
    else:
        T, V = _log_int(rng, 1, 2048), _log_int(rng, 1000, 262144)
        while T * V > 2048 * 32000:
            T = max(1, T // 2)
        c = _logprobs(None, T, V, rng.choice(["f32", "f16", "bf16"]), rng.choice([0, 1, 3, 8, 20, 32]),
                      rng.randint(0, 5), rng.random() < 0.4, rng.choice([0, 0, 0, 1, 8, 37]))
    del c["name"]
    return c


def _ranks(case):
    """Adapter i has rank R, R/2 or R/4 in turn: requests bring adapters of different ranks."""
    return [max(1, case["rank"] >> (i % 3)) for i in range(case["adapters"])]


def work(case):
    T = case["T"]
    if case["op"] == "moe":
        d, f, E, k, sh = case["d"], case["f"], case["E"], case["k"], int(case["shared"])
        used = E * (1.0 - (1.0 - k / E) ** T)  # experts some token uses, expected
        nbytes = (used + sh) * 3 * d * f * 18 / 32 + (E + sh) * d * 4 + 2 * T * d * 4 + (E * 4 if case["bias"] else 0)
        return {"bytes": nbytes, "flops": T * (k + sh) * 6.0 * d * f + 2.0 * T * (E + sh) * d}
    if case["op"] == "lora":
        n_in, n_out, n, ranks = case["n_in"], case["n_out"], case["adapters"], _ranks(case)
        r = sum(ranks) / n
        used = n * (1.0 - (1.0 - 1.0 / (n + 1)) ** T)  # adapters some token uses, expected
        es = 4 if case["dtype"] == "f32" else 2
        nbytes = n_in * n_out // 32 * BLOCK_BYTES[case["q"]] + 4 * T * (n_in + n_out) + used * r * (n_in + n_out) * es + 4 * T
        return {"bytes": nbytes, "flops": 2.0 * T * n_in * n_out + 2.0 * T * r * (n_in + n_out) * n / (n + 1)}
    V, es = case["V"], 4 if case["dtype"] == "f32" else 2
    return {"bytes": T * V * es + T * (case["targets"] * 12 + 4 + 8 * case["top"]), "flops": 6.0 * T * V}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _round_half_away(v):
    """roundf of an f32 tensor, in 64 bits so that adding one half rounds nothing."""
    v = v.double()
    return torch.floor(v.abs() + 0.5) * torch.sign(v)


def _gguf(w, q):
    """GGUF blocks (uint8 [rows, cols / 32, block bytes]) of f32 weights w [rows, cols]; Q4_0 bytes hold elements
    2i (low nibble) and 2i + 1."""
    b = w.reshape(w.shape[0], -1, 32)
    if q == "q8_0":
        d = b.abs().amax(-1, keepdim=True) / 127.0
        v = torch.where(d > 0, b / d, torch.zeros_like(b))
        qs = _round_half_away(v).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    else:
        at = b.abs().argmax(-1, keepdim=True)
        d = b.gather(-1, at) / -8.0
        v = torch.where(d != 0, b / d, torch.zeros_like(b))
        nib = (v + 8.5).floor().clamp(0, 15).to(torch.uint8)
        qs = nib[..., 0::2] | (nib[..., 1::2] << 4)
    return torch.cat([d.half().view(torch.uint8), qs], -1)


def _weights(gen, rows, cols, q, std=0.02):
    raw = torch.empty(rows, cols // 32, BLOCK_BYTES[q], dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // cols)
    for r in range(0, rows, step):  # a few hundred MB of 32-bit weights at a time
        n = min(step, rows - r)
        raw[r:r + n] = _gguf(torch.randn(n, cols, device=DEV, generator=gen) * std, q)
    return raw


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    randint = lambda lo, hi, s: torch.randint(lo, hi, s, device=DEV, generator=gen)  # noqa: E731
    T, st = case["T"], dict(case)
    if case["op"] == "moe":
        d, f, E = case["d"], case["f"], case["E"]
        st["x"] = randn(T, d)
        st["router"] = randn(E, d) * 0.02
        st["router_bias"] = None
        if case["bias"]:  # a Zipf-like preference, experts in random order
            st["router_bias"] = 2.0 * torch.log(1.0 / (torch.randperm(E, device=DEV, generator=gen) + 1.0))
        st["gate"], st["up"] = _weights(gen, E * f, d, "q4_0"), _weights(gen, E * f, d, "q4_0")
        st["down"] = _weights(gen, E * d, f, "q4_0")
        st["shared_w"] = None
        if case["shared"]:
            st["shared_w"] = (_weights(gen, f, d, "q4_0"), _weights(gen, f, d, "q4_0"), _weights(gen, d, f, "q4_0"),
                              randn(d) * 0.02)
        if own:
            from powerinfer_x64_b200.moe import MoeLayer

            st["layer"] = MoeLayer(st["router"], st["gate"], st["up"], st["down"], QTYPE["q4_0"], d, f, E, case["k"],
                                   shared=st["shared_w"], router_bias=st["router_bias"])
            st["gate"] = st["up"] = st["down"] = st["shared_w"] = None  # the layer holds the weights
    elif case["op"] == "lora":
        n_in, n_out, n, R = case["n_in"], case["n_out"], case["adapters"], case["rank"]
        dt = ADAPTER_TYPES[case["dtype"]]
        st["x"] = randn(T, n_in)
        st["w"] = _weights(gen, n_out, n_in, case["q"])
        st["a"] = (randn(n, R, n_in) / math.sqrt(n_in)).to(dt)
        st["b"] = (randn(n, n_out, R) * 0.05).to(dt)
        st["ranks"] = torch.tensor(_ranks(case), dtype=torch.int32, device=DEV)
        st["scales"] = torch.rand(n, device=DEV, generator=gen) + 0.5
        st["ids"] = randint(-1, n, (T,)).int()
        if own:
            from powerinfer_x64_b200.lora import AdapterBank, SharedProjection

            st["proj"] = SharedProjection(st["w"], QTYPE[case["q"]], n_out, n_in)
            st["bank"] = AdapterBank(st["a"], st["b"], ranks=st["ranks"], scales=st["scales"])
            st["w"] = None  # the projection holds the weights
    else:
        V = case["V"]
        wide = randn(T, V + case["pad"]) * 2.5
        wide[:, :V].scatter_add_(1, randint(0, V, (T, 8)), randn(T, 8).abs() * 6.0)  # a few likely tokens a row
        if case["masked"]:  # a grammar leaves some tokens; a row may be left with none
            wide[torch.rand(wide.shape, device=DEV, generator=gen) < 0.7] = NEG_INF
            wide[T // 2] = NEG_INF
        st["logits"] = wide.to(LOGIT_TYPES[case["dtype"]])[:, :V]
        st["ids"] = randint(0, V, (T, case["targets"]))
        if case["targets"]:
            st["ids"][randint(0, 16, (T, case["targets"])) == 0] = -1  # padding: no token
        else:
            st["ids"] = None
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _dequantise(raw, q):
    """f32 [..., cols] of GGUF blocks [..., cols / 32, block bytes]."""
    d = raw[..., :2].contiguous().view(torch.float16).float()
    if q == "q8_0":
        v = raw[..., 2:].contiguous().view(torch.int8).float()
    else:
        v = torch.stack([raw[..., 2:] & 15, raw[..., 2:] >> 4], -1).flatten(-2).float() - 8.0
    return (v * d).flatten(-2)


def _quantised_activations(x):
    """x as Q8_0 holds it: per 32 values d = max|x| / 127, q = round(x (1 / d)) half away from zero, d kept in f16."""
    b = x.reshape(x.shape[0], -1, 32)
    d = b.abs().amax(-1, keepdim=True) / 127.0
    inv = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
    return (_round_half_away(b * inv).clamp(-127, 127).float() * d.half().float()).flatten(1)


def _plain_moe(st):
    x, T, d, f, E, k = st["x"], st["T"], st["d"], st["f"], st["E"], st["k"]
    h = x
    if st["norm"]:
        h = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    logits = h.double() @ st["router"].double().T  # 64 bits: the choice of experts hangs on near ties
    if st["router_bias"] is not None:
        logits = logits + st["router_bias"]
    p, order = torch.sort(torch.softmax(logits, -1), dim=-1, descending=True, stable=True)
    gates = (p[:, :k] / p[:, :k].sum(-1, keepdim=True)).float()
    idx = order[:, :k]
    gate = _dequantise(st["gate"].view(E, f, d // 32, 18)[idx], "q4_0")  # [T, k, f, d]
    up = _dequantise(st["up"].view(E, f, d // 32, 18)[idx], "q4_0")
    v = h[:, None, :, None]
    g, u = (gate @ v).squeeze(-1), (up @ v).squeeze(-1)
    del gate, up
    down = _dequantise(st["down"].view(E, d, f // 32, 18)[idx], "q4_0")  # [T, k, d, f]
    y = (down @ (g / (1.0 + torch.exp(-g)) * u)[..., None]).squeeze(-1)
    out = (gates[..., None] * y).sum(1)
    if st["shared_w"] is not None:
        gate, up, down = (_dequantise(w, "q4_0") for w in st["shared_w"][:3])
        g, u = h @ gate.T, h @ up.T
        share = 1.0 / (1.0 + torch.exp(-(h @ st["shared_w"][3])))
        out = out + share[:, None] * ((g / (1.0 + torch.exp(-g)) * u) @ down.T)
    return {"out": x + out if st["residual"] else out}


def _plain_lora(st):
    x, ids, R = st["x"], st["ids"].long(), st["rank"]
    base = _quantised_activations(x) if st["q"] == "q8_0" else x
    y = base @ _dequantise(st["w"], st["q"]).T
    a = ids.clamp(min=0)
    use = (torch.arange(R, device=DEV) < st["ranks"].long()[a][:, None]) & (ids >= 0)[:, None]
    h = (st["a"][a].float() @ x[:, :, None]).squeeze(-1)  # [T, R]
    h = torch.where(use, h, torch.zeros_like(h)) * st["scales"][a][:, None]
    return {"y": y + (st["b"][a].float() @ h[:, :, None]).squeeze(-1)}


def _plain_logprobs(st):
    x, V, n = st["logits"].float(), st["V"], st["top"]
    m = x.amax(-1, keepdim=True)
    none = m == NEG_INF  # a row whose mask leaves nothing
    t = x - torch.where(none, torch.zeros_like(m), m)
    e = torch.exp(t)
    s = e.sum(-1, keepdim=True)
    log_s = torch.where(none, torch.zeros_like(s), torch.log(s))
    w = torch.where(e > 0, t * e, torch.zeros_like(t)).sum(-1, keepdim=True)
    out = {"entropy": torch.where(none, torch.zeros_like(s), log_s - w / s).squeeze(-1)}
    if st["ids"] is not None:
        lp = t.gather(1, st["ids"].clamp(min=0)) - log_s
        out["logp"] = torch.where(st["ids"] >= 0, lp, torch.zeros_like(lp))
    if n:
        # one key a token, larger for a larger logit and, where they tie, for a lower index
        bits = (x + 0.0).contiguous().view(torch.int32).long()
        key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32) | (0x7FFFFFFF - torch.arange(V, device=DEV))
        ids = 0x7FFFFFFF - (torch.topk(key, n, dim=-1).values & 0x7FFFFFFF)
        lp = t.gather(1, ids) - log_s
        out["top_logp"] = lp
        out["top_ids"] = torch.where(lp == NEG_INF, torch.full_like(ids, -1), ids).int()
    return out


def run(state):
    if own:
        if state["op"] == "moe":
            return {"out": state["layer"].forward(state["x"], rmsnorm=state["norm"], residual=state["residual"],
                                                  path="fused")}
        if state["op"] == "lora":
            return {"y": state["proj"].forward(state["x"], state["bank"], state["ids"])}
        from powerinfer_x64_b200.logprobs import token_logprobs

        r = token_logprobs(state["logits"], targets=state["ids"], n_top=state["top"])
        out = {"entropy": r.entropy}
        if r.logp is not None:
            out["logp"] = r.logp
        if r.top_ids is not None:
            out["top_logp"], out["top_ids"] = r.top_logp, r.top_ids
        return out
    return {"moe": _plain_moe, "lora": _plain_lora, "logprobs": _plain_logprobs}[state["op"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_matrix(raw, q):
    """f64 matrix of GGUF rows [rows, cols / 32, block bytes], block element by block element."""
    rows, nb = raw.shape[:2]
    scale = (raw[:, :, 0].to(torch.int32) | (raw[:, :, 1].to(torch.int32) << 8)).to(torch.int16).view(torch.float16)
    m = torch.empty(rows, nb, 32, dtype=torch.float64, device=DEV)
    if q == "q8_0":
        v = raw[:, :, 2:].to(torch.float64)
        m[:] = torch.where(v > 127, v - 256, v)
    else:
        for i in range(16):
            m[:, :, 2 * i] = (raw[:, :, 2 + i] % 16).to(torch.float64) - 8
            m[:, :, 2 * i + 1] = torch.div(raw[:, :, 2 + i], 16, rounding_mode="floor").to(torch.float64) - 8
    m *= scale.to(torch.float64)[:, :, None]
    return m.view(rows, nb * 32)


def _exact_swiglu(x, gate, up, down):
    g, u = _exact_matrix(gate, "q4_0") @ x, _exact_matrix(up, "q4_0") @ x
    return _exact_matrix(down, "q4_0") @ (g * torch.sigmoid(g) * u)


def _exact_moe(st):
    d, f, E, k = st["d"], st["f"], st["E"], st["k"]
    outs = []
    for t in range(st["T"]):
        x = st["x"][t].double()
        h = x / torch.sqrt(x.square().sum() / d + 1e-6) if st["norm"] else x
        logit = (st["router"].double() * h).sum(1)
        if st["router_bias"] is not None:
            logit += st["router_bias"].double()
        prob = torch.exp(logit - logit.max()).cpu().tolist()
        best = sorted(sorted(range(E), key=lambda e: (-prob[e], e))[:k])
        total = sum(prob[e] for e in best)
        acc = torch.zeros(d, dtype=torch.float64, device=DEV)
        for e in best:
            acc += prob[e] / total * _exact_swiglu(h, st["gate"].view(E, f, d // 32, 18)[e],
                                                   st["up"].view(E, f, d // 32, 18)[e],
                                                   st["down"].view(E, d, f // 32, 18)[e])
        if st["shared_w"] is not None:
            gate, up, down, s = st["shared_w"]
            acc += torch.sigmoid((s.double() * h).sum()) * _exact_swiglu(h, gate, up, down)
        outs.append(acc + x if st["residual"] else acc)
    return {"out": torch.stack(outs)}


def _exact_lora(st):
    x = st["x"]
    if st["q"] == "q8_0":  # the operator's own rounding of its input: 32-bit scale and reciprocal, f16 block scale
        blocks = x.unflatten(1, (-1, 32))
        d = blocks.abs().max(-1).values / 127
        inv = torch.where(d == 0, torch.zeros_like(d), torch.reciprocal(d))
        v = (blocks * inv[..., None]).double()
        whole = torch.trunc(v)
        whole = whole + torch.where((v - whole).abs() >= 0.5, torch.sign(v), torch.zeros_like(v))
        base = (whole.clamp(-127, 127) * d.to(torch.float16).double()[..., None]).flatten(1)
    else:
        base = x.double()
    y = torch.empty(st["T"], st["n_out"], dtype=torch.float64, device=DEV)
    for r in range(0, st["n_out"], 16384):
        y[:, r:r + 16384] = base @ _exact_matrix(st["w"][r:r + 16384], st["q"]).T
    for t, a in enumerate(st["ids"].tolist()):
        if a >= 0:
            r = int(st["ranks"][a])
            low = st["a"][a, :r].double() @ x[t].double()
            y[t] += float(st["scales"][a]) * (st["b"][a, :, :r].double() @ low)
    return {"y": y}


def _exact_logprobs(st):
    out = {"entropy": [], "logp": [], "top_logp": [], "top_ids": None}
    n = st["top"]
    for t in range(st["T"]):
        x = st["logits"][t].double()
        live = x[x > NEG_INF]
        if live.numel():
            logp = x - torch.logsumexp(live, 0)
            lv = live - torch.logsumexp(live, 0)
            out["entropy"].append(-(lv.exp() * lv).sum())
        else:
            logp = x
            out["entropy"].append(torch.zeros((), dtype=torch.float64, device=DEV))
        if st["ids"] is not None:
            i = st["ids"][t]
            out["logp"].append(torch.where(i < 0, 0.0, logp[i.clamp(min=0)]))
        if n:
            out["top_logp"].append(torch.topk(logp, n).values)
    return {k: torch.stack(v) if v else None for k, v in out.items()}


def exact(case, seed):
    st = prepare(case, seed)
    return {"moe": _exact_moe, "lora": _exact_lora, "logprobs": _exact_logprobs}[case["op"]](st)
