"""The operators around the packed attention in a decode step as sized cases: products with 4-bit
weights, the quantizer that makes these weights, and sampling of the next token.

A case is a dict of plain values.  ``prepare`` makes what a program holds before the call, ``run``
is one pass: with ``own`` through the framework's entry points (``rdkv_amd.weight_quant``,
``rdkv_amd.sampling``), without it in elementary tensor operations.  ``exact`` states the same
results in 64 bits, ``work`` the bytes and operations that no implementation can leave out.

Kinds:

* ``linear``   - activation rows times a 4-bit weight matrix (a projection of a decode step, of a batch, of a prompt chunk).
* ``mlp``      - one token's MLP block over 4-bit weights: residual add + norm + gate / up, SiLU + down.
* ``quantize`` - a weight matrix quantized by groups and its values read back, as on loading a model.
* ``sample``   - the next token of every sequence from its logits, with per-sequence settings.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
TINY = 2.0 ** -120          # a group whose scale would be below this is all zeros


def listed():
    return [
        # output projection of one decoded token, 8B layer shape: launches and latency
        {"name": "linear_1x4096x4096", "kind": "linear", "rows": 1, "N": 4096, "K": 4096, "group": 128, "dtype": "f16",
         "bias": False},
        # LM head of one decoded token: a stream of a quarter gigabyte
        {"name": "linear_1x128256x4096", "kind": "linear", "rows": 1, "N": 128256, "K": 4096, "group": 128,
         "dtype": "bf16", "bias": False},
        # q/k/v projection with bias of five sequences decoded together, finer groups
        {"name": "linear_5x6144x4096", "kind": "linear", "rows": 5, "N": 6144, "K": 4096, "group": 64, "dtype": "bf16",
         "bias": True},
        # a matrix of odd sizes (a pruned or adapted model), a few rows, the finest groups
        {"name": "linear_17x4001x2027", "kind": "linear", "rows": 17, "N": 4001, "K": 2027, "group": 32, "dtype": "f16",
         "bias": True},
        # gate and up projection of 64 sequences
        {"name": "linear_64x28672x4096", "kind": "linear", "rows": 64, "N": 28672, "K": 4096, "group": 128,
         "dtype": "f16", "bias": False},
        # a prompt chunk through the down projection
        {"name": "linear_500x4096x14336", "kind": "linear", "rows": 500, "N": 4096, "K": 14336, "group": 128,
         "dtype": "bf16", "bias": False},
        # the MLP block of one decoded token, 8B layer shape
        {"name": "mlp_4096x14336", "kind": "mlp", "hidden": 4096, "inner": 14336, "group": 128, "dtype": "f16"},
        # a square projection on loading
        {"name": "quantize_4096x4096", "kind": "quantize", "N": 4096, "K": 4096, "group": 128, "dtype": "f16"},
        # gate and up on loading, rows that end inside a group
        {"name": "quantize_28672x4100", "kind": "quantize", "N": 28672, "K": 4100, "group": 32, "dtype": "bf16"},
        # one sequence, nucleus sampling over a 128k vocabulary: latency
        {"name": "sample_1x128256", "kind": "sample", "rows": 1, "vocab": 128256, "dtype": "f16", "settings": "top_p",
         "masked": 0.0},
        # a served batch, every sequence with its own settings, some of the vocabulary forbidden
        {"name": "sample_64x128256", "kind": "sample", "rows": 64, "vocab": 128256, "dtype": "f32", "settings": "mixed",
         "masked": 0.3},
        # a large batch over an odd vocabulary
        {"name": "sample_240x151937", "kind": "sample", "rows": 240, "vocab": 151937, "dtype": "bf16",
         "settings": "mixed", "masked": 0.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "linear", "mlp", "quantize", "sample", "sample", "sample"])
    if kind == "sample":
        rows = _log_int(rng, 1, 240)
        return {"kind": kind, "rows": rows, "vocab": _log_int(rng, 500, 151937), "dtype": rng.choice(["f16", "bf16", "f32"]),
                "settings": rng.choice(["top_k", "top_p", "min_p", "mixed", "mixed", "plain"]),
                "masked": rng.choice([0.0, 0.3, 0.99])}
    case = {"kind": kind, "group": rng.choice([32, 64, 128, 128]), "dtype": rng.choice(["f16", "bf16"])}
    if kind == "mlp":
        return {**case, "hidden": 512 * rng.randint(1, 16), "inner": 512 * rng.randint(2, 32)}
    N, K = _log_int(rng, 64, 28672), _log_int(rng, 64, 14336)
    if rng.random() < 0.6:                 # most models: multiples of 64
        N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
    if kind == "quantize":
        return {**case, "N": N, "K": K}
    rows = 1 if rng.random() < 0.3 else _log_int(rng, 2, 64) if rng.random() < 0.8 else _log_int(rng, 65, 500)
    most = 500 * 4096 * 14336              # no dearer than the largest listed one
    return {**case, "rows": max(1, min(rows, most // (N * K))), "N": N, "K": K, "bias": rng.random() < 0.4}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed((seed * 1_000_003 + stream) % (1 << 62))


def _rows(rows, K, gen, dtype):
    """Activations: unit normal, a few channels twenty times as large, as a residual stream has them."""
    x = torch.randn(rows, K, generator=gen, device=DEV)
    big = torch.randint(0, K, (max(1, K // 1000),), generator=gen, device=DEV)
    x[:, big] *= 20.0
    return x.to(dtype)


def _quantized(N, K, group, gen, dtype):
    """A quantized matrix as a checkpoint holds it: codes [N, K], scales and zero points [N, groups]."""
    codes = torch.randn(N, K, generator=gen, device=DEV).mul_(2.7).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
    groups = -(-K // group)
    scale = (torch.rand(N, groups, generator=gen, device=DEV) + 0.5).mul_(0.02 / math.sqrt(K / 64)).to(dtype)
    zero = torch.randint(5, 11, (N, groups), generator=gen, device=DEV, dtype=torch.uint8)
    state = {"codes": codes, "scale": scale, "zero": zero, "group": group}
    if own:                                # laid out once, as the program that decodes with it keeps it
        from rdkv_amd import weight_quant
        state["packed"] = weight_quant.pack_weight(codes, scale, zero, group)
    return state


def _settings(case, gen):
    B = case["rows"]
    u = lambda lo, hi: torch.rand(B, generator=gen, device=DEV) * (hi - lo) + lo  # noqa: E731
    temperature, top_p, min_p = u(0.6, 1.3), u(0.8, 1.0), u(0.01, 0.1)
    top_k = torch.randint(1, 200, (B,), generator=gen, device=DEV, dtype=torch.int32)
    pick = torch.randint(0, 6, (B,), generator=gen, device=DEV)
    kind = case["settings"]
    if kind == "mixed":                    # greedy, plain, one filter, or all of them
        temperature = torch.where(pick == 0, torch.zeros_like(temperature), temperature)
    on = {"top_k": (pick == 2) | (pick == 5), "top_p": (pick == 3) | (pick == 5), "min_p": (pick == 4) | (pick == 5)}
    if kind != "mixed":
        on = {k: torch.full((B,), k == kind, device=DEV) for k in on}
    return {"temperature": temperature, "top_k": torch.where(on["top_k"], top_k, torch.zeros_like(top_k)),
            "top_p": torch.where(on["top_p"], top_p, torch.ones_like(top_p)),
            "min_p": torch.where(on["min_p"], min_p, torch.zeros_like(min_p))}


def prepare(case, seed):
    gen, dtype, kind = _gen(seed, 1), DTYPES[case["dtype"]], case["kind"]
    state = {"kind": kind, "dtype": dtype}
    if kind == "linear":
        state["w"] = _quantized(case["N"], case["K"], case["group"], gen, dtype)
        state["x"] = _rows(case["rows"], case["K"], gen, dtype)
        state["bias"] = torch.randn(case["N"], generator=gen, device=DEV).to(dtype) if case["bias"] else None
    elif kind == "mlp":
        H, F = case["hidden"], case["inner"]
        state["up"] = _quantized(2 * F, H, case["group"], gen, dtype)
        state["down"] = _quantized(H, F, case["group"], gen, dtype)
        state["h"] = _rows(1, H, gen, dtype)
        state["delta"] = torch.randn(1, H, generator=gen, device=DEV).to(dtype)
        state["norm"] = (torch.rand(H, generator=gen, device=DEV) + 0.5).to(dtype)
    elif kind == "quantize":
        w = torch.randn(case["N"], case["K"], generator=gen, device=DEV)
        state["weight"] = w.mul_(0.02).to(dtype)
        state["group"] = case["group"]
    else:
        B, V = case["rows"], case["vocab"]
        logits = torch.randn(B, V, generator=gen, device=DEV).mul_(2.0)
        hot = torch.randint(0, V, (B, 24), generator=gen, device=DEV)     # what the context makes likely
        logits.scatter_(1, hot, torch.rand(B, 24, generator=gen, device=DEV) * 8 + 6)
        if case["masked"]:
            forbidden = torch.rand(B, V, generator=gen, device=DEV) < case["masked"]
            forbidden.scatter_(1, hot[:, :1], False)                      # something is always allowed
            half = torch.arange(B, device=DEV).view(B, 1) % 2 == 0        # both ways programs mask
            low = torch.where(half, float("-inf"), torch.finfo(dtype).min)
            logits = torch.where(forbidden, low, logits)
        state["logits"] = logits.to(dtype)
        state["uniform"] = torch.rand(B, generator=gen, device=DEV)
        state.update(_settings(case, gen))
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _dense(w):
    """The matrix that the codes stand for, in 32 bits."""
    K = w["codes"].shape[1]
    at = torch.arange(K, device=DEV) // w["group"]
    return (w["codes"].float() - w["zero"].float()[:, at]) * w["scale"].float()[:, at]


def _product(x, w, bias=None):
    y = x.float() @ _dense(w).t()
    if bias is not None:
        y = y + bias.float()
    return y.to(x.dtype)


def _mlp(s):
    r = (s["h"].float() + s["delta"].float()).to(s["dtype"])
    f = r.float()
    x = (s["norm"].float() * (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS))).to(s["dtype"])
    gate_up = _product(x, s["up"])
    gate, up = gate_up.float().chunk(2, dim=-1)
    act = (gate / (1 + torch.exp(-gate))).to(s["dtype"]).float()
    return [gate_up, r, _product((act * up).to(s["dtype"]), s["down"])]


def _scale20(s):
    """fp32 rounded to 20 significant bits; groups of (next to) nothing have scale 1."""
    s = ((s.view(torch.int32) + 8) & -16).view(torch.float32)
    return torch.where(s < TINY, torch.ones_like(s), s)


def _quantize(weight, group):
    N, K = weight.shape
    pad = -K % group
    w = torch.nn.functional.pad(weight.float(), (0, pad)).view(N, -1, group)
    lo, hi = w.amin(-1, keepdim=True).clamp(max=0), w.amax(-1, keepdim=True).clamp(min=0)
    s = _scale20(((hi - lo) / 15).contiguous())
    z = torch.round(-lo / s).clamp(0, 15)
    q = (torch.round(w / s) + z).clamp(0, 15)
    return ((q - z) * s).to(weight.dtype).view(N, K + pad)[:, :K].contiguous()


def _sample(s):
    l = s["logits"].double() + 0.0
    l = torch.where(torch.isnan(l), float("-inf"), l)
    t = s["temperature"].double().view(-1, 1)
    greedy = ~(t > 0)
    val, order = torch.sort(l, dim=1, descending=True, stable=True)
    m = val[:, :1]
    z = torch.where(val == m, torch.zeros_like(val), (val - m) / torch.where(greedy, torch.ones_like(t), t))
    w = torch.where(torch.isneginf(val), torch.zeros_like(z), torch.exp(z))
    place = torch.arange(l.shape[1], device=l.device).view(1, -1)
    k = s["top_k"].view(-1, 1)
    first = place == 0
    wk = torch.where((k <= 0) | (place < k), w, torch.zeros_like(w))
    cum = wk.cumsum(1)
    before = torch.cat([torch.zeros_like(m), cum[:, :-1]], 1)
    p, least = s["top_p"].double().view(-1, 1), s["min_p"].double().view(-1, 1)
    kept = first | (((p >= 1) | (before < p * cum[:, -1:])) & (w >= least))
    wk = torch.where(kept, wk, torch.zeros_like(w))
    cum = wk.cumsum(1)
    mass = cum[:, -1:]
    at = (cum <= s["uniform"].double().view(-1, 1) * mass).sum(1, keepdim=True)
    at = torch.minimum(at, ((wk > 0).sum(1, keepdim=True) - 1).clamp(min=0))
    at = torch.where(greedy, torch.zeros_like(at), at)
    token = order.gather(1, at)
    logprob = torch.where(greedy, torch.zeros_like(mass), z.gather(1, at) - torch.log(mass))
    none = torch.isneginf(m)
    token = torch.where(none, torch.full_like(token, -1), token)
    logprob = torch.where(none, torch.full_like(logprob, float("-inf")), logprob)
    return [token.view(-1), logprob.view(-1).float()]


def run(state):
    kind = state["kind"]
    if own:
        from rdkv_amd import sampling, weight_quant
        if kind == "linear":
            return weight_quant.linear(state["x"], state["w"]["packed"], state["bias"])
        if kind == "mlp":
            gate_up, r = weight_quant.norm_linear(state["h"], state["delta"], state["norm"], EPS, state["up"]["packed"])
            gate, up = gate_up.chunk(2, dim=-1)
            return [gate_up, r, weight_quant.silu_linear(gate, up, state["down"]["packed"])]
        if kind == "quantize":
            return weight_quant.dequantize_weight(weight_quant.quantize_weight(state["weight"], state["group"]))
        return list(sampling.sample_tokens(state["logits"], state["uniform"], temperature=state["temperature"],
                                           top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"]))
    if kind == "linear":
        return _product(state["x"], state["w"], state["bias"])
    if kind == "mlp":
        return _mlp(state)
    if kind == "quantize":
        return _quantize(state["weight"], state["group"])
    return _sample(state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and its results in 64 bits
# ---------------------------------------------------------------------------------------------
def _weight_bytes(N, K, group):
    return N * (K / 2 + 4 * -(-K // group))


def work(case):
    kind = case["kind"]
    if kind == "linear":
        M, N, K = case["rows"], case["N"], case["K"]
        return {"bytes": _weight_bytes(N, K, case["group"]) + 2 * (M * K + M * N + (N if case["bias"] else 0)),
                "flops": 2 * M * N * K}
    if kind == "mlp":
        H, F = case["hidden"], case["inner"]
        return {"bytes": _weight_bytes(2 * F, H, case["group"]) + _weight_bytes(H, F, case["group"]) + 2 * (5 * H + 4 * F),
                "flops": 6 * H * F}
    if kind == "quantize":
        N, K = case["N"], case["K"]
        # the matrix read, codes and scales written and read, the values written
        return {"bytes": 4 * N * K + 2 * _weight_bytes(N, K, case["group"]), "flops": 6 * N * K}
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 32), "flops": 4 * case["rows"] * case["vocab"]}


def _exact_product(x, w, bias=None):
    """[rows, N] in 64 bits, from group sums: each group's products first, then its scale."""
    codes, scale, zero, group = w["codes"], w["scale"].double(), w["zero"].double(), w["group"]
    N, K = codes.shape
    x = x.double()
    out = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    for begin in range(0, N, 4096):
        rows = slice(begin, min(begin + 4096, N))
        for g in range(scale.shape[1]):
            ks = slice(g * group, min((g + 1) * group, K))
            dots = x[:, ks] @ (codes[rows, ks].double() - zero[rows, g:g + 1]).t().contiguous()
            out[:, rows] += dots * scale[rows, g]
    return out if bias is None else out + bias.double()


def _exact_quantize(weight, group):
    out = torch.empty(weight.shape, dtype=torch.float64, device=weight.device)
    for k in range(0, weight.shape[1], group):
        w = weight[:, k:k + group].double()
        zero = torch.zeros_like(w[:, :1])
        lo, hi = torch.minimum(w.min(1, keepdim=True).values, zero), torch.maximum(w.max(1, keepdim=True).values, zero)
        step = (hi - lo) / 15
        mantissa, exponent = torch.frexp(step)
        step = torch.ldexp(torch.floor(mantissa * 2.0 ** 20 + 0.5), exponent - 20)     # 20 bits of it
        step = torch.where(step < TINY, torch.ones_like(step), step)
        z = torch.clamp(torch.round(-lo / step), 0, 15)
        q = torch.clamp(torch.round(w / step) + z, 0, 15)
        out[:, k:k + group] = (q - z) * step
    return out


def _exact_sample(s):
    logits = s["logits"].double().cpu().numpy()
    u, t, k, p, least = (s[n].double().cpu().numpy() for n in ("uniform", "temperature", "top_k", "top_p", "min_p"))
    tokens, logprobs = [], []
    for b in range(logits.shape[0]):
        x = logits[b]
        ids = np.flatnonzero(x > -np.inf)                  # (a NaN compares false)
        if ids.size == 0:
            tokens.append(-1)
            logprobs.append(-np.inf)
            continue
        ids = ids[np.argsort(-x[ids], kind="stable")]
        if not t[b] > 0:
            tokens.append(int(ids[0]))
            logprobs.append(0.0)
            continue
        top = x[ids[0]]
        z = np.zeros(ids.size)
        z[x[ids] != top] = (x[ids][x[ids] != top] - top) / t[b]
        if k[b] > 0:
            ids, z = ids[:int(k[b])], z[:int(k[b])]
        w = np.exp(z)
        n = ids.size
        if p[b] < 1:
            n = min(n, int(np.searchsorted(np.cumsum(w), p[b] * w.sum(), side="left")) + 1)
        n = max(1, min(n, int((w >= least[b]).sum())))
        cum = np.cumsum(w[:n])
        i = min(int(np.searchsorted(cum, u[b] * cum[-1], side="right")), int((w[:n] > 0).sum()) - 1)
        tokens.append(int(ids[i]))
        logprobs.append(float(z[i] - np.log(cum[-1])))
    return [np.array(tokens, dtype=np.int64), np.array(logprobs)]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "linear":
        return _exact_product(s["x"], s["w"], s["bias"])
    if kind == "quantize":
        return _exact_quantize(s["weight"], s["group"])
    if kind == "sample":
        return _exact_sample(s)
    dtype = s["dtype"]
    r = (s["h"].double() + s["delta"].double()).to(dtype)              # what a step stores in between is part of it
    x = s["norm"].double() * r.double() / torch.sqrt((r.double() ** 2).mean() + EPS)
    gate_up = _exact_product(x.to(dtype), s["up"])
    gate, up = gate_up.to(dtype).double().chunk(2, dim=-1)
    act = (gate * torch.sigmoid(gate)).to(dtype).double() * up
    return [gate_up, r.double(), _exact_product(act.to(dtype), s["down"])]
