"""Measured cases of the serving operators: attention over packed prompts and
for single tokens, the mixture-of-experts layer for a few tokens, and packed
int4/int8 products for a few tokens.

``run`` computes each operator in elementary torch operations, or, where
``own`` is true, through ``ennx_b200.ops``.  ``exact`` computes the same from
the operator's definition in 64 bits.
"""
import math

import torch

own = False

D = 128          # head width of the framework's attention
THETA = 1e6      # HybridConfig.rope_theta
DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a few short requests entering together: launch and latency bound
        {"name": "prompt_short", "op": "prompt", "lengths": "1,37,129,200", "hq": 16, "hkv": 4},
        # a batch of prompts of ordinary, ragged lengths (the 16384 tokens of the attention benchmark)
        {"name": "prompt_ragged", "op": "prompt", "hq": 16, "hkv": 4,
         "lengths": "2048,17,731,1500,4001,64,3333,1,255,1023,2048,1363"},
        # one long document
        {"name": "prompt_long", "op": "prompt", "lengths": "16384", "hq": 16, "hkv": 4},
        # one user, a short context: latency
        {"name": "token_one_user", "op": "token", "lengths": "301", "room": 1024, "hq": 16, "hkv": 4},
        # a serving batch with ragged contexts, one slot of it empty
        {"name": "token_batch", "op": "token", "room": 4096, "hq": 16, "hkv": 4,
         "lengths": "4096,1,777,2048,0,3001,1500,64,4095,129,2222,900,3600,2500,1777,410,"
                    "1024,3333,2,1200,2900,640,4000,33,1999,2750,3100,480,2047,1111,3700,1601"},
        # few users, very long contexts: the cache has to be split along its length
        {"name": "token_long", "op": "token", "lengths": "131072,65537,100001,131072", "room": 131072,
         "hq": 16, "hkv": 4},
        # the MoE layer of HybridConfig for one token, a small batch, and the most the form takes
        {"name": "moe_1", "op": "moe", "tokens": 1, "hidden": 2048, "experts": 64, "top_k": 8, "width": 768},
        {"name": "moe_8", "op": "moe", "tokens": 8, "hidden": 2048, "experts": 64, "top_k": 8, "width": 768},
        {"name": "moe_64", "op": "moe", "tokens": 64, "hidden": 2048, "experts": 64, "top_k": 8, "width": 768},
        # a packed projection for one token (int4, group 64: the decode benchmark's linears)
        {"name": "packed_qkv_1", "op": "packed", "tokens": 1, "inp": 2048, "out": 6144, "bits": 4, "group": 64,
         "moved": False},
        # the tied LM head for a small batch
        {"name": "packed_head_4", "op": "packed", "tokens": 4, "inp": 2048, "out": 151936, "bits": 4, "group": 64,
         "moved": False},
        # an int8 projection under a candidate's integer-code perturbation, an odd width that ends inside a group
        {"name": "packed_int8_16", "op": "packed", "tokens": 16, "inp": 2011, "out": 2048, "bits": 8, "group": 64,
         "moved": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "token", "moe", "packed"])
    if op == "prompt":
        hq, hkv = rng.choice([(16, 4), (16, 4), (8, 2), (4, 1), (2, 1), (4, 4)])
        total, count = _log(rng, 32, 16384), _log(rng, 1, 48)
        cuts = sorted(rng.randint(0, total) for _ in range(count - 1))
        lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
        return {"op": op, "lengths": ",".join(map(str, lengths)), "hq": hq, "hkv": hkv}
    if op == "token":
        hq, hkv = rng.choice([(16, 4), (16, 4), (8, 2), (4, 1), (4, 2), (2, 1), (16, 1)])
        batch = _log(rng, 1, 64)
        room = _log(rng, 16, min(131072, 400000 // batch))
        lengths = [rng.randint(0, room) for _ in range(batch)]
        return {"op": op, "lengths": ",".join(map(str, lengths)), "room": room, "hq": hq, "hkv": hkv}
    if op == "moe":
        experts = rng.choice([8, 16, 40, 64])
        return {"op": op, "tokens": _log(rng, 1, 64), "hidden": 64 * rng.randint(4, 32), "experts": experts,
                "top_k": rng.randint(1, 8), "width": 128 * rng.randint(1, 6)}
    inp = _log(rng, 16, 4096)
    if rng.random() < 0.6:
        inp = max(64, inp // 64 * 64)
    return {"op": op, "tokens": rng.randint(1, 16), "inp": inp, "out": _log(rng, 16, 16384), "bits": rng.choice([4, 8]),
            "group": rng.choice([16, 32, 64, 128]), "moved": rng.random() < 0.4}


def _lengths(case):
    return [int(v) for v in case["lengths"].split(",")]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(gen, *shape, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=gen, dtype=torch.float32) * std).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"op": case["op"]}
    if case["op"] == "prompt":
        ln = _lengths(case)
        total, hq, hkv = sum(ln), case["hq"], case["hkv"]
        # columns of one fused projection, as a layer has them
        qkv = _normal(gen, total, (hq + 2 * hkv) * D)
        s["q"] = qkv[:, :hq * D].unflatten(1, (hq, D))
        s["k"] = qkv[:, hq * D:(hq + hkv) * D].unflatten(1, (hkv, D))
        s["v"] = qkv[:, (hq + hkv) * D:].unflatten(1, (hkv, D))
        s["cu"] = torch.tensor([0] + ln, device=DEV).cumsum(0).to(torch.int32)
    elif case["op"] == "token":
        ln = _lengths(case)
        batch, hq, hkv = len(ln), case["hq"], case["hkv"]
        s["kc"] = torch.randn(batch, case["room"], hkv, D, device=DEV, generator=gen, dtype=torch.bfloat16)
        s["vc"] = torch.randn(batch, case["room"], hkv, D, device=DEV, generator=gen, dtype=torch.bfloat16)
        s["q"], s["k"], s["v"] = (_normal(gen, batch, h, D) for h in (hq, hkv, hkv))
        s["lengths"] = torch.tensor(ln, device=DEV, dtype=torch.int32)
    elif case["op"] == "moe":
        t, h, e, w = case["tokens"], case["hidden"], case["experts"], case["width"]
        s["top_k"] = case["top_k"]
        s["x"], s["residual"] = _normal(gen, t, h), _normal(gen, t, h)
        s["w_router"] = _normal(gen, e, h, std=1.5 / math.sqrt(h))
        # rows in blocks of 256 = [128 gate | 128 up]
        s["w_gate_up"] = torch.randn(e, 2 * w, h, device=DEV, generator=gen, dtype=torch.bfloat16).mul_(h ** -0.5)
        s["w_down"] = torch.randn(e, h, w, device=DEV, generator=gen, dtype=torch.bfloat16).mul_(w ** -0.5)
    else:
        inp, out, bits, group = case["inp"], case["out"], case["bits"], case["group"]
        row_bytes, groups = (inp * bits + 7) // 8, -(-inp // group)
        top = (1 << bits) - 1
        s["x"] = _normal(gen, case["tokens"], inp)
        s["weights"] = torch.randint(0, 256, (out * row_bytes,), device=DEV, generator=gen, dtype=torch.uint8)
        # affine codes of weights of size 1 / sqrt(inp), their zero near the middle code
        s["scales"] = (torch.rand(out * groups, device=DEV, generator=gen) + 0.5) * (3.0 / (top * math.sqrt(inp)))
        s["biases"] = -s["scales"] * (top / 2 + torch.rand(out * groups, device=DEV, generator=gen) - 0.5)
        s["linear"] = (0, 0, 0, inp, out, bits, group, 12345, 0, 0x20000000)
        s["seed"] = (0x9E3779B1 ^ seed, 0x51ED270B, int(case["moved"]))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"prompt": _prompt, "token": _token, "moe": _moe, "packed": _packed}[s["op"]](s)


def _run_own(s):
    from ennx_b200 import _abi, ops
    if s["op"] == "prompt":
        # rotated already: the projection's q and k are left as they are
        return ops.gqa_attention_packed(s["q"], s["k"], s["v"], s["cu"], rope_theta=0.0)
    if s["op"] == "token":
        o = ops.gqa_attention_decode(s["q"], s["kc"], s["vc"], s["lengths"], k=s["k"], v=s["v"], rope_theta=THETA)
        return {"out": o, "k_cache": s["kc"], "v_cache": s["vc"]}
    if s["op"] == "moe":
        y, idx, gate = ops.moe_layer_decode(s["x"], s["w_router"], s["w_gate_up"], s["w_down"], s["top_k"],
                                            residual=s["residual"], return_routing=True)
        return {"y": y, "index": idx, "gate": gate}
    return ops.packed_linear_decode(s["x"], s["weights"], s["scales"], s["biases"], _abi.PackedLinear(*s["linear"]),
                                    s["seed"])


def _prompt(s):
    q, k, v, cu = s["q"].float(), s["k"].float(), s["v"].float(), s["cu"]
    total, hq, _ = q.shape
    hkv = k.shape[1]
    pos = torch.arange(total, device=q.device)
    seq = torch.searchsorted(cu, pos.to(torch.int32), right=True)
    hidden = (seq[:, None] != seq[None, :]) | (pos[None, :] > pos[:, None])
    qh = q.view(total, hkv, hq // hkv, D).permute(1, 2, 0, 3) * (1.0 / math.sqrt(D))
    a = (qh.reshape(hkv, -1, D) @ k.permute(1, 2, 0)).view(hkv, hq // hkv, total, total)
    a.masked_fill_(hidden, float("-inf"))
    a.sub_(a.amax(-1, keepdim=True)).exp_()
    norm = a.sum(-1, keepdim=True)
    o = (a.view(hkv, -1, total) @ v.permute(1, 0, 2)).view(hkv, hq // hkv, total, D) / norm
    return o.permute(2, 0, 1, 3).reshape(total, hq, D).to(torch.bfloat16)


def _turn(x, position):
    """Rotate-half RoPE of x [B, heads, D] in 32 bits, the angles in 64."""
    freq = THETA ** (-torch.arange(D // 2, device=x.device, dtype=torch.float64) * (2.0 / D))
    angle = position.double()[:, None, None] * freq
    c, n = angle.cos().float(), angle.sin().float()
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c - b * n, b * c + a * n], -1)


def _token(s):
    q, kc, vc, ln = s["q"], s["kc"], s["vc"], s["lengths"].long()
    batch, room, hkv, _ = kc.shape
    hq = q.shape[1]
    live = torch.nonzero(ln > 0)[:, 0]
    at = (ln - 1).clamp(min=0)
    kc[live, at[live]] = _turn(s["k"], at)[live].to(torch.bfloat16)
    vc[live, at[live]] = s["v"][live]
    qh = _turn(q, at).view(batch, hkv, hq // hkv, D) * (1.0 / math.sqrt(D))
    a = qh @ kc.permute(0, 2, 3, 1).float()
    unseen = torch.arange(room, device=q.device) >= ln[:, None]
    a.masked_fill_(unseen[:, None, None, :], float("-inf"))
    top = a.amax(-1, keepdim=True)
    a = (a - torch.where(torch.isfinite(top), top, 0.0)).exp()
    norm = a.sum(-1, keepdim=True)
    o = a @ vc.permute(0, 2, 1, 3).float()
    o = torch.where(norm > 0, o / norm, 0.0)
    return {"out": o.reshape(batch, hq, D).to(torch.bfloat16), "k_cache": kc, "v_cache": vc}


def _moe(s):
    x, kk = s["x"].float(), s["top_k"]
    tokens, hidden = x.shape
    logits = s["x"].double() @ s["w_router"].double().T
    kept, idx = torch.sort(logits, dim=1, descending=True, stable=True)
    kept, idx = kept[:, :kk].float(), idx[:, :kk]
    gate = (kept - kept.amax(1, keepdim=True)).exp()
    gate = gate / gate.sum(1, keepdim=True)
    gu = s["w_gate_up"][idx.reshape(-1)].float() @ x.repeat_interleave(kk, 0)[:, :, None]
    gu = gu.view(tokens * kk, -1, 2, 128)
    g, u = gu[:, :, 0].flatten(1), gu[:, :, 1].flatten(1)
    h = g / (1.0 + torch.exp(-g)) * u
    d = (s["w_down"][idx.reshape(-1)].float() @ h[:, :, None]).view(tokens, kk, hidden)
    y = s["residual"].float() + (d * gate[:, :, None]).sum(1)
    return {"y": y.to(torch.bfloat16), "index": idx.to(torch.int32), "gate": gate}


def _packed(s):
    _, _, _, inp, out, bits, group, element, whole, threshold = s["linear"]
    row_bytes, groups, top = (inp * bits + 7) // 8, -(-inp // group), (1 << bits) - 1
    code = s["weights"].view(out, row_bytes)
    if bits == 4:
        code = torch.stack([code & 15, code >> 4], -1).view(out, -1)[:, :inp]
    if s["seed"][2]:
        code = code.to(torch.int64)
        low, high, _ = s["seed"]
        word = 0xFFFFFFFF
        r = torch.arange(out * inp, device=code.device).view(out, inp) + element & word
        r = low & word ^ (r * 0x9E3779B9 & word)
        r = (r ^ r >> 16) * 0x7FEB352D & word
        r = (r ^ r >> 15) * 0x846CA68B & word
        r = (r ^ r >> 15) ^ high
        step = whole + (r >> 1 < threshold >> 1).long()
        down = torch.where(code >= step, code - step, (code + step).clamp(max=top))
        up = torch.where(code + step <= top, code + step, (code - step).clamp(min=0))
        code = torch.where(step == 0, code, torch.where(r & 1 == 0, down, up))
    column = torch.arange(inp, device=code.device) // group
    w = code.float() * s["scales"].view(out, groups)[:, column] + s["biases"].view(out, groups)[:, column]
    return (s["x"].float() @ w.T).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# what one pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "prompt":
        ln, hq, hkv = _lengths(case), case["hq"], case["hkv"]
        return {"bytes": 2.0 * D * sum(ln) * (2 * hq + 2 * hkv),
                "flops": 4.0 * D * hq * sum(n * (n + 1) / 2 for n in ln)}
    if case["op"] == "token":
        ln, hq, hkv = _lengths(case), case["hq"], case["hkv"]
        rows = max(1, sum(ln))
        return {"bytes": 2.0 * D * (2 * hkv * rows + 2 * (hq + 2 * hkv) * len(ln)), "flops": 4.0 * D * hq * rows}
    if case["op"] == "moe":
        t, h, e, w, kk = (case[n] for n in ("tokens", "hidden", "experts", "width", "top_k"))
        used = e * (1.0 - (1.0 - kk / e) ** t)  # experts that a token picked, on average
        return {"bytes": 2.0 * (3 * used * h * w + e * h + 3 * t * h) + 8.0 * t * kk,
                "flops": 2.0 * t * h * (3 * kk * w + e)}
    t, inp, out, bits, group = (case[n] for n in ("tokens", "inp", "out", "bits", "group"))
    return {"bytes": float(out * ((inp * bits + 7) // 8) + 8 * out * -(-inp // group) + 2 * t * (inp + out)),
            "flops": 2.0 * t * inp * out}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prompt":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        group = case["hq"] // case["hkv"]
        o, first = torch.zeros_like(q), 0
        for n in _lengths(case):
            rows = slice(first, first + n)
            first += n
            causal = torch.ones(n, n, device=DEV, dtype=torch.bool).tril()
            for h in range(case["hq"]):
                a = q[rows, h] @ k[rows, h // group].T / math.sqrt(D)
                o[rows, h] = torch.softmax(torch.where(causal, a, -math.inf), -1) @ v[rows, h // group]
        return o
    if case["op"] == "token":
        kc, vc = s["kc"].double(), s["vc"].double()
        group = case["hq"] // case["hkv"]
        o = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
        unit = torch.polar(torch.ones(D // 2, device=DEV, dtype=torch.float64),
                           torch.pow(THETA, -torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D))

        def turned(x, p):
            z = torch.complex(x[:, :D // 2].double(), x[:, D // 2:].double())
            z = z * torch.polar(torch.ones_like(unit.real), unit.angle() * p)
            return torch.cat([z.real, z.imag], 1)

        for b, n in enumerate(_lengths(case)):
            if n == 0:
                continue
            kc[b, n - 1], vc[b, n - 1] = turned(s["k"][b], n - 1), s["v"][b].double()
            q = turned(s["q"][b], n - 1)
            for j in range(case["hkv"]):
                a = q[j * group:(j + 1) * group] @ kc[b, :n, j].T / math.sqrt(D)
                o[b, j * group:(j + 1) * group] = torch.softmax(a, -1) @ vc[b, :n, j]
        return {"out": o, "k_cache": kc, "v_cache": None}
    if case["op"] == "moe":
        x, y, gates = s["x"].double(), s["residual"].double(), []
        score = torch.einsum("th,eh->te", x, s["w_router"].double())
        for t in range(case["tokens"]):
            ranked = sorted(range(case["experts"]), key=lambda e, row=score[t].tolist(): (-row[e], e))[:case["top_k"]]
            gates.append(torch.softmax(score[t, ranked], 0))
            for r, e in enumerate(ranked):
                both = (s["w_gate_up"][e].double() @ x[t]).view(-1, 256)
                h = torch.nn.functional.silu(both[:, :128]).reshape(-1) * both[:, 128:].reshape(-1)
                y[t] += gates[-1][r] * (s["w_down"][e].double() @ h)
        return {"y": y, "index": None, "gate": torch.stack(gates)}
    return _exact_packed(s, case)


def _exact_packed(s, case):
    inp, out, bits, group = case["inp"], case["out"], case["bits"], case["group"]
    row_bytes, groups, top = (inp * bits + 7) // 8, -(-inp // group), 2 ** bits - 1
    low, high, moved = s["seed"]
    element, whole, threshold = s["linear"][7:]
    y = torch.empty(case["tokens"], out, device=DEV, dtype=torch.float64)
    column = torch.arange(inp, device=DEV)
    for first in range(0, out, 8192):
        last = min(out, first + 8192)
        byte = s["weights"][first * row_bytes:last * row_bytes].view(-1, row_bytes).to(torch.int64)
        code = byte[:, column * bits // 8] // (2 ** (column * bits % 8)) % (top + 1)
        if moved:
            index = (torch.arange(first, last, device=DEV)[:, None] * inp + column + element) % 2 ** 32
            v = torch.bitwise_xor((index * 0x9E3779B9) % 2 ** 32, torch.tensor(low % 2 ** 32, device=DEV))
            for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
                v = (torch.bitwise_xor(v, v // 2 ** shift) * factor) % 2 ** 32
            v = torch.bitwise_xor(torch.bitwise_xor(v, v // 2 ** 15), torch.tensor(high, device=DEV))
            amount = whole + (v // 2 < threshold // 2).to(torch.int64)
            sign = torch.where(v % 2 == 0, -amount, amount)
            there, back = code + sign, code - sign
            inside = (there >= 0) & (there <= top)
            code = torch.where(inside, there, back.clamp(0, top))
        scale = s["scales"].view(out, groups)[first:last].double()
        bias = s["biases"].view(out, groups)[first:last].double()
        w = code.double() * scale[:, column // group] + bias[:, column // group]
        y[:, first:last] = s["x"].double() @ w.T
    return y
