"""Measured cases of the attention-block operators: rotary positions, differential attention, group norm (channels last).

``run`` makes one pass through one operator: its plain form from elementary torch operations in 32 bits (``own = False``), or the
framework's entry points (``own = True``).  ``exact`` restates every operator in 64 bits, apart from the plain form, with the
gradients written out as formulas.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- the cases ---------------------------------------------------------------------------------------------------------
def _rotary(batch, n, heads, kv_heads, width, part, layout, type, start, scaling, grad):
    return dict(op="rotary", batch=batch, n=n, heads=heads, kv_heads=kv_heads, width=width, part=part, layout=layout, type=type,
                start=start, scaling=scaling, grad=grad)


def _norm(batch, n, channels, groups, activation, type, lengths, grad):
    return dict(op="norm", batch=batch, n=n, channels=channels, groups=groups, activation=activation, type=type, lengths=lengths,
                grad=grad)


def _diff(batch, nq, nk, heads, kv_heads, d, dv, type, causal, lengths, grad):
    return dict(op="diff", batch=batch, nq=nq, nk=nk, heads=heads, kv_heads=kv_heads, d=d, dv=dv, type=type, causal=causal,
                lengths=lengths, grad=grad)


def listed():
    cases = {
        # one new token for each of 8 sequences, far into a long context whose frequencies were stretched four times
        "rotary_token": _rotary(8, 1, 32, 8, 64, 64, "half", "bf16", 1_000_000, "yarn", False),
        # the residue sequences of one training batch (128 complexes, 283 positions), the models' 64 channels as two half heads
        "rotary_residues": _rotary(128, 283, 2, 2, 32, 32, "interleaved", "fp32", 0, "none", True),
        # long training sequences, grouped keys, half of each head rotated
        "rotary_long": _rotary(4, 8192, 32, 8, 128, 64, "half", "bf16", 0, "linear", True),
        # each residue's heads normalised on their own behind the attention (128 complexes of 190 nodes, 8 heads of 64 channels)
        "norm_heads": _norm(128 * 190, 1, 512, 8, "none", "bf16", "full", True),
        # node features of one training batch of padded residue graphs, statistics over each graph's own nodes
        "norm_graphs": _norm(128, 190, 64, 8, "silu", "fp32", "ragged", True),
        # a few peptides at inference: 11 residues
        "norm_peptides": _norm(4, 11, 64, 4, "gelu", "fp32", "full", False),
        # feature maps of long inputs
        "norm_long": _norm(2, 65536, 512, 32, "silu", "bf16", "full", True),
        # node attention of one training batch: 128 padded graphs of 190 nodes, 64 channels, one head
        "diff_nodes": _diff(128, 190, 190, 1, 1, 32, 64, "fp32", "none", "ragged", True),
        # inference on full residue sequences (283 positions), 8 heads
        "diff_residues": _diff(32, 283, 283, 8, 8, 32, 64, "fp16", "none", "ragged", False),
        # causal training on long sequences with grouped keys
        "diff_long": _diff(2, 4096, 4096, 16, 4, 64, 128, "bf16", "start", "full", True),
        # one new token for each of 16 sequences over caches that are filled differently
        "diff_token": _diff(16, 1, 16384, 16, 4, 64, 128, "bf16", "end", "ragged", False),
        # odd sizes, wide heads, queries and keys of different lengths, one sequence without keys
        "diff_odd": _diff(5, 517, 1531, 6, 2, 128, 256, "fp16", "none", "empty", True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, low, high):
    """a whole number of [low, high], even over its logarithm"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    type = rng.choice(["fp32", "bf16", "fp16"])
    op = rng.choice(["rotary", "norm", "diff", "diff"])
    limit = {c["name"]: work(c) for c in listed()}
    while True:
        if op == "rotary":
            width = rng.choice([16, 24, 32, 64, 80, 128])
            kv = rng.choice([1, 2, 4, 8])
            grad = rng.random() < 0.6
            case = _rotary(_spread(rng, 1, 128), 1 if rng.random() < 0.2 else _spread(rng, 2, 8192), kv * rng.choice([1, 2, 3, 4]), kv,
                           width, rng.choice([width, width // 2]), rng.choice(["half", "interleaved"]), type,
                           rng.choice([0, 0, rng.randrange(1, 1_000_000)]), rng.choice(["none", "linear", "ntk", "yarn"]), grad)
            top = "rotary_long"
        elif op == "norm":
            groups = rng.choice([1, 2, 4, 8, 16, 32])
            n = 1 if rng.random() < 0.25 else _spread(rng, 2, 65536)
            case = _norm(_spread(rng, 1, 20000 if n == 1 else 128), n, groups * rng.choice([2, 5, 8, 16, 24, 32, 64]), groups,
                         rng.choice(["none", "silu", "gelu", "relu"]), type, "full" if n == 1 else rng.choice(["full", "ragged", "empty"]),
                         rng.random() < 0.7)
            top = "norm_long"
        else:
            kv = rng.choice([1, 2, 4])
            d = rng.choice([8, 16, 24, 32, 48, 64]) if type == "fp32" else rng.choice([8, 16, 32, 40, 64, 96, 128])
            heads = kv * rng.choice([1, 2, 3, 4])
            causal = rng.choice(["none", "none", "start", "end"])
            if rng.random() < 0.3:      # a few new tokens over a cache
                case = _diff(_spread(rng, 1, 32), rng.choice([1, 1, 2, 5]), _spread(rng, 64, 16384), heads, kv, d, 2 * d, type, "end",
                             "ragged", False)
            else:
                nk = _spread(rng, 2, 4096)
                nq = nk if causal == "start" or rng.random() < 0.6 else _spread(rng, 1, 2048)
                case = _diff(_spread(rng, 1, 128), nq, nk, heads, kv, d, 2 * d, type, causal, rng.choice(["full", "ragged", "empty"]),
                             rng.random() < 0.6)
            top = "diff_long"
        need = work(case)
        # (the plain attention holds several full score matrices in 32 bits)
        scores = case["batch"] * case["heads"] * 2 * case["nq"] * case["nk"] if op == "diff" else 0
        most = limit[top]["flops"] / (16 if type == "fp32" else 1)
        if 0 < need["flops"] <= most and need["bytes"] <= limit[top]["bytes"] and scores <= 2 ** 30:
            return case


def _lengths(case):
    """valid rows (keys) of each sample: all, a spread over the upper two thirds, or the same with one sample that has none"""
    n = case["nk"] if case["op"] == "diff" else case["n"]
    if case["lengths"] == "full":
        return [n] * case["batch"]
    low = max(1, n // 3)
    out = [n - (i * 7919) % (n - low + 1) for i in range(case["batch"])]
    if case["lengths"] == "empty" and case["batch"] > 1:
        out[-1] = 0
    return out


def _ends(case, length):
    """how many keys each query of a sample sees: all, those up to its own position, or as the last positions of the sample"""
    nq = case["nq"]
    if case["causal"] == "start":
        return [min(length, i + 1) for i in range(nq)]
    if case["causal"] == "end":
        return [max(0, length - nq + 1 + i) for i in range(nq)]
    return [length] * nq


def work(case):
    size = _BYTES[case["type"]]
    if case["op"] == "rotary":
        elements = case["batch"] * case["n"] * (case["heads"] + case["kv_heads"]) * case["width"]
        turned = elements * case["part"] // case["width"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * 2 * elements * size + case["batch"] * case["n"] * 8, "flops": passes * 3 * turned}
    if case["op"] == "norm":
        whole = case["batch"] * case["n"] * case["channels"]
        valid = sum(_lengths(case)) * case["channels"]
        if case["grad"]:
            return {"bytes": (2 * valid + 2 * whole) * size + 4 * case["channels"] * 4, "flops": 24 * valid}
        return {"bytes": (valid + whole) * size + 2 * case["channels"] * 4, "flops": 8 * valid}
    b, nq, nk, h, hk, d, dv = (case[k] for k in ("batch", "nq", "nk", "heads", "kv_heads", "d", "dv"))
    lengths = _lengths(case)
    seen = {length: sum(_ends(case, length)) for length in set(lengths)}
    pairs = h * sum(seen[length] for length in lengths)
    q, o = b * nq * h * 2 * d, b * nq * h * dv
    valid = sum(lengths)
    kv, kv_whole = valid * hk * (2 * d + dv), b * nk * hk * (2 * d + dv)
    if case["grad"]:
        return {"bytes": (2 * q + 2 * o + kv + kv_whole) * size, "flops": pairs * (4 * d + 2 * dv + 8 * d + 4 * dv)}
    return {"bytes": (q + o + kv) * size, "flops": pairs * (4 * d + 2 * dv)}


# ---- inputs ------------------------------------------------------------------------------------------------------------
_SCALING = {"none": None, "linear": dict(kind="linear", factor=4.0), "ntk": dict(kind="ntk", factor=4.0),
            "yarn": dict(kind="yarn", factor=4.0, original_length=4096)}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    type = _TYPES[case["type"]]

    def normal(*shape, mean=0.0, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(type)

    if case["op"] == "rotary":
        b, n, w = case["batch"], case["n"], case["width"]
        start = torch.randint(0, 64, (b, 1), generator=gen, device="cuda") + case["start"]
        s = {"q": normal(b, n, case["heads"], w), "k": normal(b, n, case["kv_heads"], w),
             "positions": start + torch.arange(n, device="cuda")}
        if case["grad"]:
            s["dq"], s["dk"] = normal(b, n, case["heads"], w), normal(b, n, case["kv_heads"], w)
        return s
    if case["op"] == "norm":
        b, n, c = case["batch"], case["n"], case["channels"]
        s = {"x": normal(b, n, c, mean=0.3, std=1.5), "weight": normal(c, mean=1.0, std=0.2), "bias": normal(c, std=0.2)}
        if case["grad"]:
            s["dy"] = normal(b, n, c)
    else:
        b, nq, nk, h, hk, d, dv = (case[k] for k in ("batch", "nq", "nk", "heads", "kv_heads", "d", "dv"))
        s = {"q": normal(b, nq, 2 * h, d), "k": normal(b, nk, 2 * hk, d), "v": normal(b, nk, hk, dv),
             "lam": normal(h, mean=0.5, std=0.1)}
        if case["grad"]:
            s["do"] = normal(b, nq, h, dv)
    s["lengths"] = None if case["lengths"] == "full" else torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own and case["op"] == "rotary":
        from immunostruct_amd.nn import RotaryEmbedding
        state["embedding"] = RotaryEmbedding(case["part"], layout=case["layout"], scaling=_SCALING[case["scaling"]])
    if case["grad"]:
        for name in {"rotary": ("q", "k"), "norm": ("x", "weight", "bias"), "diff": ("q", "k", "v", "lam")}[case["op"]]:
            state[name].requires_grad_(True)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------
def _plain_frequencies(part, scaling):
    """turning rate of every pair (radians a position, 64 bits) and the amplitude"""
    p = torch.arange(part // 2, dtype=torch.float64, device="cuda")
    base = 10000.0
    if scaling == "ntk":
        base *= 4.0 ** (part / (part - 2.0))
    f = base ** (-2.0 * p / part)
    if scaling == "linear":
        f = f / 4.0
    if scaling == "yarn":
        # pairs that turn more than 32 times over the original length stay, those below one turn are stretched, a ramp between
        low, high = (part * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), part - 1)
        stretch = ((p - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f * (1 - stretch) + f / 4.0 * stretch
        return f, 0.1 * math.log(4.0) + 1.0
    return f, 1.0


def _plain_turn(x, positions, case):
    f, amplitude = _plain_frequencies(case["part"], case["scaling"])
    angle = positions.double()[:, :, None, None] * f
    c, s = (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()
    part, half = case["part"], case["part"] // 2
    t = x.float()
    a, b = (t[..., :half], t[..., half:part]) if case["layout"] == "half" else (t[..., 0:part:2], t[..., 1:part:2])
    a, b = a * c - b * s, a * s + b * c
    turned = torch.cat([a, b], dim=-1) if case["layout"] == "half" else torch.stack([a, b], dim=-1).flatten(-2)
    return torch.cat([turned, t[..., part:]], dim=-1).to(x.dtype)


def _plain_activation(z, kind):
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z.clamp(min=0) if kind == "relu" else z


def _plain_norm(x, weight, bias, lengths, case):
    b, n, c = x.shape
    g = case["groups"]
    t = x.float().view(b, n, g, c // g)
    if lengths is None:
        valid = torch.ones(b, n, 1, 1, device=x.device)
    else:
        valid = (torch.arange(n, device=x.device) < lengths[:, None]).float()[:, :, None, None]
    count = (valid.sum(dim=1, keepdim=True) * (c // g)).clamp(min=1)
    mean = (t * valid).sum(dim=(1, 3), keepdim=True) / count
    off = (t - mean) * valid
    var = (off * off).sum(dim=(1, 3), keepdim=True) / count
    z = (off / torch.sqrt(var + 1e-5)).view(b, n, c) * weight.float() + bias.float()
    return (_plain_activation(z, case["activation"]) * valid[:, :, 0]).to(x.dtype)


def _plain_diff(q, k, v, lam, lengths, case):
    b, nq, nk, h, hk, d, dv = (case[key] for key in ("batch", "nq", "nk", "heads", "kv_heads", "d", "dv"))
    j = torch.arange(nk, device=q.device)
    length = torch.full((b,), nk, device=q.device) if lengths is None else lengths.long()
    seen = (j < length[:, None, None]).expand(b, nq, nk)
    if case["causal"] != "none":
        last = torch.arange(nq, device=q.device)[None, :].expand(b, nq)
        if case["causal"] == "end":
            last = last + length[:, None] - nq
        seen = seen & (j <= last[:, :, None])
    seen = seen[:, None]
    heads = torch.arange(h, device=q.device) // (h // hk)
    value = v.float()[:, :, heads].transpose(1, 2).contiguous()
    maps = []
    for m in range(2):
        query = q.float().view(b, nq, h, 2, d)[:, :, :, m].transpose(1, 2).contiguous()
        key = k.float().view(b, nk, hk, 2, d)[:, :, heads, m].permute(0, 2, 3, 1).contiguous()
        s = (torch.matmul(query, key) * d ** -0.5).masked_fill(~seen, float("-inf"))
        top = s.detach().amax(dim=-1, keepdim=True)
        e = torch.exp(s - top.masked_fill(top == float("-inf"), 0.0))
        total = e.sum(dim=-1, keepdim=True)
        maps.append(e / total.masked_fill(total == 0, 1.0))
    out = torch.matmul(maps[0] - lam.float()[:, None, None] * maps[1], value)
    return out.transpose(1, 2).to(q.dtype)


def run(state):
    case = state["case"]
    with torch.set_grad_enabled(case["grad"]):
        if case["op"] == "rotary":
            q, k = state["q"], state["k"]
            if own:
                out = state["embedding"](q, k, state["positions"])
            else:
                out = tuple(_plain_turn(x, state["positions"], case) for x in (q, k))
            if not case["grad"]:
                return out
            return out + torch.autograd.grad(out, (q, k), (state["dq"], state["dk"]))
        if case["op"] == "norm":
            x, weight, bias = state["x"], state["weight"], state["bias"]
            if own:
                from immunostruct_amd import functional as HF
                out = HF.group_norm(x, case["groups"], weight, bias, activation=case["activation"], lengths=state["lengths"])
            else:
                out = _plain_norm(x, weight, bias, state["lengths"], case)
            if not case["grad"]:
                return out
            return (out,) + torch.autograd.grad(out, (x, weight, bias), state["dy"])
        q, k, v, lam = (state[name] for name in ("q", "k", "v", "lam"))
        if own:
            from immunostruct_amd import functional as HF
            out = HF.differential_attention(q, k, v, lam, lengths=state["lengths"], causal=None if case["causal"] == "none" else case["causal"])
        else:
            out = _plain_diff(q, k, v, lam, state["lengths"], case)
        if not case["grad"]:
            return out
        return (out,) + torch.autograd.grad(out, (q, k, v, lam), state["do"])


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------
def _exact_rotary(case, s):
    part, scaling = case["part"], case["scaling"]
    half = part // 2
    rates = []
    for p in range(half):
        theta = 10000.0 * (4.0 ** (part / (part - 2.0)) if scaling == "ntk" else 1.0)
        rate = math.exp(-2.0 * p / part * math.log(theta))
        if scaling == "linear":
            rate /= 4.0
        if scaling == "yarn":
            def pair_of(turns):
                return half * math.log(4096 / (2 * math.pi * turns)) / math.log(theta)
            first, last = max(0, math.floor(pair_of(32.0))), min(part - 1, math.ceil(pair_of(1.0)))
            ramp = min(1.0, max(0.0, (p - first) / max(last - first, 0.001)))
            rate = rate * (1.0 - ramp) + rate * ramp / 4.0
        rates.append(rate)
    angle = s["positions"].double().unsqueeze(-1) * torch.tensor(rates, dtype=torch.float64, device="cuda")
    amplitude = 1.0 + 0.1 * math.log(4.0) if scaling == "yarn" else 1.0
    first = list(range(half)) if case["layout"] == "half" else list(range(0, part, 2))
    second = [i + half for i in first] if case["layout"] == "half" else [i + 1 for i in first]

    def turn(x, sign):
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.full_like(angle, amplitude), sign * angle)[:, :, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = (turn(s["q"], 1.0), turn(s["k"], 1.0))
    return out + (turn(s["dq"], -1.0), turn(s["dk"], -1.0)) if case["grad"] else out


def _exact_norm(case, s):
    x, w, bias = s["x"].double(), s["weight"].double(), s["bias"].double()
    b, n, c = x.shape
    g = case["groups"]
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    dw, db = torch.zeros_like(w), torch.zeros_like(w)
    lengths = torch.tensor(_lengths(case), device="cuda")
    # samples of equal length together, a bounded number of elements at a time
    for length in sorted(set(_lengths(case)) - {0}):
        rows = (lengths == length).nonzero()[:, 0]
        for at in rows.split(max(1, 2 ** 26 // (length * c))):
            part = x[at, :length].reshape(len(at), length, g, c // g)
            var, mean = torch.var_mean(part, dim=(1, 3), correction=0, keepdim=True)
            r = torch.rsqrt(var + 1e-5)
            hat = ((part - mean) * r).reshape(len(at), length, c)
            z = hat * w + bias
            kind = case["activation"]
            if kind == "silu":
                sig = torch.sigmoid(z)
                value, slope = z * sig, sig + z * sig * (1 - sig)
            elif kind == "gelu":
                cdf = torch.special.ndtr(z)
                value, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
            elif kind == "relu":
                slope = (z > 0).double()
                value = z * slope
            else:
                value, slope = z, torch.ones_like(z)
            y[at, :length] = value
            if case["grad"]:
                dz = s["dy"][at, :length].double() * slope
                dw += (dz * hat).sum(dim=(0, 1))
                db += dz.sum(dim=(0, 1))
                t, hat = (dz * w).view_as(part), hat.view_as(part)
                t = t - t.mean(dim=(1, 3), keepdim=True) - hat * (t * hat).mean(dim=(1, 3), keepdim=True)
                dx[at, :length] = (t * r).view(len(at), length, c)
    return (y, dx, dw, db) if case["grad"] else y


def _exact_diff(case, s):
    b, nq, nk, h, hk, d, dv = (case[key] for key in ("batch", "nq", "nk", "heads", "kv_heads", "d", "dv"))
    q, k, v, lam = (s[name].double() for name in ("q", "k", "v", "lam"))
    out = torch.zeros(b, nq, h, dv, dtype=torch.float64, device="cuda")
    dq, dk, dv_, dlam = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(lam)
    for i, length in enumerate(_lengths(case)):
        start = max(0, nq - length) if case["causal"] == "end" else 0      # the queries before it see nothing
        if length == 0 or start >= nq:
            continue
        hidden = None
        if case["causal"] != "none":
            shift = length - nq + start if case["causal"] == "end" else 0
            hidden = torch.ones(nq - start, length, dtype=torch.bool, device="cuda").triu(shift + 1)
        for head in range(h):
            kv = head // (h // hk)
            value = v[i, :length, kv]
            p = []
            for m in range(2):
                score = (q[i, start:, 2 * head + m] @ k[i, :length, 2 * kv + m].t()) / math.sqrt(d)
                if hidden is not None:
                    score[hidden] = -math.inf
                p.append(torch.softmax(score, dim=-1))
            each = [x @ value for x in p]
            out[i, start:, head] = each[0] - lam[head] * each[1]
            if not case["grad"]:
                continue
            do = s["do"][i, start:, head].double()
            dv_[i, :length, kv] += (p[0] - lam[head] * p[1]).t() @ do
            dp = do @ value.t()
            dlam[head] -= (each[1] * do).sum()
            for m, sign in ((0, 1.0), (1, -lam[head])):
                ds = sign * p[m] * (dp - (each[m] * do).sum(dim=-1, keepdim=True)) / math.sqrt(d)
                dq[i, start:, 2 * head + m] = ds @ k[i, :length, 2 * kv + m]
                dk[i, :length, 2 * kv + m] += ds.t() @ q[i, start:, 2 * head + m]
    return (out, dq, dk, dv_, dlam) if case["grad"] else out


def exact(case, seed):
    with torch.no_grad():
        return {"rotary": _exact_rotary, "norm": _exact_norm, "diff": _exact_diff}[case["op"]](case, _inputs(case, seed))
