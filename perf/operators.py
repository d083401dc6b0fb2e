"""Workloads of the layer and optimizer operators: products grouped by type, group norm with an activation, AdamW.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes a case's inputs on the device, ``run()``
computes one pass -- in elementary torch operations, or through ``dgcnn_amd`` where ``own`` is set -- and ``exact()`` says in 64 bits
what the pass should return.  ``work()`` is what a pass cannot do without: every input read once, every output written once.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
BLOCK = 256            # elements of a tensor that share one scale of an 8-bit state
E4M3_MAX = 448.0
TINY = 2.0 ** -110     # a block whose largest value is below this is held as zeros
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 1e-2

# parameters of the framework's model for COLLAB (one input feature, three classes), in the order of its flat layout
MODEL_TENSORS = [32, 32, 1024, 32, 1024, 32, 32, 1, 1552, 16, 2560, 32, 45056, 128, 384, 3]


def listed():
    return [
        # MUTAG: a batch of 50 molecules (17.9 atoms each), one 32-wide layer with a matrix for each of its 7 atom types; one training step
        dict(name="linear_atoms", op="linear", rows=895, pad=0, groups=7, k=32, n=32, skew=1.0, dtype="fp32", grad=True),
        # answering a few nodes at a time through a layer of 8 experts: the weights are the work
        dict(name="linear_few_rows", op="linear", rows=48, pad=0, groups=8, k=1024, n=1024, skew=0.5, dtype="bf16", grad=False),
        # 2048 COLLAB graphs (74.5 nodes each), three relations, the model's 97 concatenated channels in: odd rows, ordinary fp32 training
        dict(name="linear_odd_fp32", op="linear", rows=152576, pad=0, groups=3, k=97, n=128, skew=0.7, dtype="fp32", grad=True),
        # a wide expert layer over a large batch of nodes, training in bf16
        dict(name="linear_experts_bf16", op="linear", rows=131072, pad=0, groups=16, k=512, n=512, skew=0.5, dtype="bf16", grad=True),
        # one evaluation batch of 50 COLLAB graphs at the model's width: latency
        dict(name="norm_small", op="norm", samples=50, rows=3725, pad=0, c=32, groups=4, act="relu", skew=0.6, ragged=True, dtype="fp32", grad=False),
        # 2048 COLLAB graphs at the classifier's width, training in bf16
        dict(name="norm_graphs_bf16", op="norm", samples=2048, rows=152576, pad=0, c=128, groups=8, act="silu", skew=0.6, ragged=True, dtype="bf16", grad=True),
        # 50 DD proteins (284.3 nodes on average, some many times that) over all 97 concatenated channels, one group
        dict(name="norm_dd", op="norm", samples=50, rows=14216, pad=0, c=97, groups=1, act="tanh", skew=1.2, ragged=True, dtype="fp32", grad=True),
        # 16 feature maps of 64 x 64 x 512, the common 32 groups
        dict(name="norm_maps_bf16", op="norm", samples=16, rows=65536, pad=0, c=512, groups=32, act="silu", skew=0.0, ragged=False, dtype="bf16", grad=True),
        # the framework's own model: 16 small tensors, one call
        dict(name="adamw_model", op="adamw", layout="model", tensors=16, numel=51944, dtype="fp32", master=False, bits=32),
        # a mid-sized network held in bf16 with fp32 copies, sizes from biases to matrices
        dict(name="adamw_master_bf16", op="adamw", layout="mixed", tensors=60, numel=24000000, dtype="bf16", master=True, bits=32),
        # a large network, everything fp32
        dict(name="adamw_large", op="adamw", layout="mixed", tensors=40, numel=200000000, dtype="fp32", master=False, bits=32),
        # the same held in bf16, states in 8 bits
        dict(name="adamw_large_8bit", op="adamw", layout="mixed", tensors=40, numel=200000000, dtype="bf16", master=False, bits=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "norm", "adamw"])
    if op == "linear":
        while True:
            rows, k, n, groups = _log(rng, 1, 160000), _log(rng, 8, 1024), _log(rng, 8, 1024), _log(rng, 1, 64)
            if rows * k * n <= 131072 * 512 * 512 and rows * (k + n) <= 160000 * 1024:
                break
        return dict(op="linear", rows=rows, pad=rng.choice([0, 0, rng.randint(1, 100)]), groups=groups, k=k, n=n, skew=rng.uniform(0.0, 1.5),
                    dtype=rng.choice(["fp32", "bf16", "fp16"]), grad=rng.random() < 0.6)
    if op == "norm":
        ragged = rng.random() < 0.7
        while True:
            samples, mean, c = _log(rng, 1, 2048), _log(rng, 1, 4096), _log(rng, 8, 512)
            if samples * mean * c <= 65536 * 512:
                break
        groups = rng.choice([g for g in range(1, 33) if c % g == 0])
        grad = rng.random() < 0.6                           # (relu's gradient jumps where its argument's last bit decides: forward only)
        return dict(op="norm", samples=samples, rows=samples * mean, pad=rng.choice([0, rng.randint(1, 100)]) if ragged else 0, c=c, groups=groups,
                    act=rng.choice(["none", "silu", "gelu", "tanh"] + ["relu"] * (not grad)), skew=rng.uniform(0.0, 1.3) if ragged else 0.0,
                    ragged=ragged, dtype=rng.choice(["fp32", "bf16", "fp16"]), grad=grad)
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    return dict(op="adamw", layout="mixed", tensors=_log(rng, 1, 200), numel=_log(rng, 50000, 100000000), dtype=dtype,
                master=dtype != "fp32" and rng.random() < 0.5, bits=rng.choice([8, 32]))


def work(case):
    s = SIZE[case["dtype"]]
    if case["op"] == "linear":
        m, e, k, n = case["rows"], case["groups"], case["k"], case["n"]
        used = min(e, m)                                    # groups that can have rows
        data, flops = s * (m * k + used * n * (k + 1) + m * n) + 8 * (e + 1), 2 * m * n * k
        if case["grad"]:                                    # dy in, dx, dW, db out
            data, flops = data + s * (m * n + m * k + e * n * (k + 1)), 3 * flops
        return {"bytes": data, "flops": flops}
    if case["op"] == "norm":
        x = case["rows"] * case["c"]
        return {"bytes": s * x * (4 if case["grad"] else 2) + 16 * case["c"], "flops": x * (30 if case["grad"] else 10)}
    n = sum(_sizes(case))
    each = 2 * s + s - (s if case["master"] else 0) + (8 if case["master"] else 0) + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)
    return {"bytes": each * n, "flops": 20 * n}


# ---- inputs -------------------------------------------------------------------------------------------------------------------------
def _split(gen, total, parts, skew):
    """``parts`` sizes that sum to ``total``: log-normal shares (skew 0: as equal as can be); some may be empty."""
    share = torch.exp(skew * torch.randn(parts, generator=gen, dtype=torch.float64))
    at = torch.round(torch.cumsum(share, 0) / share.sum() * total).long()
    at[-1] = total
    return torch.cat([torch.zeros(1, dtype=torch.int64), at])


def _sizes(case):
    """Element counts of the tensors of an optimizer case: alternating matrices and their short rows, odd ones among them."""
    if case["layout"] == "model":
        return list(MODEL_TENSORS)
    t, n = case["tensors"], case["numel"]
    small = [max(1, min(4097, n // (8 * t))) + 3 * i % 7 for i in range(t // 2)]
    big = t - t // 2
    left = max(big, n - sum(small))
    weight = [1 + (i * 5) % 11 for i in range(big)]
    large = [max(1, left * w // sum(weight)) for w in weight]
    return [s for i in range(big) for s in ([large[i]] + ([small[i]] if i < len(small) else []))]


def _splitmix(seed, index):
    """32 random bits of (seed, index): one key for each tensor's random numbers."""
    mask = (1 << 64) - 1
    z = (seed + 0x9E3779B97F4A7C15 * (index + 1)) & mask
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
    return (z ^ (z >> 31)) & 0xFFFFFFFF


def prepare(case, seed):
    cpu = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32) * scale + shift).to(dt)

    if case["op"] == "linear":
        e, k, n, rows = case["groups"], case["k"], case["n"], case["rows"] + case["pad"]
        ptr = _split(cpu, case["rows"], e, case["skew"])
        s = dict(case=case, x=rand(rows, k), weight=rand(e, n, k, scale=k ** -0.5), bias=rand(e, n, scale=0.1), ptr=ptr.to(DEVICE),
                 sizes=(ptr[1:] - ptr[:-1]).tolist())
        if case["grad"]:
            s["dy"] = rand(rows, n, scale=n ** -0.5)
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(True)
        return s
    if case["op"] == "norm":
        c, rows, b = case["c"], case["rows"] + case["pad"], case["samples"]
        ptr = _split(cpu, case["rows"], b, case["skew"])
        x = (torch.randn(rows, c, generator=gen, device=DEVICE) * (0.5 + torch.rand(c, generator=gen, device=DEVICE))
             + 0.5 * torch.randn(c, generator=gen, device=DEVICE)).to(dt)
        s = dict(case=case, weight=rand(c, scale=0.1, shift=1.0), bias=rand(c, scale=0.1), ptr=ptr.to(DEVICE))
        s["x"] = x if case["ragged"] else x.view(b, -1, c)
        if case["grad"]:
            s["dy"] = rand(*s["x"].shape)
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(True)
        return s
    # every tensor starts on a block of its own in one buffer, as a program that keeps its parameters together has them
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    first = [0]
    for b in blocks:
        first.append(first[-1] + b)
    total = first[-1] * BLOCK
    inside = torch.zeros(total, dtype=torch.bool, device=DEVICE)
    for n, f in zip(sizes, first):
        inside[f * BLOCK:f * BLOCK + n] = True

    def flat(scale, low=False):
        v = torch.randn(total, generator=gen, device=DEVICE, dtype=torch.float32)
        v = (v.square() if low else v) * scale
        return v.masked_fill_(~inside, 0.0)

    def views(t):
        return [t[f * BLOCK:f * BLOCK + n] for n, f in zip(sizes, first)]

    # gradients differ in size from tensor to tensor, and from element to element within one
    level = torch.exp(torch.randn(len(sizes), generator=cpu)).to(DEVICE)
    level = level.repeat_interleave(torch.tensor(blocks, device=DEVICE)).repeat_interleave(BLOCK)
    grad = flat(1e-2) * level
    s = dict(case=case, step=100, seed=seed, sizes=sizes, grad=grad.to(dt))
    p = flat(0.05)
    if case["master"]:
        s["master"] = p
    s["param"] = p.to(dt)
    m, v = flat(3e-3) * level, flat(1e-4, low=True) * level.square()
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        for name, t in (("m", m), ("r", v.sqrt())):
            t = t.view(-1, BLOCK)
            top = t.abs().amax(1)
            s[name + "_scale"] = top / E4M3_MAX
            t = (t * torch.where(top > TINY, E4M3_MAX / top, 0.0).unsqueeze(1)).clamp(-E4M3_MAX, E4M3_MAX)
            if name == "r":
                t = torch.where(t > 0, t.clamp_min(2.0 ** -9), t)
            s[name] = t.to(torch.float8_e4m3fn).view(-1)
        s["key"] = torch.tensor([_splitmix(seed, i) for i in range(len(sizes))], device=DEVICE).repeat_interleave(torch.tensor(blocks, device=DEVICE))
        s["place"] = (torch.arange(first[-1], device=DEVICE) - torch.tensor(first[:-1], device=DEVICE).repeat_interleave(torch.tensor(blocks, device=DEVICE))) * BLOCK
    s["views"] = {k: views(s[k]) for k in ("param", "grad", "master", "m", "v", "r") if k in s}
    if case["bits"] == 8:
        s["views"].update({k: [s[k][f:f + b] for f, b in zip(first, blocks)] for k in ("m_scale", "r_scale")})
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return {"linear": _own_linear, "norm": _own_norm, "adamw": _own_adamw}[op](s)
    return {"linear": _linear, "norm": _norm, "adamw": _adamw}[op](s)


def _own_linear(s):
    from dgcnn_amd import layers
    y = layers.grouped_linear(s["x"], s["weight"], s["ptr"], s["bias"])
    if not s["case"]["grad"]:
        return y
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _own_norm(s):
    from dgcnn_amd import layers
    c = s["case"]
    y = layers.group_norm(s["x"], c["groups"], s["weight"], s["bias"], ptr=s["ptr"] if c["ragged"] else None, act=c["act"])
    if not c["grad"]:
        return y
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _own_adamw(s):
    from dgcnn_amd import optim
    c, v = s["case"], s["views"]
    s["step"] += 1
    more = dict(masters=v["master"]) if c["master"] else {}
    if c["bits"] == 8:
        optim.adamw_step(v["param"], v["grad"], v["m"], v["r"], exp_avg_scales=v["m_scale"], exp_avg_sq_scales=v["r_scale"], seed=s["seed"],
                         step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, **more)
    else:
        optim.adamw_step(v["param"], v["grad"], v["m"], v["v"], step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, **more)
    return _state(s)


def _state(s):
    return {k: s[k] for k in ("param", "master", "m", "v", "r", "m_scale", "r_scale") if k in s}


def _linear(s):
    with torch.no_grad():
        c, dt = s["case"], s["x"].dtype
        rows, sizes, at = c["rows"], s["sizes"], 0
        x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
        y = torch.zeros(x.shape[0], c["n"], device=x.device)
        for e, m in enumerate(sizes):
            torch.addmm(b[e], x[at:at + m], w[e].t(), out=y[at:at + m])
            at += m
        if not c["grad"]:
            return y.to(dt)
        dy, at = s["dy"].float(), 0
        dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
        for e, m in enumerate(sizes):
            torch.mm(dy[at:at + m], w[e], out=dx[at:at + m])
            torch.mm(dy[at:at + m].t(), x[at:at + m], out=dw[e])
            torch.sum(dy[at:at + m], 0, out=db[e])
            at += m
        return {"y": y.to(dt), "dx": dx.to(dt), "dweight": dw.to(dt), "dbias": db.to(dt)}


def _act(z, act):
    """The activation and its derivative."""
    if act == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if act == "silu":
        g = 1 / (1 + torch.exp(-z))
        return z * g, g * (1 + z * (1 - g))
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    return z, torch.ones_like(z)


def _norm(s):
    with torch.no_grad():
        c, dt = s["case"], s["x"].dtype
        ch, g, rows, ptr = c["c"], c["groups"], c["rows"], s["ptr"]
        x = s["x"].reshape(-1, ch)[:rows].float().view(rows, g, ch // g)
        w, bias = s["weight"].float().view(g, -1), s["bias"].float().view(g, -1)
        seg = torch.searchsorted(ptr, torch.arange(rows, device=x.device), right=True) - 1
        count = ((ptr[1:] - ptr[:-1]) * (ch // g)).double().unsqueeze(1)

        def mean(t):                                        # over the rows of a sample and the channels of a group, for each row
            if not c["ragged"]:
                total = t.double().sum(2).view(c["samples"], -1, g).sum(1)
            else:
                upto = torch.nn.functional.pad(t.double().sum(2).t().contiguous().cumsum(1), (1, 0)).t()
                total = upto[ptr[1:]] - upto[ptr[:-1]]
            return (total / count)[seg].unsqueeze(2)

        mid = (x - mean(x)).float()
        rstd = (1 / torch.sqrt(mean(mid * mid) + 1e-5)).float()
        h = mid * rstd
        y, slope = _act(h * w + bias, c["act"])
        whole = torch.zeros(rows + c["pad"], ch, dtype=dt, device=x.device)
        whole[:rows] = y.view(rows, ch).to(dt)
        y = whole.view(s["x"].shape)
        if not c["grad"]:
            return y
        q = s["dy"].reshape(-1, ch)[:rows].float().view(rows, g, -1) * slope
        db, dw = q.double().sum(0), (q * h).double().sum(0)
        q = q * w
        dx = rstd * (q - mean(q).float() - h * mean(q * h).float())
        whole = torch.zeros_like(whole)
        whole[:rows] = dx.view(rows, ch).to(dt)
        return {"y": y, "dx": whole.view(s["x"].shape), "dweight": dw.view(ch).to(dt), "dbias": db.view(ch).to(dt)}


def _round_e4m3(t, noise):
    """``t`` (at most 448 in magnitude) on the grid of e4m3: up with the probability of its distance from the lower neighbour."""
    a = t.abs()
    step = (((a.clamp_min(2.0 ** -6).view(torch.int32) >> 23) - 3) << 23).view(torch.float32)      # an eighth of the power of two below
    return torch.copysign(torch.floor(a / step + noise) * step, t).clamp(-E4M3_MAX, E4M3_MAX)


def _noise(s):
    """Two random numbers in [0, 1) with 16 bits for each element: a hash of its tensor's key and its place in the tensor."""
    low = 0xFFFFFFFF
    at = s["place"].unsqueeze(1) + torch.arange(BLOCK, device=s["place"].device)
    h = (at * 0x9E3779B1 + s["key"].unsqueeze(1) + s["step"] * 0x632BE5AB) & low
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & low
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & low
    h = h ^ (h >> 16)
    return (h & 0xFFFF).float() * 2.0 ** -16, (h >> 16).float() * 2.0 ** -16


def _adamw(s):
    c = s["case"]
    s["step"] += 1
    bc1, bc2 = 1 - BETA1 ** s["step"], 1 - BETA2 ** s["step"]
    g = s["grad"].float()
    p = s["master"] if c["master"] else s["param"].float()
    if c["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"].unsqueeze(1)).view(-1)
        r = (s["r"].float().view(-1, BLOCK) * s["r_scale"].unsqueeze(1)).view(-1)
        v = r * r
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    r = torch.sqrt(v)
    p = p * (1 - LR * DECAY) - (m / (r * (1 / math.sqrt(bc2)) + EPS)) * (LR / bc1)
    s["param"].copy_(p)
    if c["master"]:
        s["master"].copy_(p)
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return _state(s)
    for name, t, noise in zip(("m", "r"), (m, r), _noise(s)):
        t = t.view(-1, BLOCK)
        top = t.abs().amax(1)
        top = torch.where(top >= TINY, top, 0.0)
        t = t * torch.where(top > 0, E4M3_MAX / top, 0.0).unsqueeze(1)
        q = _round_e4m3(t, noise)
        if name == "r":
            q = torch.where(t > 0, q.clamp_min(2.0 ** -9), q)
        s[name].copy_(q.view(-1))
        s[name + "_scale"].copy_(top * (1 / E4M3_MAX))
    return _state(s)


# ---- what a pass returns, in 64 bits -------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](s)


def _with_gradients(s, y, x, w, b):
    if not s["case"]["grad"]:
        return y.detach()
    y.backward(s["dy"].double())
    return {"y": y.detach(), "dx": x.grad, "dweight": w.grad, "dbias": b.grad}


def _leaves(s):
    return [s[k].detach().double().requires_grad_(s["case"]["grad"]) for k in ("x", "weight", "bias")]


def _exact_linear(s):
    x, w, b = _leaves(s)
    parts = list(torch.split(x, s["sizes"] + [s["case"]["pad"]]))
    out = [part @ w[e].t().contiguous() + b[e] for e, part in enumerate(parts[:-1])]
    out.append(torch.zeros(parts[-1].shape[0], s["case"]["n"], dtype=torch.float64, device=x.device))
    return _with_gradients(s, torch.cat(out), x, w, b)


def _exact_norm(s):
    c = s["case"]
    x, w, b = _leaves(s)
    at, out = s["ptr"].tolist(), []
    for lo, hi in zip(at[:-1], at[1:]):
        if hi > lo:
            t = x.reshape(-1, c["c"])[lo:hi].reshape(hi - lo, c["groups"], -1)
            var, mean = torch.var_mean(t, dim=(0, 2), correction=0, keepdim=True)
            out.append(((t - mean) / torch.sqrt(var + 1e-5)).reshape(hi - lo, -1))
    z = torch.cat(out) * w + b
    f = torch.nn.functional
    y = {"none": lambda t: t, "relu": f.relu, "silu": f.silu, "gelu": f.gelu, "tanh": torch.tanh}[c["act"]](z)
    y = torch.cat([y, y.new_zeros(c["pad"], c["c"])])
    return _with_gradients(s, y.view(s["x"].shape), x, w, b)


def _exact_adamw(s):
    c, t = s["case"], s["step"] + 1
    g, p = s["grad"].double(), (s["master"] if c["master"] else s["param"]).double()
    wide = lambda name: s[name].double() * s[name + "_scale"].double().repeat_interleave(BLOCK)  # noqa: E731
    m = s["m"].double() if c["bits"] == 32 else wide("m")
    v = s["v"].double() if c["bits"] == 32 else wide("r") ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    update = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    p = p - LR * DECAY * p - LR * update
    out = {"param": p}
    if c["master"]:
        out["master"] = p
    if c["bits"] == 32:
        out.update(m=m, v=v)
        return out
    # e4m3: 8 steps to a factor of two down to 2^-6, then steps of 2^-9 to zero
    h = s["key"].repeat_interleave(BLOCK) + t * 0x632BE5AB
    h = (h + (s["place"].repeat_interleave(BLOCK) + torch.arange(BLOCK, device=h.device).repeat(s["place"].numel())) * 0x9E3779B1) % 2 ** 32
    for shift, factor in ((16, 0x85EBCA6B), (13, 0xC2B2AE35)):
        h = ((h ^ (h >> shift)) * factor) & (2 ** 32 - 1)
    h ^= h >> 16
    for name, x, u in (("m", m, h % 2 ** 16), ("r", v.sqrt(), h // 2 ** 16)):
        top = x.abs().view(-1, BLOCK).amax(1)
        x = x / (top / E4M3_MAX).clamp_min(1e-300).repeat_interleave(BLOCK)
        exponent = (torch.frexp(x)[1] - 1).clamp_min(-6)
        fine = torch.ldexp(x.abs(), 3 - exponent)
        q = torch.ldexp(torch.floor(fine + u.double() / 2 ** 16), exponent - 3) * x.sign()
        if name == "r":
            q = torch.where(x > 0, q.clamp_min(2.0 ** -9), q)
        out[name], out[name + "_scale"] = q.clamp(-E4M3_MAX, E4M3_MAX), top / E4M3_MAX
    return out
