"""AdamW over many tensors (dgcnn_amd.optim.adamw_step, AdamW) against the formula in 64 bits.

Tolerances: an fp32 step of m, v and p is fewer than 8 rounded operations, each off by at most half a step (2^-24 of its result): 8 * 2^-24 of
the largest term.  A result held in bf16 / fp16 is off by half a step of that type (2^-8, 2^-11) more.  8-bit codes are checked for lying on one of
the two neighbours of the exact value, and for the one that the documented hash picks wherever the 64-bit value is not within 2^-12 of a code step of the border."""
import math

import numpy as np
import pytest
import torch

from dgcnn_amd import _lib, optim

gpu = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BLOCK = optim.STATE_BLOCK


def make(sizes, dtype, gdtype, bits, master, seed=0, dev="cuda", offset=0):
    g = torch.Generator().manual_seed(seed)
    t = {k: [] for k in ("p", "g", "m", "v", "ms", "vs", "master")}

    def put(x):
        if not offset:
            return x.to(dev)
        buf = torch.empty(x.numel() + offset, dtype=x.dtype).to(dev)
        out = buf[offset:]
        out.copy_(x.to(dev))
        return out

    for n in sizes:
        p = torch.randn(n, generator=g) * 0.1
        t["p"].append(put(p.to(dtype)))
        t["g"].append(put((torch.randn(n, generator=g) * 10.0 ** float(torch.randint(-4, 1, (1,), generator=g))).to(gdtype)))
        if master:
            t["master"].append(put(p))
        m, v = torch.randn(n, generator=g) * 0.01, torch.randn(n, generator=g).square() * 1e-4
        if bits == 32:
            t["m"].append(put(m)); t["v"].append(put(v))
        else:
            for key, x in (("m", m), ("v", v.sqrt())):
                nb = -(-n // BLOCK)
                pad = torch.zeros(nb * BLOCK); pad[:n] = x
                top = pad.view(nb, BLOCK).abs().amax(1)
                q = (pad.view(nb, BLOCK) / (top / 448).clamp_min(1e-30).unsqueeze(1)).clamp(-448, 448).view(-1)[:n].to(torch.float8_e4m3fn)
                t[key].append(put(q.view(torch.uint8)).view(torch.float8_e4m3fn)); t[key + "s"].append((top / 448).to(dev))
    return t


def call(t, bits, master, **kw):
    more = {}
    if bits == 8:
        more.update(exp_avg_scales=t["ms"], exp_avg_sq_scales=t["vs"])
    if master:
        more["masters"] = t["master"]
    optim.adamw_step(t["p"], t["g"], t["m"], t["v"], **more, **kw)


def wide(q, s):
    n = q.numel()
    return q.cpu().float().double() * s.cpu().double().repeat_interleave(BLOCK)[:n]


def formula(t, i, bits, master, step, lr, betas, eps, wd):
    g = t["g"][i].cpu().double()
    p = (t["master"] if master else t["p"])[i].cpu().double()
    m = t["m"][i].cpu().double() if bits == 32 else wide(t["m"][i], t["ms"][i])
    v = t["v"][i].cpu().double() if bits == 32 else wide(t["v"][i], t["vs"][i]) ** 2
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    upd = lr / (1 - betas[0] ** step) * m / (v.sqrt() / math.sqrt(1 - betas[1] ** step) + eps)
    big_m = (betas[0] * t["m"][i].cpu().double().abs() if bits == 32 else m.abs()) + (1 - betas[0]) * g.abs()
    return p * (1 - lr * wd) - upd, m, v, upd.abs(), big_m


def hash_bits(n, tensor, seed, step):
    """the documented random numbers: two of 16 bits for each element"""
    mask = (1 << 64) - 1
    z = (seed + 0x9E3779B97F4A7C15 * (tensor + 1)) & mask
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
    key = (z ^ (z >> 31)) & 0xFFFFFFFF
    h = (np.arange(n, dtype=np.uint64) * np.uint64(0x9E3779B1) + np.uint64(key) + np.uint64((step * 0x632BE5AB) & 0xFFFFFFFF)) & np.uint64(0xFFFFFFFF)
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x85EBCA6B)) & np.uint64(0xFFFFFFFF)
    h = ((h ^ (h >> np.uint64(13))) * np.uint64(0xC2B2AE35)) & np.uint64(0xFFFFFFFF)
    h = h ^ (h >> np.uint64(16))
    return torch.from_numpy((h & np.uint64(0xFFFF)).astype(np.float64) / 65536), torch.from_numpy((h >> np.uint64(16)).astype(np.float64) / 65536)


def check_codes(q, scale, x, noise, root):
    n = x.numel()
    pad = torch.zeros(scale.numel() * BLOCK, dtype=torch.float64); pad[:n] = x.abs()
    top = pad.view(-1, BLOCK).amax(1)
    assert torch.allclose(scale.cpu().double(), top / 448, rtol=12 * 2.0 ** -24, atol=0)
    s = (top / 448).repeat_interleave(BLOCK)[:n]
    a = torch.where(s > 0, x.abs() / s.clamp_min(1e-300), torch.zeros_like(x))
    exponent = (torch.frexp(a)[1] - 1).clamp_min(-6).double()
    step = torch.exp2(exponent - 3)
    fine = a / step + noise
    want = torch.floor(fine) * step
    if root:
        want = torch.where(a > 0, want.clamp_min(2.0 ** -9), want)
    want = want.clamp_max(448)
    got = q.cpu().float().double()
    sure = (fine - torch.round(fine)).abs() > 2.0 ** -12
    assert (torch.sign(got) * torch.sign(x) >= 0).all()
    assert torch.equal(got.abs()[sure], want[sure])
    assert ((got.abs() - want).abs() <= step * 1.001 + 1e-12).all()
    assert float(sure.double().mean()) > 0.99


SIZES = [1, 7, 8, 255, 256, 257, 2048, 2049, 5000]
KW = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,gdtype,master", [(torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False),
                                                 (torch.bfloat16, torch.float32, True), (torch.float16, torch.float16, True),
                                                 (torch.float16, torch.float32, False), (torch.bfloat16, torch.bfloat16, True)])
@pytest.mark.parametrize("offset", [0, 1])
def test_step_against_the_formula(dtype, gdtype, master, bits, offset):
    """every type, sizes around the vector and block widths, tensors that start in the middle of a vector (offset 1); two steps"""
    t = make(SIZES, dtype, gdtype, bits, master, offset=offset)
    for step in (1, 2):
        want = [formula(t, i, bits, master, step, KW["lr"], KW["betas"], KW["eps"], KW["weight_decay"]) for i in range(len(SIZES))]
        call(t, bits, master, step=step, seed=5, **KW)
        for i, (p, m, v, upd, big) in enumerate(want):
            tol = 8 * 2.0 ** -24 * (p.abs() + 2 * upd) + 1e-30
            if master:
                assert ((t["master"][i].cpu().double() - p).abs() <= tol).all(), i
                assert torch.equal(t["p"][i].cpu(), t["master"][i].cpu().to(dtype))
            else:
                assert ((t["p"][i].cpu().double() - p).abs() <= tol + (HALF[dtype] * p.abs() + 2.0 ** -25 if dtype != torch.float32 else 0)).all(), i
            if bits == 32:
                assert ((t["m"][i].cpu().double() - m).abs() <= 4 * 2.0 ** -24 * big + 1e-38).all()
                assert ((t["v"][i].cpu().double() - v).abs() <= 6 * 2.0 ** -24 * v + 1e-38).all()
            else:
                nm, nv = hash_bits(SIZES[i], i, 5, step)
                check_codes(t["m"][i], t["ms"][i], m, nm, False)
                check_codes(t["v"][i], t["vs"][i], v.sqrt(), nv, True)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_does_not_depend_on_the_list_or_the_alignment(bits):
    """130 tensors (three launches): bit for bit what each gives alone or unaligned; 8-bit codes follow the place in the list"""
    sizes = [1 + (37 * i) % 900 for i in range(130)]
    a, b = make(sizes, torch.float32, torch.float32, bits, False), make(sizes, torch.float32, torch.float32, bits, False, offset=3)
    call(a, bits, False, step=7, seed=3, **KW)
    call(b, bits, False, step=7, seed=3, **KW)
    for k in ("p", "m", "v", "ms", "vs"):
        for x, y in zip(a[k], b[k]):
            assert torch.equal(x.cpu().view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x.cpu(), y.cpu().view(torch.uint8) if y.dtype == torch.float8_e4m3fn else y.cpu()), k
    if bits == 32:
        c = make(sizes, torch.float32, torch.float32, bits, False)
        for i in (0, 64, 129):
            one = {k: v[i:i + 1] for k, v in c.items()}
            call(one, bits, False, step=7, **KW)
            assert torch.equal(one["p"][0].cpu(), a["p"][i].cpu()) and torch.equal(one["v"][0].cpu(), a["v"][i].cpu())


@gpu
def test_8bit_states_of_zeros_tiny_and_non_finite_values():
    n = 3 * BLOCK
    t = make([n], torch.float32, torch.float32, 8, False)
    for k in ("m", "v"):
        t[k][0].copy_(torch.zeros(n).to(torch.float8_e4m3fn))
        t[k + "s"][0].zero_()
    g = torch.zeros(n)
    g[BLOCK] = 1e-30                          # v underflows to 0, m is below 2^-110 * 448: held as zeros
    g[BLOCK + 1] = -1e-40
    g[2 * BLOCK:] = torch.linspace(-1, 1, BLOCK)
    g[2 * BLOCK + 3], g[2 * BLOCK + 5] = float("nan"), float("inf")
    g[2 * BLOCK + 9] = 1e-7                   # v > 0 and far below the block's largest: the smallest code, not 0
    t["g"][0].copy_(g)
    before = t["p"][0].cpu().clone()
    call(t, 8, False, step=1, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    p, m, r = t["p"][0].cpu(), t["m"][0].cpu().float(), t["v"][0].cpu().float()
    assert torch.equal(p[:BLOCK], before[:BLOCK]) and not m[:BLOCK].any() and not r[:BLOCK].any()
    assert float(t["ms"][0][0]) == 0 and float(t["vs"][0][0]) == 0
    assert torch.isfinite(p[:2 * BLOCK]).all() and torch.isfinite(t["ms"][0].cpu()).all() and torch.isfinite(t["vs"][0].cpu()).all()
    bad = torch.zeros(n, dtype=torch.bool); bad[2 * BLOCK + 3] = bad[2 * BLOCK + 5] = True
    assert torch.equal(torch.isnan(m), bad) and torch.equal(torch.isnan(r), bad)
    assert torch.equal(torch.isnan(p), bad)
    assert abs(float(t["ms"][0][2]) * 448 - 0.1) < 1e-6
    assert float(r[2 * BLOCK + 9]) == 2.0 ** -9


@gpu
def test_8bit_second_moment_does_not_stall():
    """a constant gradient of 1: v_t = 1 - b2^t exactly.  Rounded to nearest the root's code stops after about ten steps (0.1 at 300 steps: a hundredth of v);
    stochastic rounding keeps the mean of 2048 elements within 4 standard errors: a code step is at most 1/8, its rounding error's deviation at most
    1/16 of the value a step, and errors of a step decay with b2, so the mean of v is off by less than 10 % at 4 sigma for any t here."""
    n = 2048
    p = [torch.zeros(n).to("cuda")]
    opt = optim.AdamW([torch.nn.Parameter(p[0])], lr=1e-3, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8, seed=11)
    q = opt.param_groups[0]["params"][0]
    spread = torch.linspace(0.5, 1.0, n).to("cuda")
    for _ in range(300):
        q.grad = spread.clone()
        opt.step()
    st = opt.state[q]
    v = wide(st["exp_avg_sq"], st["exp_avg_sq_scale"]) ** 2
    want = spread.cpu().double() ** 2 * (1 - 0.999 ** 300)
    assert abs(float((v / want).mean()) - 1) < 0.1
    m = wide(st["exp_avg"], st["exp_avg_scale"])
    assert abs(float((m / spread.cpu().double()).mean()) - 1) < 0.05


@gpu
def test_optimizer_follows_torchs_adamw_in_64_bits():
    """16 tensors of the model's kind, 12 steps with changing gradients, one of them without a gradient every third step, one channels-last"""
    torch.manual_seed(0)
    shapes = [(32, 1), (32,), (16, 1, 97), (128, 352), (3, 128), (3,), (8, 4, 3, 3)]
    ref = [torch.nn.Parameter(torch.randn(s).double() * 0.1) for s in shapes]
    mine = [torch.nn.Parameter(r.detach().float().to("cuda")) for r in ref]
    mine[-1].data = mine[-1].data.contiguous(memory_format=torch.channels_last)
    a = torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.1)
    b = optim.AdamW(mine, lr=1e-2, weight_decay=0.1)
    for k in range(12):
        for i, (r, m) in enumerate(zip(ref, mine)):
            g = torch.randn(r.shape)
            r.grad, m.grad = (None, None) if i == 1 and k % 3 == 0 else (g.double(), g.to("cuda"))
        a.step(); b.step()
    for r, m in zip(ref, mine):
        # 12 steps of at most 8 rounded operations; an update moves p by at most lr / (1 - b1) = 10 lr
        assert float((m.detach().cpu().double() - r.detach()).abs().max()) <= 12 * 8 * 2.0 ** -24 * (float(r.detach().abs().max()) + 0.1)
    assert b.state[mine[1]]["step"] == 8 and b.state[mine[0]]["step"] == 12


@gpu
@pytest.mark.parametrize("bits,dtype", [(32, torch.float32), (8, torch.float32), (32, torch.bfloat16), (8, torch.bfloat16)])
def test_state_dict_round_trip_continues_bit_for_bit(bits, dtype):
    torch.manual_seed(1)
    start = [torch.randn(300), torch.randn(40, 7)]
    grads = [[torch.randn_like(s) for s in start] for _ in range(4)]

    def run(n, opt_state=None, params=None):
        ps = params or [torch.nn.Parameter(s.clone().to(dtype).to("cuda")) for s in start]
        o = optim.AdamW(ps, lr=1e-2, state_bits=bits, master_weights=dtype != torch.float32, seed=9)
        if opt_state is not None:
            o.load_state_dict(opt_state)
        for g in n:
            for p, x in zip(ps, g):
                p.grad = x.to(dtype).to("cuda")
            o.step()
        return ps, o

    whole, _ = run(grads)
    half, o = run(grads[:2])
    saved = o.state_dict()
    again, o2 = run(grads[2:], saved, [torch.nn.Parameter(p.detach().clone()) for p in half])
    for x, y in zip(whole, again):
        assert torch.equal(x.detach().cpu(), y.detach().cpu())
    assert o2.state[again[0]]["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.float8_e4m3fn)


@gpu
def test_state_of_torchs_adamw_loads():
    p = torch.nn.Parameter(torch.randn(50).to("cuda"))
    q = torch.nn.Parameter(p.detach().clone())
    a, b = torch.optim.AdamW([p], lr=1e-2, foreach=False), optim.AdamW([q], lr=1e-2)
    g = torch.randn(50).to("cuda")
    for _ in range(3):
        p.grad = g
        a.step()
    q.data.copy_(p.data)
    b.load_state_dict(a.state_dict())
    assert b.param_groups[0]["state_bits"] == 32 and b.param_groups[0]["lr"] == 1e-2
    for o, x in ((a, p), (b, q)):
        x.grad = g
        o.step()
    assert b.state[q]["step"] == 4
    assert float((p - q).detach().abs().max()) <= 16 * 2.0 ** -24 * (float(p.detach().abs().max()) + 0.1)


@gpu
def test_master_weights_carry_small_updates():
    """an update of lr = 2^-13 at |p| = 1 is below half a step of bf16: lost without the copy, kept with it"""
    for master in (False, True):
        p = torch.nn.Parameter(torch.ones(64, dtype=torch.bfloat16).to("cuda"))
        o = optim.AdamW([p], lr=2.0 ** -13, weight_decay=0.0, master_weights=master)
        for _ in range(64):
            p.grad = torch.ones(64, dtype=torch.bfloat16).to("cuda")
            o.step()
        moved = 1 - float(p.detach().cpu().float()[0])
        assert moved == 0.0 if not master else abs(moved - 2.0 ** -7) <= 2.0 ** -9


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts_on_the_device_in_a_subprocess_free_graph(bits):
    """capturable=True: replays equal eager steps bit for bit, with eager work and a changed learning rate between them"""
    if not torch.cuda.is_available():
        pytest.skip("graphs need the GPU")
    torch.manual_seed(2)
    start, gs = torch.randn(5000), [torch.randn(5000) for _ in range(6)]
    lr = torch.tensor([1e-2], device="cuda")

    def new():
        p = torch.nn.Parameter(start.clone().to("cuda"))
        p.grad = torch.zeros_like(p)
        return p, optim.AdamW([p], lr=lr, state_bits=bits, capturable=True, seed=4)

    p, o = new()
    q, e = new()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        p.grad.copy_(gs[0])
        o.step()
    torch.cuda.current_stream().wait_stream(side)
    q.grad.copy_(gs[0]); e.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o.step()
    for k, g in enumerate(gs[1:]):
        if k == 2:
            lr.fill_(5e-3)
        p.grad.copy_(g); q.grad.copy_(g)
        graph.replay(); e.step()
        torch.cuda.synchronize()
        assert torch.equal(p.detach(), q.detach()), k
    assert int(o.state[p]["step"]) == 6 == int(e.state[q]["step"])


@gpu
def test_refuses_a_host_counter_while_capturing():
    if not torch.cuda.is_available():
        pytest.skip("graphs need the GPU")
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    p.grad = torch.zeros_like(p)
    o, c = optim.AdamW([p]), optim.AdamW([p], capturable=True)
    o.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x = torch.zeros(1, device="cuda")      # (a graph is not empty)
        with pytest.raises(_lib.DgcnnError):
            o.step()
        with pytest.raises(_lib.DgcnnError):   # no state yet
            c.step()
    del x


@gpu
def test_another_stream_than_the_current_one_is_not_used():
    """the step runs on the stream that is current where it is called: ordered behind the work that wrote the gradient there"""
    if not torch.cuda.is_available():
        pytest.skip("second streams are not emulated")
    n = 1 << 20
    a, b = (torch.nn.Parameter(torch.zeros(n, device="cuda")) for _ in range(2))
    oa, ob = optim.AdamW([a], lr=1e-2), optim.AdamW([b], lr=1e-2)
    g = torch.randn(n, device="cuda")
    b.grad = g
    ob.step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a.grad = torch.zeros(n, device="cuda")
        for _ in range(50):
            a.grad.add_(g / 50)
        a.grad.copy_(g)
        oa.step()
    s.synchronize()
    assert torch.equal(a.detach(), b.detach())


@gpu
def test_refusals_on_device_tensors():
    t = make([10, 20], torch.float32, torch.float32, 32, False)
    ok = dict(step=1, **KW)
    for change in (dict(g=t["g"][:1]), dict(m=[t["m"][0], t["m"][0]]), dict(p=[t["p"][0], t["p"][0]], g=[t["g"][0]] * 2, m=[t["m"][0]] * 2, v=[t["v"][0]] * 2),
                   dict(g=[x.to(torch.bfloat16) for x in t["g"]]), dict(p=[x.to(torch.float64) for x in t["p"]])):
        with pytest.raises(_lib.DgcnnError):
            call({**t, **change}, 32, False, **ok)
    with pytest.raises(_lib.DgcnnError):
        call(t, 32, False, **{**ok, "step": 0})
    with pytest.raises(_lib.DgcnnError):
        call(t, 32, False, **{**ok, "betas": (1.0, 0.9)})
    with pytest.raises(_lib.DgcnnError):
        call({**t, "master": t["p"]}, 32, True, **ok)                                   # masters of fp32 parameters
    with pytest.raises(_lib.DgcnnError):
        optim.adamw_step(t["p"], t["g"], t["m"], t["v"], exp_avg_scales=t["m"], **ok)   # one scale list
    with pytest.raises(_lib.DgcnnError):
        x = torch.zeros(8, 8).to("cuda")[:, :4]
        optim.adamw_step([x], [x], [x], [x], **ok)                                      # not dense
    optim.adamw_step([], [], [], [], **ok)
    call(make([0, 5, 0], torch.float32, torch.float32, 32, False), 32, False, **ok)     # empty tensors are skipped


# ---- CPU ------------------------------------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    t = make([10], torch.float32, torch.float32, 32, False, dev="cpu")
    with pytest.raises(_lib.DgcnnError):
        call(t, 32, False, step=1, **KW)
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(_lib.DgcnnError):
        optim.AdamW([p]).step()


def test_constructor_refusals():
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw in (dict(amsgrad=True), dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            optim.AdamW(p, **kw)


@gpu
@pytest.mark.parametrize("capturable", [False, True])
def test_parameters_without_gradients_keep_their_count(capturable):
    """b has a gradient in two steps of three: its bias corrections are those of its own second step"""
    init = [torch.linspace(-1, 1, 300), torch.linspace(1, 2, 70)]
    ours = [torch.nn.Parameter(t.clone().to("cuda")) for t in init]
    plain = [torch.nn.Parameter(t.double()) for t in init]
    a, b = optim.AdamW(ours, lr=1e-2, capturable=capturable), torch.optim.AdamW(plain, lr=1e-2)
    for k in range(3):
        for i, (p, q) in enumerate(zip(ours, plain)):
            g = None if (i, k) == (1, 1) else torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * k + i))
            p.grad, q.grad = (None, None) if g is None else (g.to("cuda"), g.double())
        a.step(); b.step()
    assert [int(a.state[p]["step"]) for p in ours] == [3, 2]
    for p, q in zip(ours, plain):      # three steps of a few roundings of values up to 2, and of updates up to 1e-2 a step
        assert (p.detach().cpu().double() - q.detach()).abs().max() <= 3 * 4 * 2.0 * 2 ** -24


@gpu
def test_states_load_into_parameters_of_another_layout():
    x = torch.randn(4, 3, 5, 5, generator=torch.Generator().manual_seed(3))
    p, q = (torch.nn.Parameter(x.clone().to("cuda").contiguous(memory_format=f)) for f in (torch.contiguous_format, torch.channels_last))
    a, b = optim.AdamW([p]), optim.AdamW([q])
    for _ in range(2):
        p.grad = torch.ones_like(p) * x.to("cuda")
        a.step()
    q.data.copy_(p.data)
    b.load_state_dict(a.state_dict())
    for o, t in ((a, p), (b, q)):
        t.grad = torch.empty_like(t).copy_(x)
        o.step()
    assert torch.equal(p, q) and torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])
    small = optim.AdamW([p], state_bits=8)
    small.step()
    with pytest.raises(ValueError):
        optim.AdamW([q], state_bits=8).load_state_dict(small.state_dict())


def test_states_of_other_variants_are_refused():
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        with pytest.raises(ValueError):
            optim.AdamW(p).load_state_dict(torch.optim.AdamW(p, **kw).state_dict())


def test_c_entry_refuses_bad_arguments():
    """argument checks come before any launch: they run without a GPU"""
    import ctypes
    L = _lib.lib()
    t = (_lib.AdamwTensor * 1)()
    ptr = ctypes.addressof((ctypes.c_float * 64)())

    def rc(tensor=None, **kw):
        a = _lib.AdamwArgs(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1, state_bits=32, count=1)
        t[0] = _lib.AdamwTensor(**{**dict(param=ptr, grad=ptr, exp_avg=ptr, exp_avg_sq=ptr, numel=4), **(tensor or {})})
        a.tensors = ctypes.addressof(t)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.dgcnn_adamw_step(ctypes.byref(a), None)

    assert L.dgcnn_adamw_step(None, None) == -1
    for kw in (dict(count=-1), dict(tensors=None), dict(param_dtype=7), dict(param_dtype=1, grad_dtype=2), dict(state_bits=16), dict(step=0), dict(beta1=1.0),
               dict(beta2=-0.1), dict(beta2=float("nan")), dict(eps=-1.0), dict(step_dev=ptr), dict(state_bits=8)):
        assert rc(**kw) == -1, kw
    for tensor in (dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(numel=-1), dict(master=ptr)):
        assert rc(tensor) == -1, tensor
    assert rc(dict(numel=1 << 41)) == -3
    assert rc(count=0) == 0 and rc(dict(numel=0, param=None)) == 0
