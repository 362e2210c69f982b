"""MultiTensorAdamW (csrc/adamw_multi.hip) against the update rule in 64 bits, the 8-bit states byte for byte."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
SIZES = [1, 0, 3, 255, 256, 257, 1000, 4095, 4096, 4097, 9001, 16, 64]


def tensors(sizes, pdtype, gdtype, seed, at=0):
    """Parameters and gradients as views `at` values into their buffers (at % 4 != 0: no 16-byte alignment)."""
    g = torch.Generator().manual_seed(seed)
    ps, gs = [], []
    for i, n in enumerate(sizes):
        ps.append((0.1 * torch.randn(n + at, generator=g)).to(pdtype).to(DEV)[at:])
        gs.append((torch.randn(n + at, generator=g) * 10.0 ** (i % 5 - 4) * torch.exp(2 * torch.randn(n + at, generator=g))).to(gdtype).to(DEV)[at:])
    return [torch.nn.Parameter(p) for p in ps], gs


# ---- the rule in 64 bits
def e4m3_table():
    c = torch.arange(127, dtype=torch.float64)
    e, m = torch.div(c, 8, rounding_mode="floor"), c % 8
    return torch.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0 ** -6)


TABLE = e4m3_table()


def small(t, lowest):
    """64-bit values -> (codes 0..126 with a sign bit, scales): nearest, ties to even."""
    n = t.numel()
    pad = torch.zeros((n + 255) // 256 * 256, dtype=torch.float64)
    pad[:n] = t
    rows = pad.view(-1, 256)
    scale = (rows.abs().amax(1) / 448.0).float()
    a = torch.where(scale[:, None] > 0, rows.abs() / scale.double()[:, None], 0.0).clamp_max(448.0).reshape(-1)
    mids = (TABLE[1:] + TABLE[:-1]) / 2
    c = torch.searchsorted(mids, a)
    tie = (c < 126) & (mids[c.clamp(max=125)] == a)
    c = torch.where(tie & (c % 2 == 1), c + 1, c)
    if lowest:
        c = torch.where((pad > 0) & (c == 0), 1, c)
    return (c + 128 * (torch.signbit(pad))).to(torch.uint8), scale


def value(codes, scale, n):
    v = TABLE[(codes.long() & 127)] * torch.where(codes >= 128, -1.0, 1.0)
    return (v.view(-1, 256) * scale.double()[:, None]).reshape(-1)[:n]


class Rule:
    """AdamW of one tensor in 64 bits on the CPU; the states are rounded to their own type after every step."""

    def __init__(self, p, bits):
        self.p, self.bits, self.t, self.dtype = p.detach().double().cpu(), bits, 0, p.dtype
        n = p.numel()
        if bits == 8:
            z = torch.zeros((n + 255) // 256 * 256, dtype=torch.uint8)
            self.m = self.r = (z, torch.zeros(z.numel() // 256))
        else:
            self.m = self.v = torch.zeros(n, dtype=torch.float64)

    def step(self, g, lr, b1, b2, eps, wd, scale=1.0):
        """Returns (p before rounding, magnitude of the terms of p)."""
        n = self.p.numel()
        g = (g.detach().float().cpu() * scale).double()
        self.t += 1
        if self.bits == 8:
            m, r = value(*self.m, n), value(*self.r, n)
            m, v = b1 * m + (1 - b1) * g, b2 * r * r + (1 - b2) * g * g
            self.m, self.r = small(m, False), small(v.sqrt(), True)
        else:
            m = self.m = b1 * self.m + (1 - b1) * g
            v = self.v = b2 * self.v + (1 - b2) * g * g
        u = lr / (1 - b1 ** self.t) * m / (v.sqrt() / math.sqrt(1 - b2 ** self.t) + eps)
        self.p = self.p * (1 - lr * wd) - u
        return self.p.abs() + 2 * u.abs()


def close_p(got, rule, mag, steps):
    """fp32 arithmetic: at most 12 roundings of the terms a step (moments, root, two divisions, the products and the sum),
    then half a step of the parameter's type per update (none for fp32 beyond those)."""
    tol = steps * 12 * U * mag + 1e-30
    if got.dtype != torch.float32:
        tol = tol + steps * torch.finfo(got.dtype).eps / 2 * mag * 1.01 + steps * torch.finfo(got.dtype).smallest_normal
    d = (got.detach().double().cpu() - rule.p).abs()
    assert (d <= tol).all(), (d / tol).max()


def regions(opt, key, i):
    o, n = opt.offsets[i], opt.params[i].numel()
    if "scale" in key:
        return opt.state[key][o // 256:o // 256 + (n + 255) // 256].cpu()
    t = opt.state[key][o:o + (n + 255) // 256 * 256]
    return (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t).cpu()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("at", [0, 1])
@pytest.mark.parametrize("pdtype,gdtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float16),
                                           (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
def test_update_rule(pdtype, gdtype, at, bits):
    import noise_amd as na
    hyper = dict(lr=3e-3, betas=(0.8, 0.97), eps=1e-8, weight_decay=0.1)
    params, grads = tensors(SIZES, pdtype, gdtype, 3, at)
    rules = [Rule(p, bits) for p in params]
    opt = na.MultiTensorAdamW(params, state_bits=bits, **hyper)
    for step in range(1, 4):
        gs = [(g.float() * (1 + 0.5 * step)).to(gdtype) for g in grads]
        opt.step(grads=gs)
        for i, (p, g, rule) in enumerate(zip(params, gs, rules)):
            mag = rule.step(g, hyper["lr"], *hyper["betas"], hyper["eps"], hyper["weight_decay"])
            if p.numel() == 0:
                continue
            close_p(p, rule, mag, 1)
            rule.p = p.detach().double().cpu()           # each step's rounding is judged by itself
            n = p.numel()
            if bits == 8:
                for key, (codes, scale) in (("exp_avg", rule.m), ("exp_avg_sq_root", rule.r)):
                    assert torch.equal(regions(opt, key + "_scale", i), scale), (key, i)
                    got = regions(opt, key, i)
                    same = (got == codes) | ((got & 127 == 0) & (codes & 127 == 0))      # -0 and +0
                    assert same.all(), (key, i, (~same).nonzero()[:4])
            else:
                m, v = regions(opt, "exp_avg", i), regions(opt, "exp_avg_sq", i)
                assert not m[n:].any() and not v[n:].any()
                # two products and a sum a step on states that started equal: 3 roundings of the terms' magnitudes
                gm = g.double().cpu().abs()
                assert ((m[:n].double() - rule.m).abs() <= 8 * U * (rule.m.abs() + gm) + 1e-38).all()
                assert ((v[:n].double() - rule.v).abs() <= 12 * U * rule.v + 1e-38).all()
                rule.m, rule.v = m[:n].double(), v[:n].double()
    assert (opt.step_count == 3).all()


def test_matches_the_flat_optimizer():
    """The same numbers through FusedAdamW's kernel: the two differ by the rounding of a few products."""
    import noise_amd as na
    from noise_amd import _lib
    n = 5000
    g = torch.Generator().manual_seed(1)
    p0, gr = torch.randn(n, generator=g).to(DEV), torch.randn(n, generator=g).to(DEV)
    q = torch.nn.Parameter(p0.clone())
    opt = na.MultiTensorAdamW([q], lr=1e-2)
    p, m, v, step = p0.clone(), torch.zeros(n, device=DEV), torch.zeros(n, device=DEV), torch.zeros((), dtype=torch.int64, device=DEV)
    for _ in range(4):
        opt.step(grads=[gr])
        _lib.call("noise_adamw_step", *(_lib.ptr(t) for t in (p, gr, m, v, step)), n, 1e-2, 0.9, 0.999, 1e-8, 1e-2, 1.0, _lib.stream())
    assert ((p - q.detach()).abs() <= 4 * 24 * U * (p.abs() + 0.02)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_missing_gradients_and_mixed_types(bits):
    """More tensors than one launch holds, of two types in one list, some without a gradient: those keep their values, states
    and step count."""
    import noise_amd as na
    sizes = [(i * 37) % 700 for i in range(230)]
    params, grads = tensors(sizes, torch.float32, torch.float32, 11)
    for i in range(0, 230, 3):
        params[i] = torch.nn.Parameter(params[i].detach().bfloat16())
        grads[i] = grads[i].bfloat16()
    before = [p.detach().clone() for p in params]
    rules = [Rule(p, bits) for p in params]
    opt = na.MultiTensorAdamW(params, lr=1e-2, state_bits=bits)
    for step in range(2):
        gs = [None if (i + step) % 5 == 0 else g for i, g in enumerate(grads)]
        for p, g in zip(params, gs):
            p.grad = g
        opt.step()
        for i, (p, g) in enumerate(zip(params, gs)):
            if g is None:
                if step == 0:
                    assert torch.equal(p.detach(), before[i]) and not regions(opt, "exp_avg", i).any()
            elif p.numel():
                close_p(p, rules[i], rules[i].step(g, 1e-2, 0.9, 0.999, 1e-8, 1e-2), 1)
                rules[i].p = p.detach().double().cpu()
    want = torch.tensor([sum((i + s) % 5 != 0 for s in range(2)) for i in range(230)])
    assert torch.equal(opt.step_count.cpu(), want)
    opt.zero_grad()
    assert all(p.grad is None for p in params)
    opt.step()                                          # nothing to do
    assert torch.equal(opt.step_count.cpu(), want)


@pytest.mark.parametrize("bits", [32, 8])
def test_grad_scale_checkpoint_and_versions(bits):
    import noise_amd as na
    params, grads = tensors([300, 1000], torch.float32, torch.float32, 5)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt = na.MultiTensorAdamW(params, lr=1e-2, state_bits=bits)
    version = params[0]._version
    opt.step(grad_scale=0.25, grads=[4 * g for g in grads])     # powers of two: exact
    assert params[0]._version > version
    other = na.MultiTensorAdamW(twin, lr=1e-2, state_bits=bits)
    other.step(grads=grads)
    assert all(torch.equal(a, b) for a, b in zip(params, twin))
    third = na.MultiTensorAdamW([torch.nn.Parameter(p.detach().clone()) for p in params], state_bits=bits)
    sd = {k: (v.cpu() if torch.is_tensor(v) else v) for k, v in opt.state_dict().items()}
    third.load_state_dict(sd)
    assert third.lr == 1e-2
    for o in (opt, third):
        o.step(grads=grads)
    assert all(torch.equal(a, b) for a, b in zip(opt.params, third.params))
    assert all(torch.equal(opt.state[k].view(torch.uint8), third.state[k].view(torch.uint8)) for k in opt.state)
    with pytest.raises(ValueError, match="-bit states"):
        na.MultiTensorAdamW(twin, state_bits=40 - bits).load_state_dict(sd)
    with pytest.raises(ValueError, match="state 'exp_avg'"):
        na.MultiTensorAdamW(twin[:1], state_bits=bits).load_state_dict(sd)


@pytest.mark.parametrize("bits", [32, 8])
def test_extreme_gradients(bits):
    """Zeros, tiny and huge gradients; a NaN reaches only its own value (32 bits) or its block of 256 (8 bits)."""
    import noise_amd as na
    n = 1024
    p = torch.nn.Parameter(torch.ones(n, device=DEV))
    g = torch.zeros(n, device=DEV)
    g[256:512] = torch.logspace(-18, 18, 256, device=DEV)
    g[512] = float("nan")
    g[768:] = 1e-20
    opt = na.MultiTensorAdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits)
    opt.step(grads=[g])
    assert (p[:256] == 1).all() and torch.isfinite(p[:512]).all() and torch.isnan(p[512]) and torch.isfinite(p[513:]).all()
    # first step: every update is lr * g / (|g| + eps sqrt(1 - b2) ...), never more than lr
    assert ((p[256:512] - 1).abs() <= 1e-3 * (1 + 1e-4)).all()
    opt.step(grads=[torch.zeros_like(g)])
    bad = torch.isnan(p.detach()).cpu()
    assert bad[512] and not bad[:512].any() and not bad[768:].any()
    assert bad.sum() == (1 if bits == 32 else 256)
    # a positive second moment is never stored as zero: no step of a later small gradient exceeds a few lr
    assert ((p[256:512] - 1).abs() < 5e-3).all()


def test_refusals():
    import noise_amd as na
    p, g = tensors([8, 12], torch.float32, torch.float32, 1)
    with pytest.raises(ValueError, match="twice"):
        na.MultiTensorAdamW([p[0], p[0]])
    with pytest.raises(TypeError, match="float64"):
        na.MultiTensorAdamW([torch.nn.Parameter(torch.zeros(3, device=DEV, dtype=torch.float64))])
    with pytest.raises(ValueError, match="contiguous"):
        na.MultiTensorAdamW([torch.nn.Parameter(torch.zeros(4, 6, device=DEV).t())])
    opt = na.MultiTensorAdamW(p)
    with pytest.raises(ValueError, match="gradients for"):
        opt.step(grads=g[:1])
    with pytest.raises(ValueError, match="gradient 1"):
        opt.step(grads=[g[0], g[0]])
    with pytest.raises(TypeError, match="cannot take"):
        opt.step(grads=[g[0].double(), g[1]])
    with pytest.raises(ValueError, match="gradient 0"):
        opt.step(grads=[g[0].cpu(), g[1]])
    assert not opt.step_count.any()
    half = na.MultiTensorAdamW([torch.nn.Parameter(torch.zeros(8, device=DEV, dtype=torch.bfloat16))])
    with pytest.raises(TypeError, match="cannot take"):
        half.step(grads=[g[0]])
    # a transposed gradient is read through a packed copy
    q = torch.nn.Parameter(torch.zeros(4, 6, device=DEV))
    gt = torch.randn(6, 4, device=DEV).t()
    a, b = na.MultiTensorAdamW([q]), na.MultiTensorAdamW([torch.nn.Parameter(torch.zeros(4, 6, device=DEV))])
    a.step(grads=[gt])
    b.step(grads=[gt.contiguous()])
    assert torch.equal(q, b.params[0])


def test_parameters_that_were_rebound_or_share_memory():
    """A parameter with other values behind its old address is refused; one with new memory of the same kind is followed."""
    import noise_amd as na
    make = lambda: [torch.nn.Parameter(torch.ones(1000, device=DEV)), torch.nn.Parameter(torch.ones(64, device=DEV))]
    grads = [torch.ones(1000, device=DEV), torch.ones(64, device=DEV)]
    for rebind in (lambda t: t[:500], lambda t: t[:0], lambda t: t.view(torch.bfloat16)[:1000], lambda t: t.view(torch.float16)):
        for some in (grads, [grads[0], None]):
            p = make()
            opt = na.MultiTensorAdamW(p)
            p[0].data = rebind(p[0].data)
            with pytest.raises(RuntimeError, match="after the optimizer was built"):
                opt.step(grads=some)
            assert not opt.step_count.any() and (p[1] == 1).all()
    p = make()
    opt = na.MultiTensorAdamW(p, lr=1e-2, weight_decay=0.0)
    p[0].data = torch.full((1000,), 2.0, device=DEV)
    opt.step(grads=grads)
    assert ((p[0] - 1.99).abs() < 1e-5).all() and ((p[1] - 0.99).abs() < 1e-5).all()
    p[0].data = torch.ones(1064, device=DEV)[:1000]
    p[1].data = p[0].data[936:]
    with pytest.raises(ValueError, match="share memory"):
        opt.step(grads=grads)
    both = torch.ones(100, device=DEV)
    with pytest.raises(ValueError, match="share memory"):
        na.MultiTensorAdamW([torch.nn.Parameter(both[:60]), torch.nn.Parameter(both[59:])])
    na.MultiTensorAdamW([torch.nn.Parameter(both[:60]), torch.nn.Parameter(both[60:]), torch.nn.Parameter(both[:0])])


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays(bits):
    import noise_amd as na
    params, grads = tensors([100, 5000, 7], torch.float32, torch.float32, 21)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = na.MultiTensorAdamW(params, lr=1e-2, state_bits=bits), na.MultiTensorAdamW(twin, lr=1e-2, state_bits=bits)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        a.step(grads=grads)
    assert not a.step_count.any()
    for k in range(4):
        for g in grads:
            g.mul_(1.0 - 0.1 * k)
        graph.replay()
        b.step(grads=grads)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(params, twin)) and (a.step_count == k + 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_mask_holds(bits):
    """4096 tensors are what one launch of the step counter covers; a list beyond that, whole and with gaps."""
    import noise_amd as na
    n = 4300
    g = torch.Generator().manual_seed(2)
    base, grad = torch.randn(n, 4, generator=g).to(DEV), torch.randn(n, 4, generator=g).to(DEV)
    params = [torch.nn.Parameter(base[i, :1 + i % 3].clone()) for i in range(n)]
    opt = na.MultiTensorAdamW(params, lr=1e-2, state_bits=bits)
    rules = [Rule(p, bits) for p in params]
    for step, gap in enumerate((0, 7)):
        grads = [None if gap and i % gap == 3 else grad[i, :1 + i % 3] for i in range(n)]
        opt.step(grads=grads)
        now = [p.detach().cpu() for p in params]
        for i, gr in enumerate(grads):
            if gr is not None:
                close_p(now[i], rules[i], rules[i].step(gr, 1e-2, 0.9, 0.999, 1e-8, 1e-2), 1)
                rules[i].p = now[i].double()
            else:
                assert torch.equal(now[i].double(), rules[i].p)
    want = torch.tensor([1 if i % 7 == 3 else 2 for i in range(n)])
    assert torch.equal(opt.step_count.cpu(), want)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_waveform_model_trains_with_it(bits):
    """Steps of the waveform-domain U-Net: its separate gradients go in, the rule holds for every parameter, and the next
    step runs on the new weights (a second model given them computes the same loss and gradients)."""
    import copy
    import noise_amd as na
    import test_gpu_wave as W
    x1, clean = (torch.from_numpy(W.G9[f"narrow_{k}"]).to(DEV) for k in ("x1", "val_clean"))
    m = W.build("narrow", linear_gain=1.0).to(DEV).eval()
    m(x1)
    m.train()
    m.attn_keep_masks = W.g10_masks("narrow", 2)
    opt = na.MultiTensorAdamW(m.parameters(), lr=1e-3, state_bits=bits)
    rules = [Rule(p.detach().view(-1), bits) for p in m.parameters()]
    for step in range(3):
        opt.zero_grad()
        loss = m.training_step((x1, clean, None), 0)
        loss.backward()
        if step:
            fresh = W.build("narrow", linear_gain=1.0).to(DEV).eval()
            fresh(x1)
            fresh.load_state_dict(before)
            fresh.train()
            fresh.attn_keep_masks = W.g10_masks("narrow", 2)
            other = fresh.training_step((x1, clean, None), 0)
            other.backward()
            assert torch.equal(loss, other)
            assert all(torch.equal(p.grad, q.grad) for p, q in zip(m.parameters(), fresh.parameters()))
        opt.step()
        before = copy.deepcopy(m.state_dict())
        for p, r in zip(m.parameters(), rules):
            close_p(p.detach().view(-1), r, r.step(p.grad.reshape(-1), 1e-3, 0.9, 0.999, 1e-8, 1e-2), 1)
            r.p = p.detach().view(-1).double().cpu()
    assert (opt.step_count == 3).all()


def codes_of(values):
    """e4m3 values (exact ones) -> their bytes."""
    c = torch.searchsorted(TABLE, values.abs().double())
    assert torch.equal(TABLE[c], values.abs().double())
    return (c + 128 * (values < 0)).to(torch.uint8)


@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.5, 0.25), (0.8, 0.0)])
def test_small_states_on_rounding_borders(betas, gdtype):
    """First moments that are whole numbers in units of the scale, on the very border between two codes, and scales halfway between
    two floats: sums of short numbers get there even where 1 - b1 is no short number, so the bytes are those of the rule's own
    64-bit operations and of no others."""
    import noise_amd as na
    b1 = betas[0]
    g = torch.Generator().manual_seed(8)
    blocks = 400
    ints = TABLE[(TABLE == TABLE.round()) & (TABLE <= 448) & (TABLE > 0)]
    mids = (TABLE[1:] + TABLE[:-1]) / 2
    mids = mids[(mids == mids.round()) & (mids < 448)]
    pick = lambda t: t[torch.randint(0, len(t), (blocks, 256), generator=g)] * torch.where(torch.rand(blocks, 256, generator=g) < 0.5, -1.0, 1.0)
    unit = 2.0 ** torch.randint(-30, -10, (blocks, 1), generator=g).double()
    # b1 m + (1 - b1) g = y: where b1 is a multiple of 1 / 10, g = (10 y - 10 b1 m) / (10 - 10 b1) is a whole number for enough of them
    m, y = pick(ints), pick(mids)
    m[:, 0], y[:, 0] = 448.0, 448.0
    need = (10 * y - round(10 * b1) * m) / round(10 - 10 * b1)
    grad = torch.where(need == need.to(gdtype).double(), need, 0.0)
    params, states = [torch.nn.Parameter(torch.ones(blocks * 256, device=DEV))], dict(m=codes_of(m.view(-1)), scale=unit.view(-1).float())
    grads = [(grad * unit).view(-1).to(gdtype).to(DEV)]
    assert torch.equal(grads[0].double().cpu().view(blocks, 256), grad * unit)
    opt = na.MultiTensorAdamW(params, betas=betas, state_bits=8)
    sd = opt.state_dict()
    sd["exp_avg"], sd["exp_avg_scale"] = states["m"].view(torch.float8_e4m3fn).to(DEV), states["scale"].to(DEV)
    r = TABLE[torch.randint(1, 127, (blocks * 256,), generator=g)]
    sd["exp_avg_sq_root"], sd["exp_avg_sq_root_scale"] = codes_of(r).view(torch.float8_e4m3fn).to(DEV), (unit.view(-1) / 7).float().to(DEV)
    opt.load_state_dict(sd)
    rule = Rule(params[0], 8)
    rule.m, rule.r = (states["m"], states["scale"]), (codes_of(r), (unit.view(-1) / 7).float())
    on_border = 0
    for step in range(3):
        opt.step(grads=grads)
        mag = rule.step(grads[0], 1e-4, *betas, 1e-8, 1e-2)
        for key, (codes, scale) in (("exp_avg", rule.m), ("exp_avg_sq_root", rule.r)):
            assert torch.equal(regions(opt, key + "_scale", 0), scale), (key, (regions(opt, key + "_scale", 0) != scale).sum())
            got = regions(opt, key, 0)
            same = (got == codes) | ((got & 127 == 0) & (codes & 127 == 0))
            assert same.all(), (key, (~same).sum())
        if step == 0:
            new = b1 * value(states["m"], states["scale"], blocks * 256) + (1 - b1) * grads[0].double().cpu()
            x = new.view(-1, 256).abs() / rule.m[1].double()[:, None]
            on_border = torch.isin(x, mids).sum()
    assert on_border > 500


def test_small_state_scales_halfway_between_floats():
    """The largest moment is 448 t with t halfway between two floats, in every block: t goes to the even one."""
    import noise_amd as na
    blocks = 2000
    g = torch.Generator().manual_seed(3)
    odd = (1 << 24) + 1 + 2 * torch.randint(0, 1 << 23, (blocks,), generator=g)          # 25 bits: no float
    old = ((odd - 1).double() * 2.0 ** -29)                                              # 24 bits
    assert torch.equal(old.float().double(), old)
    p = torch.nn.Parameter(torch.ones(blocks * 256, device=DEV))
    grad = torch.zeros(blocks, 256, dtype=torch.float64)
    grad[:, 5] = 448 * 2.0 ** -29                    # 0.5 (448 old + grad) = 448 odd 2^-30
    codes = torch.zeros(blocks, 256, dtype=torch.uint8)
    codes[:, 5] = 126
    opt = na.MultiTensorAdamW([p], betas=(0.5, 0.75), state_bits=8)
    sd = opt.state_dict()
    sd["exp_avg"], sd["exp_avg_scale"] = codes.view(-1).view(torch.float8_e4m3fn).to(DEV), old.float().to(DEV)
    opt.load_state_dict(sd)
    opt.step(grads=[grad.view(-1).float().to(DEV)])
    want = torch.where(odd % 4 == 1, odd - 1, odd + 1).double() * 2.0 ** -30              # the neighbour with an even last bit
    assert torch.equal(opt.state["exp_avg_scale"].cpu().double(), want)
    assert torch.equal(opt.state["exp_avg"].view(torch.uint8).cpu().view(-1, 256), codes)


def test_first_step_of_short_gradients():
    """From zero states the roots are sqrt(1 - b2) |g|: ratios of short gradients lie next to borders, a float's rounding away."""
    import noise_amd as na
    n = 256 * 4000
    g = torch.Generator().manual_seed(5)
    p = torch.nn.Parameter(torch.ones(n, device=DEV))
    grad = (torch.randint(1, 256, (n,), generator=g).double() * 2.0 ** torch.randint(-3, 4, (n,), generator=g)).to(torch.bfloat16)
    opt, rule = na.MultiTensorAdamW([p], state_bits=8), Rule(p, 8)
    opt.step(grads=[grad.to(DEV)])
    rule.step(grad, 1e-4, 0.9, 0.999, 1e-8, 1e-2)
    for key, (codes, scale) in (("exp_avg", rule.m), ("exp_avg_sq_root", rule.r)):
        assert torch.equal(regions(opt, key + "_scale", 0), scale), key
        assert torch.equal(regions(opt, key, 0), codes), (key, (regions(opt, key, 0) != codes).sum())
