"""The token operators of noise_amd as measured workloads: layer norm, decay attention (linear attention with a decay for
each head) and AdamW over many tensors.  `own` selects the framework's kernels; otherwise `run` is the plain form, made of
elementary torch operations in 32 bits (64 where a value is rounded next to a border)."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-6
CHUNK = 128          # tokens per chunk of the plain decay attention
BLOCK = 256          # values per scale of the 8-bit optimizer states
LR, BETAS, ADAM_EPS, DECAY, STEP0 = 1e-4, (0.9, 0.999), 1e-8, 1e-2, 1000


def listed():
    return [
        # the bottleneck tokens of one half-second clip (55 tokens of width 64): latency
        dict(name="norm forward - one clip", op="norm_fwd", rows=55, dim=64, dtype="fp32", pad=0),
        # a long batch of wide half-precision tokens: bandwidth
        dict(name="norm forward - wide tokens", op="norm_fwd", rows=65536, dim=2048, dtype="bf16", pad=0),
        # the bottleneck tokens of a training batch of 1280 segments
        dict(name="norm backward - train batch", op="norm_bwd", rows=70400, dim=64, dtype="fp32", pad=0),
        # one new token of one stream, the head sizes of the spectral model's bottleneck (6 heads of 10)
        dict(name="decay token - one stream", op="decay_step", B=1, T=1, H=6, dk=10, dv=10, dtype="fp32", packed=False, ragged=False),
        # one new token of each of 1024 streams
        dict(name="decay token - 1024 streams", op="decay_step", B=1024, T=1, H=8, dk=64, dv=64, dtype="bf16", packed=False, ragged=False),
        # a few clips of 55 tokens, q, k and v in one projection's output
        dict(name="decay forward - clips", op="decay_fwd", B=8, T=55, H=6, dk=10, dv=10, dtype="fp32", packed=True, ragged=False),
        # a padded batch of clips of about ten seconds (100 tokens a second)
        dict(name="decay forward - padded batch", op="decay_fwd", B=64, T=1001, H=8, dk=64, dv=64, dtype="bf16", packed=True, ragged=True),
        # one recording of ten minutes: few rows, a long axis
        dict(name="decay forward - recording", op="decay_fwd", B=1, T=60001, H=16, dk=128, dv=128, dtype="bf16", packed=False, ragged=False),
        # forward and backward of a training batch in fp32, 8 heads of 16 (model width 128)
        dict(name="decay training - fp32 heads", op="decay_train", B=64, T=1001, H=8, dk=16, dv=16, dtype="fp32", packed=True, ragged=True),
        # forward and backward with wide heads in half precision
        dict(name="decay training - wide heads", op="decay_train", B=8, T=4096, H=16, dk=128, dv=128, dtype="bf16", packed=False, ragged=False),
        # the 76146 parameters of the spectral model
        dict(name="adamw 32 bits - spectral model", op="adamw", tensors=128, numel=76146, bits=32, dtype="fp32", gdtype="fp32"),
        # a large model with small states
        dict(name="adamw 8 bits - large model", op="adamw", tensors=300, numel=150_000_000, bits=8, dtype="fp32", gdtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges: every size over its range, most of them odd."""
    op = rng.choice(["norm_fwd", "norm_bwd", "decay_step", "decay_fwd", "decay_train", "decay_fwd", "decay_train", "adamw"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op.startswith("norm"):
        dim = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, max(2, min(100000, (1 << 27) // dim)))
        return dict(op=op, rows=rows, dim=dim, dtype=dtype, pad=rng.choice([0, 0, 8, 3]))
    if op == "adamw":
        numel = _log_int(rng, 1000, 100_000_000)
        bits = rng.choice([8, 32])
        gdtype = rng.choice(["fp32", dtype]) if dtype == "fp32" else dtype
        return dict(op=op, tensors=_log_int(rng, 1, min(600, max(2, numel // 16))), numel=numel, bits=bits, dtype=dtype, gdtype=gdtype)
    H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    dk = rng.choice([8, 10, 16, 24, 32, 40, 64, 64, 80, 96, 128, 128])
    dv = dk if rng.random() < 0.7 else rng.choice([8, 16, 33, 64, 128])
    if op == "decay_step":
        return dict(op=op, B=_log_int(rng, 1, max(1, min(2048, (1 << 26) // (H * dk * dv)))), T=1, H=H, dk=dk, dv=dv, dtype=dtype,
                    packed=False, ragged=False)
    T = _log_int(rng, 1, 20000)
    most = max(1, int(3e7 // (T * H * (dk + dv))))
    B = _log_int(rng, 1, min(256, most))
    return dict(op=op, B=B, T=T, H=H, dk=dk, dv=dv, dtype=dtype, packed=dk == dv and rng.random() < 0.5, ragged=B > 1 and rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------------------- inputs
def _sizes(tensors, numel):
    """`tensors` sizes that add up to `numel`: a few large ones, many small ones, as in a model's parameter list."""
    w = [(1 + (i * 7) % 11) ** 4 for i in range(tensors)]
    total = sum(w)
    sizes = [max(1, numel * x // total) for x in w]
    sizes[-1] = max(1, sizes[-1] + numel - sum(sizes))
    return sizes


def _padded(sizes):
    """Offsets of the tensors in a flat state buffer: each begins a block of 256 values."""
    offs, o = [], 0
    for s in sizes:
        offs.append(o)
        o += (s + BLOCK - 1) // BLOCK * BLOCK
    return offs, o


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev).to(dtype)

    s = dict(case=dict(case), op=case["op"])
    dt = DTYPES[case["dtype"]]
    if case["op"].startswith("norm"):
        R, D = case["rows"], case["dim"]

        def rows():
            # rows of a wider buffer where the case says so (a column slice of a projection's output)
            return (randn(R, D + case["pad"]) * (0.5 + torch.rand(R, 1, generator=g, device=dev)) + 0.3).to(dt)[:, :D]
        s["x"] = rows()
        s["w"], s["b"] = 1 + 0.1 * randn(D), 0.1 * randn(D)
        if case["op"] == "norm_bwd":
            x = s["x"].double()
            mean = x.mean(1)
            s["mean"] = mean.float()
            s["rstd"] = ((x - mean[:, None]).square().mean(1) + EPS).rsqrt().float()
            s["dy"] = randn(R, D, dtype=dt)
        return s
    if case["op"] == "adamw":
        sizes = _sizes(case["tensors"], case["numel"])
        offs, total = _padded(sizes)
        blocks = total // BLOCK
        inside = torch.zeros(total, dtype=torch.bool, device=dev)
        for o, n in zip(offs, sizes):
            inside[o:o + n] = True
        p, grad = randn(total) * 0.05, randn(total) * torch.exp(randn(total)) * 1e-3
        # per-block magnitudes spread over two decades, moments as after many steps
        mag = torch.exp(1.5 * randn(blocks)).repeat_interleave(BLOCK)
        grad = torch.where(inside, grad * mag, 0.0)
        s["p"] = torch.where(inside, p, 0.0).to(dt)
        s["g"] = grad.to(DTYPES[case["gdtype"]])
        m, r = torch.where(inside, grad * 0.1 + randn(total) * 1e-4 * mag, 0.0), torch.where(inside, (randn(total).abs() + 0.05) * 1e-3 * mag, 0.0)
        if case["bits"] == 8:
            for key, t in (("m", m), ("r", r)):
                scale = t.view(blocks, BLOCK).abs().amax(1) / 448.0
                s[key + "_scale"] = scale
                s[key] = torch.where(scale[:, None] > 0, t.view(blocks, BLOCK) / scale[:, None], 0.0).clamp(-448, 448).view(-1).to(torch.float8_e4m3fn)
        else:
            s["m"], s["v"] = m, r * r
        s["step"] = torch.full((), STEP0, dtype=torch.int64, device=dev)
        if own:
            from noise_amd import MultiTensorAdamW
            params = [torch.nn.Parameter(s["p"][o:o + n]) for o, n in zip(offs, sizes)]
            opt = MultiTensorAdamW(params, lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"])
            moments = (dict(exp_avg=s["m"], exp_avg_scale=s["m_scale"], exp_avg_sq_root=s["r"], exp_avg_sq_root_scale=s["r_scale"])
                       if case["bits"] == 8 else dict(exp_avg=s["m"], exp_avg_sq=s["v"]))
            opt.load_state_dict(dict(opt.state_dict(), step=torch.full((len(params),), STEP0, dtype=torch.int64, device=dev), **moments))
            s["opt"], s["grads"] = opt, [s["g"][o:o + n] for o, n in zip(offs, sizes)]
        return s
    B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
    shape = (B, T) if case["op"] != "decay_step" else (B,)
    if case["packed"]:
        qkv = randn(*shape, 3, H, dk, dtype=dt)
        s["q"], s["k"], s["v"] = qkv.unbind(-3)
        s["k"].mul_(dk ** -0.5)
    else:
        s["q"], s["k"], s["v"] = randn(*shape, H, dk, dtype=dt), (randn(*shape, H, dk) * dk ** -0.5).to(dt), randn(*shape, H, dv, dtype=dt)
    # memories of 8 to 2048 tokens over the heads
    s["log_decay"] = torch.log1p(-torch.exp2(-3.0 - 8.0 * torch.arange(H, device=dev, dtype=torch.float64) / max(1, H - 1))).float()
    s["state"] = randn(B, H, dk, dv)
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        s["lengths"][0] = T
    if case["op"] == "decay_train":
        s["do"] = randn(B, T, H, dv, dtype=dt)
        s["d_state"] = randn(B, H, dk, dv)
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_norm_fwd(x, w, b):
    xf = x.float()
    mean = xf.mean(1, keepdim=True)
    c = xf - mean
    rstd = (c.square().mean(1, keepdim=True) + EPS).rsqrt()
    return (c * rstd * w + b).to(x.dtype), mean[:, 0], rstd[:, 0]


def _plain_norm_bwd(dy, x, mean, rstd, w):
    g = dy.float()
    xhat = (x.float() - mean[:, None]) * rstd[:, None]
    gw = g * w
    dx = rstd[:, None] * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
    return dx.to(x.dtype), (g * xhat).sum(0), g.sum(0)


def _powers(log_decay, n):
    """exp(log_decay * n) for whole n, exponents in 64 bits, as float32; n broadcasts behind the head axis."""
    return torch.exp(log_decay.double().view(-1, *([1] * n.dim())) * n).float()


def _plain_decay(q, k, v, log_decay, state, lengths, scale):
    """Chunked form, all chunks at once: products inside the chunks, states between them by a triangular product."""
    B, T, H, dk = q.shape
    dv, dev = v.shape[-1], q.device
    n = -(-T // CHUNK)
    C = min(T, CHUNK)
    n = -(-T // C)

    def chunks(t):
        t = t.float().transpose(1, 2)
        t = torch.nn.functional.pad(t, (0, 0, 0, n * C - T))
        return t.reshape(B, H, n, C, t.shape[-1])

    valid = torch.ones(B, T, 1, 1, dtype=torch.bool, device=dev) if lengths is None else (
        torch.arange(T, device=dev)[None, :] < lengths[:, None])[:, :, None, None]
    qc, kc, vc = (chunks(torch.where(valid, t, 0)) for t in (q, k, v))
    i = torch.arange(C, device=dev)
    away = i[:, None] - i[None, :]
    inside = torch.where(away >= 0, _powers(log_decay, away.clamp_min(0)), 0.0)               # (H, C, C)
    a = (qc @ kc.transpose(-1, -2)) * inside[None, :, None]
    o = a @ vc
    kv = (kc * _powers(log_decay, C - 1 - i)[None, :, None, :, None]).transpose(-1, -2) @ vc   # (B, H, n, dk, dv)
    j = torch.arange(n, device=dev)
    back = j[:, None] - 1 - j[None, :]
    between = torch.where(back >= 0, _powers(log_decay, back.clamp_min(0) * C), 0.0)          # (H, n, n)
    s_in = (between[None] @ kv.reshape(B, H, n, dk * dv)).reshape(B, H, n, dk, dv)
    s_in = s_in + _powers(log_decay, j * C)[None, :, :, None, None] * state[:, :, None]
    o = (o + (qc * _powers(log_decay, i + 1)[None, :, None, :, None]) @ s_in) * scale
    o = o.reshape(B, H, n * C, dv)[:, :, :T].transpose(1, 2)
    o = torch.where(valid, o, 0.0).to(q.dtype)
    ends = torch.full((B,), T, device=dev) if lengths is None else lengths.long()
    t = torch.arange(n * C, device=dev)
    left = ends[:, None] - 1 - t[None, :]                                                      # (B, T)
    weight = torch.where(left[:, None] >= 0, _powers(log_decay, left.clamp_min(0)).transpose(0, 1), 0.0)   # (B, H, T)
    kall, vall = kc.reshape(B, H, n * C, dk), vc.reshape(B, H, n * C, dv)
    end = (kall * weight[..., None]).transpose(-1, -2) @ vall + _powers(log_decay, ends).transpose(0, 1)[:, :, None, None] * state
    return o, end


def _plain_decay_step(q, k, v, log_decay, state, scale):
    state.mul_(torch.exp(log_decay.double()).float()[None, :, None, None]).add_(k.float()[..., :, None] * v.float()[..., None, :])
    return ((q.float()[..., :, None] * state).sum(-2) * scale).to(q.dtype), state


def _plain_e4m3(x):
    """Nearest e4m3 value, ties to even, of |x| <= 448 in 64 bits."""
    a = x.abs()
    step = torch.ldexp(torch.ones_like(a), (torch.frexp(a)[1] - 1).clamp_min(-6) - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp_max(448.0)


def _plain_small(t, lowest):
    """(e4m3 values, scales) of a flat 64-bit tensor, one scale per block."""
    t = t.view(-1, BLOCK)
    scale = (t.abs().amax(1) / 448.0).float()
    inverse = torch.where(scale > 0, 1.0 / scale.double(), 0.0)
    c = _plain_e4m3((t * inverse[:, None]).clamp(-448.0, 448.0))
    if lowest:
        c = torch.where((t > 0) & (c == 0), 2.0 ** -9, c)
    return c.view(-1).float().to(torch.float8_e4m3fn), scale


def _plain_adamw(s):
    case = s["case"]
    b1, b2 = BETAS
    s["step"] += 1
    t = s["step"].double()
    size, root = (LR / (1 - b1 ** t)).float(), torch.sqrt(1 - b2 ** t).float()
    p = s["p"].float()
    if case["bits"] == 8:
        g = s["g"].double()
        m = b1 * (s["m"].double().view(-1, BLOCK) * s["m_scale"].double()[:, None]).view(-1) + (1 - b1) * g
        r = (s["r"].double().view(-1, BLOCK) * s["r_scale"].double()[:, None]).view(-1)
        r = torch.sqrt(b2 * r * r + (1 - b2) * g * g)
        p = p * (1 - LR * DECAY) - size * (m.float() / (r.float() / root + ADAM_EPS))
        (s["m"], s["m_scale"]), (s["r"], s["r_scale"]) = _plain_small(m, False), _plain_small(r, True)
    else:
        g = s["g"].float()
        s["m"].mul_(b1).add_(g, alpha=1 - b1)
        s["v"].mul_(b2).add_(g * g, alpha=1 - b2)
        p = p * (1 - LR * DECAY) - size * (s["m"] / (s["v"].sqrt() / root + ADAM_EPS))
    s["p"].copy_(p)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    keys = ("p", "m", "m_scale", "r", "r_scale") if s["case"]["bits"] == 8 else ("p", "m", "v")
    return {k: s[k] for k in keys}


# ------------------------------------------------------------------------------------------------------------------ run
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_plain(s):
    op = s["op"]
    if op == "norm_fwd":
        return _plain_norm_fwd(s["x"], s["w"], s["b"])
    if op == "norm_bwd":
        return _plain_norm_bwd(s["dy"], s["x"], s["mean"], s["rstd"], s["w"])
    if op == "adamw":
        return _plain_adamw(s)
    scale = s["case"]["dk"] ** -0.5
    if op == "decay_step":
        return _plain_decay_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], scale)
    if op == "decay_fwd":
        return _plain_decay(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["lengths"], scale)
    leaves = [s[n].detach().requires_grad_(True) for n in ("q", "k", "v", "state")]
    q, k, v, state = leaves
    o, end = _plain_decay(q, k, v, s["log_decay"], state, s["lengths"], scale)
    grads = torch.autograd.grad([o, end], leaves, [s["do"], s["d_state"]])
    return dict(o=o.detach(), state=end.detach(), dq=grads[0], dk=grads[1], dv=grads[2], d_state=grads[3])


def _run_own(s):
    import noise_amd as na
    op = s["op"]
    if op == "norm_fwd":
        return na.layer_norm_fwd(s["x"], s["w"], s["b"], EPS)
    if op == "norm_bwd":
        return na.layer_norm_bwd(s["dy"], s["x"], s["mean"], s["rstd"], s["w"])
    if op == "adamw":
        s["opt"].step(grads=s["grads"])
        st = s["opt"].state
        if s["case"]["bits"] == 8:
            return dict(p=s["p"], m=st["exp_avg"], m_scale=st["exp_avg_scale"], r=st["exp_avg_sq_root"], r_scale=st["exp_avg_sq_root_scale"])
        return dict(p=s["p"], m=st["exp_avg"], v=st["exp_avg_sq"])
    if op == "decay_step":
        return na.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"]), s["state"]
    args = (s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["lengths"])
    o, end = na.decay_attention_fwd(*args)
    if op == "decay_fwd":
        return o, end
    dq, dk, dv, d_state = na.decay_attention_bwd(s["do"], *args, d_state=s["d_state"])
    return dict(o=o, state=end, dq=dq, dk=dk, dv=dv, d_state=d_state)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op == "norm_fwd":
        n = case["rows"] * case["dim"]
        return dict(bytes=2 * e * n + 8 * case["rows"] + 8 * case["dim"], flops=8 * n)
    if op == "norm_bwd":
        n = case["rows"] * case["dim"]
        return dict(bytes=3 * e * n + 8 * case["rows"] + 12 * case["dim"], flops=14 * n)
    if op == "adamw":
        n = case["numel"]
        states = 4 + 4 * 4 / BLOCK if case["bits"] == 8 else 16
        return dict(bytes=int(n * (2 * e + BYTES[case["gdtype"]] + states)), flops=16 * n)
    B, T, H, dk, dv = (case[k] for k in ("B", "T", "H", "dk", "dv"))
    t = B * T * H
    states = B * H * dk * dv
    if op == "decay_train":
        # forward: q, k, v -> o; backward: q, k, v, do -> dq, dk, dv; the states and their gradients once each
        return dict(bytes=e * t * (2 * dk + 2 * dv + 4 * dk + 3 * dv) + 4 * 5 * states, flops=14 * t * dk * dv)
    return dict(bytes=e * t * (2 * dk + 2 * dv) + 4 * 2 * states, flops=4 * t * dk * dv)


# ---------------------------------------------------------------------------------------------------------------- exact
def _exact_small(t, lowest):
    """Nearest of the 127 non-negative e4m3 values by search, ties to the even code."""
    codes = torch.arange(127, device=t.device)
    e, m = codes // 8, (codes % 8).double()
    table = torch.where(e > 0, (1 + m / 8) * torch.exp2((e - 7).double()), m / 8 * 2.0 ** -6)
    mids = (table[1:] + table[:-1]) / 2
    rows = t.reshape(-1, BLOCK)
    scale = (rows.abs().max(dim=1).values / 448.0).float()
    a = (rows.abs() / torch.where(scale > 0, scale.double(), 1.0)[:, None]).reshape(-1)
    c = torch.searchsorted(mids, a)
    tie = (c < 126) & (mids[c.clamp(max=125)] == a)
    c = torch.where(tie & (c % 2 == 1), c + 1, c)
    if lowest:
        c = torch.where((t.reshape(-1) > 0) & (c == 0), 1, c)
    return table[c] * torch.where(t.reshape(-1) < 0, -1.0, 1.0), scale.double()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = 1 / torch.sqrt(var + EPS)
        y = (x - mean[:, None]) * rstd[:, None]
        return y * s["w"].double() + s["b"].double(), mean, rstd
    if op == "norm_bwd":
        x, g, w = s["x"].double(), s["dy"].double(), s["w"].double()
        mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
        xhat = (x - mean) * rstd
        a, D = g * w, case["dim"]
        dx = rstd / D * (D * a - a.sum(1, keepdim=True) - xhat * (a * xhat).sum(1, keepdim=True))
        return dx, (g * xhat).sum(0), g.sum(0)
    if op == "adamw":
        b1, b2 = BETAS
        t = STEP0 + 1
        g = s["g"].double()
        if case["bits"] == 8:
            m = s["m"].double() * s["m_scale"].double().repeat_interleave(BLOCK)
            v = (s["r"].double() * s["r_scale"].double().repeat_interleave(BLOCK)) ** 2
        else:
            m, v = s["m"].double(), s["v"].double()
        m, v = m * b1 + g * (1 - b1), v * b2 + g ** 2 * (1 - b2)
        mhat, vhat = m / (1 - b1 ** t), v / (1 - b2 ** t)
        p = s["p"].double()
        p = p - LR * DECAY * p - LR * mhat / (vhat.sqrt() + ADAM_EPS)
        if case["bits"] == 32:
            return dict(p=p, m=m, v=v)
        (mc, ms), (rc, rs) = _exact_small(m, False), _exact_small(v.sqrt(), True)
        return dict(p=p, m=mc, m_scale=ms, r=rc, r_scale=rs)
    # the recurrence, token by token
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    scale = case["dk"] ** -0.5
    S = s["state"].double().clone()
    lam = torch.exp(s["log_decay"].double())[None, :, None, None]
    if op == "decay_step":
        S = lam * S + k[..., :, None] * v[..., None, :]
        return torch.einsum("bhk,bhkv->bhv", q, S) * scale, S
    B, T, H, dk, dv = (case[n] for n in ("B", "T", "H", "dk", "dv"))
    lengths = torch.full((B,), T, device=q.device) if s["lengths"] is None else s["lengths"].long()
    train = op == "decay_train"
    live = (torch.arange(T, device=q.device)[:, None] < lengths[None, :]).double()      # (T, B)
    ragged = s["lengths"] is not None
    o, dq = torch.zeros_like(v), torch.zeros_like(q)
    do = s["do"].double() if train else None
    for t in range(T):
        new = torch.addcmul(lam * S, k[:, t, :, :, None], v[:, t, :, None, :])
        S = torch.where(live[t, :, None, None, None] > 0, new, S) if ragged else new
        torch.matmul(q[:, t, :, None, :], S, out=o[:, t, :, None, :]) if not ragged else o[:, t].copy_((q[:, t, :, None, :] @ S)[:, :, 0])
        if train:
            dq[:, t] = (S @ do[:, t, :, :, None])[..., 0]
    o = o * scale * live.t()[:, :, None, None]
    if not train:
        return o, S
    end = S
    dq = dq * scale * live.t()[:, :, None, None]
    dkk, dvv = torch.zeros_like(k), torch.zeros_like(v)
    G = s["d_state"].double().clone()       # gradient of the state behind token t; a clip's own end comes first
    for t in range(T - 1, -1, -1):
        on = live[t, :, None, None, None]
        new = G + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
        dkk[:, t] = (new @ v[:, t, :, :, None])[..., 0] * on[..., 0]
        dvv[:, t] = (k[:, t, :, None, :] @ new)[:, :, 0] * on[..., 0]
        G = torch.where(on > 0, lam * new, G) if ragged else lam * new
    return dict(o=o, state=end, dq=dq, dk=dkk, dv=dvv, d_state=G)
