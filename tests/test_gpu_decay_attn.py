"""Decay attention (csrc/decay_attn.hip) against its recurrence in 64 bits: clips, gradients, single tokens, and the calls it
refuses."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def half(dtype):
    """Half a step of the type, relative; fp32 results are counted with the arithmetic."""
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def tiny(dtype):
    fi = torch.finfo(dtype)
    return 0.0 if dtype == torch.float32 else fi.smallest_normal * fi.eps


def make(B, T, H, dk, dv, dtype, seed, packed=False, ragged=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    if packed:
        assert dk == dv
        q, k, v = r(B, T, 3, H, dk).to(dtype).to(DEV).unbind(2)
    else:
        q, k, v = (r(B, T, H, d).to(dtype).to(DEV) for d in (dk, dk, dv))
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        lengths[0] = T
        if B > 1:
            lengths[1] = 0
        lengths = lengths.to(DEV)
    decay = torch.tensor([[-0.5, -0.03, 0.0, -1e-3, -4.0, -float("inf")][h % 6] for h in range(H)], device=DEV)
    return dict(q=q, k=k, v=v, log_decay=decay, state=r(B, H, dk, dv).to(DEV), lengths=lengths,
                do=r(B, T, H, dv).to(dtype).to(DEV), d_state=r(B, H, dk, dv).to(DEV))


def recurrence(c, scale, magnitude=False):
    """All outputs and gradients from the definition, token by token, in 64 bits.  magnitude: the same with every input
    replaced by its absolute value, i.e. the sum of the magnitudes of all terms that a result adds up."""
    f = (lambda t: t.double().abs()) if magnitude else (lambda t: t.double())
    q, k, v, do = (f(c[n]) for n in ("q", "k", "v", "do"))
    B, T, H, dk = q.shape
    S, G = f(c["state"]).clone(), f(c["d_state"]).clone()
    lam = torch.exp(c["log_decay"].double()).view(1, H, 1, 1)
    n = torch.full((B,), T, device=DEV) if c["lengths"] is None else c["lengths"].long()
    live = torch.arange(T, device=DEV)[:, None] < n[None, :]
    o, dq, dkk, dvv = torch.zeros_like(v), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    z = torch.zeros((), device=DEV, dtype=torch.float64)
    for t in range(T):
        on = live[t].view(B, 1, 1, 1)
        S = torch.where(on, lam * S + torch.where(on, k[:, t, :, :, None] * v[:, t, :, None, :], z), S)
        o[:, t] = torch.where(on[..., 0], (torch.where(on[..., 0], q[:, t], z)[..., None] * S).sum(-2) * scale, z)
        dq[:, t] = torch.where(on[..., 0], (S * torch.where(on[..., 0], do[:, t], z)[:, :, None, :]).sum(-1) * scale, z)
    for t in range(T - 1, -1, -1):
        on = live[t].view(B, 1, 1, 1)
        new = G + scale * torch.where(on, q[:, t, :, :, None] * do[:, t, :, None, :], z)
        dkk[:, t] = torch.where(on[..., 0], (new * v[:, t, :, None, :]).sum(-1), z)
        dvv[:, t] = torch.where(on[..., 0], (new * k[:, t, :, :, None]).sum(-2), z)
        G = torch.where(on, lam * new, G)
    return dict(o=o, end=S, dq=dq, dk=dkk, dv=dvv, d_state=G)


def tolerance(name, want, mag, dtype, T, dk, dv):
    """A result is a sum over at most T tokens of sums over a head axis; each term passes through at most T + max(dk, dv) fp32
    additions and, beside them, 16 roundings (decay powers: exponent and exponential, weights, state decay; the powers of a
    long memory are products of at most T / 32 rounded ones).  In 16-bit types the weights and the state are rounded to the
    type on their way into the matrix products (one half step each of the terms' magnitudes), and o, dq, dk, dv once more; the
    carried states are not rounded below fp32."""
    n = (T + max(dk, dv)) + 16 + 2 * (T // 32 + 1)
    t = n * U * mag + 1e-30
    if name in ("o", "dq", "dk", "dv"):
        h = half(dtype)
        t = t + 2.02 * h * mag * (1 + h) + h * want.abs() * 1.01 + tiny(dtype)
    return t


def check(c, got, scale, dtype):
    B, T, H, dk = c["q"].shape
    dv = c["v"].shape[-1]
    want, mag = recurrence(c, scale), recurrence(c, scale, True)
    for name, g in got.items():
        w, m = want[name], mag[name]
        assert g.shape == w.shape and g.dtype == (torch.float32 if name in ("end", "d_state") else dtype), name
        t = tolerance(name, w, m, dtype, T, dk, dv)
        d = (g.double() - w).abs()
        assert (d <= t).all(), (name, (d / t).max().item(), (d.norm() / w.norm()).item())


def run_all(c, scale=None):
    import noise_amd as na
    args = (c["q"], c["k"], c["v"], c["log_decay"], c["state"], c["lengths"])
    o, end = na.decay_attention_fwd(*args, scale=scale)
    dq, dk, dv, d_state = na.decay_attention_bwd(c["do"], *args, scale=scale, d_state=c["d_state"])
    return dict(o=o, end=end, dq=dq, dk=dk, dv=dv, d_state=d_state)


SHAPES = [(1, 1, 1, 1, 1), (2, 2, 3, 10, 10), (3, 31, 2, 16, 16), (2, 32, 2, 17, 5), (2, 33, 3, 32, 32), (3, 64, 2, 24, 40), (2, 65, 6, 64, 64),
          (2, 100, 2, 128, 128), (2, 129, 2, 128, 33), (1, 200, 2, 7, 100), (2, 530, 2, 64, 64), (1, 777, 3, 16, 16), (1, 1100, 2, 128, 128),
          (2, 600, 3, 33, 128), (70, 40, 8, 10, 10)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("B,T,H,dk,dv", SHAPES)
def test_clips_and_gradients(B, T, H, dk, dv, ragged, dtype):
    c = make(B, T, H, dk, dv, dtype, B * 1000 + T + dk, packed=dk == dv and T % 2 == 0, ragged=ragged)
    got = run_all(c)
    check(c, got, dk ** -0.5, dtype)
    again = run_all(c)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_defaults_without_states(dtype):
    """No state, no gradient of the end, an explicit scale."""
    import noise_amd as na
    c = make(2, 70, 3, 20, 20, dtype, 4)
    o, end = na.decay_attention_fwd(c["q"], c["k"], c["v"], c["log_decay"], scale=0.3)
    dq, dk, dv, d_state = na.decay_attention_bwd(c["do"], c["q"], c["k"], c["v"], c["log_decay"], scale=0.3)
    c["state"], c["d_state"] = torch.zeros_like(c["state"]), torch.zeros_like(c["d_state"])
    check(c, dict(o=o, end=end, dq=dq, dk=dk, dv=dv, d_state=d_state), 0.3, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_padding_is_never_read(dtype):
    """NaN and infinity in the padded rows change nothing; rows behind the end are zero, an empty clip keeps its state."""
    c = make(4, 300, 2, 48, 64, dtype, 8, ragged=True)
    want = run_all(c)
    pad = torch.arange(300, device=DEV)[None, :] >= c["lengths"][:, None]
    assert pad[1].all()
    for n in ("q", "k", "v", "do"):
        c[n][pad] = float("nan") if n != "v" else float("inf")
    got = run_all(c)
    assert all(torch.equal(want[n], got[n]) for n in want)
    for n in ("o", "dq", "dk", "dv"):
        assert not got[n][pad].any()
    assert torch.equal(got["end"][1], c["state"][1]) and torch.equal(got["d_state"][1], c["d_state"][1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q,k,v,state,do", [(6, -8, 9, 14, -6), (-9, 7, -10, -30, -12), (5, 5, 0, 20, 0), (0, 0, -14, 0, 10), (7, 4, 12, -100, 3)])
def test_magnitudes_far_from_one(q, k, v, state, do, dtype):
    """Inputs scaled by powers of two up to the type's ends, and a piece of silence: the 16-bit operands inside carry their own
    scales, so the error stays relative to the terms.  Results that leave the type's range are left out."""
    c = make(2, 300, 2, 64, 40, dtype, 17)
    for n, e in (("q", q), ("k", k), ("v", v), ("do", do)):
        c[n] = (c[n].double() * 2.0 ** e).to(dtype)
    c["v"][:, 70:200] = 0
    c["state"], c["d_state"] = c["state"] * 2.0 ** state, c["d_state"] * 2.0 ** state
    c["log_decay"] = torch.tensor([-0.02, 0.0], device=DEV)
    got = run_all(c)
    want, mag = recurrence(c, 64 ** -0.5), recurrence(c, 64 ** -0.5, True)
    top = torch.finfo(dtype).max
    for name, g in got.items():
        fits = want[name].abs() < (0.9 * top if name in ("o", "dq", "dk", "dv") else float("inf"))
        t = tolerance(name, want[name], mag[name], dtype, 300, 64, 40)
        assert ((g.double() - want[name]).abs() <= t)[fits].all(), (name, ((g.double() - want[name]).abs() / t)[fits].max())


def test_views_strides_and_orders():
    """Packed projections, a (B, H, T, D) layout, a sliced axis, a broadcast clip and a last axis with a stride: the numbers of
    packed copies."""
    import noise_amd as na
    g = torch.Generator().manual_seed(3)
    B, T, H, D = 3, 77, 4, 20
    decay = torch.tensor([-0.1, -0.01, 0.0, -1.0], device=DEV)
    big = torch.randn(B, T, H, 3 * D + 1, generator=g).to(DEV)
    bhtd = torch.randn(3, B, H, T, D, generator=g).to(DEV)
    last = torch.randn(3, B, T, H, D, 2, generator=g).to(DEV)
    one = torch.randn(3, 1, T, H, D, generator=g).to(DEV).expand(3, B, T, H, D)
    for q, k, v in ([big[..., 1 + i * D:1 + (i + 1) * D] for i in range(3)], bhtd.transpose(2, 3).unbind(0), last[..., 1].unbind(0), one.unbind(0),
                    torch.randn(3, B, 2 * T, H, D, generator=g).to(DEV)[:, :, ::2].unbind(0)):
        a = na.decay_attention_fwd(q, k, v, decay)
        b = na.decay_attention_fwd(q.contiguous(), k.contiguous(), v.contiguous(), decay)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        do = v.transpose(1, 2).contiguous().transpose(1, 2)
        a = na.decay_attention_bwd(do, q, k, v, decay)
        b = na.decay_attention_bwd(do.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), decay)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (1, 6, 10, 10), (5, 3, 64, 64), (2, 2, 128, 128), (3, 2, 128, 6), (2, 3, 33, 100), (40, 8, 16, 32)])
def test_single_tokens(B, H, dk, dv, dtype):
    import noise_amd as na
    c = make(B, 3, H, dk, dv, dtype, B + dk, packed=dk == dv)
    state = c["state"].clone()
    lam = torch.exp(c["log_decay"].double()).view(1, H, 1, 1)
    for t in range(3):
        before = state.double()
        o = na.decay_attention_step(c["q"][:, t], c["k"][:, t], c["v"][:, t], c["log_decay"], state)
        k, v, q = (c[n][:, t].double() for n in "kvq")
        want = lam * before + k[..., :, None] * v[..., None, :]
        mag = lam * before.abs() + (k[..., :, None] * v[..., None, :]).abs()
        assert ((state.double() - want).abs() <= 6 * U * mag).all()          # decay, its product, k v, the sum
        wo = (q[..., None] * want).sum(-2) * dk ** -0.5
        mo = (q.abs()[..., None] * mag).sum(-2) * dk ** -0.5
        assert ((o.double() - wo).abs() <= (dk + 10) * U * mo + half(dtype) * wo.abs() * 1.01 + tiny(dtype) + 1e-30).all()
    out = torch.empty(B, H, dv, device=DEV, dtype=dtype)
    assert na.decay_attention_step(c["q"][:, 0], c["k"][:, 0], c["v"][:, 0], c["log_decay"], state, out=out) is out


def test_pieces_equal_the_whole_and_tokens_equal_clips():
    """A clip in pieces of odd sizes, then token by token, carrying the state: the fp32 results of one pass, up to the
    rounding both may make."""
    import noise_amd as na
    c = make(2, 150, 3, 32, 24, torch.float32, 12)
    c["lengths"] = None
    whole, end = na.decay_attention_fwd(c["q"], c["k"], c["v"], c["log_decay"], c["state"])
    state, outs, t = c["state"], [], 0
    for n in (1, 37, 64, 40):
        o, state = na.decay_attention_fwd(c["q"][:, t:t + n], c["k"][:, t:t + n], c["v"][:, t:t + n], c["log_decay"], state)
        outs.append(o)
        t += n
    state = state.clone()
    while t < 150:
        outs.append(na.decay_attention_step(c["q"][:, t], c["k"][:, t], c["v"][:, t], c["log_decay"], state)[:, None])
        t += 1
    mag = recurrence(c, 32 ** -0.5, True)
    tol = 2 * (150 + 32 + 28)
    assert ((torch.cat(outs, 1) - whole).abs().double() <= tol * U * mag["o"]).all()
    assert ((state - end).abs().double() <= tol * U * mag["end"]).all()


def test_autograd_against_differences():
    """Central differences of a weighted sum of both outputs in 64 bits along a random direction."""
    import noise_amd as na
    g = torch.Generator().manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    B, T, H, dk, dv = 2, 45, 2, 12, 9
    x = [r(B, T, H, dk), r(B, T, H, dk), r(B, T, H, dv), r(B, H, dk, dv)]
    u = [r(*t.shape) for t in x]
    cw, ce = r(B, T, H, dv), r(B, H, dk, dv)
    decay = torch.tensor([-0.2, -0.01])

    def f(t):
        q, k, v, S = (a + t * b for a, b in zip(x, u))
        lam, total = decay.double().exp().view(1, H, 1, 1), 0.0
        for i in range(T):
            S = lam * S + k[:, i, :, :, None] * v[:, i, :, None, :]
            total = total + (cw[:, i] * (q[:, i, :, :, None] * S).sum(-2) * dk ** -0.5).sum()
        return (total + (ce * S).sum()).item()
    want = (f(1e-5) - f(-1e-5)) / 2e-5
    leaves = [t.float().to(DEV).requires_grad_(True) for t in x]
    o, end = na.decay_attention(*leaves[:3], decay.to(DEV), leaves[3])
    ((o * cw.float().to(DEV)).sum() + (end * ce.float().to(DEV)).sum()).backward()
    parts = [(l.grad.double().cpu() * d) for l, d in zip(leaves, u)]
    got, scale = sum(p.sum().item() for p in parts), sum(p.abs().sum().item() for p in parts)
    # fp32 inputs (one rounding), the arithmetic of at most T + dk + 30 terms, differences exact to ~1e-8 of the scale
    assert abs(got - want) <= scale * ((T + dk + 30) * U * 4 + 1e-7)
    # an unused end state, and an output that is broadcast back
    for l in leaves:
        l.grad = None
    na.decay_attention(*leaves[:3], decay.to(DEV), leaves[3])[0].sum().backward()
    assert all(torch.isfinite(l.grad).all() for l in leaves)


def test_refusals():
    import noise_amd as na
    c = make(2, 5, 3, 8, 8, torch.float32, 1)
    q, k, v, g, s = c["q"], c["k"], c["v"], c["log_decay"], c["state"]
    z = lambda *a, **kw: torch.zeros(*a, device=DEV, **kw)
    for args, kind, text in (((q, k[:, :4], v, g), ValueError, "q, k must be"), ((q[0], k[0], v[0], g), ValueError, "q, k must be"),
                             ((q, k.half(), v, g), TypeError, "share one"), ((q.double(), k.double(), v.double(), g), TypeError, "share one"),
                             ((z(1, 2, 1, 129), z(1, 2, 1, 129), z(1, 2, 1, 8), z(1)), ValueError, "head sizes"),
                             ((q, k, v, g[:2]), ValueError, "log_decay"), ((q, k, v, g.double()), ValueError, "log_decay"),
                             ((q, k, v, g, s[:1]), ValueError, "state"), ((q, k, v, g, s.half()), ValueError, "state"),
                             ((q, k, v, g, s, z(3, dtype=torch.int32)), ValueError, "lengths"), ((q, k, v, g, s, z(2)), ValueError, "lengths")):
        with pytest.raises(kind, match=text):
            na.decay_attention(*args)
    with pytest.raises(ValueError, match="no gradient"):
        na.decay_attention(q, k, v, g.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="do must be"):
        na.decay_attention_bwd(c["do"][:, :2], q, k, v, g)
    with pytest.raises(ValueError, match="d_state"):
        na.decay_attention_bwd(c["do"], q, k, v, g, d_state=s[:, :1])
    one = (q[:, 0], k[:, 0], v[:, 0], g)
    with pytest.raises(ValueError, match="needs the streams' state"):
        na.decay_attention_step(*one, None)
    with pytest.raises(ValueError, match="packed"):
        na.decay_attention_step(*one, s.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(RuntimeError, match="no backward"):
        na.decay_attention_step(q[:, 0].clone().requires_grad_(True), k[:, 0], v[:, 0], g, s)
    with pytest.raises(ValueError, match="out must be"):
        na.decay_attention_step(*one, s, out=z(2, 3, 7))


def test_a_step_over_a_saved_state_is_noticed():
    """A state that a graph holds for its backward pass and a step then overwrites: the backward pass refuses."""
    import noise_amd as na
    c = make(1, 4, 2, 8, 8, torch.float32, 2)
    q = c["q"].clone().requires_grad_(True)
    state = c["state"].clone()
    o, _ = na.decay_attention(q, c["k"], c["v"], c["log_decay"], state)
    na.decay_attention_step(c["q"][:, 0], c["k"][:, 0], c["v"][:, 0], c["log_decay"], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    with torch.inference_mode():       # states made in inference mode have no version and need none
        s2 = torch.zeros(1, 2, 8, 8, device=DEV)
        na.decay_attention_step(c["q"][:, 0], c["k"][:, 0], c["v"][:, 0], c["log_decay"], s2)


def test_calls_on_two_streams_at_once():
    """Two different calls in flight together: nothing is shared between them."""
    import noise_amd as na
    cs = [make(1, 3000, 2, 64, 64, torch.bfloat16, 3), make(1, 2500, 2, 64, 64, torch.bfloat16, 4)]
    want = [run_all(c) for c in cs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cs], [None, None]
    for _ in range(3):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                got[i] = run_all(c)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w[n], g[n]) for n in w)


def test_no_tokens():
    import noise_amd as na
    c = make(2, 5, 3, 8, 6, torch.float32, 1)
    e = lambda t: t[:, :0]
    o, end = na.decay_attention_fwd(e(c["q"]), e(c["k"]), e(c["v"]), c["log_decay"], c["state"])
    assert o.shape == (2, 0, 3, 6) and torch.equal(end, c["state"]) and end.data_ptr() != c["state"].data_ptr()
    dq, dk, dv, ds = na.decay_attention_bwd(e(c["do"]), e(c["q"]), e(c["k"]), e(c["v"]), c["log_decay"], c["state"], d_state=c["d_state"])
    assert dq.shape == (2, 0, 3, 8) and torch.equal(ds, c["d_state"])
    assert na.decay_attention_step(c["q"][:0, 0], c["k"][:0, 0], c["v"][:0, 0], c["log_decay"], c["state"][:0]).shape == (0, 3, 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_other_stream_and_captured_graph(dtype):
    """Two shapes (one walk, and one cut into segments) on another stream and through a graph replayed over changed inputs."""
    import noise_amd as na
    for shape in ((3, 90, 2, 32, 32), (1, 900, 2, 64, 64)):
        c = make(*shape, dtype, 5, ragged=shape[0] > 1)
        want = run_all(c)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = run_all(c)
        s.synchronize()
        assert all(torch.equal(want[n], got[n]) for n in want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run_all(c)
            step_state = c["state"].clone()
            step = na.decay_attention_step(c["q"][:, 0], c["k"][:, 0], c["v"][:, 0], c["log_decay"], step_state)
        for i in range(3):
            c["q"].mul_(-1)
            c["state"].add_(0.25)
            graph.replay()
            eager = run_all(c)
            st = c["state"].clone()
            eo = na.decay_attention_step(c["q"][:, 0], c["k"][:, 0], c["v"][:, 0], c["log_decay"], st)
            torch.cuda.synchronize()
            assert all(torch.equal(eager[n], held[n]) for n in eager) and torch.equal(eo, step) and torch.equal(st, step_state)


@pytest.mark.parametrize("T", [40, 900])
def test_lengths_outside_of_the_clip(T):
    """int64 and int32 lengths, below zero and far above T: those of the limits, forwards and backwards."""
    c = make(6, T, 2, 16, 16, torch.float32, 9)
    c["lengths"] = torch.tensor([T, T, 0, 0, T, 11], dtype=torch.int32, device=DEV)
    want = run_all(c)
    big = torch.iinfo(torch.int64)
    for lengths in (torch.tensor([2 ** 40, big.max, big.min, -3, T + 1, 11]), torch.tensor([T, 2 ** 32 + 5, -2 ** 32 + 7, 0, 2 ** 31, 11]),
                    torch.tensor([2 ** 31 - 1, T + 1, -1, -2 ** 31, T, 11], dtype=torch.int32)):
        c["lengths"] = lengths.to(DEV)
        got = run_all(c)
        assert all(torch.equal(want[n], got[n]) for n in want)


def test_step_into_its_own_arguments():
    """out over q, k or v row for row gives the same numbers; over the state it is refused and the state stays."""
    import noise_amd as na
    c = make(5, 1, 3, 16, 16, torch.bfloat16, 2)
    one = [c[n][:, 0].contiguous() for n in "qkv"]
    state = c["state"].clone()
    want = na.decay_attention_step(*one, c["log_decay"], state)
    for i in range(3):
        again, s = [t.clone() for t in one], c["state"].clone()
        assert na.decay_attention_step(*again, c["log_decay"], s, out=again[i]) is again[i]
        assert torch.equal(again[i], want) and torch.equal(s, state)
    f = [t.float() for t in one]
    s = c["state"].clone()
    with pytest.raises(RuntimeError, match="shares memory"):
        na.decay_attention_step(*f, c["log_decay"], s, out=s.view(-1)[:5 * 3 * 16].view(5, 3, 16))
    assert torch.equal(s, c["state"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,D", [(3, 77, 20), (2, 129, 24), (1, 700, 64), (2, 90, 128)])
def test_layouts_of_every_type(B, T, D, dtype):
    """Layouts that are read in place, and those that are copied first (a broadcast token axis, overlapping windows, a last axis
    with a stride): the numbers of packed copies, forwards and backwards."""
    import noise_amd as na
    g = torch.Generator().manual_seed(T)
    H = 3
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)
    decay = torch.tensor([-0.1, -0.01, 0.0], device=DEV)
    big, line = r(B, T, H, 3 * D + 1), r(B, H, 3, T + D)
    layouts = [[big[..., 1 + i * D:1 + (i + 1) * D] for i in range(3)],               # rows off any 16-byte border
               [big[..., i * D:(i + 1) * D] for i in range(3)],
               r(3, B, H, T, D).transpose(2, 3).unbind(0),                             # heads outside of tokens
               r(3, B, T, H, D, 2)[..., 1].unbind(0),                                  # a strided last axis
               r(3, 1, T, H, D).expand(3, B, T, H, D).unbind(0),                       # one clip for all
               r(3, B, T, 1, D).expand(3, B, T, H, D).unbind(0),                       # one head for all
               r(3, B, 1, H, D).expand(3, B, T, H, D).unbind(0),                       # one token for all: copied
               line.unfold(-1, D, 1)[..., :T, :].permute(2, 0, 3, 1, 4).unbind(0),     # windows that overlap: copied
               r(3, B, 2 * T, H, D)[:, :, ::2].unbind(0)]
    state = torch.randn(B, H, D, D, generator=g).to(DEV)
    for q, k, v in layouts:
        assert q.shape == k.shape == v.shape == (B, T, H, D)
        packed = [t.contiguous() for t in (q, k, v)]
        a, b = (na.decay_attention_fwd(*t, decay, state) for t in ((q, k, v), packed))
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        a = na.decay_attention_bwd(k, q, k, v, decay, state)
        b = na.decay_attention_bwd(packed[1], *packed, decay, state)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("e,v", [(64, 0), (70, -14), (75, 0), (90, -10), (110, 0), (118, -14), (123, 5)])
@pytest.mark.parametrize("T", [130, 900])
def test_states_up_to_the_end_of_fp32(T, e, v, dtype):
    """States and their gradients of 2^e beside ordinary and small tokens: what fp32 can hold stays finite, whatever units the
    fp16 kernel carries the state in.  Results beyond their type's range are left out; e = 123 leaves room for four sigma."""
    c = make(1, T, 3, 32, 24, dtype, e + T)
    c["log_decay"] = torch.tensor([-3.0, -0.4, 0.0], device=DEV)
    c["v"] = (c["v"].double() * 2.0 ** v).to(dtype)
    c["do"] = (c["do"].double() * 2.0 ** v).to(dtype)
    c["state"], c["d_state"] = (c[n].clamp(-4, 4) * 2.0 ** e for n in ("state", "d_state"))
    got = run_all(c)
    want, mag = recurrence(c, 32 ** -0.5), recurrence(c, 32 ** -0.5, True)
    top = torch.finfo(dtype).max
    for name, g in got.items():
        if name in ("o", "dq", "dk", "dv"):
            # a product of 16-bit rounded weights and states can leave the type's range where its magnitude sum does
            fits = mag[name] < 0.9 * top
            if dtype != torch.float16:
                # the product of a row with the state before its chunk of up to 64 tokens is formed in fp32 without its scale and
                # decay, and has to fit itself: elements of at most 4 2^e, decayed up to that chunk, plus what the tokens add
                row = c[{"o": "q", "dq": "do", "dk": "v", "dv": "k"}[name]].double().abs().sum(-1, keepdim=True)
                t = torch.arange(T, device=DEV) if name in ("o", "dq") else torch.arange(T, device=DEV).flip(0)
                lam = torch.exp(c["log_decay"].double().view(1, 3) * (t - 64).clamp_min(0).view(T, 1)).view(1, T, 3, 1)
                fits &= row * (4 * 2.0 ** e * lam + 2.0 ** 40) < 0.9 * torch.finfo(torch.float32).max
        else:
            fits = torch.ones_like(g, dtype=torch.bool)
            assert torch.isfinite(g).all(), name
        # a decay over d tokens is 2^(g2 d), g2 = g log2(e): log2(e), g2 and the product are rounded, 3 U of an exponent of |g| d
        # (in units of e), so 3 U |g| d of the power.  With states this large a power counts that would vanish otherwise
        g3 = 3 * c["log_decay"].double().abs() * T * U
        t = tolerance(name, want[name], mag[name], dtype, T, 32, 24) + mag[name] * (g3.view(3, 1) if g.shape[1] == T else g3.view(3, 1, 1))
        assert fits.any() and ((g.double() - want[name]).abs() <= t)[fits].all(), (name, ((g.double() - want[name]).abs() / t)[fits].max())


def poison(c, places):
    for name, b, t, h, col, value in places:
        c[name][b, t, h, col] = value
    return c


def check_poisoned(c, dtype):
    """What the definition leaves finite is finite and as exact as ever; what it does not is not."""
    B, T, H, dk = c["q"].shape
    dv = c["v"].shape[-1]
    got, want, mag = run_all(c), recurrence(c, dk ** -0.5), recurrence(c, dk ** -0.5, True)
    for name, g in got.items():
        ok = torch.isfinite(want[name])
        assert torch.equal(torch.isfinite(g), ok), (name, (torch.isfinite(g) != ok).nonzero()[:4])
        t = tolerance(name, want[name], mag[name], dtype, T, dk, dv)
        assert ((g.double() - want[name]).abs() <= t)[ok].all(), (name, ((g.double() - want[name]).abs() / t)[ok].max())
    return got


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,dk,dv", [(2, 7, 10, 10), (2, 150, 16, 16), (2, 130, 33, 24), (2, 200, 64, 64), (1, 1100, 64, 40), (2, 140, 128, 128),
                                       (1, 900, 128, 100)])
@pytest.mark.parametrize("name", ["q", "k", "v", "do"])
def test_a_token_that_is_not_finite(name, B, T, dk, dv, dtype):
    """One, two neighbouring, and several values of a tensor that are not finite, at the ends of chunks and inside them: neither a
    token before it (behind it in the gradients that run backwards) nor another column feels them."""
    n = dv if name in ("v", "do") else dk
    for i, places in enumerate(([(T // 2, 3, NAN)], [(T - 1, 0, INF), (0, n - 1, -INF)], [(T // 3, 2, INF), (T // 3 + 1, 1, NAN), (T // 3 + 2, n - 2, INF)],
                                [(t, (5 * t) % n, -INF) for t in (1, 31, 32, 63, 64, 65, 96, 127, 128) if t < T])):
        c = make(B, T, 2, dk, dv, dtype, 100 * i + T + dk)
        c["log_decay"] = torch.tensor([-0.05, 0.0], device=DEV)
        check_poisoned(poison(c, [(name, B - 1, t, 1, col, x) for t, col, x in places]), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_poison_everywhere_and_nowhere_else(dtype):
    """Tokens of every tensor and elements of the states at once, a clip whose tokens are all poisoned in one column, padding, and
    layouts without 16-byte rows; clips and heads beside them keep the very bits they have without."""
    c = make(4, 260, 3, 40, 40, dtype, 6, packed=True, ragged=True)
    c["lengths"][:] = torch.tensor([260, 100, 177, 0])
    c["log_decay"] = torch.tensor([-0.1, 0.0, -1.0], device=DEV)
    clean = run_all(c)
    poison(c, [("v", 0, t, 1, 7, NAN) for t in range(260)] + [("k", 2, 40, 0, 3, INF), ("q", 2, 50, 2, 0, NAN), ("do", 2, 60, 2, 5, INF),
                                                             ("v", 2, 33, 1, 39, -INF), ("v", 2, 34, 1, 38, INF), ("v", 2, 176, 1, 0, NAN),
                                                             ("state", 1, 0, 2, 4, INF), ("d_state", 1, 1, 3, 9, NAN)])
    pad = torch.arange(260, device=DEV)[None, :] >= c["lengths"][:, None]
    for n in ("q", "k", "v", "do"):
        c[n][pad] = NAN
    got = check_poisoned(c, dtype)
    touched = torch.zeros(4, 3, dtype=torch.bool)
    for b, h in ((0, 1), (2, 0), (2, 2), (2, 1), (1, 0), (1, 1)):
        touched[b, h] = True
    for n, g in got.items():
        heads = (lambda t: t.transpose(1, 2)) if n in ("o", "dq", "dk", "dv") else (lambda t: t)
        assert torch.equal(heads(g)[~touched.to(DEV)], heads(clean[n])[~touched.to(DEV)]), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,H,dk,dv", [(1, 1, 1, 8, 8), (1, 3, 2, 8, 8), (2, 5, 2, 128, 128), (4, 20, 4, 16, 16), (3, 33, 3, 10, 10), (2, 100, 2, 33, 64),
                                         (2, 300, 4, 64, 64), (2, 300, 3, 128, 100), (1, 1500, 2, 128, 128), (1, 2000, 2, 24, 24)])
def test_16_bit_results_are_rounded_once(B, T, H, dk, dv, dtype):
    """Two terms of a 16-bit type leave 2^-15 (bf16: the first is cut, 2^-7 of the value, the second rounded, 2^-8 of that) or 2^-22 (fp16:
    2^-11 twice) of each weight and of each state element as it enters a product; a term of a result passes through one of them.
    fp16 is scaled to 2^14 by a bound, below 2^-14 its steps are 2^-24: 2^-39 of a bound that is far less than 2^16 times the
    magnitudes that are added up here.  Beside that the fp32 roundings as ever, and one rounding of the result."""
    c = make(B, T, H, dk, dv, dtype, B + 7 * T + dk)
    c["log_decay"] = torch.tensor([-0.125, -4e-4, -0.01, 0.0][:H], device=DEV)
    got, scale = run_all(c), dk ** -0.5
    want, mag = recurrence(c, scale), recurrence(c, scale, True)
    left = 2.0 ** -15 if dtype == torch.bfloat16 else 2.0 ** -22 + 2.0 ** -23
    n = (T + max(dk, dv)) + 16 + 2 * (T // 32 + 1)
    for name in ("o", "dq", "dk", "dv"):
        t = (n * U + 1.01 * left) * mag[name] + half(dtype) * want[name].abs() * 1.01 + tiny(dtype) + 1e-30
        d = (got[name].double() - want[name]).abs()
        assert (d <= t).all(), (name, (d / t).max().item())
