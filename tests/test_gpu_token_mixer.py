"""layer_norm, decay_attention and MultiTensorAdamW together, as a causal token mixer uses them: training on clips through
autograd, and the same weights run one token at a time."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, D = 4, 48                       # heads, model width (heads of 12)


class Mixer(torch.nn.Module):
    """y = x + W_o decay_attention(W_qkv layer_norm(x)), then a layer norm."""

    def __init__(self, seed):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        p = lambda *s: torch.nn.Parameter(torch.randn(*s, generator=g) * s[-1] ** -0.5)
        self.w_qkv, self.w_o = p(3 * D, D), p(D, D)
        self.ln1_w, self.ln1_b = torch.nn.Parameter(torch.ones(D)), torch.nn.Parameter(torch.zeros(D))
        self.ln2_w, self.ln2_b = torch.nn.Parameter(torch.ones(D)), torch.nn.Parameter(torch.zeros(D))
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-2.0 - torch.arange(H, dtype=torch.float32))))

    def qkv(self, x):
        import noise_amd as na
        y = na.layer_norm(x, self.ln1_w, self.ln1_b)
        return (y @ self.w_qkv.t().to(x.dtype)).view(*x.shape[:-1], 3, H, D // H).unbind(-3)

    def out(self, x, o):
        import noise_amd as na
        return na.layer_norm(x + o.reshape(x.shape) @ self.w_o.t().to(x.dtype), self.ln2_w, self.ln2_b)

    def forward(self, x, state=None, lengths=None):
        import noise_amd as na
        o, end = na.decay_attention(*self.qkv(x), self.log_decay, state, lengths)
        return self.out(x, o), end

    @torch.no_grad()
    def step(self, x, state):
        import noise_amd as na
        return self.out(x, na.decay_attention_step(*self.qkv(x), self.log_decay, state))


def reference(params, x, target, lengths, log_decay):
    """Loss of the mixer and its gradients in 64 bits on the CPU, the attention by its recurrence."""
    P = {k: v.detach().double().cpu().requires_grad_(True) for k, v in params.items()}
    x = x.double().cpu()
    ln = lambda t, w, b: (t - t.mean(-1, keepdim=True)) * ((t - t.mean(-1, keepdim=True)) ** 2).mean(-1, keepdim=True).add(1e-6).rsqrt() * w + b
    q, k, v = (ln(x, P["ln1_w"], P["ln1_b"]) @ P["w_qkv"].t()).view(*x.shape[:-1], 3, H, D // H).unbind(-3)
    B, T = x.shape[:2]
    S, o = torch.zeros(B, H, D // H, D // H, dtype=torch.float64), []
    lam = log_decay.double().cpu().exp().view(1, H, 1, 1)
    for t in range(T):
        on = (t < lengths.cpu()).view(B, 1, 1, 1).double()
        S = torch.where(on > 0, lam * S + k[:, t, :, :, None] * v[:, t, :, None, :], S)
        o.append((q[:, t, :, :, None] * S).sum(-2) * (D // H) ** -0.5 * on[..., 0])
    y = ln(x + torch.stack(o, 1).reshape(B, T, D) @ P["w_o"].t(), P["ln2_w"], P["ln2_b"])
    live = (torch.arange(T)[None, :] < lengths.cpu()[:, None]).double()[..., None]
    loss = (((y - target.double().cpu()) * live) ** 2).sum() / live.sum()
    loss.backward()
    return loss.item(), {k: v.grad for k, v in P.items()}


def batch(seed, B=3, T=70):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, T, D, generator=g).to(DEV), torch.randn(B, T, D, generator=g).to(DEV),
            torch.tensor([T, 33, 5], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(bits):
    """Three optimizer steps; the gradients of each against 64 bits at the current weights.  Bound: fp32 sums of at most T (B T
    for the parameters) terms behind two normalisations; 2^-24 * 4 * (T + B T + 3 D) of the largest gradient."""
    import noise_amd as na
    m = Mixer(0).to(DEV)
    opt = na.MultiTensorAdamW(m.parameters(), lr=1e-3, state_bits=bits)
    for step in range(3):
        x, target, lengths = batch(step)
        live = (torch.arange(x.shape[1], device=DEV)[None, :] < lengths[:, None])[..., None]
        opt.zero_grad()
        y, _ = m(x, lengths=lengths)
        loss = (((y - target) * live) ** 2).sum() / live.sum()
        loss.backward()
        want, grads = reference(dict(m.named_parameters()), x, target, lengths, m.log_decay)
        eps = 2.0 ** -24 * 4 * (70 + 210 + 3 * D)
        assert abs(loss.item() - want) <= eps * abs(want)
        for n, p in m.named_parameters():
            assert (p.grad.double().cpu() - grads[n]).abs().max() <= eps * grads[n].abs().max(), n
        before = [p.detach().clone() for p in m.parameters()]
        opt.step()
        assert all((p - b).abs().max() > 0 for p, b in zip(m.parameters(), before))
    assert (opt.step_count == 3).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_streams_follow_the_clip(dtype):
    """A clip in one pass, and the same clip as a prefix followed by single tokens from the state that the prefix leaves.  Bound:
    in fp32 the sums' roundings as above; in bf16 the pass rounds its weights and states to bf16 on the way into the products and
    both round qkv, o and y: at most eight half steps (2^-8) of values of order 8 (normalised rows have rms 1)."""
    m = Mixer(1).to(DEV).eval()
    x = batch(9)[0].to(dtype)
    for p in (m.ln2_w, m.ln2_b):
        p.requires_grad_(False)
    with torch.no_grad():
        whole, _ = m(x)
        y, state = m(x[:, :40])
        outs = [y]
        for t in range(40, x.shape[1]):
            outs.append(m.step(x[:, t], state)[:, None])
    got = torch.cat(outs, 1)
    tol = 2.0 ** -24 * 8 * (70 + 3 * D) * 8 if dtype == torch.float32 else 8 * 2.0 ** -8 * 8
    assert (got.float() - whole.float()).abs().max() <= tol
    assert (got.float() - whole.float()).norm() <= (1e-5 if dtype == torch.float32 else 2.0 ** -6) * whole.float().norm()
