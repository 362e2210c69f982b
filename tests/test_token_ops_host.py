"""Argument checks of the token operators that need no GPU: what they refuse, before any launch."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    import noise_amd as na
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        na.layer_norm(x, torch.ones(8), torch.zeros(8))
    with pytest.raises(RuntimeError, match="GPU"):
        na.layer_norm_bwd(x, x, torch.zeros(2), torch.ones(2))
    with pytest.raises(RuntimeError, match="GPU"):
        na.MultiTensorAdamW([torch.nn.Parameter(x)])
    t = torch.zeros(1, 3, 2, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        na.decay_attention(t, t, t, torch.zeros(2))
    with pytest.raises(RuntimeError, match="GPU"):
        na.decay_attention_step(t[:, 0], t[:, 0], t[:, 0], torch.zeros(2), torch.zeros(1, 2, 8, 8))


def test_optimizer_arguments():
    import noise_amd as na
    p = [torch.nn.Parameter(torch.zeros(3))]
    with pytest.raises(ValueError, match="empty"):
        na.MultiTensorAdamW([])
    with pytest.raises(ValueError, match="state_bits"):
        na.MultiTensorAdamW(p, state_bits=16)
    for kw in (dict(lr=-1), dict(eps=-1e-8), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(weight_decay=-1), dict(lr=float("nan"))):
        with pytest.raises(ValueError, match="need lr"):
            na.MultiTensorAdamW(p, **kw)


def test_c_entry_points_refuse_bad_arguments():
    """Bad sizes, types and null pointers come back as errors: nothing is launched."""
    from noise_amd import _lib
    one = ctypes.c_void_p(16)
    for args, text in (((None, 8, None, None, 1e-6, one, None, None, 1, 8, 0, 0, None), "null"),
                       ((one, 8, None, None, 1e-6, one, None, None, 0, 8, 0, 0, None), "rows"),
                       ((one, 8, None, None, 1e-6, one, None, None, 1, 0, 0, 0, None), "rows"),
                       ((one, -8, None, None, 1e-6, one, None, None, 1, 8, 0, 0, None), "stride"),
                       ((one, 8, None, None, 1e-6, one, None, None, 1, 8, 3, 0, None), "type"),
                       ((one, 8, None, None, 1e-6, one, None, None, 1, 8, 1, 2, None), "type")):
        with pytest.raises(RuntimeError, match=text):
            _lib.call("noise_layer_norm_fwd", *args)
    with pytest.raises(RuntimeError, match="null"):
        _lib.call("noise_layer_norm_bwd", one, 8, one, 8, None, one, None, one, None, None, None, 1, 8, 0, 0, None)
    with pytest.raises(RuntimeError, match="slab"):
        _lib.call("noise_layer_norm_bwd", one, 8, one, 8, one, one, None, one, one, None, None, 1, 8, 0, 0, None)
    assert _lib.lib.noise_layer_norm_bwd_rows(10 ** 6, 64) == 1024 and _lib.lib.noise_layer_norm_bwd_rows(5, 64) == 5
    assert _lib.lib.noise_layer_norm_bwd_rows(10 ** 6, 1 << 20) == 64
    with pytest.raises(RuntimeError, match="bad argument"):
        _lib.call("noise_adamw_multi_begin", None, None, None, 1, 1e-3, 0.9, 0.99, None)
    import array
    st = array.array("l", [64, 8, 8] * 7)
    sp = ctypes.c_void_p(st.buffer_info()[0])
    low = array.array("l", [64, 7, 8] * 7)
    lp = ctypes.c_void_p(low.buffer_info()[0])

    def fwd(q=one, strides=sp, B=1, T=8, H=1, dk=8, dv=8, dtype=0):
        _lib.call("noise_decay_attn_fwd", q, one, one, one, strides, one, None, None, None, None, 1.0, B, T, H, dk, dv, dtype, None)

    def bwd(go=one, strides=sp, B=1, T=8, H=1, dk=8, dv=8, dtype=0):
        _lib.call("noise_decay_attn_bwd", go, one, one, one, one, one, one, strides, one, None, None, None, None, None, 1.0, B, T, H, dk, dv,
                  dtype, None)
    for f, first in ((fwd, "q"), (bwd, "go")):
        for kw, text in ((dict(B=0), "empty"), (dict(T=0), "empty"), (dict(H=0), "empty"), (dict(dk=0), "head sizes"), (dict(dk=129), "head sizes"),
                         (dict(dv=129), "head sizes"), (dict(dtype=3), "element type"), (dict(B=1 << 22, H=2), "pairs"), (dict(strides=lp), "token stride"),
                         (dict(strides=None), "null"), ({first: None}, "null"), (dict(T=100000), "workspace")):
            with pytest.raises(RuntimeError, match=text):
                f(**kw)
    for args, text in (((None, 1, 1, 8, 8, 0), "null"), ((one, 0, 1, 8, 8, 0), "head sizes"), ((one, 1, 1, 129, 8, 0), "head sizes"), ((one, 1, 1, 8, 8, 7), "element type")):
        with pytest.raises(RuntimeError, match=text):
            _lib.call("noise_decay_attn_step", args[0], one, one, sp, one, one, one, 1.0, *args[1:], None)
    assert _lib.lib.noise_decay_attn_workspace(1, 8, 1, 8, 8, 0, 0) == 0 and _lib.lib.noise_decay_attn_workspace(1, 100000, 1, 8, 8, 0, 1) > 0
    assert _lib.lib.noise_decay_attn_workspace(1, 8, 1, 200, 8, 0, 0) == 0
    q, l, i = array.array("Q", [64]), array.array("l", [4]), array.array("i", [0])
    a = lambda x: ctypes.c_void_p(x.buffer_info()[0])
    off = array.array("l", [0])
    tail = (one, one, None, one, None, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1.0, None)
    for pd, gd, bits, text in ((0, 0, 16, "32 bits"), (0, 0, 8, "32 bits"), (1, 2, 32, "type"), (3, 3, 32, "type"), (1, 0, 32, "type")):
        with pytest.raises(RuntimeError, match=text):
            _lib.call("noise_adamw_multi", a(q), a(q), a(l), a(off), a(i), 1, pd, gd, bits, *tail)
    for bad in (dict(off=array.array("l", [100])), dict(l=array.array("l", [-1])), dict(q=array.array("Q", [0]))):
        with pytest.raises(RuntimeError, match="tensor 0"):
            _lib.call("noise_adamw_multi", a(bad.get("q", q)), a(q), a(bad.get("l", l)), a(bad.get("off", off)), a(i), 1, 0, 0, 32, *tail)


@pytest.fixture
def on_cpu(monkeypatch):
    """The wrappers' own work on CPU tensors: calls of the library go to the list that this returns as (name, arguments) or, when
    `during` is set, to that function."""
    import contextlib
    from noise_amd import _lib

    class Calls(list):
        during = None

    calls = Calls()

    def call(name, *args, nbytes=0):
        calls.append((name, args))
        if calls.during is not None:
            calls.during(name, args)

    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "on_device", lambda *t: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream", lambda: ctypes.c_void_p(0))
    monkeypatch.setattr(_lib, "call", call)
    return calls


@pytest.mark.parametrize("form", ["step", "fwd", "bwd"])
def test_copies_live_until_the_kernel_is_launched(on_cpu, monkeypatch, form):
    """Every tensor whose address goes to a kernel is held until the call has returned, packed copies of strided arguments too:
    memory that is free before the launch can be handed out and written ahead of it by another thread on the same stream."""
    import weakref
    from noise_amd import decay_attn as da
    seen = []

    def ptr(t):
        if t is not None:
            seen.append(weakref.ref(t))
        return None if t is None else ctypes.c_void_p(t.data_ptr())

    dead = []
    on_cpu.during = lambda name, args: dead.extend(r for r in seen if r() is None)
    monkeypatch.setattr(da, "ptr", ptr)
    strided = lambda *s: torch.zeros(*s, 2)[..., 0]
    q, k, v = (strided(2, 3, 4, 8) for _ in range(3))
    g, state, lengths = strided(4), strided(2, 4, 8, 8), torch.zeros(2, 2, dtype=torch.int64)[:, 0]
    if form == "step":
        da.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state.contiguous())
    elif form == "fwd":
        da.decay_attention_fwd(q, k, v, g, state, lengths)
    else:
        da.decay_attention_bwd(v, q, k, v, g, state, lengths, d_state=state)
    assert len(on_cpu) == 1 and len(seen) >= 6 and not dead


def test_copies_of_the_older_wrappers_live_until_the_launch(on_cpu, monkeypatch):
    """The same for the inverse transform's backward pass, whose two copies would share memory if the first went before the second
    was made, the activity measure and the activity label."""
    import weakref
    from noise_amd import STFT, _lib, losses, mixer
    seen, dead, got = [], [], {}

    def ptr(t):
        if t is not None:
            seen.append(weakref.ref(t))
            got[t.data_ptr()] = t.is_contiguous()
        return None if t is None else ctypes.c_void_p(t.data_ptr())

    on_cpu.during = lambda name, args: dead.extend(r for r in seen if r() is None)
    monkeypatch.setattr(_lib, "ptr", ptr)
    monkeypatch.setattr(losses, "ptr", ptr)
    lm, ph = torch.zeros(2, 1, 5, 161).transpose(2, 3), torch.zeros(2, 5, 161).transpose(1, 2)
    stft = STFT(20, 320, 160, 320, "hann")
    d_lm = stft._inverse_bwd(torch.zeros(2, 1, 1, 640), torch.zeros(2, 1, 1, 640), lm, ph)
    assert len(on_cpu) == 1 and not dead and d_lm.shape == lm.shape and all(got.values())
    seen.clear()
    mixer.activity_batch(torch.zeros(800, 3, dtype=torch.float64).t())
    seen.clear()
    clean = torch.zeros(800, 3).t()
    monkeypatch.setattr(losses, "smooth_l1_loss", lambda *a, **k: 0.0)
    monkeypatch.setattr(losses, "multi_resolution_stft_loss", lambda *a, **k: 0.0)
    monkeypatch.setattr(losses, "_check_pair", lambda *a: None)
    losses.waveform_loss(clean, clean, torch.zeros(3))
    assert len(on_cpu) == 3 and not dead


def test_dual_tensors_are_refused(on_cpu):
    """Forward-mode differentiation: a result without a tangent would be read as a derivative of zero."""
    import torch.autograd.forward_ad as fwad
    import noise_amd as na
    x, w, s = torch.zeros(3, 8), torch.ones(8), torch.zeros(3)
    t, g, state, one = torch.zeros(1, 3, 2, 8), torch.zeros(2), torch.zeros(1, 2, 8, 8), torch.zeros(1, 2, 8)
    calls = [(na.layer_norm, (x, w, w)), (na.layer_norm_fwd, (x, w, w)), (na.layer_norm_bwd, (x, x, s, s, w)),
             (na.decay_attention, (t, t, t, g, state)), (na.decay_attention_fwd, (t, t, t, g, state)),
             (na.decay_attention_bwd, (t, t, t, t, g, state, None, 1.0, state)), (na.decay_attention_step, (one, one, one, g, state))]
    for f, args in calls:
        with fwad.dual_level():
            f(*args)                    # plain tensors inside a level: as ever
            done = len(on_cpu)
            for i, a in enumerate(args):
                if torch.is_tensor(a):
                    dual = fwad.make_dual(a, torch.ones_like(a))
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        f(*args[:i], dual, *args[i + 1:])
                    with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                        f(*args[:i], dual, *args[i + 1:])
            assert len(on_cpu) == done


def test_lengths_are_limited_before_they_are_narrowed(on_cpu):
    """int64 lengths beyond 32 bits mean what they say: all tokens, or none."""
    import noise_amd as na
    seen = []
    on_cpu.during = lambda name, args: seen.append(list((ctypes.c_int * 12).from_address(args[6 if name.endswith("fwd") else 9].value)))
    big = torch.iinfo(torch.int64)
    lengths = torch.tensor([2 ** 40, 2 ** 32, 2 ** 32 + 3, big.max, big.min, -2 ** 32 + 2, -1, 0, 3, 7, 8, 2 ** 31])
    t, g = torch.zeros(12, 7, 1, 8), torch.zeros(1)
    na.decay_attention_fwd(t, t, t, g, None, lengths)
    na.decay_attention_bwd(t, t, t, t, g, None, lengths)
    assert seen == [[min(max(n, 0), 7) for n in lengths.tolist()]] * 2


def test_decay_attention_entries_refuse_outputs_over_inputs():
    """Workgroups of one launch read what such an output would write: refused before any launch."""
    import array
    from noise_amd import _lib
    st = array.array("l", [64, 8, 8] * 7)
    sp = ctypes.c_void_p(st.buffer_info()[0])
    at = lambda n: ctypes.c_void_p(n)
    n = 4 * 2 * 8 * 8          # bytes of a state: one clip, two heads

    def fwd(state, end):
        _lib.call("noise_decay_attn_fwd", at(16), at(16), at(16), at(16), sp, at(16), None, state, end, None, 1.0, 1, 8, 2, 8, 8, 0, None)

    def bwd(state=None, d_end=None, d_state=None, ins=(16, 32, 48, 64), outs=(80, 96, 112)):
        _lib.call("noise_decay_attn_bwd", *map(at, ins), *map(at, outs), sp, at(16), None, state, d_end, d_state, None, 1.0, 1, 8, 2, 8, 8, 0, None)
    for other in (1 << 20, (1 << 20) + n - 4, (1 << 20) - n + 4):
        with pytest.raises(RuntimeError, match="share"):
            fwd(at(1 << 20), at(other))
        with pytest.raises(RuntimeError, match="shares"):
            bwd(d_end=at(1 << 20), d_state=at(other))
        with pytest.raises(RuntimeError, match="shares"):
            bwd(state=at(1 << 20), d_state=at(other))
    for i in range(4):
        for o in range(3):
            outs = [80, 96, 112]
            outs[o] = 16 * (i + 1)
            with pytest.raises(RuntimeError, match="over an input"):
                bwd(outs=tuple(outs))
    # neighbours are no overlap: these reach the workspace check of a shape cut into segments
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.call("noise_decay_attn_fwd", at(16), at(16), at(16), at(16), sp, at(16), None, at(1 << 20), at((1 << 20) + n // 2), None, 1.0, 1, 100000,
                  1, 8, 8, 0, None)


def test_a_parameter_as_log_decay(on_cpu):
    """A module may hold log_decay as a parameter and run without gradients; while gradients are recorded it is refused."""
    import noise_amd as na
    t, g = torch.zeros(1, 3, 2, 8), torch.nn.Parameter(torch.zeros(2))
    with pytest.raises(ValueError, match="no gradient"):
        na.decay_attention(t, t, t, g)
    assert not on_cpu
    with torch.no_grad():
        na.decay_attention(t, t, t, g)
    with torch.inference_mode():
        na.decay_attention(t, t, t, g)
    na.decay_attention(t, t, t, g.detach())
    assert [name for name, _ in on_cpu] == ["noise_decay_attn_fwd"] * 3


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints_of_other_parameter_lists_are_refused(on_cpu, bits):
    """Lists of equal totals in another order own other parts of the flat states; a checkpoint that lacks something, or holds a bad
    number, leaves the optimizer as it was."""
    import noise_amd as na
    make = lambda *sizes, **kw: na.MultiTensorAdamW([torch.nn.Parameter(torch.zeros(n)) for n in sizes], state_bits=bits, **kw)
    fill = lambda opt: [t.view(torch.uint8).fill_(17) for t in opt.state.values()] + [opt.step_count.fill_(5)]
    src = make(300, 1000, lr=0.5, betas=(0.5, 0.75), eps=0.25, weight_decay=0.125)
    fill(src)
    sd = src.state_dict()
    untouched = lambda o: (o.lr == 1e-4 and o.betas == (0.9, 0.999) and not o.step_count.any()
                           and not any(t.view(torch.uint8).any() for t in o.state.values()))
    for sizes in ((1000, 300), (301, 999)):       # both pad to 1536 values of two tensors
        other = make(*sizes)
        with pytest.raises(ValueError, match="other sizes"):
            other.load_state_dict(sd)
        assert untouched(other)
    for key in ("lr", "betas", "eps", "weight_decay", "step", "exp_avg", "state_bits"):
        twin = make(300, 1000)
        with pytest.raises(ValueError):
            twin.load_state_dict({k: v for k, v in sd.items() if k != key})
        assert untouched(twin)
    for bad in (dict(lr=-1.0), dict(betas=(0.5,)), dict(betas=(0.5, 1.0)), dict(eps=float("nan"))):
        twin = make(300, 1000)
        with pytest.raises(ValueError, match="need lr"):
            twin.load_state_dict({**sd, **bad})
        assert untouched(twin)
    for d in (sd, {k: v for k, v in sd.items() if k != "sizes"}):        # the sizes were not always kept
        twin = make(300, 1000)
        twin.load_state_dict(d)
        assert (twin.lr, twin.betas, twin.eps, twin.weight_decay) == (0.5, (0.5, 0.75), 0.25, 0.125) and (twin.step_count == 5).all()
        assert all((t.view(torch.uint8) == 17).all() for t in twin.state.values())


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
def test_buffers_are_fp32_whatever_the_default_type(on_cpu, default):
    """The kernels read and write the states and coefficients as fp32: in half the bytes they would leave them."""
    import noise_amd as na
    t, g, x = torch.zeros(2, 3, 2, 8), torch.zeros(2), torch.zeros(3, 8)
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        for bits in (32, 8):
            opt = na.MultiTensorAdamW([torch.nn.Parameter(torch.zeros(300, dtype=torch.float32))], state_bits=bits)
            assert opt._coef.dtype == torch.float32 and opt.step_count.dtype == torch.int64
            for k, v in opt.state.items():
                assert v.dtype == (torch.float8_e4m3fn if bits == 8 and not k.endswith("scale") else torch.float32), k
        for n in (0, 3):
            a = t[:, :n]
            assert na.decay_attention_fwd(a, a, a, g)[1].dtype == na.decay_attention_bwd(a, a, a, a, g)[3].dtype == torch.float32
            y = na.layer_norm_fwd(x[:n], x[0], x[1])
            assert [s.dtype for s in y] == [torch.float32] * 3
            assert [s.dtype for s in na.layer_norm_bwd(x[:n], x[:n], y[1], y[2])] == [torch.float32] * 3
    finally:
        torch.set_default_dtype(before)


def test_no_tokens_return_a_packed_state(on_cpu):
    """The state behind no token is a new packed tensor, ready for single tokens, whatever the strides of the one given."""
    import noise_amd as na
    t, g = torch.zeros(2, 0, 3, 8), torch.zeros(3)
    state = torch.arange(2 * 3 * 64, dtype=torch.float32).view(2, 3, 8, 8).transpose(2, 3)
    o, end = na.decay_attention_fwd(t, t, t, g, state)
    assert end.is_contiguous() and torch.equal(end, state) and end.data_ptr() != state.data_ptr()
    na.decay_attention_step(t.new_zeros(2, 3, 8), t.new_zeros(2, 3, 8), t.new_zeros(2, 3, 8), g, end)
    assert not na.decay_attention_fwd(t, t, t, g)[1].any()


def test_sizes_beyond_the_entry_points_numbers_are_refused(on_cpu):
    """A size that 32 bits cannot carry would arrive as another one; views of one value stand for the large tensors."""
    import noise_amd as na
    from noise_amd import _lib
    z = torch.zeros(())
    for shape in ((1, 2 ** 30 + 1, 1, 1), (1, 2 ** 32 + 5, 1, 1), (2 ** 22 + 1, 1, 1, 1), (2 ** 32 + 2, 1, 1, 1), (1, 1, 2 ** 32 + 1, 1)):
        t = z.expand(shape)
        with pytest.raises(ValueError, match="too many"):
            na.decay_attention_fwd(t, t, t, z.expand(shape[2]))
        with pytest.raises(ValueError, match="too many"):
            na.decay_attention_bwd(t, t, t, t, z.expand(shape[2]))
    for shape in ((2 ** 23 + 1, 1, 1), (2 ** 32 + 1, 1, 1), (1, 2 ** 32 + 3, 1)):
        t = z.expand(shape)
        with pytest.raises(ValueError, match="too many"):
            na.decay_attention_step(t, t, t, z.expand(shape[1]), z.expand(*shape, 1))
    for shape in ((2, 2 ** 24 + 1), (1, 2 ** 32 + 8), (2 ** 31, 4)):
        t = z.expand(shape)
        with pytest.raises(ValueError, match="rows of at most"):
            na.layer_norm_fwd(t)
        with pytest.raises(ValueError, match="rows of at most"):
            na.layer_norm_bwd(t, t, z.expand(shape[:-1]), z.expand(shape[:-1]))
    assert not on_cpu
    import array
    st = array.array("l", [1 << 31, 8, 8] * 7)
    one, sp = ctypes.c_void_p(16), ctypes.c_void_p(st.buffer_info()[0])
    assert _lib.lib.noise_decay_attn_workspace(1, (1 << 30) + 1, 1, 8, 8, 0, 0) == 0
    assert _lib.lib.noise_decay_attn_workspace(1, 1 << 30, 1, 8, 8, 0, 0) > 0
    with pytest.raises(RuntimeError, match="2.30 tokens"):
        rc = _lib.lib.noise_decay_attn_fwd(one, one, one, one, sp, one, None, None, None, None, 1.0, 1, (1 << 30) + 1, 1, 8, 8, 0, None)
        raise RuntimeError(f"{rc} {_lib.lib.noise_last_error().decode()}")


def test_step_output_over_other_arguments():
    """o may be q, k or v itself, row for row, but no part of the state nor a shifted piece of another argument.  What is allowed
    gets as far as the launch, which needs a GPU; nothing is launched here."""
    import array
    from noise_amd import _lib
    if torch.cuda.is_available():
        pytest.skip("addresses of no memory: for machines without a GPU")
    B, H, D = 2, 3, 8
    row, q, k, v, state = 4 * B * H * D, 1 << 20, 2 << 20, 3 << 20, 4 << 20

    def step(o, q=q, k=k, v=v, strides=(H * D, D) * 3, dk=D, B=B):
        st = array.array("l", strides)
        a = [ctypes.c_void_p(x) for x in (q, k, v, st.buffer_info()[0], 16, state, o)]
        _lib.call("noise_decay_attn_step", *a, 1.0, B, H, dk, D, 0, None)
    for o in (q, k, v, v + row, v - row, state - row, state + D * row):
        with pytest.raises(RuntimeError, match="no ROCm-capable device"):
            step(o)
    for o in (state, state + D * row - row, state + D * row - 4, state - 4, q + 4, k - 4, v + row - 4):
        with pytest.raises(RuntimeError, match="shares memory"):
            step(o)
    wide = (2 * H * D, 2 * D) + (H * D, D) * 2      # q with gaps: its rows go on behind a packed one's end
    for o in (q, q + row):
        with pytest.raises(RuntimeError, match="shares memory"):
            step(o, strides=wide)
    with pytest.raises(RuntimeError, match="shares memory"):
        step(q, dk=D - 1)
    for strides in ((5, D, 7, D, 9, D), (0, D) * 3):      # one stream: its stride says nothing
        with pytest.raises(RuntimeError, match="no ROCm-capable device"):
            step(q, strides=strides, B=1)


def test_a_step_that_cannot_run_leaves_the_step_counts(on_cpu):
    """A tensor beyond one launch is refused at construction, and a grad_scale that is no number before the counts advance; a
    number of another kind counts as one."""
    import numpy as np
    import noise_amd as na
    big = lambda n: torch.nn.Parameter(torch.empty(n, device="meta", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="at most"):
        na.MultiTensorAdamW([big(8), big((1 << 33) + 1)])
    na.MultiTensorAdamW([big(1 << 33)], state_bits=8)
    p, g = torch.nn.Parameter(torch.zeros(4)), torch.ones(4)
    opt = na.MultiTensorAdamW([p])
    for bad in (None, "x", torch.ones(2)):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            opt.step(grad_scale=bad, grads=[g])
        assert not on_cpu
    for scale in (torch.tensor(0.5), np.float32(0.5), 0.5):
        opt.step(grad_scale=scale, grads=[g])
        name, args = on_cpu[-1]
        assert name == "noise_adamw_multi" and type(args[-2]) is float and args[-2] == 0.5
