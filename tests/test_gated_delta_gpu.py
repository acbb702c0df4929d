"""The gated delta rule (gated_delta, gated_delta_forward, gated_delta_step) against its definition in
float64 on the CPU, step by step, with gradients by autograd through those steps and by differences.

Tolerances are relative in the 2-norm, from the roundings a call makes: the result's own, at most u =
2^-8 (bf16), 2^-11 (fp16) or 2^-24 (fp32) of each value; of the operands, 2^-17 a value in the half
types and 2^-25 in fp32, of which a chunk's chain has about ten; for bf16 gradients the kept states
and errors, 2^-12 of a block's largest value, so up to 2^-10 of a typical one. Sums over n terms in
fp32 add about sqrt(n) 2^-24. The decays' gradients are differences of sums several times as large.
"""
import math

import pytest
import torch

import fpscan_amd

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device (MI355X)"),
]

DEVICE = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
OUT_TOL = {torch.float32: 3e-6, torch.float16: 2.0 ** -11 + 1e-4, torch.bfloat16: 2.0 ** -8 + 1e-4}
GRAD_TOL = {torch.float32: 6e-6, torch.float16: 2.0 ** -11 + 2e-4, torch.bfloat16: 2.0 ** -8 + 2.0 ** -10}
DECAY_TOL = {torch.float32: 4e-5, torch.float16: 2.0 ** -11 + 8e-4, torch.bfloat16: 2.0 ** -8 + 2.0 ** -8}
STATE_TOL = 3e-6
NAMES = ("q", "k", "v", "log_decay", "beta")


def inputs(B, L, Hk, H, Dk, Dv, dtype, seed=0, decay=0.1):
    gen = torch.Generator().manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)

    q, k = (torch.nn.functional.normalize(randn(B, L, Hk, Dk), dim=-1) for _ in range(2))
    g = -decay * torch.nn.functional.softplus(randn(B, L, H))
    t = {"q": q, "k": k, "v": randn(B, L, H, Dv), "log_decay": g, "beta": torch.sigmoid(randn(B, L, H))}
    return {n: x.to(dtype) for n, x in t.items()}


def rule(t, state=None, scale=None):
    """(out, last state) by the definition, in float64."""
    q, k, v, g, beta = (t[n].double() for n in NAMES)
    B, L, H, Dv = v.shape
    R = H // k.shape[2]
    q, k = q.repeat_interleave(R, 2), k.repeat_interleave(R, 2)
    S = torch.zeros(B, H, k.shape[-1], Dv, dtype=torch.float64) if state is None else state.double()
    out = []
    for i in range(L):
        S = torch.exp(g[:, i])[..., None, None] * S
        u = beta[:, i, :, None] * (v[:, i] - (k[:, i, :, :, None] * S).sum(-2))
        S = S + k[:, i, :, :, None] * u[:, :, None]
        out.append((q[:, i, :, :, None] * S).sum(-2))
    scale = k.shape[-1] ** -0.5 if scale is None else scale
    return torch.stack(out, 1) * scale, S


def gpu(t):
    return [t[n].to(DEVICE) for n in NAMES]


def check(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    norm = want.norm()
    err = (got - want).norm() / norm if norm > 0 else got.norm()
    assert err <= tol, f"{what}: {err:.3e} > {tol:.3e}"


SHAPES = [  # batch, seqlen, key heads, heads, key dim, value dim
    (1, 1, 1, 1, 64, 64), (2, 2, 1, 1, 8, 8), (1, 63, 2, 2, 64, 16), (2, 64, 1, 2, 128, 128),
    (1, 65, 2, 4, 72, 104), (3, 130, 1, 3, 40, 24), (1, 200, 9, 9, 128, 72), (1, 333, 1, 1, 128, 264),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, dtype):
    t = inputs(*shape, dtype)
    leaves = {n: x.double().requires_grad_() for n, x in t.items()}
    want, _ = rule(leaves)
    go = torch.randn(want.shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64).to(dtype)
    grads = torch.autograd.grad(want, [leaves[n] for n in NAMES], go.double(), allow_unused=True)
    on = [x.requires_grad_() for x in gpu(t)]
    out = fpscan_amd.gated_delta(*on)
    got = torch.autograd.grad(out, on, go.to(DEVICE))
    with torch.no_grad():
        check(fpscan_amd.gated_delta(*on), want, OUT_TOL[dtype], "out without gradients")
    check(out, want, OUT_TOL[dtype], "out")
    for n, x, y in zip(NAMES, got, grads):
        y = torch.zeros_like(leaves[n]) if y is None else y
        assert x.dtype == dtype
        check(x, y, DECAY_TOL[dtype] if n == "log_decay" else GRAD_TOL[dtype], "grad_" + n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_continued_state(shape, dtype):
    B, L, Hk, H, Dk, Dv = shape
    t = inputs(*shape, dtype, seed=3)
    s0 = torch.randn(B, H, Dk, Dv, generator=torch.Generator().manual_seed(4))
    want, last = rule(t, s0, scale=0.5)
    for call in (fpscan_amd.gated_delta_forward, fpscan_amd.gated_delta_step):
        state = s0.to(DEVICE)
        out = call(*gpu(t), state=state, scale=0.5)
        check(out, want, OUT_TOL[dtype], call.__name__)
        check(state, last, STATE_TOL, call.__name__ + " state")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1300, 1, 2, 64, 40), (2, 2049, 1, 1, 128, 72)])
def test_long_sequences_of_few_heads(shape, dtype):
    """Long enough, and few enough heads, that segments of the sequence are walked side by side."""
    B, L, Hk, H, Dk, Dv = shape
    t = inputs(*shape, dtype, seed=21, decay=0.02)
    t["log_decay"][:, 700] = -math.inf
    leaves = {n: x.double().requires_grad_() for n, x in t.items()}
    want, _ = rule(leaves)
    go = torch.randn(want.shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64).to(dtype)
    grads = torch.autograd.grad(want, [leaves[n] for n in NAMES], go.double())
    on = [x.requires_grad_() for x in gpu(t)]
    out = fpscan_amd.gated_delta(*on)
    check(out, want, OUT_TOL[dtype], "out")
    for n, x, y in zip(NAMES, torch.autograd.grad(out, on, go.to(DEVICE)), grads):
        y = torch.where(t[n] == -math.inf, 0, y) if n == "log_decay" else y
        check(x, y, DECAY_TOL[dtype] if n == "log_decay" else GRAD_TOL[dtype], "grad_" + n)
    s0 = torch.randn(B, H, Dk, Dv, generator=torch.Generator().manual_seed(22))
    want, last = rule(t, s0)
    state = s0.to(DEVICE)
    check(fpscan_amd.gated_delta_forward(*(x.detach() for x in on), state=state), want, OUT_TOL[dtype],
          "continued")
    check(state, last, STATE_TOL, "state")


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_of_a_prompt_and_tokens_make_the_whole(dtype):
    """A prompt in two parts, then token by token, is the whole sequence at once."""
    t = inputs(2, 150, 2, 4, 64, 64, dtype, seed=5)
    want, last = rule(t)
    on = gpu(t)
    state = torch.zeros(2, 4, 64, 64, device=DEVICE)
    parts = [fpscan_amd.gated_delta_forward(*(x[:, :100] for x in on), state=state),
             fpscan_amd.gated_delta_forward(*(x[:, 100:147] for x in on), state=state)]
    parts += [fpscan_amd.gated_delta_step(*(x[:, i:i + 1] for x in on), state=state)
              for i in range(147, 150)]
    check(torch.cat(parts, 1), want, OUT_TOL[dtype], "out")
    check(state, last, STATE_TOL, "state")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("none", [-math.inf, "lowest", -104.5])
def test_decays_of_zero_start_the_state_anew(dtype, none):
    """Packed documents: the state before a log_decay whose exp is 0 leaves no trace, and the results
    after it keep their precision; gradients do not cross it."""
    t = inputs(1, 200, 1, 2, 64, 64, dtype, seed=6)
    starts = [0, 7, 8, 64, 127, 150]
    value = torch.finfo(dtype).min if none == "lowest" else none
    t["log_decay"][:, starts] = value
    leaves = {n: x.double().requires_grad_() for n, x in t.items()}
    parts = [rule({n: x[:, a:b] for n, x in leaves.items()})[0]
             for a, b in zip(starts, starts[1:] + [200])]
    want = torch.cat(parts, 1)
    go = torch.randn(want.shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64).to(dtype)
    grads = torch.autograd.grad(want, [leaves[n] for n in NAMES], go.double())
    on = [x.requires_grad_() for x in gpu(t)]
    out = fpscan_amd.gated_delta(*on)
    check(out, want, OUT_TOL[dtype], "out")
    for n, x, y in zip(NAMES, torch.autograd.grad(out, on, go.to(DEVICE)), grads):
        if n == "log_decay":
            assert (x[:, starts] == 0).all()
            y = y.clone()
            y[:, starts] = 0
        check(x, y, DECAY_TOL[dtype] if n == "log_decay" else GRAD_TOL[dtype], "grad_" + n)
    state = torch.full((1, 2, 64, 64), 1e30, device=DEVICE)
    check(fpscan_amd.gated_delta_step(*(x.detach() for x in on), state=state), want, OUT_TOL[dtype],
          "steps")


@pytest.mark.parametrize("dtype", DTYPES)
def test_strong_decays_and_no_writes(dtype):
    """Decays of up to e^-40 a step, then steps that neither decay nor write (padding): the state
    stays as it is bit for bit in the recurrent form, and to its precision in the chunked one."""
    t = inputs(2, 130, 2, 2, 64, 32, dtype, seed=7, decay=20.0)
    want, _ = rule(t)
    check(fpscan_amd.gated_delta_forward(*gpu(t)), want, OUT_TOL[dtype], "strong decays")
    t["log_decay"].zero_()
    t["beta"].zero_()
    s0 = torch.randn(2, 2, 64, 32, generator=torch.Generator().manual_seed(8))
    state = s0.to(DEVICE)
    out = fpscan_amd.gated_delta_step(*gpu(t), state=state)
    assert torch.equal(state.cpu(), s0)
    check(out, rule(t, s0)[0], OUT_TOL[dtype], "reads")
    state = s0.to(DEVICE)
    fpscan_amd.gated_delta_forward(*gpu(t), state=state)
    assert torch.equal(state.cpu(), s0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_zero_beta_has_its_gradient(dtype):
    t = inputs(1, 100, 1, 2, 64, 64, dtype, seed=10)
    t["beta"][:, ::3] = 0
    leaves = {n: x.double().requires_grad_() for n, x in t.items()}
    want, _ = rule(leaves)
    grad = torch.autograd.grad(want.square().sum() / 2, leaves["beta"])[0]
    on = [x.requires_grad_() for x in gpu(t)]
    out = fpscan_amd.gated_delta(*on)
    got = torch.autograd.grad(out, on[4], want.detach().to(DEVICE, dtype))[0]
    check(got[:, ::3], grad[:, ::3], 2 * GRAD_TOL[dtype], "grad_beta at 0")


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_a_fused_projection_and_broadcasts(dtype):
    """q, k and v as slices of one tensor, v's batch and k's heads expanded (stride 0), log_decay and
    beta transposed; and a gradient that is one value for all (of a sum)."""
    B, L, H, D = 2, 70, 2, 64
    gen = torch.Generator().manual_seed(11)
    fused = (0.125 * torch.randn(B, L, H, 3 * D, generator=gen)).to(dtype)
    t = dict(zip("qkv", fused.split(D, -1)))
    t["k"] = t["k"][:, :, :1].expand(B, L, H, D)
    t["v"] = t["v"][:1].expand(B, L, H, D)
    for n in ("log_decay", "beta"):
        t[n] = (torch.rand(B, H, L, generator=gen) * (1 if n == "beta" else -0.2)).to(dtype).transpose(1, 2)
    leaves = {n: x.double().requires_grad_() for n, x in t.items()}
    want, _ = rule(leaves)
    grads = torch.autograd.grad(want.sum(), [leaves[n] for n in NAMES])
    on_fused = fused.to(DEVICE)
    on = dict(zip("qkv", on_fused.split(D, -1)))
    on["k"] = on["k"][:, :, :1].expand(B, L, H, D)
    on["v"] = on["v"][:1].expand(B, L, H, D)
    for n in ("log_decay", "beta"):
        on[n] = t[n].transpose(1, 2).contiguous().to(DEVICE).transpose(1, 2)
    on = [on[n].detach().requires_grad_() for n in NAMES]
    assert not on[0].is_contiguous() and on[1].stride(2) == 0 and on[2].stride(0) == 0
    out = fpscan_amd.gated_delta(*on)
    check(out, want, OUT_TOL[dtype], "out")
    for n, x, y in zip(NAMES, torch.autograd.grad(out.sum(), on), grads):
        check(x, y, DECAY_TOL[dtype] if n == "log_decay" else GRAD_TOL[dtype], "grad_" + n)


def test_gradients_against_differences():
    """The gradient along a random direction against the central difference of the float64 rule."""
    t = inputs(1, 70, 1, 2, 32, 16, torch.float32, seed=12)
    go = torch.randn(1, 70, 2, 16, generator=torch.Generator().manual_seed(13))
    on = [x.requires_grad_() for x in gpu(t)]
    got = torch.autograd.grad(fpscan_amd.gated_delta(*on), on, go.to(DEVICE))
    for i, n in enumerate(NAMES):
        d = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(14 + i), dtype=torch.float64)
        h = 1e-5
        f = [(rule({**t, n: t[n].double() + s * h * d})[0] * go).sum() for s in (1, -1)]
        want = float((f[0] - f[1]) / (2 * h))
        # the projection's own rounding: its terms' norm, not its value, which may cancel
        scale = float((got[i].double().cpu() * d).norm())
        assert abs(float((got[i].double().cpu() * d).sum()) - want) <= 1e-4 * scale, n


def test_slots_of_a_pool():
    t = inputs(4, 2, 2, 4, 64, 64, torch.bfloat16, seed=15)
    pool = torch.randn(7, 4, 64, 64, generator=torch.Generator().manual_seed(16))
    slots = [5, -1, 0, 7]
    state = pool.to(DEVICE)
    out = fpscan_amd.gated_delta_step(*gpu(t), state=state,
                                      slots=torch.tensor(slots, dtype=torch.int32, device=DEVICE))
    expect = pool.clone()
    for b, s in enumerate(slots):
        if not 0 <= s < 7:
            assert (out[b] == 0).all()
            continue
        want, last = rule({n: x[b:b + 1] for n, x in t.items()}, pool[s:s + 1])
        check(out[b:b + 1], want, OUT_TOL[torch.bfloat16], f"sequence {b}")
        check(state[s:s + 1], last, STATE_TOL, f"slot {s}")
        expect[s] = state[s].cpu()
    assert torch.equal(state.cpu(), expect)


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 values, and a sequence whose steps lie 16 MiB apart."""
    n = (1 << 18) + 8
    state = torch.empty(n, 1, 128, 128, device=DEVICE)
    state[-1].normal_()
    s0 = state[-1:].cpu()
    t = inputs(1, 1, 1, 1, 128, 128, torch.float32, seed=17)
    out = fpscan_amd.gated_delta_step(*gpu(t), state=state,
                                      slots=torch.tensor([n - 1], dtype=torch.int32, device=DEVICE))
    want, last = rule(t, s0)
    check(out, want, OUT_TOL[torch.float32], "out")
    check(state[-1:], last, STATE_TOL, "state")
    del state
    t = inputs(1, 300, 1, 1, 64, 64, torch.bfloat16, seed=18)
    wide = torch.empty(1, 300, 1, 1 << 23, dtype=torch.bfloat16, device=DEVICE)
    wide[..., -64:] = t["v"].to(DEVICE)
    on = gpu(t)
    on[2] = wide[..., -64:]
    check(fpscan_amd.gated_delta_forward(*on), rule(t)[0], OUT_TOL[torch.bfloat16], "wide rows")


def test_nan_stays_in_its_head_and_after():
    t = inputs(1, 200, 1, 2, 64, 64, torch.bfloat16, seed=19)
    want, _ = rule(t)
    t["v"][0, 140, 1, 3] = math.nan
    out = fpscan_amd.gated_delta_forward(*gpu(t))
    check(out[:, :, 0], want[:, :, 0], OUT_TOL[torch.bfloat16], "the other head")
    check(out[:, :128, 1], want[:, :128, 1], OUT_TOL[torch.bfloat16], "the chunks before")
    assert torch.isnan(out[0, 140:, 1, 3]).all()


def test_calls_repeat_bit_for_bit_and_run_on_other_streams():
    t = inputs(2, 300, 2, 4, 128, 128, torch.bfloat16, seed=20)
    on = [x.requires_grad_() for x in gpu(t)]

    def step():
        out = fpscan_amd.gated_delta(*on)
        return (out, *torch.autograd.grad(out, on, out.detach()))

    first = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    torch.cuda.synchronize()
    for a, b, c in zip(first, step(), other):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("shape", [(0, 5, 1, 1, 64, 64), (2, 0, 1, 1, 64, 64), (2, 5, 0, 0, 64, 64)])
def test_empty(shape):
    t = inputs(*shape[:4], *shape[4:], torch.float32) if shape[3] else {
        n: torch.zeros(2, 5, 0, *([64] if n in "qkv" else [])) for n in NAMES}
    on = [x.requires_grad_() for x in gpu(t)]
    out = fpscan_amd.gated_delta(*on)
    assert out.shape == t["v"].shape
    for x, g in zip(on, torch.autograd.grad(out.sum(), on)):
        assert g.shape == x.shape
    state = torch.ones(shape[0], shape[3], 64, 64, device=DEVICE)
    for call in (fpscan_amd.gated_delta_forward, fpscan_amd.gated_delta_step):
        assert call(*(x.detach() for x in on), state=state).shape == t["v"].shape
        assert (state == 1).all()


def test_refusals():
    def call(fn=fpscan_amd.gated_delta, **change):
        t = {n: x.to(DEVICE) for n, x in inputs(2, 5, 2, 4, 64, 64, torch.bfloat16).items()}
        extra = {n: change.pop(n) for n in list(change) if n not in NAMES}
        t.update({n: f(t[n]) for n, f in change.items()})
        return fn(*(t[n] for n in NAMES), **extra)

    with pytest.raises(RuntimeError, match="CUDA tensor"):
        call(q=lambda x: x.cpu())
    with pytest.raises(RuntimeError, match="dtype of v"):
        call(beta=lambda x: x.float())
    with pytest.raises(RuntimeError, match="float16 or bfloat16 or float32"):
        call(**{n: (lambda x: x.double()) for n in NAMES})
    with pytest.raises(RuntimeError, match="4-d"):
        call(v=lambda x: x[0])
    with pytest.raises(RuntimeError, match="shape of k"):
        call(q=lambda x: x[..., :32])
    with pytest.raises(RuntimeError, match="multiple of k's"):
        call(v=lambda x: x[:, :, :3], log_decay=lambda x: x[:, :, :3], beta=lambda x: x[:, :, :3])
    with pytest.raises(RuntimeError, match="multiple of 8"):
        call(q=lambda x: x[..., :60], k=lambda x: x[..., :60])
    with pytest.raises(RuntimeError, match="must have shape"):
        call(log_decay=lambda x: x[:, :4])
    with pytest.raises(RuntimeError, match="contiguous last axis"):
        call(v=lambda x: x.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(RuntimeError, match="16-byte vectors"):
        call(v=lambda x: torch.zeros(2, 5, 4, 68, dtype=x.dtype, device=DEVICE)[..., 4:])
    with pytest.raises(RuntimeError, match="must not overlap"):
        call(v=lambda x: x[:, :1].expand(2, 5, 4, 64))
    fwd, step = fpscan_amd.gated_delta_forward, fpscan_amd.gated_delta_step
    good = torch.zeros(2, 4, 64, 64, device=DEVICE)
    for fn in (fwd, step):
        with pytest.raises(RuntimeError, match="state must have shape"):
            call(fn, state=good[:1])
        with pytest.raises(RuntimeError, match="float32"):
            call(fn, state=good.half())
        with pytest.raises(RuntimeError, match="contiguous"):
            call(fn, state=good.transpose(2, 3))
        with pytest.raises(RuntimeError, match="no gradient"):
            call(fn, state=good.clone().requires_grad_())
        with pytest.raises(RuntimeError, match="out must"):
            call(fn, state=good, out=torch.zeros(2, 5, 4, 32, dtype=torch.bfloat16, device=DEVICE))
    with pytest.raises(RuntimeError, match="int32"):
        call(step, state=good, slots=torch.zeros(2, dtype=torch.int64, device=DEVICE))
    v = torch.zeros(2, 5, 4, 64, dtype=torch.bfloat16, device=DEVICE)
    with pytest.raises(RuntimeError, match="overlap"):
        call(fwd, v=lambda x: v, out=v)
