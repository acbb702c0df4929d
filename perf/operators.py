"""Cases of the layer operators: the gated delta rule and the group norm that follows it.

Each case is one pass on tensors already on the GPU, in one of two forms that give the same
outputs: the plain form (elementary torch operations in 32 bits, rounded once at the end) and,
where `own` is true, this package's operators:

  delta_train   gated_delta, then its gradients for a given grad_out (a training step)
  delta_fill    gated_delta_forward with a state that is continued in place (a prompt)
  delta_step    gated_delta_step: a few tokens of every sequence, states in place (decoding)
  norm          group_norm_channel_last
  norm_train    the same, then its gradients for a given grad_out

The gated delta rule keeps, for every sequence and head, a (key_dim, value_dim) state S:

  S' = exp(log_decay[t]) S[t-1];  u = beta[t] (v[t] - k[t]^T S');  S[t] = S' + k[t] u^T
  out[t] = scale q[t]^T S[t]

q and k have `key_heads` heads, each shared by heads / key_heads value heads. Inputs are those of
such a layer: unit keys and queries, decays exp(-softplus(N(0,1)) * rate) with rates between
0.001 and 1, writing strengths sigmoid(N(0,1)), values and output gradients N(0,1).
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}

# steps per block of the plain form
BLOCK = 64
# steps between the states that the 64-bit gradients start again from
KEEP = 64


def _delta(op, dtype, batch, seqlen, key_heads, heads, key_dim, value_dim):
    return {"op": op, "dtype": dtype, "batch": batch, "seqlen": seqlen, "key_heads": key_heads,
            "heads": heads, "key_dim": key_dim, "value_dim": value_dim}


def _norm(op, dtype, batch, seqlen, dim, groups, gate):
    return {"op": op, "dtype": dtype, "batch": batch, "seqlen": seqlen, "dim": dim,
            "groups": groups, "gate": gate}


def listed():
    cases = [
        # the smallest training step, in fp32: width 256 as four heads of 64
        _delta("delta_train", "f32", 2, 256, 4, 4, 64, 64),
        # an ordinary layer of a language model: 8 sequences of 2048 steps, width 1024
        _delta("delta_train", "bf16", 8, 2048, 8, 8, 128, 128),
        # sizes that are not round: 3 sequences of 1000 steps, keys shared by two heads
        _delta("delta_train", "f16", 3, 1000, 4, 8, 72, 104),
        # the largest training step: 8 sequences of 16384 steps, width 1024
        _delta("delta_train", "bf16", 8, 16384, 8, 8, 128, 128),
        # a single prompt at the longest length
        _delta("delta_fill", "bf16", 1, 65536, 8, 8, 128, 128),
        # a few prompts of an odd length, keys shared by four heads
        _delta("delta_fill", "f16", 5, 777, 4, 16, 128, 128),
        # decoding for one user: one token of one sequence, where latency counts
        _delta("delta_step", "bf16", 1, 1, 8, 8, 128, 128),
        # decoding for many users: one token of 256 sequences
        _delta("delta_step", "bf16", 256, 1, 16, 32, 128, 128),
        # the norm of a layer's heads, token by token, times an activated gate
        _norm("norm_train", "bf16", 16384, 1, 1024, 8, True),
        # the norm over whole sequences, a call of few rows in fp32
        _norm("norm", "f32", 2, 256, 256, 32, False),
        # the same with sizes that are not round: groups of 97 channels
        _norm("norm_train", "f16", 3, 1000, 776, 8, False),
        # the largest norm: 8 sequences of 16384 steps, width 1024
        _norm("norm_train", "bf16", 8, 16384, 1024, 32, False),
    ]
    for c in cases:
        if c["op"].startswith("delta"):
            c["name"] = "{op}_{dtype}_b{batch}_l{seqlen}_h{key_heads}-{heads}_d{key_dim}-{value_dim}"
        else:
            c["name"] = "{op}_{dtype}_b{batch}_l{seqlen}_d{dim}_g{groups}"
        c["name"] = c["name"].format(**c)
    return cases


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["delta_train", "delta_train", "delta_fill", "delta_step", "norm",
                     "norm_train"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op.startswith("norm"):
        dim = 8 * _log(rng, 4, 256)
        groups = rng.choice([g for g in (1, 2, 4, 8, 16, 32, 64) if dim % g == 0 and dim // g >= 8])
        most = (1 << 27) // dim
        if rng.random() < 0.5:  # token by token
            return _norm(op, dtype, _log(rng, 1, min(most, 65536)), 1, dim, groups,
                         rng.random() < 0.5)
        batch = _log(rng, 1, 64)
        return _norm(op, dtype, batch, _log(rng, 2, min(16384, most // batch)), dim, groups,
                     rng.random() < 0.5)
    key_heads = _log(rng, 1, 16)
    heads = key_heads * rng.choice([1, 1, 2, 4])
    key_dim, value_dim = 8 * rng.randint(4, 16), 8 * rng.randint(4, 16)
    if rng.random() < 0.5:
        key_dim = value_dim = rng.choice([64, 128])
    # no more steps of heads than the largest case of the kind
    if op == "delta_step":
        batch = _log(rng, 1, min(512, 8192 // heads))
        return _delta(op, dtype, batch, _log(rng, 1, 4), key_heads, heads, key_dim, value_dim)
    most = (1 << 20 if op == "delta_train" else 1 << 19) // heads
    batch = _log(rng, 1, 8)
    seqlen = _log(rng, 1, min(16384 if op == "delta_train" else 65536, most // batch))
    return _delta(op, dtype, batch, seqlen, key_heads, heads, key_dim, value_dim)


# ------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """The case's tensors by name, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    B, L = case["batch"], case["seqlen"]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"].startswith("norm"):
        D = case["dim"]
        got = {"x": (randn(B, L, D) + 0.5 * randn(D)).to(dtype),
               "weight": 1 + 0.1 * randn(D), "bias": 0.1 * randn(D)}
        if case["gate"]:
            got["gate"] = randn(B, L, D).to(dtype)
        if case["op"].endswith("train"):
            got["grad_out"] = randn(B, L, D).to(dtype)
        return got

    Hk, H, Dk, Dv = case["key_heads"], case["heads"], case["key_dim"], case["value_dim"]

    def unit(x):
        return (x * torch.rsqrt((x * x).sum(-1, keepdim=True))).to(dtype)

    rate = torch.exp(math.log(1e-3) * torch.rand(H, generator=gen, device="cuda"))
    got = {"q": unit(randn(B, L, Hk, Dk)), "k": unit(randn(B, L, Hk, Dk)),
           "v": randn(B, L, H, Dv).to(dtype),
           "log_decay": (-torch.log1p(torch.exp(randn(B, L, H))) * rate).to(dtype),
           "beta": torch.sigmoid(randn(B, L, H)).to(dtype)}
    if case["op"] == "delta_train":
        got["grad_out"] = randn(B, L, H, Dv).to(dtype)
    else:
        got["state"] = randn(B, H, Dk, Dv) * Dk ** -0.5
    return got


LEAVES = {"delta_train": ("q", "k", "v", "log_decay", "beta"),
          "norm_train": ("x", "weight", "bias", "gate")}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["leaves"] = [n for n in LEAVES.get(case["op"], ()) if n in state]
    for name in state["leaves"]:
        state[name].requires_grad_()
    state["op"], state["groups"] = case["op"], case.get("groups")
    return state


# -------------------------------------------------------------------------------- pass
def run(state):
    op = state["op"]
    if op.startswith("norm"):
        out = (_own_norm if own else _plain_norm)(state)
    elif op == "delta_train":
        out = (_own_delta if own else _plain_delta)(state)
    else:
        return {"out": (_own_continued if own else _plain_continued)(state),
                "state": state["state"]}
    if not state["leaves"]:
        return {"out": out}
    grads = torch.autograd.grad(out, [state[n] for n in state["leaves"]], state["grad_out"])
    return {"out": out, **{"grad_" + n: g for n, g in zip(state["leaves"], grads)}}


def _own_delta(s):
    import fpscan_amd

    return fpscan_amd.gated_delta(s["q"], s["k"], s["v"], s["log_decay"], s["beta"])


def _own_continued(s):
    import fpscan_amd

    if s["op"] == "delta_step":
        return fpscan_amd.gated_delta_step(s["q"], s["k"], s["v"], s["log_decay"], s["beta"],
                                           s["state"])
    return fpscan_amd.gated_delta_forward(s["q"], s["k"], s["v"], s["log_decay"], s["beta"],
                                          state=s["state"])


def _own_norm(s):
    import fpscan_amd

    return fpscan_amd.group_norm_channel_last(s["x"], s["groups"], s["weight"], s["bias"],
                                              gate=s.get("gate"), activation="silu")


# ------------------------------------------------------------------------- plain forms
def _heads_first(x, heads):
    """(batch, seqlen, h, ...) in 32 bits as (batch, heads, seqlen, ...), shared heads repeated."""
    x = x.float().transpose(1, 2)
    if x.shape[1] != heads:
        x = x.repeat_interleave(heads // x.shape[1], 1)
    return x


def _blocks(x):
    """(batch, heads, seqlen, ...) in blocks of BLOCK steps, the last one filled with zeros."""
    B, H, L = x.shape[:3]
    n = -(-L // BLOCK)
    if n * BLOCK != L:
        x = torch.cat([x, x.new_zeros(B, H, n * BLOCK - L, *x.shape[3:])], 2)
    return x.reshape(B, H, n, BLOCK, *x.shape[3:])


def _plain_rule(s, S):
    """The gated delta rule from the state S, in blocks of steps: within a block the writes u solve
    a unit lower triangular system, whose inverse is a product of doublings (its strict part is
    nilpotent); from block to block only the state is handed on."""
    H = s["v"].shape[2]
    scale = s["q"].shape[-1] ** -0.5
    L = s["v"].shape[1]
    q, k, v, g, beta = (_blocks(_heads_first(s[n], H))
                        for n in ("q", "k", "v", "log_decay", "beta"))
    G = g.cumsum(-1)
    lower = torch.ones(BLOCK, BLOCK, dtype=torch.bool, device=v.device).tril()
    decay = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~lower, -math.inf))
    kt = k.transpose(-1, -2).contiguous()
    strict = (beta[..., None] * decay * (k @ kt)).tril(-1)
    inverse = torch.eye(BLOCK, device=v.device) - strict
    power, span = strict, 2
    while span < BLOCK:
        power = power @ power
        inverse = inverse + power @ inverse
        span *= 2
    u0 = inverse @ (beta[..., None] * v)
    w = inverse @ ((beta * torch.exp(G))[..., None] * k)
    scores = scale * decay * (q @ kt)
    from_state = scale * torch.exp(G)[..., None] * q
    end = G[..., -1:]
    writes = (kt * torch.exp(end - G)[..., None, :]).contiguous()
    keep = torch.exp(end)[..., None]
    states, us = [], []
    for c in range(v.shape[2]):
        u = u0[:, :, c] - w[:, :, c] @ S
        states.append(S)
        us.append(u)
        S = keep[:, :, c] * S + writes[:, :, c] @ u
    out = from_state @ torch.stack(states, 2) + scores @ torch.stack(us, 2)
    B, H, n = out.shape[:3]
    out = out.reshape(B, H, n * BLOCK, -1)[:, :, :L].transpose(1, 2)
    return out.to(s["v"].dtype).contiguous(), S


def _plain_delta(s):
    B, _, H, Dv = s["v"].shape
    zero = torch.zeros(B, H, s["k"].shape[-1], Dv, device=s["v"].device)
    return _plain_rule(s, zero)[0]


def _plain_steps(s, S):
    H = s["v"].shape[2]
    q, k, v, g, beta = (_heads_first(s[n], H) for n in ("q", "k", "v", "log_decay", "beta"))
    out = []
    for t in range(v.shape[2]):
        kt, qt = k[:, :, t, :, None], q[:, :, t, :, None]
        S = torch.exp(g[:, :, t, None, None]) * S
        u = beta[:, :, t, None] * (v[:, :, t] - (kt * S).sum(-2))
        S = S + kt * u[:, :, None]
        out.append((qt * S).sum(-2))
    return (torch.stack(out, 1) * q.shape[-1] ** -0.5).to(s["v"].dtype), S


def _plain_continued(s):
    out, S = (_plain_steps if s["op"] == "delta_step" else _plain_rule)(s, s["state"])
    s["state"].copy_(S)
    return out


def _plain_norm(s):
    B, L, D = s["x"].shape
    x = s["x"].float().reshape(B, L, s["groups"], -1)
    x = x - x.mean((1, 3), keepdim=True)
    x = x * torch.rsqrt((x * x).mean((1, 3), keepdim=True) + 1e-5)
    x = x.reshape(B, L, D) * s["weight"] + s["bias"]
    z = s["gate"].float() if "gate" in s else x
    act = z / (1 + torch.exp(-z))
    return (x * act if "gate" in s else act).to(s["x"].dtype)


# ------------------------------------------------------------------------ bytes, flops
def work(case):
    """What one pass cannot do without: every input read once and every output written once. A
    step of the rule decays the state, reads it twice and writes to it once: 7 operations for each
    of its values; its gradient, 16."""
    n = SIZE[case["dtype"]]
    if case["op"].startswith("norm"):
        e = case["batch"] * case["seqlen"] * case["dim"]
        gate = 1 if case["gate"] else 0
        if case["op"] == "norm":
            return {"bytes": (2 + gate) * e * n + 8 * case["dim"], "flops": 15 * e}
        return {"bytes": (4 + 2 * gate) * e * n + 16 * case["dim"], "flops": 45 * e}
    steps = case["batch"] * case["seqlen"]
    per_step = 2 * case["key_heads"] * case["key_dim"] + case["heads"] * (case["value_dim"] + 2)
    out = case["heads"] * case["value_dim"]
    cells = case["heads"] * case["key_dim"] * case["value_dim"]
    if case["op"] == "delta_train":
        return {"bytes": n * steps * (2 * per_step + 2 * out), "flops": 23 * steps * cells}
    return {"bytes": n * steps * (per_step + out) + 8 * case["batch"] * cells,
            "flops": 7 * steps * cells}


# ------------------------------------------------------------------- results in 64 bits
def _exact_norm(case, s):
    B, L, D = s["x"].shape
    G = case["groups"]
    n = L * (D // G)
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()

    def mean(t):
        """The mean over each sequence and group, for every channel."""
        m = t.sum(1).view(B, G, -1).sum(-1) / n
        return m.repeat_interleave(D // G, 1)[:, None]

    d = x - mean(x)
    r = 1 / torch.sqrt(mean(d * d) + 1e-5)
    h = d * r
    y = h * w + b
    z = s["gate"].double() if "gate" in s else y
    sig = torch.sigmoid(z)
    got = {"out": y * z * sig if "gate" in s else z * sig}
    if "grad_out" not in s:
        return got
    go = s["grad_out"].double()
    slope = sig * (1 + z * (1 - sig))
    gy = go * (z * sig if "gate" in s else slope)
    if "gate" in s:
        got["grad_gate"] = go * y * slope
    gh = gy * w
    got["grad_x"] = r * (gh - mean(gh) - h * mean(gh * h))
    got["grad_weight"], got["grad_bias"] = (gy * h).sum((0, 1)), gy.sum((0, 1))
    return got


def _exact_rule(case, s):
    """Step by step from the definition; the gradients by its adjoint, from states kept every KEEP
    steps."""
    L, H = case["seqlen"], case["heads"]
    shared = H // case["key_heads"]
    scale = case["key_dim"] ** -0.5

    def steps_first(x):
        x = x.double().movedim(1, 0)
        return x.contiguous()

    q, k = (steps_first(s[n]).repeat_interleave(shared, 2) for n in ("q", "k"))
    v, beta = steps_first(s["v"]), steps_first(s["beta"])[..., None]
    a = torch.exp(steps_first(s["log_decay"]))[..., None, None]
    out = torch.empty_like(v)
    S = s["state"].double() if "state" in s else v.new_zeros(*v.shape[1:3], k.shape[-1],
                                                             v.shape[-1])

    def read(x, S):
        return (x[..., None, :] @ S)[..., 0, :]

    def step(t, S):
        D = a[t] * S
        e = v[t] - read(k[t], D)
        return D, e, torch.addcmul(D, k[t][..., None], (beta[t] * e)[..., None, :])

    kept = []
    for t in range(L):
        if t % KEEP == 0:
            kept.append(S)
        S = step(t, S)[2]
        out[t] = scale * read(q[t], S)
    if case["op"] != "delta_train":
        return {"out": out.movedim(0, 1).contiguous(), "state": S}

    go = steps_first(s["grad_out"])
    gq, gk, gv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ga, gb = torch.empty_like(a), torch.empty_like(beta)
    R = torch.zeros_like(S)
    for c in reversed(range(len(kept))):
        part, S = [], kept.pop()
        for t in range(c * KEEP, min(L, (c + 1) * KEEP)):
            D, e, N = step(t, S)
            part.append((t, S, D, e, N))
            S = N
        for t, P, D, e, N in reversed(part):
            gq[t] = scale * (N @ go[t][..., None])[..., 0]
            R = torch.addcmul(R, q[t][..., None], (scale * go[t])[..., None, :])
            gu = read(k[t], R)
            gb[t] = (gu * e).sum(-1, keepdim=True)
            gv[t] = beta[t] * gu
            gk[t] = (R @ (beta[t] * e)[..., None] - D @ gv[t][..., None])[..., 0]
            R = torch.addcmul(R, k[t][..., None], gv[t][..., None, :], value=-1)
            ga[t] = (R * P).sum((-1, -2), keepdim=True)
            R = R * a[t]
        del part

    def back(x):
        return x.movedim(0, 1).contiguous()

    def heads(x):
        return back(x).unflatten(2, (H // shared, shared)).sum(3)

    return {"out": back(out), "grad_q": heads(gq), "grad_k": heads(gk), "grad_v": back(gv),
            "grad_log_decay": back((ga * a)[..., 0, 0]), "grad_beta": back(gb[..., 0])}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"].startswith("norm"):
        return _exact_norm(case, s)
    # about 60 microseconds of calls a step without gradients, 300 with them, and the states' memory
    cells = case["batch"] * case["heads"] * case["key_dim"] * case["value_dim"]
    train = case["op"] == "delta_train"
    if case["seqlen"] * ((300e-6 if train else 60e-6) + cells * (1.2e-10 if train else 2e-11)) > 18:
        return None
    return _exact_rule(case, s)
