"""A recurrent layer of a language model on the gated delta rule, as it is trained and served.

The layer projects its input to queries, keys, values, decays, writing strengths and an output gate,
runs the gated delta rule over the sequence, normalises every head of the result times the activated
gate, and projects back. Training runs whole sequences with gradients; a prompt runs whole sequences
into a state; decoding runs one token at a time on that state, or on a pool of states.

    python examples/gated_delta_layer.py

trains a small model on a recall task (pairs of a key and a value token, then keys whose values it has
to name) and then decodes from a prompt, checking that prompt and decoding give what the whole
sequence gives. Needs an MI355X.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import fpscan_amd  # noqa: E402


class GatedDeltaLayer(torch.nn.Module):
    """(batch, seqlen, width) -> the same. `heads` value heads of head_dim, each group of heads /
    key_heads sharing a key head."""

    def __init__(self, width, heads, head_dim, key_heads=None, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.heads, self.head_dim = heads, head_dim
        self.key_heads = heads if key_heads is None else key_heads
        qk, v = self.key_heads * head_dim, heads * head_dim
        self.splits = [qk, qk, v]
        options = {"dtype": dtype, "device": device}
        # q, k and v are taken as slices of one projection; the norm's gate is a tensor of its own
        self.inward = torch.nn.Linear(width, sum(self.splits), bias=False, **options)
        self.gate = torch.nn.Linear(width, v, bias=False, **options)
        self.control = torch.nn.Linear(width, 2 * heads, bias=False, **options)
        self.outward = torch.nn.Linear(v, width, bias=False, **options)
        # decays of a head: exp(-softplus(z) rate), rates from 0.001 to 0.1
        rates = torch.exp(torch.linspace(-6.9, -2.3, heads, device=device))
        self.log_rate = torch.nn.Parameter(rates.log())
        self.weight = torch.nn.Parameter(torch.ones(v, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(v, device=device))

    def new_state(self, slots):
        """States of zero for `slots` sequences."""
        return torch.zeros(slots, self.heads, self.head_dim, self.head_dim,
                           device=self.log_rate.device)

    def _project(self, x):
        q, k, v = self.inward(x).split(self.splits, -1)
        decay, beta = self.control(x).chunk(2, -1)
        unit = torch.nn.functional.normalize
        q = unit(q.unflatten(-1, (self.key_heads, self.head_dim)), dim=-1)
        k = unit(k.unflatten(-1, (self.key_heads, self.head_dim)), dim=-1)
        v = v.unflatten(-1, (self.heads, self.head_dim))  # a view of the projection, taken as it is
        decay = -torch.nn.functional.softplus(decay.float()) * torch.exp(self.log_rate)
        return (q, k, v, decay.to(x.dtype), torch.sigmoid(beta)), self.gate(x)

    def _finish(self, out, gate):
        shape = gate.shape
        out = fpscan_amd.group_norm_channel_last(out.reshape(-1, 1, shape[-1]), self.heads, self.weight,
                                                 self.bias, gate=gate.reshape(-1, 1, shape[-1]))
        return self.outward(out.view(shape))

    def forward(self, x):
        """Whole sequences from states of zero, differentiable."""
        rule, gate = self._project(x)
        return self._finish(fpscan_amd.gated_delta(*rule), gate)

    @torch.no_grad()
    def prompt(self, x, state):
        """Whole sequences (or the next parts of them) from `state`, which is brought up to date."""
        rule, gate = self._project(x)
        return self._finish(fpscan_amd.gated_delta_forward(*rule, state=state), gate)

    @torch.no_grad()
    def step(self, x, state, slots=None):
        """The next tokens (batch, 1, width) of sequences whose states are state[slots]."""
        rule, gate = self._project(x)
        return self._finish(fpscan_amd.gated_delta_step(*rule, state=state, slots=slots), gate)


class RecallModel(torch.nn.Module):
    def __init__(self, tokens, width=128, heads=2, head_dim=64, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.embed = torch.nn.Embedding(tokens, width, dtype=dtype, device=device)
        self.layer = GatedDeltaLayer(width, heads, head_dim, dtype=dtype, device=device)
        self.head = torch.nn.Linear(width, tokens, bias=False, dtype=dtype, device=device)

    def forward(self, ids):
        x = self.embed(ids)
        return self.head(x + self.layer(x)).float()


def recall_batch(batch, pairs, keys, values, gen, device="cuda"):
    """Sequences k1 v1 k2 v2 .. of distinct keys (one token a pair: key * values + value), then every key
    again in another order; the answers are the values."""
    order = torch.stack([torch.randperm(keys, generator=gen)[:pairs] for _ in range(batch)])
    given = torch.randint(values, (batch, pairs), generator=gen)
    again = torch.stack([torch.randperm(pairs, generator=gen) for _ in range(batch)])
    ids = torch.cat([order * values + given, keys * values + order.gather(1, again)], 1)
    return ids.to(device), given.gather(1, again).to(device)


def train(steps=200, seed=0, verbose=True):
    keys, values, pairs = 32, 8, 16
    torch.manual_seed(seed)
    gen = torch.Generator().manual_seed(seed)
    model = RecallModel(keys * values + keys)
    optimiser = torch.optim.AdamW(model.parameters(), lr=4e-3, weight_decay=0.0)
    losses = []
    for step in range(steps):
        ids, answers = recall_batch(64, pairs, keys, values, gen)
        logits = model(ids)[:, pairs:, :values]
        loss = torch.nn.functional.cross_entropy(logits.flatten(0, 1), answers.flatten())
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
        if verbose and step % 20 == 0:
            print(f"step {step}: loss {float(loss.detach()):.3f}", flush=True)
    return model, [float(x) for x in torch.stack(losses).cpu()]


@torch.no_grad()
def decode_difference(model, seed=1):
    """The largest difference, over the largest value, between the layer's output for whole sequences
    and for a prompt in two parts followed by single tokens in a pool of states."""
    torch.manual_seed(seed)
    layer = model.layer
    x = torch.randn(3, 150, layer.inward.in_features, device="cuda").to(layer.inward.weight.dtype)
    whole = layer(x)
    state = layer.new_state(3)
    parts = [layer.prompt(x[:, :90], state), layer.prompt(x[:, 90:140], state)]
    pool, slots = layer.new_state(8), torch.tensor([6, 1, 3], dtype=torch.int32, device="cuda")
    pool[slots.long()] = state
    parts += [layer.step(x[:, t:t + 1], pool, slots) for t in range(140, 150)]
    return float((torch.cat(parts, 1) - whole).abs().max() / whole.abs().max())


if __name__ == "__main__":
    model, losses = train()
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f}")
    print(f"prompt and decoding against whole sequences: {decode_difference(model):.1e} of the largest value")
