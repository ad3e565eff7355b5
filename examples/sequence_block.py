"""A small sequence model of pre-norm recurrence blocks, trained and then served.

    python examples/sequence_block.py [--steps 150] [--channels 128] [--layers 2]

Each block is  x + W_out scan(W_in norm(x)):  layer norm, one projection whose halves are the
recurrence's inputs and gates, the gated recurrence, and a projection back.  The model learns
to output a slowly decaying memory of one input feature that a second one switches (which a
model without state cannot); then it runs prompts of unlike lengths at once and goes on token by
token, with the states of all sequences in one pool, and the outputs are compared with those of
the whole sequences in one pass.

Training uses thunderfft_amd.layer_norm and thunderfft_amd.gated_scan (torch functions with
gradients); serving the calls on device buffers, whose shapes and buffers are kept.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import thunderfft_amd as thff  # noqa: E402

FEATURES = 4
# The operators hold states and weights in float32, whatever torch's default type is; so do the values here.
FLOAT = dict(device="cuda", dtype=torch.float32)


class Model:
    def __init__(self, channels: int, layers: int, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(rows, cols):
            return (torch.randn(rows, cols, generator=gen, **FLOAT) / rows ** 0.5).requires_grad_()

        self.channels = channels
        self.embed = matrix(FEATURES, channels)
        self.blocks = [dict(weight=torch.ones(channels, requires_grad=True, **FLOAT),
                            bias=torch.zeros(channels, requires_grad=True, **FLOAT),
                            w_in=matrix(channels, 2 * channels), w_out=matrix(channels, channels))
                       for _ in range(layers)]
        self.head = matrix(channels, 1)

    def parameters(self):
        return [self.embed, self.head] + [p for b in self.blocks for p in b.values()]

    def __call__(self, features, lengths=None):
        """(outputs (batch, n, 1), the blocks' last states) of features (batch, n, FEATURES)."""
        x, states = features @ self.embed, []
        for b in self.blocks:
            inner = thff.layer_norm(x, b["weight"], b["bias"]) @ b["w_in"]
            y, state = thff.gated_scan(inner[..., :self.channels], inner[..., self.channels:], lengths=lengths)
            x = x + y @ b["w_out"]
            states.append(state)
        return x @ self.head, states


class Server:
    """Runs a trained model's tokens; each block has a pool with a state for each slot."""

    def __init__(self, model: Model, slots: int, batch: int):
        self.model, self.batch, c = model, batch, model.channels
        self.pools = [torch.zeros(slots, c, **FLOAT) for _ in model.blocks]
        self.shape = thff.ScanShape("float", batch, 1, c, x_stride=2 * c, gate_stride=2 * c, states=slots)
        self.normed, self.mixed = torch.empty(batch, c, **FLOAT), torch.empty(batch, c, **FLOAT)
        self.inner = torch.empty(batch, 2 * c, **FLOAT)

    def fill(self, slots, states):
        """Puts a prompt's last states into the slots."""
        for pool, state in zip(self.pools, states):
            pool[slots.long()] = state

    def token(self, features, slots):
        """One step of each sequence (batch, FEATURES); slots: int32, -1 for an empty place."""
        c, stream = self.model.channels, torch.cuda.current_stream()
        x = features @ self.model.embed
        for b, pool in zip(self.model.blocks, self.pools):
            thff.ThunderFFT_layer_norm_async("float", x, b["weight"], b["bias"], 1e-5, self.normed, self.batch, c,
                                             stream=stream)
            torch.mm(self.normed, b["w_in"], out=self.inner)
            thff.ThunderFFT_gated_scan_async(self.shape, self.inner, self.inner[:, c:], self.mixed, d_state_in=pool,
                                             d_state_out=pool, d_slots=slots, stream=stream)
            x = x + self.mixed @ b["w_out"]
        return x @ self.model.head


def sample(batch: int, n: int, gen):
    """Features and the memory to learn: it takes up feature 0 where feature 1 is on, and decays."""
    features = torch.randn(batch, n, FEATURES, generator=gen, **FLOAT)
    on = (features[..., 1] > 1.0).float()
    target, memory = torch.empty(batch, n, **FLOAT), torch.zeros(batch, **FLOAT)
    for t in range(n):
        memory = torch.where(on[:, t] > 0, features[:, t, 0], 0.97 * memory)
        target[:, t] = memory
    return features, target.unsqueeze(2)


def train(model: Model, steps: int, batch: int = 16, n: int = 100, seed: int = 1):
    """The mean squared errors of the steps."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    data = [sample(batch, n, gen) for _ in range(8)]
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for step in range(steps):
        features, target = data[step % len(data)]
        outputs, _ = model(features)
        loss = (outputs - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if step % 25 == 0 or step == steps - 1:
            print(f"step {step:4d}  mean squared error {losses[-1]:.4f}", flush=True)
    return losses


@torch.no_grad()
def serve(model: Model, lengths=(40, 1, 77, 13), tokens: int = 24, seed: int = 2):
    """The largest difference between tokens served one by one and whole sequences."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    batch, most = len(lengths), max(lengths)
    features = torch.randn(batch, most + tokens, FEATURES, generator=gen, **FLOAT)
    ends = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    # Prompts of unlike lengths in one pass; what lies past an end reaches no state.
    _, states = model(features[:, :most].contiguous(), ends)
    server = Server(model, slots=2 * batch, batch=batch + 1)
    slots = torch.arange(batch, dtype=torch.int32, device="cuda") * 2 + 1
    server.fill(slots, states)
    slots = torch.cat([slots, torch.full((1,), -1, dtype=torch.int32, device="cuda")])  # an empty place
    rows, worst = torch.arange(batch, device="cuda"), 0.0
    for step in range(tokens):
        now = torch.cat([features[rows, ends.long() + step], features.new_zeros(1, FEATURES)])
        served = server.token(now, slots)[:batch]
        for b, length in enumerate(lengths):
            whole, _ = model(features[b:b + 1, :length + step + 1].contiguous())
            worst = max(worst, float((whole[0, -1] - served[b]).abs()))
    return worst


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=150)
    ap.add_argument("--channels", type=int, default=128)
    ap.add_argument("--layers", type=int, default=2)
    args = ap.parse_args(argv)
    model = Model(args.channels, args.layers)
    losses = train(model, args.steps)
    worst = serve(model)
    print(f"token by token against whole sequences: largest difference {worst:.2e}")
    return losses, worst


if __name__ == "__main__":
    main()
