"""A small sequence model of state space blocks, trained and then served.

    python examples/state_space_block.py [--steps 150] [--channels 64] [--layers 2]

Each block takes what the block before it has put out and the residual stream, adds and norms them,
and projects the result to the halves of a row: values, which go through a short causal convolution,
and a gate.  A second projection of the convolved values gives the steps, inputs and outputs of a state
space scan, which the gate ends; a third leads back.  The model learns to add up one input feature
where a second one is on, and to forget where a third one is; then it runs prompts of unlike lengths
at once and goes on token by token, with the convolution's and the scan's states of all sequences in
pools, and the outputs are compared with those of the whole sequences in one pass.

Training uses thunderfft_amd.rms_norm, short_conv and state_scan (torch functions with gradients);
serving the calls on device buffers, whose shapes and buffers are kept.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import thunderfft_amd as thff  # noqa: E402

FEATURES, ORDER, WIDTH, EPS = 4, 16, 4, 1e-5
# The operators hold states and weights in float32, whatever torch's default type is; so do the values here.
FLOAT = dict(device="cuda", dtype=torch.float32)


class Model:
    def __init__(self, channels: int, layers: int, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(rows, cols):
            return (torch.randn(rows, cols, generator=gen, **FLOAT) / rows ** 0.5).requires_grad_()

        def leaf(v):
            return v.to(**FLOAT).contiguous().requires_grad_()

        self.channels = channels
        self.embed = matrix(FEATURES, channels)
        self.blocks = []
        for _ in range(layers):
            # Steps from a thousandth to a tenth; rates from one to ORDER.
            dt = torch.exp(torch.rand(channels, generator=gen, **FLOAT) * 4.6 - 6.9)
            self.blocks.append(dict(
                norm=leaf(torch.ones(channels)), w_in=matrix(channels, 2 * channels),
                taps=leaf(torch.randn(channels, WIDTH, generator=gen, **FLOAT) / WIDTH ** 0.5), bias=leaf(torch.zeros(channels)),
                w_state=matrix(channels, channels + 2 * ORDER), delta_bias=leaf(dt + torch.log(-torch.expm1(-dt))),
                log_a=leaf(torch.log(torch.arange(1, ORDER + 1, **FLOAT)).expand(channels, ORDER)),
                skip=leaf(torch.ones(channels)), w_out=matrix(channels, channels)))
        self.norm = leaf(torch.ones(channels))
        self.head = matrix(channels, 1)

    def parameters(self):
        return [self.embed, self.norm, self.head] + [p for b in self.blocks for p in b.values()]

    def __call__(self, features, lengths=None):
        """(outputs (batch, n, 1), the blocks' last states) of features (batch, n, FEATURES)."""
        c, states = self.channels, []
        stream = features @ self.embed
        more = torch.zeros_like(stream)
        for b in self.blocks:
            x, stream = thff.rms_norm(more, b["norm"], stream, EPS)
            inner = x @ b["w_in"]
            x, conv = thff.short_conv(inner[..., :c], b["taps"], b["bias"], lengths=lengths)
            rows = x @ b["w_state"]
            y, state = thff.state_scan(x, rows[..., :c], -torch.exp(b["log_a"]), rows[..., c:c + ORDER], rows[..., c + ORDER:],
                                       b["skip"], inner[..., c:], b["delta_bias"], lengths=lengths)
            more = y @ b["w_out"]
            states.append((conv, state))
        x, _ = thff.rms_norm(more, self.norm, stream, EPS)
        return x @ self.head, states


class Server:
    """Runs a trained model's tokens; each block has pools with the states of each slot."""

    def __init__(self, model: Model, slots: int, batch: int):
        self.model, self.batch, c = model, batch, model.channels
        self.pools = [(torch.zeros(slots, WIDTH - 1, c, **FLOAT), torch.zeros(slots, c, ORDER, **FLOAT)) for _ in model.blocks]
        self.rates = [-torch.exp(b["log_a"]) for b in model.blocks]
        self.conv = thff.ConvShape("float", batch, 1, c, WIDTH, x_stride=2 * c, states=slots)
        row = c + 2 * ORDER
        self.scan = thff.StateShape("float", batch, 1, c, ORDER, delta_stride=row, gate_stride=2 * c, b_stride=row, c_stride=row,
                                    states=slots)
        self.stream, self.normed, self.mixed, self.out = (torch.empty(batch, c, **FLOAT) for _ in range(4))
        self.inner, self.rows = torch.empty(batch, 2 * c, **FLOAT), torch.empty(batch, row, **FLOAT)

    def fill(self, slots, states):
        """Puts a prompt's last states into the slots."""
        for pools, last in zip(self.pools, states):
            for pool, state in zip(pools, last):
                pool[slots.long()] = state

    def norm(self, more, weight):
        """The norm of stream + more, the sums in the stream's place."""
        thff.ThunderFFT_rms_norm_async("float", more, weight, EPS, self.normed, self.batch, self.model.channels,
                                       d_residual=self.stream, d_sum=self.stream, stream=torch.cuda.current_stream())

    def token(self, features, slots):
        """One step of each sequence (batch, FEATURES); slots: int32, -1 for an empty place."""
        c, stream = self.model.channels, torch.cuda.current_stream()
        torch.mm(features, self.model.embed, out=self.stream)
        more = self.out.zero_()
        for b, (conv, state), rates in zip(self.model.blocks, self.pools, self.rates):
            self.norm(more, b["norm"])
            torch.mm(self.normed, b["w_in"], out=self.inner)
            thff.ThunderFFT_short_conv_async(self.conv, self.inner, b["taps"], b["bias"], self.mixed, d_state_in=conv,
                                             d_state_out=conv, d_slots=slots, stream=stream)
            torch.mm(self.mixed, b["w_state"], out=self.rows)
            thff.ThunderFFT_state_scan_async(self.scan, self.mixed, self.rows, rates, self.rows[:, c:], self.rows[:, c + ORDER:],
                                             self.normed, d_skip=b["skip"], d_gate=self.inner[:, c:],
                                             d_delta_bias=b["delta_bias"], d_state_in=state, d_state_out=state, d_slots=slots,
                                             stream=stream)
            more = torch.mm(self.normed, b["w_out"], out=self.out)
        self.norm(more, self.model.norm)
        return self.normed @ self.model.head


def sample(batch: int, n: int, gen):
    """Features and the sum to learn: of feature 0 where feature 1 is on, from where feature 2 was on last."""
    features = torch.randn(batch, n, FEATURES, generator=gen, **FLOAT)
    on, reset = features[..., 1] > 1.0, features[..., 2] > 1.7
    target, total = torch.empty(batch, n, **FLOAT), torch.zeros(batch, **FLOAT)
    for t in range(n):
        total = torch.where(reset[:, t], torch.zeros_like(total), 0.98 * total) + torch.where(on[:, t], features[:, t, 0], 0.0)
        target[:, t] = total
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
    ap.add_argument("--channels", type=int, default=64)
    ap.add_argument("--layers", type=int, default=2)
    args = ap.parse_args(argv)
    model = Model(args.channels, args.layers)
    losses = train(model, args.steps)
    worst = serve(model)
    print(f"token by token against whole sequences: largest difference {worst:.2e}")
    return losses, worst


if __name__ == "__main__":
    main()
