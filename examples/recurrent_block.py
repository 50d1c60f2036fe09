"""A small gated recurrent language model: training on packed documents, then decoding token by token.

PyTorch holds the parameters, the matrix products and the optimizer; between the products run this library's
operators, on the same memory (DLPack, no copies):

    embedding -> dropout -> per block: products of y give the recurrence's input, its gates and the output gate
                 h = gated_scan(input, gates, reset=document starts, kind="blend")
                 r, y = norm_residual(h, r, gate=output gate, ...)      # norm, gate, dropout, residual scale, next norm
              -> product with the embedding

The task needs the recurrence: every token of a document is to be answered with the document's first token.

    python examples/recurrent_block.py [--steps 200] [--width 128] [--blocks 2] [--length 96]
"""
import argparse
import os
import sys

import torch  # first, so that both libraries share its HIP runtime

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import musapy_amd as ms  # noqa: E402

CLASSES = 8  # first tokens; the others of a document come from the rest of the vocabulary
VOCABULARY = 32
DROPOUT = 0.1


def arr(t):
    return None if t is None else ms.from_dlpack(t.detach().contiguous())


def ten(a):
    return None if a is None else torch.from_dlpack(a)


class GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, reset):
        h, _ = ms.gated_scan(arr(x), arr(gate), reset=arr(reset), axis=1, kind="blend")
        h = ten(h)
        ctx.save_for_backward(x, gate, reset, h)
        return h

    @staticmethod
    def backward(ctx, dh):
        x, gate, reset, h = ctx.saved_tensors
        dx, dgate, _ = ms.gated_scan_grad(arr(dh), arr(x), arr(gate), arr(h), reset=arr(reset), axis=1, kind="blend")
        return ten(dx), ten(dgate), None


class NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, gate, w1, scale, w2, p, seed, offset):
        ctx.args = dict(p=p, seed=seed, offset=offset)
        r, y = ms.norm_residual(arr(x), arr(residual), gate=arr(gate), post_weight=arr(w1), scale=arr(scale), pre_weight=arr(w2),
                                **ctx.args)
        r, y = ten(r), ten(y)
        ctx.save_for_backward(x, r, gate, w1, scale, w2)
        return r, y

    @staticmethod
    def backward(ctx, dr, dy):
        x, r, gate, w1, scale, w2 = ctx.saved_tensors
        dx, dres, dgate, dw1, dscale, dw2 = ms.norm_residual_grad(
            arr(dr), arr(dy), arr(x), arr(r), gate=arr(gate), post_weight=arr(w1), scale=arr(scale), pre_weight=arr(w2), **ctx.args)
        return ten(dx), ten(dres), ten(dgate), ten(dw1), ten(dscale), ten(dw2), None, None, None


class Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset):
        ctx.args = (p, seed, offset)
        return ten(ms.dropout(arr(x), *ctx.args))

    @staticmethod
    def backward(ctx, dy):  # the same bits drop the same elements
        return ten(ms.dropout(arr(dy), *ctx.args)), None, None, None


class Model:
    def __init__(self, width, blocks, seed=0, dtype=torch.bfloat16):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape, std):
            return (torch.randn(shape, device="cuda", generator=g) * std).requires_grad_()

        def full(value):
            return torch.full((width,), value, device="cuda").requires_grad_()

        self.dtype, self.width = dtype, width
        self.embedding = weight(VOCABULARY, width, std=1.0)
        self.blocks = [{"products": weight(width, 3 * width, std=width ** -0.5), "bias": full(2.0), "post": full(1.0),
                        "scale": full(0.5), "pre": full(1.0)} for _ in range(blocks)]

    def parameters(self):
        return [self.embedding] + [w for b in self.blocks for w in b.values()]

    def products(self, b, y):
        """The recurrence's input and gates, and the output gate, of normed activations."""
        x, g, o = (y.flatten(0, -2) @ b["products"].to(self.dtype)).view(*y.shape[:-1], 3, self.width).unbind(-2)
        return x.contiguous(), (g + b["bias"].to(self.dtype)).contiguous(), o.contiguous()

    def logits(self, y):
        return (y.flatten(0, -2) @ self.embedding.to(self.dtype).t()).float().view(*y.shape[:-1], VOCABULARY) * self.width ** -0.5

    def forward(self, tokens, reset, p=0.0, seed=0, step=0):
        r = self.embedding[tokens]  # the residual stream stays in 32 bits
        y = r.to(self.dtype)
        if p > 0:
            y = Dropout.apply(y, p, seed, step * 64)
        for i, b in enumerate(self.blocks):
            x, g, o = self.products(b, y)
            h = GatedScan.apply(x, g, reset)
            r, y = NormResidual.apply(h, r, o, b["post"], b["scale"], b["pre"], p, seed, step * 64 + 1 + i)
        return self.logits(y)

    @torch.no_grad()
    def step(self, token, states):
        """Logits behind one more token of each sequence; the states are carried on in place of the sequence."""
        r = self.embedding[token][:, None]
        y = r.to(self.dtype)
        for i, b in enumerate(self.blocks):
            x, g, o = self.products(b, y)
            h, state = ms.gated_scan(arr(x), arr(g), arr(states[i]), axis=1, kind="blend")
            states[i] = ten(state)
            r, y = (ten(v) for v in ms.norm_residual(h, arr(r), gate=arr(o), post_weight=arr(b["post"]), scale=arr(b["scale"]),
                                                     pre_weight=arr(b["pre"])))
        return self.logits(y)[:, 0]


def documents(batch, length, generator):
    """Rows of documents of 8 to 32 tokens: (tokens, answers, document starts)."""
    tokens = torch.randint(CLASSES, VOCABULARY, (batch, length), device="cuda", generator=generator)
    starts = torch.zeros(batch, length, 1, dtype=torch.bool, device="cuda")
    answers = torch.empty_like(tokens)
    for b in range(batch):
        at = 0
        while at < length:
            n = int(torch.randint(8, 33, (1,), device="cuda", generator=generator))
            first = int(torch.randint(0, CLASSES, (1,), device="cuda", generator=generator))
            tokens[b, at], starts[b, at], answers[b, at:at + n] = first, True, first
            at += n
    return tokens, answers, starts


def train(model, steps, length, batch=8, report=None):
    generator = torch.Generator(device="cuda").manual_seed(1)
    optimizer = torch.optim.AdamW(model.parameters(), lr=5e-3, weight_decay=0.0)
    losses = []
    for step in range(steps):
        tokens, answers, starts = documents(batch, length, generator)
        logits = model.forward(tokens, starts, DROPOUT, seed=17, step=step)
        loss = torch.nn.functional.cross_entropy(logits.flatten(0, 1), answers.flatten())
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
        if report and (step + 1) % report == 0:
            print(f"step {step + 1}: loss {losses[-1]:.4f}", flush=True)
    return losses


@torch.no_grad()
def decode(model, tokens):
    """Logits of every position, one token at a time."""
    states = [torch.zeros(tokens.shape[0], model.width, device="cuda") for _ in model.blocks]
    return torch.stack([model.step(tokens[:, t], states) for t in range(tokens.shape[1])], 1)


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--steps", type=int, default=200)
    p.add_argument("--width", type=int, default=128)
    p.add_argument("--blocks", type=int, default=2)
    p.add_argument("--length", type=int, default=96)
    a = p.parse_args()
    model = Model(a.width, a.blocks)
    train(model, a.steps, a.length, report=max(1, a.steps // 10))
    generator = torch.Generator(device="cuda").manual_seed(2)
    tokens = torch.randint(CLASSES, VOCABULARY, (16, 24), device="cuda", generator=generator)
    tokens[:, 0] = torch.arange(16, device="cuda") % CLASSES
    answers = decode(model, tokens).argmax(-1)
    print(f"decoded token by token: {float((answers == tokens[:, :1]).float().mean()):.1%} of the answers right")


if __name__ == "__main__":
    main()
