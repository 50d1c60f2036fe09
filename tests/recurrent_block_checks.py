"""The gated recurrent example's checks: its operators together, in training and token by token.  Run by
test_gpu_recurrent_block.py in a process that imports torch first, so that both libraries share one HIP runtime."""
import torch


def check_training_learns_and_decoding_agrees():
    from examples import recurrent_block as E

    torch.manual_seed(0)
    model = E.Model(width=64, blocks=2, dtype=torch.float32)
    losses = E.train(model, steps=60, length=64)
    # a model that knows the eight classes but not which one has a loss of log 8 = 2.08
    assert sum(losses[-5:]) / 5 < 1.5 < losses[0], (losses[0], losses[-5:])

    # The same sequence in one call and token by token.  Products of 64 terms and norms in 32 bits, summed in another
    # order: a relative error of some 2^-24 x 64 a block, on logits of a size of about 10.
    tokens = torch.randint(E.CLASSES, E.VOCABULARY, (3, 37), device="cuda")
    tokens[:, 0] = torch.arange(3, device="cuda")
    starts = torch.zeros(3, 37, 1, dtype=torch.bool, device="cuda")
    with torch.no_grad():
        whole = model.forward(tokens, starts)
    steps = E.decode(model, tokens)
    assert float((whole - steps).abs().max()) < 1e-3


def check_packed_documents_do_not_meet():
    """A row of two documents gives each the logits that it has alone."""
    from examples import recurrent_block as E

    model = E.Model(width=64, blocks=2, dtype=torch.float32, seed=3)
    tokens = torch.randint(0, E.VOCABULARY, (2, 40), device="cuda")
    starts = torch.zeros(2, 40, 1, dtype=torch.bool, device="cuda")
    starts[:, 0] = starts[:, 23] = True
    with torch.no_grad():
        packed = model.forward(tokens, starts)
        first = model.forward(tokens[:, :23], starts[:, :23])
        second = model.forward(tokens[:, 23:], starts[:, 23:])
    assert float((packed - torch.cat([first, second], 1)).abs().max()) < 1e-3


def check_gradients_against_differences():
    """The loss's slope along a direction between the gradient's and a random one, for every parameter, with dropout, against central differences: the
    difference's own error is the third derivative's (step^2) and the loss's rounding over the step (2^-24 / 1e-2)."""
    from examples import recurrent_block as E

    model = E.Model(width=32, blocks=2, dtype=torch.float32, seed=5)
    g = torch.Generator(device="cuda").manual_seed(4)
    tokens, answers, starts = E.documents(4, 48, g)

    def loss():
        logits = model.forward(tokens, starts, 0.1, seed=3, step=7)
        return torch.nn.functional.cross_entropy(logits.flatten(0, 1).double(), answers.flatten())

    loss().backward()
    for w in model.parameters():
        d = torch.randn(w.shape, device="cuda", generator=g)
        d = d / d.norm() + w.grad / w.grad.norm()
        d /= d.norm()
        slope = float((w.grad * d).sum())
        eps = 1e-2
        with torch.no_grad():
            w += eps * d
            up = float(loss().detach())
            w -= 2 * eps * d
            down = float(loss().detach())
            w += eps * d
        assert abs((up - down) / (2 * eps) - slope) < 2e-3 + 0.02 * abs(slope), (tuple(w.shape), slope, (up - down) / (2 * eps))


if __name__ == "__main__":
    for check in (check_training_learns_and_decoding_agrees, check_packed_documents_do_not_meet, check_gradients_against_differences):
        check()
        print(check.__name__, "ok", flush=True)
