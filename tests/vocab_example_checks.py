"""The gated recurrent example's two ends, together as they are used: embedding, distillation and the choice of tokens.  Run by
test_gpu_vocab_example.py in a process that imports torch first, so that both libraries share one HIP runtime."""
import torch


def setup(seed=0, width=32, blocks=1):
    from examples import recurrent_block as E

    teacher, student = E.Model(width, 2, seed=seed, dtype=torch.float32), E.Model(width, blocks, seed=seed + 1, dtype=torch.float32)
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    tokens, answers, starts = E.documents(3, 40, g)
    with torch.no_grad():
        top, index = teacher.forward(tokens, starts).flatten(0, 1).topk(5)
    answers[0, :7] = -100
    index[3] = -1
    return E, student, tokens, answers.flatten(), starts, top, index


def plain_loss(logits, top, index, answers, temperature, weight):
    z = logits.double()
    p = torch.softmax(torch.where(index >= 0, top.double() / temperature, -torch.inf), 1).nan_to_num(0.0)
    soft = torch.log_softmax(z / temperature, 1).gather(1, index.clamp_min(0))
    first = (torch.xlogy(p, p) - p * soft).sum(1) * temperature ** 2
    second = torch.nn.functional.cross_entropy(z, answers, reduction="none", ignore_index=-100)
    return weight * first + (1 - weight) * second


def check_losses_and_their_gradients():
    """A training step's loss, and the gradients of the logits and of the tied embedding, against the same in 64 bits from plain
    operations on the same logits.  Losses of some 5 and gradients of at most 2, summed over 120 rows, 32 columns and 32 places in
    f32: relative errors of a few hundred roundings of 2^-24."""
    E, student, tokens, answers, starts, top, index = setup()
    for temperature, weight in ((2.0, 0.5), (1.0, 1.0), (3.0, 0.7)):
        logits = student.forward(tokens, starts).flatten(0, 1).detach().requires_grad_()
        loss = E.DistillLoss.apply(logits, index, top, answers, temperature, weight)
        want = plain_loss(logits, top, index, answers, temperature, weight)
        assert float((loss - want).abs().max()) < 300 * 2.0 ** -24 * 10, (temperature, weight)
        got, = torch.autograd.grad(loss.mean(), logits)
        ref, = torch.autograd.grad(want.mean(), logits)
        assert float((got - ref).abs().max()) < 300 * 2.0 ** -24 / len(answers) * 10
    table = torch.randn(E.VOCABULARY, 32, device="cuda", requires_grad=True)
    w = torch.randn(3, 40, 32, device="cuda")
    padded = torch.where(tokens == 5, -1, tokens)
    y = E.Embedding.apply(table, padded)
    plain = torch.where((padded >= 0)[..., None], table[padded.clamp_min(0)], 0.0)
    assert torch.equal(y, plain)
    got, = torch.autograd.grad((y * w).sum(), table)
    ref, = torch.autograd.grad((plain.double() * w).sum(), table)
    assert float((got - ref).abs().max()) < 120 * 2.0 ** -24 * 120


def check_the_gradient_against_differences():
    """The distillation loss's slope along a direction between the gradient's and a random one, for every parameter, against central
    differences: the difference's own error is the third derivative's (step^2) and the loss's rounding over the step."""
    E, student, tokens, answers, starts, top, index = setup(seed=4)

    def loss():
        return E.DistillLoss.apply(student.forward(tokens, starts).flatten(0, 1), index, top, answers, 2.0, 0.5).double().mean()

    loss().backward()
    g = torch.Generator(device="cuda").manual_seed(9)
    for w in student.parameters():
        d = torch.randn(w.shape, device="cuda", generator=g)
        d = d / d.norm() + w.grad / w.grad.norm()
        d /= d.norm()
        slope, eps = float((w.grad * d).sum()), 1e-2
        with torch.no_grad():
            w += eps * d
            up = float(loss().detach())
            w -= 2 * eps * d
            down = float(loss().detach())
            w += eps * d
        assert abs((up - down) / (2 * eps) - slope) < 2e-3 + 0.02 * abs(slope), (tuple(w.shape), slope, (up - down) / (2 * eps))


def check_a_student_trains():
    E, student, *_ = setup(seed=7)
    losses = E.distill(student, E.Model(32, 1, seed=8, dtype=torch.float32), steps=4, length=40)
    assert len(losses) == 4 and all(torch.isfinite(torch.tensor(losses)))


def check_generation():
    """Every token that is generated is the first of the highest of the plain form's adjusted logits, one step after the other."""
    E, student, tokens, *_ = setup(seed=11)
    prompt = tokens[:, :9]
    allowed = torch.ones(E.VOCABULARY, dtype=torch.bool, device="cuda")
    allowed[3::5] = False
    penalties = dict(repetition=1.3, presence=0.4, frequency=0.25)
    out = E.generate(student, prompt, 12, allowed, **penalties)
    assert out.shape == (3, 21) and torch.equal(out[:, :9], prompt)
    assert bool(allowed[out[:, 9:]].all())
    logits = E.decode(student, out)
    for t in range(9, 21):
        z = logits[:, t - 1].float()
        n = torch.zeros_like(z).scatter_add_(1, out[:, :t], torch.ones_like(out[:, :t], dtype=torch.float32))
        seen = torch.where(z > 0, z / 1.3, z * 1.3) - (0.25 * n + 0.4)
        z = torch.where(allowed, torch.where(n > 0, seen, z), -torch.inf)
        best = z.max(1).values
        assert bool((z.gather(1, out[:, t:t + 1])[:, 0] >= best - 2.0 ** -20 * 10).all())  # (frequency and the like: an ulp of 2^-24)


if __name__ == "__main__":
    for check in (check_losses_and_their_gradients, check_the_gradient_against_differences, check_a_student_trains, check_generation):
        check()
        print(check.__name__, "ok", flush=True)
