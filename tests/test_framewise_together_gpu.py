"""Label scores, Muon, AdamW, embedding and alignment in one training, as the example has them: it runs, its gradients are those
of the same network in 64 bits, and what it reports fits together."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_example_runs_with_muon(cuda, dtype):
    from i6_native_ops_b200.framewise import example

    seen = []
    losses, (within, alone) = example.train("monophone", steps=3, dtype=dtype, state_bits=32, width=192, seqs=3, scale=0.2, muon=True, report=seen.append)
    assert len(losses) == 4 and all(x == x and 0 < x < 1e4 for x in losses)
    got = seen[0]
    inside = got.top_labels[..., 0] != example.IGNORE
    assert inside.any() and (got.entropy[inside] >= 0).all() and not got.entropy[~inside].any()
    best = got.top_log_probs[inside]
    assert (best[:, :-1] >= best[:, 1:]).all() and (got.log_probs[inside] <= best[:, 0]).all()
    # the output layer with the loss in it and the scores off its logits (which are rounded to the type) agree
    tol = 2 * 2.0**-8 * 40 if dtype == torch.bfloat16 else 1e-3
    assert abs(float(-got.log_probs[0, 0]) - within) < tol


def test_gradients_of_the_objective(cuda):
    """Cross entropy less an entropy bonus through ``label_scores``, float32, against torch's own 64-bit autograd: each of the
    few products is off by some K 2^-24 of its magnitudes (K = 96 and 48 here, values of order one), gradients by less than
    1e-4 of their largest."""
    from i6_native_ops_b200.framewise import example

    torch.manual_seed(3)
    F, D, V, B, T = 48, 96, 41, 3, 50
    torch.backends.cuda.matmul.allow_tf32 = False
    model = example.ContextModel(F, D, V, torch.float32, cuda)
    x = torch.randn(B, T, F, device=cuda)
    targets = torch.randint(0, V, (B, T), device=cuda, dtype=torch.int32)
    lens = torch.tensor([T, 31, 0], device=cuda, dtype=torch.int32)
    left = example.left_labels(targets)
    got = model.scores(x, left, targets, lens, top=2)
    (-got.log_probs.sum() - 0.1 * got.entropy.sum() + 0.2 * got.top_log_probs.sum()).backward()
    wide = {n: p.detach().double().requires_grad_() for n, p in model.named_parameters()}
    ok = torch.arange(T, device=cuda)[None] < lens[:, None]
    context = torch.where((ok & (left != example.IGNORE))[..., None], wide["context"][left.clamp(min=0).long()] * D**0.5, 0.0)
    lp = (torch.tanh(x.double() @ wide["inner.weight"].T + wide["inner.bias"] + context) @ wide["out.weight"].T + wide["out.bias"]).log_softmax(-1)
    H = -(lp.exp() * lp).sum(-1)
    nll = lp.gather(-1, targets.long()[..., None])[..., 0]
    best = lp.gather(-1, got.top_labels.clamp(min=0).long()).sum(-1)
    (torch.where(ok, -nll - 0.1 * H + 0.2 * best, 0.0)).sum().backward()
    for n, p in model.named_parameters():
        want = wide[n].grad
        assert float((p.grad.double() - want).abs().max()) < 1e-4 * float(want.abs().max()), n


def test_a_training_step_in_a_graph(cuda):
    """Forward, backward and both optimizers, captured and replayed, against the same steps in turn."""
    from i6_native_ops_b200.framewise import Muon, label_scores

    def model():
        torch.manual_seed(1)
        return torch.nn.Linear(160, 272, device=cuda), torch.nn.Linear(272, 51, device=cuda)

    x = torch.randn(4, 30, 160, device=cuda)
    t = torch.randint(0, 51, (4, 30), device=cuda)

    def step(layers, opt):
        for w in (p for m in layers for p in m.parameters()):
            w.grad = None
        got = label_scores(layers[1](torch.tanh(layers[0](x))), t, top=1)
        (-got.log_probs.mean() - 0.01 * got.entropy.mean()).backward()
        opt.step()

    eager = model()
    opt = Muon([eager[0].weight, eager[1].weight], lr=0.01)
    for _ in range(5):
        step(eager, opt)
    layers = model()
    opt = Muon([layers[0].weight, layers[1].weight], lr=0.01)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(layers, opt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(layers, opt)
    for _ in range(3):
        graph.replay()
    for a, b in zip(eager, layers):
        assert torch.equal(a.weight, b.weight)
