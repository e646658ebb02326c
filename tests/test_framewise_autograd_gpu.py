"""What autograd has to know of the framewise operators: that the optimizer changed a tensor, what a graph keeps."""
import pytest
import torch
import torch.utils.checkpoint

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fw():
    import i6_native_ops_b200.framewise as m

    return m


def layer(cuda, dtype, B=3, T=40, V=90, D=64, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device=cuda, generator=gen)
    h = torch.randn(B, T, D, **kw).to(dtype).requires_grad_()
    w = (torch.randn(V, D, **kw) / D**0.5).to(dtype)
    t = torch.randint(0, V, (B, T), **kw)
    return h, w, t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_between_a_loss_and_its_gradients_is_an_error(fw, cuda, dtype, bits):
    """The gradients are formed from the weight that the loss was formed from: changed by the optimizer, it is refused, as
    one changed by torch is."""
    h, w, t = layer(cuda, dtype)
    w = torch.nn.Parameter(w)
    optimizer = fw.AdamW([w], lr=1e-2, betas=(0.9, 0.98), state_bits=bits)
    loss = fw.linear_cross_entropy(h, w, t).sum()
    square = (w * w).sum()  # torch's own product saves the weight as well
    w.grad = torch.ones_like(w)
    optimizer.step()
    for x in (loss, square):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            x.backward()
    # and after the step all is as usual
    fw.linear_cross_entropy(h, w, t).sum().backward()
    assert bool(h.grad.isfinite().all())


@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_moves_the_versions_of_what_it_writes(fw, cuda, bits):
    p = [torch.ones(300, device=cuda, dtype=torch.bfloat16), torch.ones(7, 5, device=cuda, dtype=torch.bfloat16)]
    g = [torch.ones_like(x) for x in p]
    master = [x.float() for x in p]
    if bits == 8:
        m, v = ([(torch.zeros(x.shape, device=cuda, dtype=kind), torch.zeros(-(-x.numel() // 256), device=cuda)) for x in p]
                for kind in (torch.int8, torch.uint8))
        states = [y for x in m + v for y in x]
    else:
        m, v = ([torch.zeros(x.shape, device=cuda) for x in p] for _ in range(2))
        states = m + v
    written, read = p + master + states, g
    before = [x._version for x in written], [x._version for x in read]
    fw.adamw_step(p, g, m, v, step=1, master=master, betas=(0.9, 0.98))
    assert all(x._version > n for x, n in zip(written, before[0]))
    assert all(x._version == n for x, n in zip(read, before[1]))
    # tensors without versions are written all the same
    with torch.inference_mode():
        q = torch.ones(300, device=cuda)
        m, v = torch.zeros(300, device=cuda), torch.zeros(300, device=cuda)
    fw.adamw_step([q], [torch.ones(300, device=cuda)], [m], [v], step=1)
    assert bool((q < 1).all())


@pytest.mark.parametrize("train", [False, True])
def test_forward_mode_derivatives_are_refused(fw, cuda, train):
    """There are none; a tangent is not lost in silence."""
    import torch.autograd.forward_ad as fwd

    h, w, t = layer(cuda, torch.float32)
    h, b = h.detach(), torch.zeros(90, device=cuda)

    def dual(x):
        return fwd.make_dual(x.detach().requires_grad_(train), torch.ones_like(x))

    with fwd.dual_level():
        for call in (lambda: fw.linear_cross_entropy(dual(h), w, t), lambda: fw.linear_cross_entropy(h, dual(w), t),
                     lambda: fw.linear_cross_entropy(h, w, t, bias=dual(b)), lambda: fw.label_embedding(t, dual(w))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        # of the incoming gradients
        for out, leaf in ((lambda x: fw.linear_cross_entropy(x, w, t), h), (lambda x: fw.label_embedding(t, x), w)):
            x = leaf.clone().requires_grad_()
            y = out(x)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, x, fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))
        # tensors without a tangent pass
        assert bool(fw.linear_cross_entropy(h, w, t).isfinite().all())
    for transform in (lambda: torch.func.jvp(lambda x: fw.linear_cross_entropy(x, w, t), (h,), (h,)),
                      lambda: torch.func.vmap(lambda x: fw.label_embedding(t, x))(w[None])):
        with pytest.raises(RuntimeError):
            transform()


def gradients(fw, h, w, t, twice=False):
    x, y = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = fw.linear_cross_entropy(x, y, t).sum()
    out = torch.autograd.grad(loss, (x, y), retain_graph=twice)
    return (out, torch.autograd.grad(loss, (x, y))) if twice else out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensor_hooks_see_all_that_is_kept(fw, cuda, dtype):
    """What the backward pass needs can be carried to the host and back; nothing of it stays on the device meanwhile."""
    h, w, t = layer(cuda, dtype, B=8, T=200, V=300, D=256)
    want = gradients(fw, h, w, t)
    with torch.autograd.graph.save_on_cpu():
        got = gradients(fw, h, w, t)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a graph whose tensors are on the host holds the loss and little else
    x, y = h.detach().requires_grad_(), w.detach().requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        loss = fw.linear_cross_entropy(x, y, t)
    assert torch.cuda.memory_allocated() - before <= loss.numel() * 4 + 65536
    loss.sum().backward()
    assert torch.equal(x.grad, want[0]) and torch.equal(y.grad, want[1])
    # the embedding's labels and lengths as well
    lens = torch.full((8,), 150, dtype=torch.int32, device=cuda)
    y.grad = None
    with torch.autograd.graph.save_on_cpu():
        out = fw.label_embedding(t, y, seq_lens=lens)
    out.backward(torch.ones_like(out))
    z = w.detach().requires_grad_()
    fw.label_embedding(t, z, seq_lens=lens).backward(torch.ones_like(out))
    assert torch.equal(y.grad, z.grad)


def test_what_hooks_give_back_is_looked_at(fw, cuda):
    h, w, t = layer(cuda, torch.float32)
    for spoil in (lambda x: x.cpu(), lambda x: x[:1], lambda x: x.double()):
        for call in (lambda: fw.linear_cross_entropy(h, w.requires_grad_(), t), lambda: fw.label_embedding(t, w.requires_grad_())):
            with torch.autograd.graph.saved_tensors_hooks(lambda x: x, spoil):
                out = call()
            with pytest.raises(RuntimeError, match="hooks"):
                out.sum().backward()


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoints(fw, cuda, reentrant):
    h, w, t = layer(cuda, torch.bfloat16)
    want = gradients(fw, h, w, t)
    x, y = h.detach().requires_grad_(), w.detach().requires_grad_()
    loss = torch.utils.checkpoint.checkpoint(lambda a, b: fw.linear_cross_entropy(a * 1, b, t), x, y, use_reentrant=reentrant)
    loss.sum().backward()
    assert torch.equal(x.grad, want[0]) and torch.equal(y.grad, want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_backward_passes_over_one_graph(fw, cuda, dtype):
    h, w, t = layer(cuda, dtype)
    first, second = gradients(fw, h, w, t, twice=True)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    x = h.detach().requires_grad_()
    loss = fw.linear_cross_entropy(x, w.detach(), t).sum()
    loss.backward()
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", [(3, 40, 90, 64), (2, 700, 1000, 300), (5, 300, 41, 256), (30, 400, 12001, 40)])
def test_gradients_are_nan_throughout_where_a_wait_ran_out(fw, cuda, dtype, sizes):
    """The mark that a wait ran out, the second word of what is kept, is set on the way from the forward to the backward
    pass: no finite value may be left, whatever CTA writes last."""
    B, T, V, D = sizes
    h, w, t = layer(cuda, dtype, B, T, V, D)
    h, w, b = h.detach().requires_grad_(), w.requires_grad_(), torch.zeros(V, dtype=dtype, device=cuda).requires_grad_()
    t[0, 3] = -100

    def mark(x):
        if x.dtype == torch.uint8:
            x = x.clone()
            assert int(x[:8].view(torch.int32)[0]) == B * T - 1 and int(x[:8].view(torch.int32)[1]) == 0
            x[:8].view(torch.int32)[1] = 1
        return x

    for _ in range(3):
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, mark):
            loss = fw.linear_cross_entropy(h, w, t, bias=b)
        for g in torch.autograd.grad(loss.sum(), (h, w, b)):
            assert bool(g.isnan().all())
