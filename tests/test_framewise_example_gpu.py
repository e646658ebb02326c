"""The operators together: a network trained on an alignment."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 8), (torch.bfloat16, 32)])
def test_training_on_an_alignment(cuda, dtype, bits):
    """From about log(classes) the loss falls: the left label and the scores tell the class of most frames.  A frame scored
    by itself has the loss it has in its batch."""
    from i6_native_ops_b200.framewise.example import train

    losses, (within, alone) = train("monophone", 30, dtype, bits, seqs=6, scale=0.4)
    assert all(math.isfinite(v) for v in losses)
    assert losses[-1] < 0.5 * losses[0]
    # the network before the loss is torch's, which may round differently at another batch size
    assert abs(within - alone) <= (1e-4 if dtype == torch.float32 else 0.1) * (1 + abs(within))


def test_the_step_against_torch(cuda):
    """One step's loss and gradients in 32 bits against torch's own operators in 64, to 2^-18 of the largest value."""
    from i6_native_ops_b200.framewise import label_embedding, linear_cross_entropy

    gen = torch.Generator(device="cuda").manual_seed(0)
    B, T, V, D = 4, 70, 500, 96
    kw = dict(device=cuda, generator=gen)
    table, out, b = torch.randn(V, D, **kw), torch.randn(V, D, **kw) / D**0.5, torch.randn(V, **kw)
    x, t = torch.randn(B, T, D, **kw), torch.randint(0, V, (B, T), **kw)
    lens = torch.tensor([70, 1, 0, 33], dtype=torch.int32, device=cuda)
    leaves = [v.clone().requires_grad_() for v in (table, out, b, x)]
    h = torch.tanh(leaves[3] + label_embedding(t, leaves[0], scale=2.0, seq_lens=lens))
    loss = linear_cross_entropy(h, leaves[1], t.roll(-1, 1), bias=leaves[2], seq_lens=lens).sum()
    got = torch.autograd.grad(loss, leaves)
    ref = [v.double().requires_grad_() for v in (table, out, b, x)]
    ok = torch.arange(T, device=cuda) < lens[:, None]
    h = torch.tanh(ref[3] + 2.0 * ref[0][t] * ok[..., None])
    z = h @ ref[1].T + ref[2]
    want_loss = torch.nn.functional.cross_entropy(z[ok], t.roll(-1, 1)[ok], reduction="sum")
    want = torch.autograd.grad(want_loss, ref)
    assert abs(float(loss.detach()) - float(want_loss.detach())) <= 2.0**-18 * abs(float(want_loss.detach()))
    for a, c in zip(got, want):
        assert float((a - c).abs().max()) <= 2.0**-18 * float(c.abs().max())
