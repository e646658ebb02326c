"""Plain 64-bit forms of the operators of framewise training, and how far 32-bit or 16-bit results may be from them.

Bounds are derived, per value, not fitted.  u = 2^-24 is the rounding of one 32-bit operation, r that of the result's
type, half of its last place (``finfo.eps / 2``: 2^-24, bf16 2^-8).  A sum of K products formed in 32 bits, in any order and whether
rounded or cut off, is off by at most (K + c) 2u times the sum of the products' magnitudes; here the terms come 16 at
a time, so K / 16 + 16 steps count, and for f32 inputs in six parts of three bf16 each, which leave out 4u of a product.
"""
import torch

U = 2.0**-24


def kept(labels, lens, ignore):
    ok = labels != ignore
    if lens is not None:
        ok = ok & (torch.arange(labels.shape[-1], device=labels.device) < lens[:, None])
    return ok


def step_error(K, dtype):
    return (K / 16 + 16) * (6 if dtype == torch.float32 else 1) * 2 * U + 4 * U


def ce_reference(hidden, weight, bias, targets, lens, ignore, g):
    """Losses and gradients in 64 bits, and a bound of each."""
    f64 = torch.float64
    dtype, D, V = hidden.dtype, hidden.shape[-1], weight.shape[0]
    r = torch.finfo(dtype).eps / 2
    ok = kept(targets, lens, ignore).reshape(-1)
    x = hidden.detach().reshape(-1, D)[ok].to(f64)
    t = targets.reshape(-1)[ok].long()
    gg = g.reshape(-1)[ok].to(f64)
    w = weight.detach().to(f64)
    b = torch.zeros(V, dtype=f64, device=w.device) if bias is None else bias.detach().to(f64)
    z = x @ w.T + b
    rows = torch.arange(len(t), device=w.device)
    lse = z.logsumexp(1)
    p = (z - lse[:, None]).exp()
    nll = lse - z[rows, t]
    # a logit's error; +-inf biases are exact
    fin = torch.where(b.isfinite(), b.abs(), 0.0)
    dz = step_error(D, dtype) * (x.abs() @ w.abs().T) + 2 * U * ((x @ w.T).abs() + fin)
    # exp of a difference d: its rounding, that of its product with log2 e, the exponential's (2^-22)
    spread = torch.where(p > 0, (z - z.amax(1, keepdim=True)), 0.0).abs()
    de = dz + (4 * spread + 8) * U
    row = (p * de).sum(1) + (V / 32 + 64) * U
    dloss = row + dz[rows, t] + 4 * U * (nll.abs() + z.amax(1).abs() + z[rows, t].abs() + 1)
    q = p.clone()
    q[rows, t] -= 1
    q = q * gg[:, None]
    dq = (p * (de + row[:, None] + 4 * U)) * gg.abs()[:, None] + 4 * U * q.abs()
    held = q.abs() * (r if dtype != torch.float32 else 2 * U)  # q itself is rounded to bf16, or to three parts
    N = int(ok.numel())

    def back(v, shape):
        full = torch.zeros((N,) + tuple(v.shape[1:]), dtype=f64, device=v.device)
        full[ok] = v
        return full.reshape(shape)

    hid = q @ w
    wei = q.T @ x
    err = dq + held
    out = {
        "loss": (back(nll, targets.shape), back(dloss, targets.shape)),
        "hidden": (back(hid, hidden.shape),
                   back(err @ w.abs() + step_error(V, dtype) * (q.abs() @ w.abs()) + r * hid.abs(), hidden.shape)),
        "weight": (wei, err.T @ x.abs() + (step_error(len(t), dtype) + 64 * U) * (q.abs().T @ x.abs()) + r * wei.abs()),
        "bias": (q.sum(0), dq.sum(0) + (len(t) / 32 + 64) * U * q.abs().sum(0) + r * q.sum(0).abs()),
    }
    return out


def close(got, want, name=""):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    got = got.double()
    off = (got - value).abs()
    # infinities and NaN have to be the same
    same = (got == value) | (got.isnan() & value.isnan())
    bad = ~(same | (off <= bound + 1e-37))
    if bad.any():
        i = int((torch.where(bad, off / (bound + 1e-37), 0.0)).nan_to_num(posinf=1e30).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values off; worst {got.reshape(-1)[i]:.9g} "
                             f"for {value.reshape(-1)[i]:.9g}, bound {bound.expand_as(value).reshape(-1)[i]:.3g}")


def adamw_reference(p, g, m, v, step, lr, betas, eps, decay):
    f64 = torch.float64
    p, g, m, v = (x.to(f64) for x in (p, g, m, v))
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    p = p * (1 - lr * decay) - lr * (m / (1 - betas[0] ** step)) / ((v / (1 - betas[1] ** step)).sqrt() + eps)
    return p, m, v


def codes_of(x, top, block=256):
    """8-bit codes and steps of 32-bit values, by the definition."""
    n = x.numel()
    flat = torch.nn.functional.pad(x.reshape(-1), (0, -n % block)).reshape(-1, block)
    k = flat.abs().amax(1, keepdim=True) * torch.tensor(1.0 / (top * top), device=x.device)
    k = torch.where(k < 2.0**-120, torch.zeros_like(k), k)
    c = (flat.abs() * (torch.ones_like(k) / k)).sqrt().round().clamp(max=top)
    if top == 255:
        c = torch.where(flat > 0, c.clamp(min=1), c)
    c = torch.where(k > 0, c, torch.zeros_like(c)) * flat.sign()
    kind = torch.int8 if top == 127 else torch.uint8
    return c.reshape(-1)[:n].reshape(x.shape).to(kind), k.reshape(-1)


def values_of(codes, steps, block=256):
    n = codes.numel()
    c = torch.nn.functional.pad(codes.reshape(-1), (0, -n % block)).reshape(-1, block).float()
    return ((c * c.abs()) * steps[:, None]).reshape(-1)[:n].reshape(codes.shape)
