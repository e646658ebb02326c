"""More operators of framewise training whose speed counts: what a program reads off a distribution over the
classes that is in memory, and the optimizer step of the hidden layers' matrices
(``i6_native_ops_b200.framewise``).

A case is a dict of

  op      ``scores`` (``label_scores``: log probabilities of given labels, entropies and the best alternatives),
          ``orth`` (``orthogonalize``: matrices to the nearest orthogonal ones by Newton-Schulz products),
          ``muon`` (``muon_step``: momentum, orthogonalisation and update of all matrices of a model)
  entry   ``score`` (the forward pass alone), ``train`` (and its gradients), ``step``
  dtype   ``f32`` or ``bf16``, of logits, matrices, parameters and gradients
  B T     ``scores``: sequences and positions of the padded batch, ``tlo`` the shortest length drawn
  V       ``scores``: classes; ``top`` alternatives; ``mask`` the share of classes that are impossible (-inf);
          ``skip`` the share of positions inside the sequences that are left out (the ignored label)
  M N     ``orth``: rows and columns of ``count`` matrices
  D       ``muon``: width of a model of ``layers`` layers of two matrices each

Inputs are synthetic and drawn from a seed.  Where ``own`` is false, ``run`` computes the operators in
elementary steps, in 32 bits.
"""
import math

import torch

own = False

IGNORE = -100  # the label of positions that are left out
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, BETA, DECAY = 0.02, 0.95, 0.01


def scores(name, entry, dtype, B, T, tlo, V, top, skip=0.0, mask=0.0):
    return {"name": name, "op": "scores", "entry": entry, "dtype": dtype, "B": B, "T": T, "tlo": tlo, "V": V, "top": top,
            "skip": skip, "mask": mask}


def orth(name, dtype, count, M, N):
    return {"name": name, "op": "orth", "entry": "score", "dtype": dtype, "count": count, "M": M, "N": N}


def muon(name, dtype, layers, D):
    return {"name": name, "op": "muon", "entry": "step", "dtype": dtype, "layers": layers, "D": D}


def listed():
    return [
        # the next label of eight hypotheses with its eight alternatives: one position each, the smallest call
        scores("scores_next_label", "score", "f32", 8, 1, 1, 10025, 8),
        # the same for the hypotheses of a large beam, some classes ruled out, in 16 bits
        scores("scores_beam", "score", "bf16", 256, 1, 1, 10025, 16, mask=0.1),
        # held-out frames of a lattice system, an odd length: how sure the model is of its alignment
        scores("scores_heldout", "score", "f32", 8, 1777, 1000, 5000, 4),
        # the scores of a whole triphone batch, those that fbw and the alignment take: the largest
        scores("scores_triphone", "score", "f32", 64, 1500, 1200, 12001, 8),
        # labels of a large vocabulary: likelihood and an entropy bonus, in 16 bits
        scores("scores_bpe_train", "train", "bf16", 256, 100, 20, 10025, 0),
        # frames of a triphone system trained on its alignment and five alternatives, some frames left out
        scores("scores_triphone_train", "train", "f32", 17, 1499, 1200, 12001, 5, skip=0.05),
        # one update of a small layer: launches and the host's time are everything
        orth("orth_one", "bf16", 1, 256, 64),
        # matrices of sizes that divide nothing, in 32 bits
        orth("orth_odd", "f32", 6, 500, 2001),
        # a small model's step, in 32 bits
        muon("muon_small", "f32", 2, 64),
        # an encoder of medium width in 16 bits
        muon("muon_encoder", "bf16", 8, 512),
        # the same width class in 32 bits, sizes that are no powers of two
        muon("muon_encoder_f32", "f32", 6, 500),
        # a large model in 16 bits
        muon("muon_large", "bf16", 4, 2048),
    ]


def draw(rng):
    """A case of the listed ranges, sizes spread over their logarithm."""

    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["f32", "bf16"])
    op = rng.choice(["scores", "scores", "orth", "muon"])
    if op == "muon":
        return {"op": op, "entry": "step", "dtype": dtype, "layers": rng.randint(1, 6),
                "D": 64 * spread(1, 16) if rng.random() < 0.5 else spread(20, 1100)}
    if op == "orth":
        M, N = spread(1, 2048), spread(1, 4096)
        count = max(1, min(spread(1, 24), (1 << 25) // (M * N)))
        return {"op": op, "entry": "score", "dtype": dtype, "count": count, "M": M, "N": N}
    V = spread(41, 12001)
    B = spread(1, 256)
    T = max(1, min(spread(1, 1500), 96000 // B))
    entry = rng.choice(["score", "train"])
    if entry == "train":
        T = max(1, min(T, 300_000_000 // (B * V)))
    return {"op": "scores", "entry": entry, "dtype": dtype, "B": B, "T": T, "tlo": rng.randint(0, T), "V": V,
            "top": min(rng.choice([0, 1, spread(2, 16), 32]), V // 4), "skip": rng.choice([0.0, 0.02, 0.3]),
            "mask": rng.choice([0.0, 0.0, 0.15])}


# ------------------------------------------------------------------------------------------------ inputs


def shapes(case):
    """A layer's two matrices: to four times the width and back."""
    D = case["D"]
    return [(4 * D, D), (D, 4 * D)] * case["layers"]


def update(shape, kw):
    """What a gradient looks like: some directions far stronger than the others, rows of their own sizes, noise."""
    m, n = shape[-2:]
    rank = max(1, min(m, n) // 8)
    left, right = torch.randn(*shape[:-1], rank, **kw), torch.randn(*shape[:-2], rank, n, **kw)
    left *= torch.logspace(0, -1.5, rank, device="cuda")
    rows = (0.7 * torch.randn(*shape[:-1], 1, **kw)).exp()
    return (left @ right / math.sqrt(rank) + 0.5 * torch.randn(shape, **kw)) * rows * 1e-3


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kw = {"device": "cuda", "generator": gen}
    dt = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "orth":
        state["x"] = update((case["count"], case["M"], case["N"]), kw).to(dt)
        return state
    if case["op"] == "muon":
        sh = shapes(case)
        state["params"] = [(torch.randn(s, **kw) / math.sqrt(s[-1])).to(dt) for s in sh]
        state["grads"] = [update(s, kw).to(dt) for s in sh]
        # after some steps: the momentum remembers most of what the gradient says
        state["momentum"] = [0.6 * g.float() + 0.5 * update(g.shape, kw) for g in state["grads"]]
        return state
    B, T, V = case["B"], case["T"], case["V"]
    lens = torch.randint(case["tlo"], T + 1, (B,), **kw).to(torch.int32)
    lens[int(seed) % B] = T  # a batch is as long as its longest sequence
    labels = torch.randint(0, V, (B, T), **kw)
    logits = torch.randn(B, T, V, **kw)
    logits *= 1.5
    # a model partly sure of its labels
    sure = 14.0 * torch.rand(B, T, 1, **kw)
    logits.scatter_add_(2, labels[..., None], sure)
    if case["mask"]:
        never = torch.rand(V, **kw) < case["mask"]
        never[labels[0, 0]] = False
        never[0] = False
        labels = torch.where(never[labels], 0, labels)
        logits.masked_fill_(never, -math.inf)
    labels = labels.to(torch.int32)
    if case["skip"]:
        labels = torch.where(torch.rand(B, T, **kw) < case["skip"], IGNORE, labels).to(torch.int32)
    state |= {"lens": lens, "labels": labels, "logits": logits.to(dt)}
    if case["entry"] == "train":
        state["logits"].requires_grad_(True)
        state["grads"] = [-(torch.rand(B, T, **kw) + 0.5), -0.1 * (torch.rand(B, T, **kw) + 0.5)]
        if case["top"]:
            state["grads"].append(-0.2 * torch.rand(B, T, case["top"], **kw))
    return state


# ------------------------------------------------------------------------------------------------ plain forms


def kept(labels, lens):
    """Which positions count: those inside their sequence whose label is not the ignored one."""
    inside = torch.arange(labels.shape[1], device=labels.device)[None, :] < lens[:, None]
    return inside & (labels != IGNORE)


def plain_scores(s):
    case, dt = s["case"], s["logits"].dtype
    B, T, V = s["logits"].shape
    ok = kept(s["labels"], s["lens"]).reshape(-1, 1)
    t = torch.where(ok, s["labels"].reshape(-1, 1).long(), 0)
    z = s["logits"].reshape(-1, V).float()
    z = z - z.amax(1, keepdim=True)
    p = z.exp()
    total = p.sum(1, keepdim=True)
    z -= total.log()
    p /= total
    z_or_0 = torch.where(p > 0, z, 0.0)
    entropy = -(p * z_or_0).sum(1, keepdim=True)
    shape = lambda x: torch.where(ok, x, 0.0).reshape(B, T)  # noqa: E731
    out = {"log_probs": shape(z.gather(1, t)), "entropy": shape(entropy)}
    if case["top"]:
        rest, values, labels = z.clone(), [], []
        for _ in range(case["top"]):  # the first of the largest
            best, at = rest.max(1, keepdim=True)
            values.append(best)
            labels.append(at)
            rest.scatter_(1, at, -math.inf)
        values, labels = torch.cat(values, 1), torch.cat(labels, 1)
        out["top_log_probs"] = torch.where(ok, values, 0.0).reshape(B, T, -1)
        out["top_labels"] = torch.where(ok, labels, IGNORE).to(torch.int32).reshape(B, T, -1)
    if case["entry"] == "train":
        g, h = s["grads"][0].reshape(-1, 1), s["grads"][1].reshape(-1, 1)
        d = (z_or_0 + entropy).mul_(-h)
        d -= g
        if case["top"]:
            d -= s["grads"][2].reshape(B * T, -1).sum(1, keepdim=True)
        d *= p
        d.scatter_add_(1, t, g)
        if case["top"]:
            d.scatter_add_(1, labels, s["grads"][2].reshape(B * T, -1))
        out["logits"] = torch.where(ok, d, 0.0).to(dt).reshape(B, T, V)
    return out


def plain_orthogonalize(x):
    """Newton-Schulz products of a batch of matrices, in 32 bits."""
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


def plain_muon(s):
    grads = [g.float() for g in s["grads"]]
    s["momentum"] = [v + (g - v) * (1 - BETA) for v, g in zip(s["momentum"], grads)]
    # all matrices of a model are alike once they lie: one batch
    u = [g + (v - g) * BETA for v, g in zip(s["momentum"], grads)]
    x = plain_orthogonalize(torch.stack([w.mT if w.shape[0] > w.shape[1] else w for w in u]))
    for p, w, o in zip(s["params"], u, x):
        o = o.mT if w.shape[0] > w.shape[1] else o
        rate = LR * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        p.copy_(p.float() * (1 - LR * DECAY) - rate * o)
    return {"params": s["params"], "momentum": s["momentum"]}


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            if case["op"] == "scores":
                return plain_scores(state)
            if case["op"] == "orth":
                return {"out": plain_orthogonalize(state["x"].float()).to(state["x"].dtype)}
            return plain_muon(state)
    from i6_native_ops_b200 import framewise

    if case["op"] == "orth":
        return {"out": framewise.orthogonalize(state["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)}
    if case["op"] == "muon":
        framewise.muon_step(state["params"], state["grads"], state["momentum"], lr=LR, beta=BETA, nesterov=True,
                            weight_decay=DECAY, steps=STEPS, coefficients=COEFFICIENTS, eps=EPS, adjust_lr="original")
        return {"params": state["params"], "momentum": state["momentum"]}
    got = framewise.label_scores(state["logits"], state["labels"], top=case["top"], seq_lens=state["lens"],
                                 ignore_index=IGNORE)
    names = ("log_probs", "entropy") + (("top_log_probs",) if case["top"] else ())
    out = {n: getattr(got, n).detach() for n in names}
    if case["top"]:
        out["top_labels"] = got.top_labels
    if case["entry"] == "train":
        out["logits"] = torch.autograd.grad([getattr(got, n) for n in names], state["logits"], state["grads"])[0]
    return out


def work(case):
    size = {"f32": 4, "bf16": 2}[case["dtype"]]
    if case["op"] in ("orth", "muon"):
        sh = [(case["M"], case["N"])] * case["count"] if case["op"] == "orth" else shapes(case)
        flops = 0
        for m, n in sh:
            m, n = min(m, n), max(m, n)
            flops += STEPS * (3 * m * m * n + m * m * m)  # of the symmetric products (X X^T and its square) a half
        values = sum(m * n for m, n in sh)
        return {"bytes": values * (2 * size if case["op"] == "orth" else 3 * size + 8), "flops": flops}
    B, T, V, top = case["B"], case["T"], case["V"], case["top"]
    rows = B * T
    used = max(1.0, B * (case["tlo"] + T) / 2 * (1 - case["skip"]))  # positions that count
    train = case["entry"] == "train"
    b = size * V * used + 4 * rows + 8 * rows * (1 + top)
    b += size * V * rows + 4 * rows * (2 + top) if train else 0
    return {"bytes": b, "flops": V * used * (14 if train else 6)}


# ------------------------------------------------------------------------------------------------ 64 bits


def polynomial_of_gram(x):
    """What STEPS steps make of x, by the m x m matrices alone: every step's factor is a polynomial of x x^T, so
    all of them commute."""
    if x.shape[0] > x.shape[1]:
        return polynomial_of_gram(x.t()).t()
    x = x / max(float(x.pow(2).sum()) ** 0.5, EPS)
    eye = torch.eye(x.shape[0], dtype=x.dtype, device=x.device)
    gram, q = torch.einsum("ik,jk->ij", x, x), eye
    for _ in range(STEPS):
        f = COEFFICIENTS[0] * eye + COEFFICIENTS[1] * gram + COEFFICIENTS[2] * torch.einsum("ik,kj->ij", gram, gram)
        q = torch.einsum("ik,kj->ij", f, q)
        gram = torch.einsum("ik,kl,lj->ij", f, gram, f)
    return torch.einsum("ik,kj->ij", q, x)


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "orth":
        return {"out": torch.stack([polynomial_of_gram(x.to(f64)) for x in s["x"]])}
    if case["op"] == "muon":
        out = {"params": [], "momentum": []}
        for p, g, v in zip(s["params"], s["grads"], s["momentum"]):
            g = g.to(f64)
            v = BETA * v.to(f64) + (1 - BETA) * g
            o = polynomial_of_gram((1 - BETA) * g + BETA * v)
            out["params"].append((1 - LR * DECAY) * p.to(f64) - LR * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * o)
            out["momentum"].append(v)
        return out
    B, T, V, top = case["B"], case["T"], case["V"], case["top"]
    train = case["entry"] == "train"
    rows = [(b, t) for b, n in enumerate(s["lens"].tolist()) for t in range(n)]
    at = torch.tensor([b * T + t for b, t in rows], device="cuda", dtype=torch.long)
    at = at[s["labels"].flatten()[at] != IGNORE]
    got = {"log_probs": torch.zeros(B * T, dtype=f64, device="cuda"), "entropy": torch.zeros(B * T, dtype=f64, device="cuda")}
    if top:
        got["top_log_probs"] = torch.zeros(B * T, top, dtype=f64, device="cuda")
        got["top_labels"] = torch.full((B * T, top), IGNORE, dtype=torch.int32, device="cuda")
    if train:
        got["logits"] = torch.zeros(B * T, V, dtype=f64, device="cuda")
    step = max(1, (1 << 27) // V)
    for a in range(0, len(at), step):
        i = at[a : a + step]
        n = torch.arange(len(i), device="cuda")
        t = s["labels"].flatten()[i].long()
        z = s["logits"].detach().view(B * T, V)[i].to(f64)
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        p = lp.exp()
        plogp = torch.special.entr(p)
        h = plogp.sum(1)
        got["log_probs"][i] = lp[n, t]
        got["entropy"][i] = h
        if top:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
            got["top_log_probs"][i] = lp.gather(1, order)
            got["top_labels"][i] = order.to(torch.int32)
        if train:
            g, gh = s["grads"][0].flatten()[i].to(f64), s["grads"][1].flatten()[i].to(f64)
            # dH/dz = -p (log p + H) = entr(p) - p H
            dz = gh[:, None] * (plogp - p * h[:, None])
            onehot = torch.zeros_like(p)
            onehot[n, t] += g
            total = g
            if top:
                gt = s["grads"][2].view(B * T, top)[i].to(f64)
                onehot.scatter_add_(1, order, gt)
                total = g + gt.sum(1)
            got["logits"][i] = dz + onehot - total[:, None] * p
    return {k: v.view(B, T, *v.shape[1:]) for k, v in got.items()}
