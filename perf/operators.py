"""The operators of framewise training whose speed counts: what a program that trains a network on the
alignments and label sequences of this package asks of ``i6_native_ops_b200.framewise``.

A case is a dict of

  op      ``ce`` (``linear_cross_entropy``: output layer and cross entropy over the classes, in one),
          ``embed`` (``label_embedding``: scaled rows of a table), ``adamw`` (``AdamW.step``)
  entry   ``score`` / ``lookup`` (the forward pass alone), ``train`` (and its gradients), ``step``
  dtype   ``f32`` or ``bf16``, of parameters, activations and gradients
  B T     sequences and positions of the padded batch, ``tlo`` the shortest length drawn
  V D     classes (or labels) and width; ``bias`` whether the output layer has one; ``skip`` the share of
          positions inside the sequences that are left out (the ignored label)
  zipf    exponent of the label frequencies (0: alike)
  layers  ``adamw``: layers of the model, of four tensors each; ``bits`` of the optimizer's states

Inputs are synthetic and drawn from a seed.  Where ``own`` is false, ``run`` computes the operators in
elementary steps, in 32 bits.
"""
import math

import torch

own = False

IGNORE = -100  # the label of positions that are left out
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.98), 1e-8, 0.01


def ce(name, entry, dtype, B, T, tlo, V, D, bias=True, skip=0.0, zipf=0.0):
    return {"name": name, "op": "ce", "entry": entry, "dtype": dtype, "B": B, "T": T, "tlo": tlo, "V": V, "D": D,
            "bias": bias, "skip": skip, "zipf": zipf}


def embed(name, entry, dtype, B, T, tlo, V, D, skip=0.0, zipf=0.0):
    return {"name": name, "op": "embed", "entry": entry, "dtype": dtype, "B": B, "T": T, "tlo": tlo, "V": V, "D": D,
            "bias": False, "skip": skip, "zipf": zipf}


def adamw(name, dtype, bits, layers, V, D):
    return {"name": name, "op": "adamw", "entry": "step", "dtype": dtype, "bits": bits, "layers": layers, "V": V, "D": D}


def listed():
    return [
        # the next label of eight hypotheses is scored: one position each, the smallest call
        ce("ce_score_labels", "score", "bf16", 8, 1, 1, 10025, 512),
        # a handful of short utterances with a character vocabulary
        ce("ce_tiny_train", "train", "f32", 4, 50, 40, 41, 256),
        # held-out frames scored with a lattice system's 5000 classes, in 32 bits, an odd length
        ce("ce_heldout_score", "score", "f32", 8, 1777, 1000, 5000, 512),
        # labels of a large vocabulary, all utterances of a batch, in 32 bits
        ce("ce_bpe_train", "train", "f32", 256, 100, 20, 10025, 512, zipf=1.1),
        # frames of a tied-state triphone system at a batch that leaves room for an encoder beside it;
        # sizes that divide nothing, some frames left out
        ce("ce_triphone_train", "train", "bf16", 17, 1499, 1200, 12001, 500, skip=0.05),
        # the full batch of that system, the largest case
        ce("ce_triphone_large", "train", "bf16", 64, 1500, 1200, 12001, 1024),
        # embedding of the last label of every hypothesis: one position each
        embed("embed_last_labels", "lookup", "bf16", 256, 1, 1, 10025, 512),
        # label sequences of a large vocabulary, frequent units first
        embed("embed_bpe_train", "train", "bf16", 256, 100, 20, 10025, 512, zipf=1.1),
        # left context of every frame of an alignment: many positions, few labels
        embed("embed_context_train", "train", "f32", 64, 1500, 1200, 121, 256, skip=0.01),
        # a small model's step: launches and the host's time are everything
        adamw("adamw_small", "f32", 32, 2, 41, 64),
        # a model kept in 16 bits with 8-bit states
        adamw("adamw_states8", "bf16", 8, 4, 12001, 1024),
        # a large model in 32 bits throughout
        adamw("adamw_large", "f32", 32, 4, 12001, 2048),
    ]


def draw(rng):
    """A case of the listed ranges, sizes spread over their logarithm."""

    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["ce", "ce", "embed", "adamw"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "adamw":
        D = spread(40, 1600)
        return {"op": op, "entry": "step", "dtype": dtype, "bits": rng.choice([8, 32]), "layers": rng.randint(1, 4),
                "V": spread(41, 12001), "D": D}
    V = spread(41, 12001)
    D = 64 * spread(1, 16) if rng.random() < 0.6 else spread(40, 1024)
    B = spread(1, 256)
    T = spread(1, 1500)
    most = 96000 if op == "embed" else min(96000, 1 * 96000 * 12001 * 1024 // (V * D * (6 if dtype == "f32" else 1)))
    T = max(1, min(T, most // B))
    entry = rng.choice(["score", "train", "train"]) if op == "ce" else rng.choice(["lookup", "train", "train"])
    return {"op": op, "entry": entry, "dtype": dtype, "B": B, "T": T, "tlo": rng.randint(0, T), "V": V, "D": D,
            "bias": op == "ce" and rng.random() < 0.7, "skip": rng.choice([0.0, 0.02, 0.3]),
            "zipf": rng.choice([0.0, 1.1])}


# ------------------------------------------------------------------------------------------------ inputs


def shapes(case):
    """The tensors of a small model: label table, output layer and its bias, four per layer between."""
    V, D = case["V"], case["D"]
    return [(V, D), (V, D), (V,)] + [(4 * D, D), (4 * D,), (D, 4 * D), (D,)] * case["layers"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kw = {"device": "cuda", "generator": gen}
    dt = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "adamw":
        # after some hundred steps: first moments below the second's root, rows of their own sizes
        sh = shapes(case)
        state |= {"params": [], "grads": [], "exp_avg": [], "exp_avg_sq": []}
        for s in sh:
            rows = (torch.rand(s[0], **kw) * 6 - 9).exp().reshape((-1,) + (1,) * (len(s) - 1))
            p = (torch.randn(s, **kw) / math.sqrt(s[-1])).to(dt)
            state["params"].append(p)
            state["grads"].append((torch.randn(s, **kw) * rows).to(dt))
            state["exp_avg"].append(torch.randn(s, **kw) * rows * 0.2)
            state["exp_avg_sq"].append((torch.rand(s, **kw) + 0.5) * rows * rows)
        state["step"] = 400
        state["master"] = None if dt == torch.float32 else [p.float() for p in state["params"]]
        if case["bits"] == 8:
            state["exp_avg"] = [coded(x, 127) for x in state["exp_avg"]]
            state["exp_avg_sq"] = [coded(x.sqrt(), 255) for x in state["exp_avg_sq"]]
        return state
    B, T, V, D = case["B"], case["T"], case["V"], case["D"]
    lens = torch.randint(case["tlo"], T + 1, (B,), **kw).to(torch.int32)
    lens[int(seed) % B] = T  # a batch is as long as its longest sequence
    if case["zipf"]:
        p = torch.arange(1, V + 1, device="cuda", dtype=torch.float64).pow(-case["zipf"])
        edge = (p / p.sum()).cumsum(0)
        labels = torch.searchsorted(edge, torch.rand(B, T, dtype=torch.float64, **kw)).clamp_(max=V - 1)
    else:
        labels = torch.randint(0, V, (B, T), **kw)
        if case["entry"] == "train" and T > 100:  # an alignment: labels hold for some frames
            labels = labels[:, torch.arange(T, device="cuda") // 3 * 3]
    labels = labels.to(torch.int32)
    if case["skip"]:
        labels = torch.where(torch.rand(B, T, **kw) < case["skip"], IGNORE, labels).to(torch.int32)
    weight = torch.randn(V, D, **kw)
    state |= {"lens": lens, "labels": labels}
    if case["op"] == "ce":
        weight *= 2.0 / math.sqrt(D)
        hidden = torch.randn(B, T, D, **kw)
        # a model partly sure of its labels
        hidden += 2.0 * torch.rand(B, T, 1, **kw) * weight[labels.long().clamp(min=0)]
        state["hidden"] = hidden.to(dt)
        state["bias"] = (0.5 * torch.randn(V, **kw)).to(dt) if case["bias"] else None
        state["grad"] = torch.rand(B, T, **kw) + 0.5  # weights of the frames
    else:
        state["scale"] = math.sqrt(D)
        state["grad"] = torch.randn(B, T, D, **kw).to(dt)
        weight *= 1.0 / math.sqrt(D)
    state["weight"] = weight.to(dt)
    if case["entry"] == "train":
        for n in ("hidden", "weight", "bias"):
            if state.get(n) is not None:
                state[n].requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------------------ plain forms


def kept(labels, lens):
    """Which positions count: those inside their sequence whose label is not the ignored one."""
    inside = torch.arange(labels.shape[1], device=labels.device)[None, :] < lens[:, None]
    return inside & (labels != IGNORE)


def plain_ce(s):
    case, dt = s["case"], s["weight"].dtype
    B, T, D = s["hidden"].shape
    ok = kept(s["labels"], s["lens"]).reshape(-1, 1)
    t = torch.where(ok, s["labels"].reshape(-1, 1).long(), 0)
    x = torch.where(ok, s["hidden"].reshape(-1, D).float(), 0.0)
    w = s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z += s["bias"].float()
    top = z.amax(1, keepdim=True)
    target = z.gather(1, t)
    e = z.sub_(top).exp_()
    total = e.sum(1, keepdim=True)
    loss = torch.where(ok, total.log() + (top - target), 0.0).reshape(B, T)
    if case["entry"] == "score":
        return {"loss": loss}
    d = e.div_(total)
    d.scatter_add_(1, t, torch.full_like(target, -1.0))
    d *= torch.where(ok, s["grad"].reshape(-1, 1), 0.0)
    out = {"loss": loss, "hidden": (d @ w).to(dt).reshape(B, T, D), "weight": (d.t() @ x).to(dt)}
    if s["bias"] is not None:
        out["bias"] = d.sum(0).to(dt)
    return out


def plain_embed(s):
    case, dt = s["case"], s["weight"].dtype
    ok = kept(s["labels"], s["lens"])[..., None]
    t = torch.where(ok[..., 0], s["labels"].long(), 0)
    out = {"out": torch.where(ok, s["weight"].float()[t] * s["scale"], 0.0).to(dt)}
    if case["entry"] == "train":
        g = torch.where(ok, s["grad"].float() * s["scale"], 0.0)
        grad = torch.zeros(s["weight"].shape, device=g.device)
        out["weight"] = grad.index_add_(0, t.reshape(-1), g.reshape(-1, g.shape[-1])).to(dt)
    return out


BLOCK = 256  # values that share a step
TINY = 2.0**-120  # a block whose step is smaller is held as zeros


def coded(x, top):
    """A tensor in 8 bits: per block a step k and per value a whole c of at most ``top``, which stand for
    c * |c| * k.  ``top`` 127: signed values.  255: values that are not negative; one that is positive stays so."""
    flat = torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % BLOCK)).reshape(-1, BLOCK)
    k = flat.abs().amax(1, keepdim=True) / float(top * top)
    k = torch.where(k < TINY, 0.0, k)
    c = (flat.abs() * (1.0 / k)).sqrt().round().clamp(max=float(top))
    if top == 255:
        c = torch.where(flat > 0, c.clamp(min=1.0), c)
    c = torch.where(k > 0, c, 0.0) * flat.sign()
    return c.to(torch.int8 if top == 127 else torch.uint8).reshape(-1)[: x.numel()].reshape(x.shape), k.reshape(-1)


def decoded(code):
    c, k = code
    x = torch.nn.functional.pad(c.reshape(-1), (0, -c.numel() % BLOCK)).reshape(-1, BLOCK).float()
    return (x * x.abs() * k[:, None]).reshape(-1)[: c.numel()].reshape(c.shape)


def plain_adamw(s):
    b1, b2 = BETAS
    eight = s["case"]["bits"] == 8
    s["step"] += 1
    step = LR / (1 - b1 ** s["step"])
    root = 1 / math.sqrt(1 - b2 ** s["step"])
    out = {"params": s["params"], "exp_avg": [], "exp_avg_sq": []}
    for i, p in enumerate(s["params"]):
        g = s["grads"][i].float()
        m, v = s["exp_avg"][i], s["exp_avg_sq"][i]
        if eight:
            m, v = decoded(m), decoded(v).square()
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * g) * (1 - b2)
        r = v.sqrt()
        x = p if s["master"] is None else s["master"][i]
        x.copy_(x * (1 - LR * DECAY) - (m * step) / (r * root + EPS))
        if x is not p:
            p.copy_(x)
        s["exp_avg"][i], s["exp_avg_sq"][i] = (coded(m, 127), coded(r, 255)) if eight else (m, v)
        out["exp_avg"].append(decoded(s["exp_avg"][i]) if eight else m)
        out["exp_avg_sq"].append(decoded(s["exp_avg_sq"][i]).square() if eight else v)
    return out


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"ce": plain_ce, "embed": plain_embed, "adamw": plain_adamw}[case["op"]](state)
    from i6_native_ops_b200 import framewise

    if case["op"] == "adamw":
        state["step"] += 1
        states = state["exp_avg"], state["exp_avg_sq"]
        framewise.adamw_step(state["params"], state["grads"], *states, step=state["step"], master=state["master"], lr=LR,
                             betas=BETAS, eps=EPS, weight_decay=DECAY)
        exp_avg, exp_avg_sq = states if case["bits"] == 32 else framewise.adamw_values(*states)
        return {"params": state["params"], "exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq}
    if case["op"] == "embed":
        out = framewise.label_embedding(state["labels"], state["weight"], scale=state["scale"], seq_lens=state["lens"],
                                        ignore_index=IGNORE)
        if case["entry"] == "lookup":
            return {"out": out}
        return {"out": out.detach(), "weight": torch.autograd.grad(out, state["weight"], state["grad"])[0]}
    loss = framewise.linear_cross_entropy(state["hidden"], state["weight"], state["labels"], bias=state["bias"],
                                          seq_lens=state["lens"], ignore_index=IGNORE)
    if case["entry"] == "score":
        return {"loss": loss}
    names = [n for n in ("hidden", "weight", "bias") if state[n] is not None]
    grads = torch.autograd.grad(loss, [state[n] for n in names], state["grad"])
    return {"loss": loss.detach(), **dict(zip(names, grads))}


def work(case):
    size = {"f32": 4, "bf16": 2}[case["dtype"]]
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in shapes(case))
        master = 0 if size == 4 else 4
        held = 8 if case["bits"] == 32 else 2 + 8 / BLOCK
        values = 0 if case["bits"] == 32 else 8  # the states' values that are returned
        # gradient read; weights (those in 32 bits) and states read and written; the 16-bit weights written
        return {"bytes": n * (size + 2 * (master or size) + (size if master else 0) + 2 * held + values), "flops": 14 * n}
    B, T, V, D = case["B"], case["T"], case["V"], case["D"]
    rows = B * T
    used = max(1.0, B * (case["tlo"] + T) / 2 * (1 - case["skip"]))  # positions that count
    train = case["entry"] == "train"
    if case["op"] == "embed":
        n = min(V, used)  # rows of the table at least looked at
        read = size * D * n + 4 * rows
        return {"bytes": read + size * rows * D + (size * used * D + size * V * D if train else 0),
                "flops": used * D * (2 if train else 1)}
    per = size * D * used + size * V * D + (size * V if case["bias"] else 0)
    b = per + 8 * rows + ((4 * rows + size * rows * D + size * V * D + (size * V if case["bias"] else 0)) if train else 0)
    return {"bytes": b, "flops": 2.0 * used * V * D * (3 if train else 1)}


# ------------------------------------------------------------------------------------------------ 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "adamw":
        t, (b1, b2) = 401, BETAS
        out = {"params": [], "exp_avg": [], "exp_avg_sq": []}
        for i, p in enumerate(s["params"]):
            g = s["grads"][i].to(f64)
            if case["bits"] == 8:  # the moments that the codes stand for; after the step they are rounded to codes again
                at = torch.arange(p.numel(), device="cuda").view(p.shape) // BLOCK
                c, k = s["exp_avg"][i]
                m = c.to(f64).square().copysign(c.to(f64)) * k.to(f64)[at]
                c, k = s["exp_avg_sq"][i]
                v = (c.to(f64).square() * k.to(f64)[at]).square()
            else:
                m, v = s["exp_avg"][i].to(f64), s["exp_avg_sq"][i].to(f64)
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g.square()
            new = p.to(f64) * (1 - LR * DECAY) - LR * (m / (1 - b1**t)) / ((v / (1 - b2**t)).sqrt() + EPS)
            out["params"].append(new)
            out["exp_avg"].append(None if case["bits"] == 8 else m)
            out["exp_avg_sq"].append(None if case["bits"] == 8 else v)
        return out
    B, T, V, D = case["B"], case["T"], case["V"], case["D"]
    rows = [(b, t) for b, n in enumerate(s["lens"].tolist()) for t in range(n)]
    at = torch.tensor([b * T + t for b, t in rows], device="cuda", dtype=torch.long)
    label = s["labels"].flatten()[at].long()
    at, label = at[label != IGNORE], label[label != IGNORE]
    w = s["weight"].detach().to(f64)
    if case["op"] == "embed":
        out = torch.zeros(B * T, D, dtype=f64, device="cuda")
        out[at] = w[label] * s["scale"]
        got = {"out": out.view(B, T, D)}
        if case["entry"] == "train":
            got["weight"] = torch.zeros(V, D, dtype=f64, device="cuda")
            g = s["grad"].reshape(B * T, D)
            got["weight"].index_put_((label,), g[at].to(f64) * s["scale"], accumulate=True)
        return got
    loss = torch.zeros(B * T, dtype=f64, device="cuda")
    got = {"loss": loss.view(B, T)}
    if case["entry"] == "train":
        gx = torch.zeros(B * T, D, dtype=f64, device="cuda")
        got |= {"hidden": gx.view(B, T, D), "weight": torch.zeros_like(w)}
        if case["bias"]:
            got["bias"] = torch.zeros(V, dtype=f64, device="cuda")
    step = 8192
    for a in range(0, len(at), step):
        i, lab = at[a : a + step], label[a : a + step]
        x = s["hidden"].detach().view(B * T, D)[i].to(f64)
        z = torch.einsum("nd,vd->nv", x, w)
        if case["bias"]:
            z = z + s["bias"].detach().to(f64)
        lse = torch.logsumexp(z, 1)
        n = torch.arange(len(i), device="cuda")
        loss[i] = lse - z[n, lab]
        if case["entry"] == "train":
            q = (z - lse[:, None]).exp()
            q[n, lab] -= 1
            q *= s["grad"].flatten()[i].to(f64)[:, None]
            gx[i] = torch.einsum("nv,vd->nd", q, w)
            got["weight"] += torch.einsum("nv,nd->vd", q, x)
            if case["bias"]:
                got["bias"] += q.sum(0)
    return got
