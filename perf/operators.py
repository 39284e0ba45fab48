"""Cases and plain forms of the training operators for deep residual networks with large class heads:

* ``ce``    -- softmax cross entropy of a linear head, ``x W^T + b`` against class indices, without keeping the
               logits, with the gradients to x, W and b (``vae_amd.losses.linear_cross_entropy``);
* ``norm``  -- the two norms around a residual block in one pass: ``y = r + s * act(g) * norm(b)``, ``h = norm(y)``,
               with all gradients (``vae_amd.functional.gated_residual_norm``);
* ``adamw`` -- one AdamW step over many tensors with moments in 8 or 32 bits
               (``vae_amd.optim.multi_tensor_adamw_``).

``own`` selects what ``run`` computes with: False = elementary torch operations in 32 bits, True = the framework.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100
BLOCK = 256                       # elements of a quantisation block of the 8-bit moments; every tensor starts a new one
LR, BETAS, EPS, WD = 5e-4, (0.9, 0.998), 1e-7, 0.05


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a cell-property head on the latent of one training batch: microseconds, launch latency is what counts
        dict(name="ce_head_fp32", op="ce", n=512, d=30, v=17, dtype="fp32", bias=True, weight=True, ignored=0.2, train=True),
        # a head as wide as the gene axis on the hidden layer of one batch, full precision
        dict(name="ce_genes_fp32", op="ce", n=512, d=256, v=20000, dtype="fp32", bias=True, weight=False, ignored=0.0, train=True),
        # a ragged batch against a ragged vocabulary: nothing is a multiple of a tile
        dict(name="ce_ragged_bf16", op="ce", n=4093, d=1000, v=30011, dtype="bf16", bias=False, weight=False, ignored=0.1, train=True),
        # evaluation: the loss of every row, no gradients
        dict(name="ce_eval_fp16", op="ce", n=2048, d=2048, v=65536, dtype="fp16", bias=False, weight=False, ignored=0.05, train=False),
        # the largest vocabulary: the logits alone would be 4.3 GB in 32 bits
        dict(name="ce_large_bf16", op="ce", n=8192, d=4096, v=131072, dtype="bf16", bias=False, weight=False, ignored=0.02, train=True),
        # a few rows in evaluation, one launch
        dict(name="norm_rows_bf16", op="norm", n=4, d=4096, dtype="bf16", kind="rms", gate="full", act="sigmoid", post=True, scale=True,
             bias=False, train=False),
        # the hidden width and batch of the shipped networks, LayerNorm with bias, one gate per cell
        dict(name="norm_hidden_fp32", op="norm", n=512, d=256, dtype="fp32", kind="layer", gate="row", act="sigmoid", post=True, scale=True,
             bias=True, train=True),
        # odd width: rows are not aligned
        dict(name="norm_odd_fp16", op="norm", n=5003, d=1531, dtype="fp16", kind="layer", gate="full", act="tanh", post=False, scale=True,
             bias=True, train=True),
        # a large training batch
        dict(name="norm_large_bf16", op="norm", n=32768, d=4096, dtype="bf16", kind="rms", gate="full", act="sigmoid", post=True, scale=True,
             bias=False, train=True),
        # the smallest network of the benchmark: some twenty tensors, under a million parameters
        dict(name="adamw_small_8bit", op="adamw", total=850_011, tensors=24, dtype="fp32", bits=8, master=False, clip=0.0),
        # the benchmark network's 18 M parameters with gradient clipping, moments in 32 bits
        dict(name="adamw_clip_32bit", op="adamw", total=18_020_003, tensors=41, dtype="fp32", bits=32, master=False, clip=0.5),
        # a large network in bf16 with 32-bit master weights and moments in 8 bits
        dict(name="adamw_large_8bit", op="adamw", total=1_000_000_007, tensors=300, dtype="bf16", bits=8, master=True, clip=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ce", "norm", "adamw"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    if op == "ce":
        n, d, v = _log(rng, 1, 8192), _log(rng, 16, 4096), _log(rng, 2, 131072)
        if dtype == "fp32":       # 32-bit products cost more: a narrower range
            n, v = min(n, 4096), min(v, 40000)
        return dict(op="ce", n=n, d=d, v=v, dtype=dtype, bias=rng.random() < 0.5, weight=rng.random() < 0.3,
                    ignored=rng.choice((0.0, 0.1, 0.5)), train=rng.random() < 0.7)
    if op == "norm":
        n, d = _log(rng, 1, 32768), _log(rng, 16, 16384)
        n = min(n, 32768 * 4096 // d)
        return dict(op="norm", n=n, d=d, dtype=dtype, kind=rng.choice(("rms", "layer")), gate=rng.choice(("none", "row", "full")),
                    act=rng.choice(("identity", "sigmoid", "tanh")), post=rng.random() < 0.6, scale=rng.random() < 0.6,
                    bias=rng.random() < 0.5, train=rng.random() < 0.7)
    total = _log(rng, 1000, 300_000_000)
    # 8-bit codes with clipping are left to the tests: the coefficient's last bit decides a code here and there
    bits = rng.choice((8, 32))
    return dict(op="adamw", total=total, tensors=min(_log(rng, 1, 400), max(1, total // 300)), dtype=dtype, bits=bits,
                master=dtype != "fp32" and rng.random() < 0.5, clip=0.5 if bits == 32 and rng.random() < 0.5 else 0.0)


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "ce":
        n, d, v = case["n"], case["d"], case["v"]
        once = (n * d + v * d) * e + (v * e if case["bias"] else 0) + (4 * v if case["weight"] else 0) + 8 * n
        if not case["train"]:
            return {"bytes": once + 4 * n, "flops": 2 * n * d * v}
        return {"bytes": once + (n * d + v * d) * e + (v * e if case["bias"] else 0) + 4, "flops": 6 * n * d * v}
    if case["op"] == "norm":
        n, d, full = case["n"], case["d"], case["gate"] == "full"
        fwd = (2 + full + 2) * n * d * e                          # r, b, gate -> y, h
        if not case["train"]:
            return {"bytes": fwd, "flops": 20 * n * d}
        # backward: y, b, gate, dy, dh -> dr, db, dgate
        return {"bytes": fwd + (4 + full + 2 + full) * n * d * e, "flops": 60 * n * d}
    state = 4 if case["bits"] == 8 else 16                         # both moments, read and written
    per = 3 * e + state + (8 - e if case["master"] else 0)         # with master weights the low-precision ones are only written
    return {"bytes": per * case["total"] + (16 * case["total"] // BLOCK if case["bits"] == 8 else 0), "flops": 20 * case["total"]}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _prepare_ce(c, seed):
    g, t = _gen(seed), DTYPES[c["dtype"]]
    n, d, v = c["n"], c["d"], c["v"]
    w = (_randn(g, v, d) / math.sqrt(d)).to(t)
    # class frequencies fall off as a power law, as labels and words do
    u = torch.rand(n, generator=g, device=DEV)
    target = ((v ** u - 1.0) / max(v - 1, 1) * v).long().clamp_(0, v - 1)
    x = (_randn(g, n, d) + 2.0 * w[target].float()).to(t)          # rows lean towards their class
    if c["ignored"]:
        target = torch.where(torch.rand(n, generator=g, device=DEV) < c["ignored"], torch.full_like(target, IGNORE), target)
        target[0] = 0
    bias = (0.5 * _randn(g, v)).to(t) if c["bias"] else None
    weight = (0.1 + torch.rand(v, generator=g, device=DEV)) if c["weight"] else None
    return dict(x=x, w=w, target=target, bias=bias, weight=weight)


def _prepare_norm(c, seed):
    g, t = _gen(seed), DTYPES[c["dtype"]]
    n, d = c["n"], c["d"]
    s = dict(r=(2.0 * _randn(g, n, d)).to(t), b=(_randn(g, n, d) + 0.3).to(t), gate=None, post_weight=None, post_bias=None, scale=None,
             norm_weight=(1.0 + 0.1 * _randn(g, d)).to(t), norm_bias=None)
    if c["gate"] != "none":
        s["gate"] = _randn(g, n, d if c["gate"] == "full" else 1).to(t)
    if c["post"]:
        s["post_weight"] = (1.0 + 0.1 * _randn(g, d)).to(t)
    if c["scale"]:
        s["scale"] = (0.5 + 0.1 * _randn(g, d)).to(t)
    if c["bias"]:
        s["norm_bias"] = (0.1 * _randn(g, d)).to(t)
        s["post_bias"] = (0.1 * _randn(g, d)).to(t) if c["post"] else None
    if c["train"]:
        s["dy"], s["dh"] = _randn(g, n, d).to(t), _randn(g, n, d).to(t)
    return s


def _sizes(total, tensors):
    """``tensors`` sizes of several magnitudes that add up to ``total``, every one at least 1."""
    rng = random.Random(total * 1009 + tensors)
    share = [math.exp(rng.uniform(0.0, 6.0)) for _ in range(tensors)]
    got = [max(1, int(total * s / sum(share))) for s in share]
    got[got.index(max(got))] += total - sum(got)
    return got


def _prepare_adamw(c, seed):
    g, t = _gen(seed), DTYPES[c["dtype"]]
    sizes = _sizes(c["total"], c["tensors"])
    at, starts = 0, []
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    used = torch.zeros(at, dtype=torch.bool, device=DEV)
    for s, n in zip(starts, sizes):
        used[s:s + n] = True
    flat32 = (0.05 * _randn(g, at)).mul_(used)
    # magnitudes of the gradients differ from block to block
    mag = 1e-3 * torch.exp(_randn(g, at // BLOCK, 1))
    grad = (_randn(g, at // BLOCK, BLOCK) * mag).view(-1).mul_(used).to(t)
    m = (_randn(g, at // BLOCK, BLOCK) * (0.3 * mag)).view(-1).mul_(used)
    v = ((0.2 + torch.rand(at // BLOCK, BLOCK, generator=g, device=DEV)) * mag).square_().view(-1).mul_(used)
    flat = flat32.to(t)
    s = dict(flat=flat, grad=grad, params=[flat[b:b + n] for b, n in zip(starts, sizes)],
             grads=[grad[b:b + n] for b, n in zip(starts, sizes)], sizes=sizes, starts=starts, used=used, step=9,
             master=flat32 if c["master"] else None, decay=[WD if k % 2 == 0 else 0.0 for k in range(len(sizes))],
             clip=c["clip"], seed=seed, scales=None)
    if c["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        mb, ub = m.view(-1, BLOCK), v.view(-1, BLOCK).sqrt()
        sm, su = mb.abs().amax(1) / 448.0, ub.amax(1) / 448.0
        s["m"] = (mb / sm.clamp_min(1e-30)[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(-1)
        s["v"] = (ub / su.clamp_min(1e-30)[:, None]).clamp(0.0, 448.0).to(torch.float8_e4m3fn).view(-1)
        s["scales"] = torch.stack((sm, su))
    return s


def prepare(case, seed):
    return {"case": case, **{"ce": _prepare_ce, "norm": _prepare_norm, "adamw": _prepare_adamw}[case["op"]](case, seed)}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_ce(s):
    from vae_amd.losses import linear_cross_entropy
    if not s["case"]["train"]:
        with torch.no_grad():
            return {"loss": linear_cross_entropy(s["x"], s["w"], s["target"], bias=s["bias"], weight=s["weight"], ignore_index=IGNORE,
                                                 reduction="none")}
    leaf = {k: s[k].detach().requires_grad_() for k in ("x", "w", "bias") if s[k] is not None}
    loss = linear_cross_entropy(leaf["x"], leaf["w"], s["target"], bias=leaf.get("bias"), weight=s["weight"], ignore_index=IGNORE,
                                reduction="mean")
    grads = torch.autograd.grad(loss, list(leaf.values()))
    return {"loss": loss.detach(), **{"d" + k: g for k, g in zip(leaf, grads)}}


NORM_INPUTS = ("r", "b", "gate", "post_weight", "post_bias", "scale", "norm_weight", "norm_bias")


def _own_norm(s):
    from vae_amd.functional import gated_residual_norm
    c = s["case"]
    if not c["train"]:
        with torch.no_grad():
            y, h = gated_residual_norm(*[s[k] for k in NORM_INPUTS[:2]], **{k: s[k] for k in NORM_INPUTS[2:]}, kind=c["kind"],
                                       gate_act=c["act"], eps=1e-5)
        return {"y": y, "h": h}
    leaf = {k: s[k].detach().requires_grad_() for k in NORM_INPUTS if s[k] is not None}
    y, h = gated_residual_norm(leaf["r"], leaf["b"], **{k: leaf.get(k) for k in NORM_INPUTS[2:]}, kind=c["kind"], gate_act=c["act"],
                               eps=1e-5)
    grads = torch.autograd.grad([y, h], list(leaf.values()), [s["dy"], s["dh"]])
    return {"y": y.detach(), "h": h.detach(), **{"d" + k: g for k, g in zip(leaf, grads)}}


def _own_adamw(s):
    from vae_amd.optim import multi_tensor_adamw_
    s["step"] += 1
    multi_tensor_adamw_(s["params"], s["grads"], s["m"], s["v"], step=s["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=s["decay"],
                        scales=s["scales"], master=s["master"], max_grad_norm=s["clip"], seed=s["seed"])
    return {k: s[k] for k in ("flat", "master", "m", "v", "scales")}


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_ce(s):
    c = s["case"]
    x, w, target = s["x"].float(), s["w"].float(), s["target"]
    logits = x @ w.t()
    if s["bias"] is not None:
        logits = logits + s["bias"].float()
    kept = target != IGNORE
    at = torch.where(kept, target, torch.zeros_like(target))[:, None]
    top = logits.amax(1, keepdim=True)
    lse = top + (logits - top).exp().sum(1, keepdim=True).log()
    cw = kept.float() if s["weight"] is None else kept.float() * s["weight"][at[:, 0]]
    nll = cw * (lse - logits.gather(1, at))[:, 0]
    if not c["train"]:
        return {"loss": nll}
    total = cw.sum()
    g = (cw / total)[:, None]
    d = (logits - lse).exp() * g
    d.scatter_add_(1, at, -g)
    out = {"loss": nll.sum() / total, "dx": (d @ w).to(s["x"].dtype), "dw": (d.t() @ x).to(s["x"].dtype)}
    if s["bias"] is not None:
        out["dbias"] = d.sum(0).to(s["x"].dtype)
    return out


def _stats(t, kind, eps):
    """(normalised rows, 1 / their scale)"""
    if kind == "layer":
        t = t - t.mean(1, keepdim=True)
    inv = (t.square().mean(1, keepdim=True) + eps).rsqrt()
    return t * inv, inv


def _norm_back(dn, n, inv, kind):
    """Gradient through n = (t - mean) * inv (layer) or t * inv (rms)."""
    got = dn - n * (dn * n).mean(1, keepdim=True)
    if kind == "layer":
        got = got - dn.mean(1, keepdim=True)
    return got * inv


def _act(gate, kind):
    """(act(gate), act'(gate))"""
    if kind == "sigmoid":
        a = 1.0 / (1.0 + (-gate).exp())
        return a, a * (1.0 - a)
    if kind == "tanh":
        a = gate.tanh()
        return a, 1.0 - a * a
    return gate, torch.ones_like(gate)


def _norm_in(s, real):
    """The whole operator in the type ``real``: its outputs before the rounding to the inputs' type."""
    c, eps = s["case"], 1e-5
    t = {k: None if s[k] is None else s[k].to(real) for k in NORM_INPUTS}
    kind = c["kind"]
    u, inv_b = t["b"], None
    if t["post_weight"] is not None:
        nb, inv_b = _stats(t["b"], kind, eps)
        u = nb * t["post_weight"]
        if t["post_bias"] is not None:
            u = u + t["post_bias"]
    a, da = (None, None) if t["gate"] is None else _act(t["gate"], c["act"])
    k = u if t["scale"] is None else u * t["scale"]
    y = t["r"] + (k if a is None else k * a)
    ny, inv_y = _stats(y.to(s["r"].dtype).to(real), kind, eps)         # the next block reads the rounded stream
    h = ny * t["norm_weight"]
    if t["norm_bias"] is not None:
        h = h + t["norm_bias"]
    out = {"y": y, "h": h}
    if not c["train"]:
        return out
    dy, dh = s["dy"].to(real), s["dh"].to(real)
    out["dnorm_weight"] = (dh * ny).sum(0)
    if t["norm_bias"] is not None:
        out["dnorm_bias"] = dh.sum(0)
    dt = dy + _norm_back(dh * t["norm_weight"], ny, inv_y, kind)
    out["dr"] = dt
    if a is not None:
        dg = dt * k * da
        out["dgate"] = dg if c["gate"] == "full" else dg.sum(1, keepdim=True)
        dt = dt * a
    if t["scale"] is not None:
        out["dscale"] = (dt * u).sum(0)
        dt = dt * t["scale"]
    if t["post_weight"] is None:
        out["db"] = dt
    else:
        out["dpost_weight"] = (dt * nb).sum(0)
        if t["post_bias"] is not None:
            out["dpost_bias"] = dt.sum(0)
        out["db"] = _norm_back(dt * t["post_weight"], nb, inv_b, kind)
    return out


def _plain_norm(s):
    return {k: v.to(s["r"].dtype) for k, v in _norm_in(s, torch.float32).items()}


def _mix32(h):
    """Austin Appleby's 32-bit finaliser (MurmurHash3, public domain) on int64 tensors or ints that hold 32-bit values."""
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _noise(n, seed, step):
    """The 16 random bits of every element, two elements to a 32-bit hash of (seed, step, index)."""
    key = _mix32(((seed & 0xFFFFFFFF) ^ _mix32((seed >> 32) & 0xFFFFFFFF)) ^ _mix32((step * 0x9E3779B9) & 0xFFFFFFFF))
    pair = torch.arange(-(-n // 2), dtype=torch.int64, device=DEV)
    h = _mix32((pair & 0xFFFFFFFF) ^ _mix32(((pair >> 32) + key) & 0xFFFFFFFF))
    return torch.stack((h & 0xFFFF, h >> 16), 1).view(-1)[:n]


def _plain_adamw(s):
    c, blocks = s["case"], s["flat"].numel() // BLOCK
    s["step"] += 1
    b1, b2 = BETAS
    p = s["flat"].float() if s["master"] is None else s["master"]
    g = s["grad"].float()
    if s["clip"]:
        norm = g.double().square().sum().sqrt()
        g = g * (s["clip"] / (norm + 1e-6)).clamp(max=1.0).float()
    if c["bits"] == 8:
        m = (s["m"].float().view(blocks, BLOCK) * s["scales"][0][:, None]).view(-1)
        u = (s["v"].float().view(blocks, BLOCK) * s["scales"][1][:, None]).view(-1)
        v = u * u
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    u = v.sqrt()
    inv_bc2 = 1.0 / math.sqrt(1.0 - b2 ** s["step"])
    moved = (m / (u * inv_bc2 + EPS)) * (LR / (1.0 - b1 ** s["step"]))
    ends = torch.tensor([-(-n // BLOCK) * BLOCK for n in s["sizes"]], device=DEV)
    keep = torch.tensor([1.0 - LR * d for d in s["decay"]], dtype=torch.float32, device=DEV).repeat_interleave(ends, output_size=p.numel())
    p = p * keep - moved
    if s["master"] is not None:
        s["master"].copy_(p)
    s["flat"].copy_(p)
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        mb, ub = m.view(blocks, BLOCK), u.view(blocks, BLOCK)
        top = torch.stack((mb.abs().amax(1), ub.amax(1)))
        inv = torch.where(top > 1e-30, top.reciprocal() * 448.0, torch.zeros_like(top))
        s["m"].copy_((mb * inv[0][:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(-1))
        # the root of the second moment is rounded up or down at random, so that its slow decay is kept on average:
        # scaled by 2^-120 the upper 12 bits of a float are the 8 bits of the code
        bits = ((ub * inv[1][:, None]) * 2.0 ** -120).view(torch.int32).view(-1)
        code = ((bits + (_noise(bits.numel(), s["seed"], s["step"]).to(torch.int32) << 4) + 8) >> 20).clamp_(max=126)
        code = torch.maximum(code, (u > 0).to(torch.int32))            # what is not zero stays so: it divides
        s["v"].copy_(code.to(torch.uint8).view(torch.float8_e4m3fn))
        s["scales"].copy_(top * (1.0 / 448.0))
    return {k: s[k] for k in ("flat", "master", "m", "v", "scales")}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"ce": _own_ce, "norm": _own_norm, "adamw": _own_adamw}[op](state)
    with torch.no_grad():
        return {"ce": _plain_ce, "norm": _plain_norm, "adamw": _plain_adamw}[op](state)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_ce(s):
    c = s["case"]
    x, w, target = s["x"].double(), s["w"].double(), s["target"]
    n, v = c["n"], c["v"]
    bias = torch.zeros(v, dtype=torch.float64, device=DEV) if s["bias"] is None else s["bias"].double()
    wt = torch.ones(v, dtype=torch.float64, device=DEV) if s["weight"] is None else s["weight"].double()
    rows = torch.nonzero(target != IGNORE)[:, 0]
    share = torch.zeros(n, dtype=torch.float64, device=DEV)
    share[rows] = wt[target[rows]]
    nll, dx, dw, db = torch.zeros_like(share), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
    for part in torch.split(rows, max(1, (1 << 28) // v)):              # rows at a time: the logits take 8 bytes each
        z = torch.addmm(bias, x[part], w.t())
        z = z - torch.logsumexp(z, 1, keepdim=True)
        hot = target[part]
        nll[part] = -z.gather(1, hot[:, None])[:, 0] * share[part]
        if c["train"]:
            z.exp_()
            z[torch.arange(len(part), device=DEV), hot] -= 1.0
            z *= (share[part] / share.sum())[:, None]
            dx[part] = z @ w
            dw += z.t() @ x[part]
            db += z.sum(0)
    if not c["train"]:
        return {"loss": nll}
    out = {"loss": nll.sum() / share.sum(), "dx": dx, "dw": dw}
    if s["bias"] is not None:
        out["dbias"] = db
    return out


def _exact_norm(s):
    """Through torch's automatic differentiation in 64 bits, where the plain form has the gradients written out."""
    c = s["case"]
    t = {k: None if s[k] is None else s[k].double().requires_grad_(c["train"]) for k in NORM_INPUTS}

    def normed(z, weight, bias):
        if c["kind"] == "layer":
            return torch.nn.functional.layer_norm(z, z.shape[-1:], weight, bias, 1e-5)
        z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-5) * weight
        return z if bias is None else z + bias

    u = t["b"] if t["post_weight"] is None else normed(t["b"], t["post_weight"], t["post_bias"])
    if t["scale"] is not None:
        u = u * t["scale"]
    if t["gate"] is not None:
        u = u * {"sigmoid": torch.sigmoid, "tanh": torch.tanh, "identity": lambda z: z}[c["act"]](t["gate"])
    y = t["r"] + u
    seen = y + (y.detach().to(s["r"].dtype).double() - y.detach())     # the next block reads the rounded stream
    h = normed(seen, t["norm_weight"], t["norm_bias"])
    out = {"y": y.detach(), "h": h.detach()}
    if c["train"]:
        leaf = {k: v for k, v in t.items() if v is not None}
        grads = torch.autograd.grad([y, h], list(leaf.values()), [s["dy"].double(), s["dh"].double()])
        out.update({"d" + k: g for k, g in zip(leaf, grads)})
    return out


def _exact_adamw(s):
    """One step in 64 bits.  The codes of the 8-bit moments are given as the unrounded values that they round."""
    c, k = s["case"], s["step"] + 1
    b1, b2 = BETAS
    p = (s["flat"] if s["master"] is None else s["master"]).double()
    g = s["grad"].double()
    if s["clip"]:
        g = g * min(1.0, s["clip"] / (float(torch.linalg.vector_norm(g)) + 1e-6))
    if c["bits"] == 8:
        sc = s["scales"].double().repeat_interleave(BLOCK, dim=1)
        m, v = s["m"].double() * sc[0], (s["v"].double() * sc[1]) ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    for at, n, d in zip(s["starts"], s["sizes"], s["decay"]):
        p[at:at + n] *= 1 - LR * d
    p = p - LR * (m / (1 - b1 ** k)) / (torch.sqrt(v / (1 - b2 ** k)) + EPS)
    out = {"flat": p, "master": p if s["master"] is not None else None, "m": m, "v": v, "scales": None}
    if c["bits"] == 8:
        mb, ub = m.view(-1, BLOCK), v.sqrt().view(-1, BLOCK)
        top = torch.stack((mb.abs().amax(1), ub.amax(1)))
        inv = torch.where(top > 0, 448 / top, torch.zeros_like(top))
        out.update(m=(mb * inv[0][:, None]).view(-1), v=(ub * inv[1][:, None]).view(-1), scales=top / 448)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"ce": _exact_ce, "norm": _exact_norm, "adamw": _exact_adamw}[case["op"]](s)
