"""The norms around a residual block with its gate and residual scale (vae_amd.functional.gated_residual_norm,
modules.GatedResidualNorm; C ABI vae_gated_norm_fwd / _bwd) against torch's automatic differentiation in 64 bits.

Tolerances.  A sum of D terms in 32 bits, by threads of at most 32 values and then by a tree, is off by at most about
(32 + 2 log2 D) 2^-24 of the sum of magnitudes, and some twenty more roundings follow: 2e-5 of the largest value around covers
them for D up to 16384 and sums over thousands of rows.  Rounding to 16 bits adds finfo.eps / 2 of the value.  The second
output reads the first after that rounding: the oracle takes the rounded stream that the kernel wrote (checked by itself
against the exact one), since a value next to the middle of two neighbours may go to either, which moves the column sums of a
few rows by finfo.eps of a term.  The gradients of the vectors are sums over the rows that may cancel: a thread adds its rows
one by one (fewer than 32 here), at most 64 partial sums follow and 16 of these, each step off by 2^-24 of a partial
sum: 128 * 2^-24 of the sum of the magnitudes of the rows' shares is allowed on top."""
import ctypes as C

import pytest
import torch

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NAMES = ("r", "b", "gate", "post_weight", "post_bias", "scale", "norm_weight", "norm_bias")


# ---------------------------------------------------------------------------------------------------- on the CPU
def test_refusals_of_the_c_entry():
    from vae_amd import _lib
    lib = _lib.load()
    ok = dict(N=4, D=8, dtype=0, kind=0, gate_mode=0, act=0, eps=1e-5, r=4096, ld_r=8, b=8192, ld_b=8, y=16384, h=32768)

    def refused(msg, bwd=False, ws=None, n=0, **k):
        a = _lib.GatedNorm(**{**ok, **k})
        rc = lib.vae_gated_norm_bwd(C.byref(a), ws, n, None) if bwd else lib.vae_gated_norm_fwd(C.byref(a), None)
        assert rc == 1 and msg in lib.vae_last_error().decode(), lib.vae_last_error()

    refused("dtype", dtype=3)
    refused("D <=", D=0)
    refused("D <=", D=16385)
    refused("N >= 0", N=-1)
    refused("unknown norm", kind=2)
    refused("gate mode", gate_mode=3)
    refused("activation", act=3)
    refused("eps", eps=-1.0)
    refused("post_bias", post_bias=4096)
    refused("null pointer", b=None)
    refused("null pointer", gate_mode=1)
    refused("null pointer", h=None)
    refused("aligned", r=4098)
    refused("vector is not aligned", scale=4098)
    refused("vector is not aligned", dtype=1, vectors_f32=1, norm_weight=4098)
    refused("stats", stats=4100)
    refused("null pointer", bwd=True)
    full = dict(stats=65536, dr=4096, db=4096)
    refused("no rows", bwd=True, N=0, **full)
    refused("not there", bwd=True, dpost_weight=4096, **full)
    refused("workspace", bwd=True, dnorm_weight=4096, **full)
    assert lib.vae_gated_norm_fwd(C.byref(_lib.GatedNorm(**{**ok, "N": 0})), None) == 0
    assert lib.vae_gated_norm_fwd(None, None) == 1


def test_refusals_of_the_python_entry():
    from vae_amd.functional import gated_residual_norm
    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        gated_residual_norm(x, x)
    with pytest.raises(ValueError, match="kind"):
        gated_residual_norm(x, x, kind="batch")
    with pytest.raises(ValueError, match="gate_act"):
        gated_residual_norm(x, x, gate_act="relu")
    with pytest.raises(ValueError, match="r is"):
        gated_residual_norm(x[:2], x)
    with pytest.raises(ValueError, match="gate"):
        gated_residual_norm(x, x, x[:, :3])
    with pytest.raises(ValueError, match="gate"):
        gated_residual_norm(x, x, x[:2])
    with pytest.raises(TypeError, match="float64"):
        gated_residual_norm(x.double(), x.double())
    with pytest.raises(TypeError, match="r is"):
        gated_residual_norm(x.half(), x)
    with pytest.raises(TypeError, match="vectors"):
        gated_residual_norm(x, x, scale=torch.zeros(8).half())
    with pytest.raises(TypeError, match="vectors"):
        gated_residual_norm(x.half(), x.half(), scale=torch.zeros(8).half(), norm_weight=torch.zeros(8))
    with pytest.raises(ValueError, match="vector of 8"):
        gated_residual_norm(x, x, scale=torch.zeros(7))
    with pytest.raises(ValueError, match="post_bias"):
        gated_residual_norm(x, x, post_bias=torch.zeros(8))
    with pytest.raises(ValueError, match="16384"):
        gated_residual_norm(torch.zeros(1, 16385), torch.zeros(1, 16385))
    with pytest.raises(ValueError, match="columns"):
        gated_residual_norm(torch.zeros(1, 0), torch.zeros(1, 0))


def test_strides_of_vectors_are_no_reason_to_refuse():
    from vae_amd.functional import gated_residual_norm
    x, v = torch.zeros(3, 8), torch.zeros(8, 2)
    for call in (lambda: gated_residual_norm(x, x, scale=v[:, 0]), lambda: gated_residual_norm(x, x, norm_weight=torch.ones(1).expand(8))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


# ---------------------------------------------------------------------------------------------------- on the GPU
def _inputs(n, d, dtype, gate, post, scale, bias, vec32, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, v = DT[dtype], torch.float32 if vec32 else DT[dtype]
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = dict.fromkeys(NAMES)
    x["r"], x["b"] = (2 * rnd(n, d)).to(t), (rnd(n, d) + 0.5).to(t)
    if gate:
        x["gate"] = rnd(n, d if gate == "full" else 1).to(t)
    x["norm_weight"] = (1 + 0.2 * rnd(d)).to(v)
    if post:
        x["post_weight"] = (1 + 0.2 * rnd(d)).to(v)
    if scale:
        x["scale"] = (0.5 + 0.2 * rnd(d)).to(v)
    if bias:
        x["norm_bias"] = (0.2 * rnd(d)).to(v)
        x["post_bias"] = (0.2 * rnd(d)).to(v) if post else None
    return x, rnd(n, d).to(t), rnd(n, d).to(t)


def _oracle(x, dy, dh, kind, act, seen, eps=1e-5):
    """(outputs, gradients) in 64 bits; ``seen``: the rounded first output, from which the second is formed."""
    # a vector as one row of its own for every row: the gradient's terms, and so the sum of their magnitudes
    t = {k: None if v is None else (v.detach().double() if v.dim() > 1 else v.detach().double().expand(x["b"].shape).clone()).requires_grad_()
         for k, v in x.items()}

    def norm(z, w, b):
        z = z - z.mean(-1, keepdim=True) if kind == "layer" else z
        z = z / (z.square().mean(-1, keepdim=True) + eps).sqrt()
        z = z if w is None else z * w
        return z if b is None else z + b

    u = norm(t["b"], t["post_weight"], t["post_bias"]) if t["post_weight"] is not None else t["b"]
    if t["scale"] is not None:
        u = u * t["scale"]
    if t["gate"] is not None:
        u = u * {"sigmoid": torch.sigmoid, "tanh": torch.tanh, "identity": lambda z: z}[act](t["gate"])
    y = t["r"] + u
    h = norm(y + (seen.double() - y.detach()), t["norm_weight"], t["norm_bias"])
    leaf = {k: v for k, v in t.items() if v is not None}
    loss = sum((o * g.double()).sum() for o, g in ((y, dy), (h, dh)) if g is not None)
    grads = torch.autograd.grad(loss, list(leaf.values()), allow_unused=True)
    full = {k: torch.zeros_like(v) if g is None else g for (k, v), g in zip(leaf.items(), grads)}
    return (y.detach(), h.detach()), {k: (g.sum(0), g.abs().sum(0)) if x[k].dim() == 1 else (g, 0.0) for k, g in full.items()}


def _close(name, got, ref, dtype):
    ref, mag = ref if isinstance(ref, tuple) else (ref, 0.0)
    ref = ref.double()
    assert got.shape == ref.shape, name
    if not ref.numel():
        return
    eps = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    err = (got.double() - ref).abs()
    tol = 2e-5 * ref.abs().max() + eps * ref.abs() + 128 * 2.0 ** -24 * mag + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert not bool((err > tol).any()), (name, float((err - tol).max()), float(ref.abs().max()))


def _run(x, dy, dh, kind, act, eps=1e-5):
    from vae_amd.functional import gated_residual_norm
    leaf = {k: None if v is None else v.detach().requires_grad_() for k, v in x.items()}
    y, h = gated_residual_norm(leaf["r"], leaf["b"], leaf["gate"], **{k: leaf[k] for k in NAMES[3:]}, kind=kind, gate_act=act, eps=eps)
    on = {k: v for k, v in leaf.items() if v is not None}
    pairs = [(o, g) for o, g in ((y, dy), (h, dh)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(on.values()), [g for _, g in pairs], allow_unused=True)
    return (y.detach(), h.detach()), dict(zip(on, grads))


WIDTHS = [1, 2, 7, 8, 64, 255, 256, 257, 512, 513, 1000, 1531, 2048, 2049, 4096, 4100, 8192, 8195, 16384]


@pytest.mark.gpu
@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_widths(d, dtype, kind):
    """Every path over the row, odd widths, more rows than workgroups now and then."""
    n = {1: 4099, 255: 2051, 2049: 1100, 8195: 300}.get(d, 5)
    # two columns under LayerNorm are +-1 whatever they were: the gradient is a difference of equal numbers, left to the formula
    post = not (kind == "layer" and d <= 2)
    x, dy, dh = _inputs(n, d, dtype, "full", post, True, True, d % 2 == 1, seed=d)
    out, grads = _run(x, dy, dh, kind, "sigmoid")
    ref, rgrads = _oracle(x, dy, dh, kind, "sigmoid", out[0])
    _close("y", out[0], ref[0], DT[dtype])
    if d <= 2 and kind == "layer":
        assert bool(torch.isfinite(out[1]).all()) and all(bool(torch.isfinite(g).all()) for g in grads.values())
        return
    _close("h", out[1], ref[1], DT[dtype])
    for k, g in grads.items():
        _close(k, g, rgrads[k], g.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [None, "row", "full"])
@pytest.mark.parametrize("act", ["identity", "sigmoid", "tanh"])
@pytest.mark.parametrize("post,scale,bias", [(False, False, False), (True, False, True), (False, True, True), (True, True, False)])
@pytest.mark.parametrize("d,dtype", [(96, "fp32"), (700, "bf16"), (1200, "fp16")])
def test_parts(gate, act, post, scale, bias, d, dtype):
    x, dy, dh = _inputs(33, d, dtype, gate, post, scale, bias, False, seed=7)
    out, grads = _run(x, dy, dh, "layer", act)
    ref, rgrads = _oracle(x, dy, dh, "layer", act, out[0])
    for name, a, b in zip(("y", "h"), out, ref):
        _close(name, a, b, DT[dtype])
    assert set(grads) == set(rgrads)
    for k, g in grads.items():
        _close(k, g, rgrads[k], DT[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["y", "h"])
def test_one_output_used_and_no_affine(which):
    x, dy, dh = _inputs(9, 300, "fp32", "row", True, True, True, False, seed=3)
    x["norm_weight"] = x["norm_bias"] = None
    dy, dh = (dy, None) if which == "y" else (None, dh)
    out, grads = _run(x, dy, dh, "rms", "tanh")
    _, ref = _oracle(x, dy, dh, "rms", "tanh", out[0])
    for k, g in grads.items():
        _close(k, g, ref[k], torch.float32)


@pytest.mark.gpu
def test_strides_leading_dims_broadcasts_and_empty():
    from vae_amd.functional import gated_residual_norm
    from vae_amd.modules import GatedResidualNorm
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(6, 4, 50, generator=g, device="cuda")
    r, b = wide[:, :, 1:34], wide[:, :, 7:40].transpose(0, 1).contiguous().transpose(0, 1)     # odd offsets, row strides of their own
    gate = torch.randn(6, 4, 1, generator=g, device="cuda")
    y, h = gated_residual_norm(r, b, gate, kind="layer")
    y2, h2 = gated_residual_norm(r.contiguous().view(24, 33), b.contiguous().view(24, 33), gate.view(24, 1), kind="layer")
    assert torch.equal(y.view(24, 33), y2) and torch.equal(h.view(24, 33), h2) and y.shape == r.shape
    row = torch.randn(33, generator=g, device="cuda").requires_grad_()                    # one row for all: its gradient is the sum
    gt = torch.randn(1, 33, generator=g, device="cuda").requires_grad_()
    y3, h3 = gated_residual_norm(row.expand(24, 33), b.reshape(24, 33), gt.expand(24, 33), kind="rms")
    (y3.sum() + (h3 * y2).sum()).backward()                                                # dy is an expanded scalar
    x = dict.fromkeys(NAMES)
    x.update(r=row.detach().expand(24, 33), b=b.reshape(24, 33), gate=gt.detach().expand(24, 33))
    _, ref = _oracle(x, torch.ones(24, 33, device="cuda"), y2, "rms", "sigmoid", y3.detach())
    _close("r", row.grad, ref["r"][0].sum(0), torch.float32)
    _close("gate", gt.grad, ref["gate"][0].sum(0, keepdim=True), torch.float32)
    m = GatedResidualNorm(33).cuda()
    e = torch.zeros(0, 33, device="cuda", requires_grad=True)
    y, h = m(e, e.clone())
    (y.sum() + h.sum()).backward()
    assert e.grad.shape == (0, 33) and not bool(m.norm_weight.grad.any()) and not bool(m.scale.grad.any())


@pytest.mark.gpu
def test_differences():
    """The gradient against central differences of the forward pass in the direction of itself (fp32: steps of 2^-6 lose about
    2^-24 / 2^-6 of the values to cancellation and 2^-12 of the second derivative's share: 1e-2 is wide)."""
    from vae_amd.functional import gated_residual_norm
    x, dy, dh = _inputs(3, 40, "fp32", "full", True, True, True, False, seed=5)
    _, grads = _run(x, dy, dh, "layer", "sigmoid")

    def value(v):
        y, h = gated_residual_norm(v["r"], v["b"], v["gate"], **{k: v[k] for k in NAMES[3:]}, kind="layer")
        return float((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum())

    for k, g in grads.items():
        dirn = g / g.norm()
        step = 2.0 ** -6
        up, down = value({**x, k: x[k] + step * dirn}), value({**x, k: x[k] - step * dirn})
        assert abs((up - down) / (2 * step) / float(g.norm()) - 1) < 1e-2, k


@pytest.mark.gpu
def test_repeats_other_stream_and_graph():
    from vae_amd.functional import gated_residual_norm
    x, dy, dh = _inputs(700, 1000, "bf16", "full", True, True, True, False, seed=11)
    first = _run(x, dy, dh, "rms", "sigmoid")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _run(x, dy, dh, "rms", "sigmoid")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first[0], again[0])) and all(torch.equal(first[1][k], again[1][k]) for k in first[1])
    static = {k: None if v is None else v.clone() for k, v in x.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = _run(static, dy, dh, "rms", "sigmoid")
    for seed in (12, 13, 14):
        new = _inputs(700, 1000, "bf16", "full", True, True, True, False, seed=seed)[0]
        for k, v in new.items():
            if v is not None:
                static[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        want = _run(new, dy, dh, "rms", "sigmoid")
        assert all(torch.equal(a, b) for a, b in zip(out, want[0])) and all(torch.equal(grads[k], want[1][k]) for k in grads)
        y, h = gated_residual_norm(new["r"], new["b"])                 # eager work between the replays
        del y, h


@pytest.mark.gpu
def test_non_finite_rows_stay_in_their_rows():
    from vae_amd.functional import gated_residual_norm
    g = torch.Generator(device="cuda").manual_seed(2)
    r, b = torch.randn(6, 300, generator=g, device="cuda"), torch.randn(6, 300, generator=g, device="cuda")
    clean = gated_residual_norm(r, b, kind="layer", post_weight=torch.ones(300, device="cuda"))
    b[2, 5], r[4, 299] = float("nan"), float("inf")
    got = gated_residual_norm(r, b, kind="layer", post_weight=torch.ones(300, device="cuda"))
    for c, o in zip(clean, got):
        assert torch.equal(c[[0, 1, 3, 5]], o[[0, 1, 3, 5]])
        assert bool(torch.isnan(o[2]).all())
    assert bool(torch.isinf(got[0][4, 299])) and not bool(torch.isfinite(got[1][4]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("d", [40, 1000])
def test_gradients_of_vectors_that_are_taken_as_one_or_zero(d):
    """The C entry gives them as well: the gradient of an absent bias of the second norm is the sum of dh over the rows."""
    from vae_amd import _lib
    lib, n = _lib.load(), 9
    x = _inputs(n, d, "fp32", None, False, False, False, False, seed=3)[0]
    from vae_amd import ops
    y, h, stats = ops.gated_norm_fwd(x["r"], x["b"])
    dh = torch.randn(n, d, device="cuda")
    dr, db, out = torch.empty_like(y), torch.empty_like(y), torch.full((3, d), float("nan"), device="cuda")
    nbytes = lib.vae_gated_norm_workspace_bytes(n, d, 0)
    ws = torch.full((nbytes // 4,), float("nan"), device="cuda")
    a = _lib.GatedNorm(N=n, D=d, dtype=0, kind=0, gate_mode=0, act=0, eps=1e-5, r=x["r"].data_ptr(), ld_r=d, b=x["b"].data_ptr(), ld_b=d,
                       y=y.data_ptr(), h=h.data_ptr(), stats=stats.data_ptr(), dh=dh.data_ptr(), ld_dh=d, dr=dr.data_ptr(),
                       db=db.data_ptr(), dnorm_weight=out[0].data_ptr(), dnorm_bias=out[1].data_ptr(), dscale=out[2].data_ptr())
    assert lib.vae_gated_norm_bwd(C.byref(a), ws.data_ptr(), nbytes, None) == 0
    torch.cuda.synchronize()
    ny = y.double() / (y.double().square().mean(1, keepdim=True) + 1e-5).sqrt()
    for got, ref in ((out[0], dh.double() * ny), (out[1], dh.double()), (out[2], dr.double() * x["b"].double())):
        tol = 2e-5 * float(ref.abs().max()) + 128 * 2.0 ** -24 * ref.abs().sum(0)        # (as the gradients of the vectors above)
        assert bool(((got.double() - ref.sum(0)).abs() <= tol).all())


@pytest.mark.gpu
def test_strided_vectors():
    from vae_amd.functional import gated_residual_norm
    x, dy, dh = _inputs(9, 300, "bf16", "full", True, True, True, False, seed=3)
    want, grads = _run(x, dy, dh, "layer", "sigmoid")
    wide = torch.stack([x[k] for k in NAMES[3:]], 1).requires_grad_()                       # one parameter holds them side by side
    y, h = gated_residual_norm(x["r"], x["b"], x["gate"], **{k: wide[:, i] for i, k in enumerate(NAMES[3:])}, kind="layer")
    torch.autograd.backward([y, h], [dy, dh])
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    for i, k in enumerate(NAMES[3:]):
        assert torch.equal(wide.grad[:, i], grads[k]), k
    s = torch.full((1,), 0.5, device="cuda", dtype=torch.bfloat16, requires_grad=True)      # one value for all columns
    x["scale"] = torch.full((300,), 0.5, device="cuda", dtype=torch.bfloat16)
    _, grads = _run(x, dy, dh, "layer", "sigmoid")
    y, h = gated_residual_norm(x["r"], x["b"], x["gate"], scale=s.expand(300), **{k: x[k] for k in NAMES[3:] if k != "scale"}, kind="layer")
    torch.autograd.backward([y, h], [dy, dh])
    total = grads["scale"].double()
    assert abs(float(s.grad) - float(total.sum())) <= 2.0 ** -7 * float(total.abs().sum())  # (torch adds 300 of them in bf16's terms)


@pytest.mark.gpu
@pytest.mark.parametrize("d,n", [(700, 4500), (1000, 4500), (2000, 2300), (1531, 2100), (5000, 800), (8192, 700), (9001, 600), (16384, 520)])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kind,gate,bias", [("layer", "full", True), ("rms", "row", False)])
def test_workgroups_that_walk_over_several_rows(d, n, dtype, kind, gate, bias):
    """More rows than workgroups on two, four, eight and sixteen waves: loads ahead of their row, and column sums over rows."""
    x, dy, dh = _inputs(n, d, dtype, gate, True, True, bias, d % 2 == 1, seed=d)
    out, grads = _run(x, dy, dh, kind, "tanh")
    ref, rgrads = _oracle(x, dy, dh, kind, "tanh", out[0])
    for name, a, b in zip(("y", "h"), out, ref):
        _close(name, a, b, DT[dtype])
    for k, g in grads.items():
        _close(k, g, rgrads[k], g.dtype)


@pytest.mark.gpu
def test_the_kernel_entries_beside_autograd():
    """ops.gated_norm_fwd / gated_norm_bwd give what the differentiable form gives, and only what is asked for."""
    from vae_amd import ops
    x, dy, dh = _inputs(33, 300, "bf16", "full", True, True, True, False, seed=4)
    out, grads = _run(x, dy, dh, "layer", "sigmoid")
    vectors = {k: x[k] for k in NAMES[3:]}
    y, h, stats = ops.gated_norm_fwd(x["r"], x["b"], x["gate"], **vectors, kind="layer")
    assert torch.equal(y, out[0]) and torch.equal(h, out[1])
    got = ops.gated_norm_bwd(dy, dh, y, x["b"], stats, x["gate"], **vectors, kind="layer")
    assert set(got) == set(grads) and all(torch.equal(got[k], grads[k]) for k in grads)
    some = ops.gated_norm_bwd(dy, dh, y, x["b"], stats, x["gate"], **vectors, kind="layer", want=("scale",))
    assert set(some) == {"r", "b", "scale"} and all(torch.equal(some[k], grads[k]) for k in some)
