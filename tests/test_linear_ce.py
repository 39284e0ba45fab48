"""Cross entropy of a linear head without its logits (vae_amd.losses.linear_cross_entropy; C ABI vae_linear_ce_fwd / _bwd)
against the definition in 64 bits.

Tolerances.  Logits are sums of D products in 32 bits: off by a few 2^-24 of |x| |w| (norms); with the rows made here (logits of
a few units) the loss is held to 2e-6 of itself plus 1e-6.  A gradient element is a sum of terms whose d has been rounded
to the operands' type (finfo.eps / 2 of each) and that is rounded itself: its error is at most eps (the sum of the magnitudes of
its terms) / 2 plus eps / 2 of the result; the bound takes the matrices |d| |w| and |d|^T |x| for the first.  fp32: 32 * 2^-24 of
the same sums (three-term products are exact to 2^-24, sums run over thousands of terms in blocks).  For every type p itself is
off by p times the error of z - lse, two values of up to Z = max |z| that are rounded in 32 bits a few times each, 8 + 4 Z in
units of 2^-24.  z is a running sum besides: six term products for every 16 of D, S = 6 D / 16 roundings, each of at most half a
unit in the last place of a partial sum of some Z at most, that is 2^-24 Z, spread evenly on both sides: a standard deviation of
2^-24 Z sqrt(S / 3), of which the 10^7 logits of a case see 5.2, 3 sqrt(S) Z 2^-24.  (At D = 300 and Z = 5.7 a logit of 5.4 was off
by 45 * 2^-24, half an ulp of 4 * 2^-24 eleven times over, where 8 + 4 Z is 31; S is 113.)  At the target p - 1 keeps the error of p
however small p - 1 is, so this term takes the matrices of p and not those of d."""
import ctypes as C
import math

import pytest
import torch

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------- on the CPU
def test_refusals_of_the_c_entry():
    from vae_amd import _lib
    lib = _lib.load()
    ok = dict(N=4, D=8, V=160, dtype=1, x=4096, ldx=8, w=8192, ldw=8, target=16384, ignore_index=-100)

    def refused(msg, fwd=True, reduction=2, loss=4096, state=4096, ws=4096, n=1 << 40, dx=4096, db=None, **k):
        a = _lib.LinearCE(**{**ok, **k})
        rc = lib.vae_linear_ce_fwd(C.byref(a), reduction, loss, state, ws, n, None) if fwd else \
            lib.vae_linear_ce_bwd(C.byref(a), reduction, loss, state, dx, None, db, ws, n, None)
        assert rc == 1 and msg in lib.vae_last_error().decode(), lib.vae_last_error()

    for fwd in (True, False):
        refused("dtype", fwd, dtype=3)
        refused("at least 1", fwd, N=0)
        refused("at least 1", fwd, D=0)
        refused("at least 1", fwd, V=0)
        refused("at most", fwd, V=(1 << 24) + 1)
        refused("tiles", fwd, V=1 << 24, N=1 << 24)
        refused("128 classes", fwd, V=1 << 20, N=1 << 18)
        refused("128 columns", fwd, D=1 << 20, N=1 << 18, ldw=1 << 20, ldx=1 << 20)
        refused("128 columns", fwd, D=1 << 20, V=1 << 18, ldw=1 << 20, ldx=1 << 20)
        refused("null pointer", fwd, x=None)
        refused("null pointer", fwd, w=None)
        refused("null pointer", fwd, target=None)
        refused("stride", fwd, ldw=7)
        refused("stride is too large", fwd, ldw=1 << 22)
        refused("aligned to its element", fwd, w=8193)
        refused("unknown reduction", fwd, reduction=3)
        refused("null pointer", fwd, state=None)
        refused("null pointer", fwd, loss=None)
        refused("workspace", fwd, ws=None)
        refused("workspace", fwd, n=100)
        refused("workspace", fwd, ws=4100)
    refused("null pointer", False, dx=None)
    refused("not there", False, db=4096)
    assert lib.vae_linear_ce_workspace_bytes(C.byref(_lib.LinearCE(**{**ok, "N": 0})), 0) == -1
    # the backward workspace is bounded: half a gigabyte of logit gradients, whatever the vocabulary
    big = _lib.LinearCE(**{**ok, "N": 8192, "D": 4096, "V": 1 << 20, "ldx": 4096, "ldw": 4096})
    assert lib.vae_linear_ce_workspace_bytes(C.byref(big), 1) < (512 << 20) + 4 * 8192 * 4096 + 2 * 8192 * 4096 + (1 << 20)


def _workspace_bound(n, d, v, dtype, bias, packed, backward):
    """The parts that include/vae_amd.h lists, each rounded up to 256 bytes."""
    up = lambda a, b: -(-a // b) * b  # noqa: E731
    e, rows, cols, part = 6 if dtype == 0 else 2, up(n, 256), up(d, 64), 134_217_728 + 256
    total = e * rows * cols + (e * v * cols if packed else 0) + 12 * 256
    if not backward:
        return total + max(8 * rows * (up(v, 128) // 128), part) + 12 * rows
    classes = min(up(v, 256), max(256, (512 << 20) // (e * rows)))
    total += e * rows * classes + 8 * rows + (2 * rows * cols if dtype == 2 else 0)
    total += (max(4 * classes * (rows // 128), 4 * classes * (rows // 8) if rows * classes <= 1 << 26 else 0) if bias else 0)
    return total + max(part, 4 * n * d) + part + part


def test_workspaces_are_what_the_header_says():
    """Random sizes up to the limits, long batches among them (which hold 256 classes however many bytes these take)."""
    import random
    from vae_amd import _lib
    lib, rng, seen = _lib.load(), random.Random(1), 0
    sizes = [(1 << 21, 64, 1000), (1 << 20, 4096, 500), (1 << 24, 1, 100), (1, 1 << 20, 7), (64, 1 << 20, 1000), (8192, 4096, 1 << 20)]
    sizes += [tuple(int(2 ** rng.uniform(0, k)) for k in (24, 20, 24)) for _ in range(3000)]
    for n, d, v in sizes:
        tiles = [-(-a // 128) * -(-b // 128) for a, b in ((n, v), (n, d), (v, d))]
        if max(tiles) >= 1 << 24:
            continue
        seen += 1
        for dtype in range(3):
            for bias in (None, 4096):
                for backward in (0, 1):
                    ldw = d + rng.randrange(2)
                    a = _lib.LinearCE(N=n, D=d, V=v, dtype=dtype, x=4096, ldx=d, w=8192, ldw=ldw, target=4096, bias=bias, ignore_index=-100)
                    if ldw >= 1 << 22:
                        continue
                    got = lib.vae_linear_ce_workspace_bytes(C.byref(a), backward)
                    packed = dtype == 0 or d % 8 != 0 or ldw % 8 != 0
                    assert 0 <= got <= _workspace_bound(n, d, v, dtype, bias, packed, backward), (n, d, v, dtype, bias, backward, got)
    assert seen > 1000
    long = _lib.LinearCE(N=1 << 21, D=64, V=1000, dtype=1, x=4096, ldx=64, w=8192, ldw=64, target=4096, ignore_index=-100)
    assert lib.vae_linear_ce_workspace_bytes(C.byref(long), 1) > (1 << 30)               # 256 classes of 2^21 rows


def test_refusals_of_the_python_entry():
    from vae_amd.losses import linear_cross_entropy
    x, w, t = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_cross_entropy(x, w, t)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_cross_entropy(x[:0], w, t[:0])
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(ValueError, match="target"):
        linear_cross_entropy(x, w, t[:2])
    with pytest.raises(ValueError, match="int64"):
        linear_cross_entropy(x, w, t.int())
    with pytest.raises(ValueError, match="x must be"):
        linear_cross_entropy(x, w[:, :7], t)
    with pytest.raises(TypeError, match="float64"):
        linear_cross_entropy(x.double(), w.double(), t)
    with pytest.raises(TypeError, match="w is"):
        linear_cross_entropy(x, w.half(), t)
    with pytest.raises(TypeError, match="bias is"):
        linear_cross_entropy(x, w, t, bias=torch.zeros(5).half())
    with pytest.raises(TypeError, match="weight is"):
        linear_cross_entropy(x, w, t, weight=torch.zeros(5).double())
    with pytest.raises(ValueError, match="not differentiable"):
        linear_cross_entropy(x, w, t, weight=torch.zeros(5, requires_grad=True))
    with pytest.raises(ValueError, match="vector of 5"):
        linear_cross_entropy(x, w, t, weight=torch.zeros(4))


def test_strides_are_no_reason_to_refuse():
    """Targets, biases and class weights of any stride, and a column of weights that is one value: only the missing GPU stops them."""
    from vae_amd.losses import linear_cross_entropy
    x, w, t = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(6, dtype=torch.int64)[::2]
    for call in (lambda: linear_cross_entropy(x, w, t), lambda: linear_cross_entropy(x, w, t, bias=torch.zeros(10)[::2]),
                 lambda: linear_cross_entropy(x, w, t, weight=torch.zeros(1).expand(5)),
                 lambda: linear_cross_entropy(x[:, :1], torch.zeros(1, 1).expand(5, 1), t)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def _rms(t):
    return float(t.double().square().mean().sqrt())


def _expected_loss_error(z_t, lse, loss, steps):
    """Root mean square over the rows of what the roundings of a loss come to, with a quarter to spare.

    z_t: a running sum over ``steps`` of matrix instructions, each of which rounds it once or twice.  A rounding has a standard
    deviation of ulp / sqrt(12), over the mantissas 2^-25.2 of the value; the mean square of the partial sums is at most half that
    of the whole, whether it grows steadily (a third) or as a random walk (a half): 2^-25.2 sqrt(2 steps / 2) rms(z_t).
    Else: five roundings of lse's size (maximum, scaled logit and its offset, logarithm, sum), two of z_t's and one of the
    loss's, of 2^-24 / sqrt(3) each."""
    sums = 1.25 * 2.0 ** -25.2 * steps ** 0.5 * _rms(z_t)
    return (sums ** 2 + (5 * _rms(lse) ** 2 + 2 * _rms(z_t) ** 2 + _rms(loss) ** 2) * 2.0 ** -48 / 3) ** 0.5


def _three_terms(t):
    h = t.bfloat16().float()
    m = (t - h).bfloat16().float()
    return h.double(), m.double(), (t - h - m).bfloat16().double()


@pytest.mark.parametrize("d", [64, 512, 4096])
def test_the_expected_error_shows_a_missing_product_of_terms(d):
    """fp32 operands as three bf16 terms: without even the smallest of the six products the loss is off by more than that."""
    g = torch.Generator().manual_seed(0)
    n, v = 1000, 500
    w = torch.randn(v, d, generator=g) / d ** 0.5
    t = torch.randint(0, v, (n,), generator=g)
    x = torch.randn(n, d, generator=g) + 2 * w[t]
    z = x.double() @ w.double().t()
    pick = lambda q: (q.logsumexp(1), q.gather(1, t[:, None])[:, 0])  # noqa: E731
    lse, z_t = pick(z)
    bound = _expected_loss_error(z_t, lse, lse - z_t, 6 * d / 32)
    xs, ws = _three_terms(x), _three_terms(w)
    six = [(0, 0), (0, 1), (1, 0), (0, 2), (2, 0), (1, 1)]
    for left_out in (None, (1, 1), (0, 2), (2, 0)):
        a, b = pick(sum(xs[i] @ ws[j].t() for i, j in six if (i, j) != left_out))
        assert (_rms(a - b - lse + z_t) > bound) == (left_out is not None), left_out


def test_class_weights_keep_their_bits():
    """A head that is moved to 16 bits takes its parameters along, not the class weights."""
    from vae_amd.losses import LinearCrossEntropyLoss
    c = torch.rand(40)
    for to in (lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: torch.nn.Sequential(m).half()[0]):
        m = to(LinearCrossEntropyLoss(32, 40, weight=c.clone()))
        assert m.linear.weight.dtype != torch.float32 and m.weight.dtype == torch.float32 and torch.equal(m.weight, c)
    assert m.to("meta").weight.device.type == "meta" and LinearCrossEntropyLoss(32, 40).half().weight is None


# ---------------------------------------------------------------------------------------------------- on the GPU
def _inputs(n, d, v, dtype, bias, weight, ignored, seed, off=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DT[dtype]
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = (rnd(v, d + off) / d ** 0.5).to(t)[:, off:]
    target = torch.randint(0, v, (n,), generator=g, device="cuda")
    x = torch.zeros(n, d + off, dtype=t, device="cuda")[:, off:]
    x.copy_(rnd(n, d) + 2 * w[target].float())
    if ignored:
        target[torch.rand(n, generator=g, device="cuda") < ignored] = -100
    return dict(x=x, w=w, target=target, bias=(0.5 * rnd(v)).to(t) if bias else None,
                weight=0.1 + torch.rand(v, generator=g, device="cuda") if weight else None)


def _oracle(s, reduction, up=None, ignore=-100):
    """(loss, {grad: (value, sum of the magnitudes of its terms, error that p brings)}) in 64 bits."""
    x, w, t = s["x"].double(), s["w"].double(), s["target"]
    z = x @ w.t() + (0 if s["bias"] is None else s["bias"].double())
    kept = t != ignore
    at = t.clamp(min=0)
    cw = kept.double() * (1 if s["weight"] is None else s["weight"].double()[at])
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    nll = torch.where(kept, -logp.gather(1, at[:, None])[:, 0] * cw, torch.zeros_like(cw))
    loss = {"none": nll, "sum": nll.sum(), "mean": nll.sum() / cw.sum()}[reduction]
    g = cw * (1.0 if up is None else up.double())
    g = g / cw.sum() if reduction == "mean" else g
    d = logp.exp()
    per_z = max(4.0, 3 * (6 * x.shape[1] / 16) ** 0.5)
    p = torch.where(kept[:, None], d * g[:, None], torch.zeros_like(d)) * (8 + per_z * z.abs().amax()) * 2.0 ** -24
    d.scatter_add_(1, at[:, None], -torch.ones_like(d[:, :1]))
    d = torch.where(kept[:, None], d * g[:, None], torch.zeros_like(d))
    clean = torch.where(kept[:, None], x, torch.zeros_like(x))
    return loss, {"x": (d @ w, d.abs() @ w.abs(), p @ w.abs()), "w": (d.t() @ clean, d.abs().t() @ clean.abs(), p.t() @ clean.abs()),
                  "bias": (d.sum(0), d.abs().sum(0), p.sum(0))}


def _check(s, reduction, got_loss, grads, up=None):
    loss, ref = _oracle(s, reduction, up)
    assert got_loss.dtype == torch.float32
    err = (got_loss.double() - loss).abs()
    assert bool((err <= 2e-6 * loss.abs() + 1e-6 * (1 if reduction != "sum" else len(s["x"]))).all()), float(err.max())
    t = s["x"].dtype
    eps = torch.finfo(t).eps / 2
    for k, g in grads.items():
        val, mag, off = ref[k]
        assert g.dtype == t and g.shape == val.shape
        k_len = s["w"].shape[0] if k == "x" else s["x"].shape[0]
        tol = off + max(32.0, 2 * (6 * k_len / 16) ** 0.5) * 2.0 ** -24 * mag + (0 if t == torch.float32 else eps * mag + 1.01 * eps * val.abs())
        if t == torch.float16:
            tol = tol + 2.0 ** -25          # half the smallest subnormal
        bad = (g.double() - val).abs() - tol - 1e-30
        assert float(bad.max()) <= 0, (k, float(bad.max()), float(val.abs().max()))


def _run(s, reduction, up=None, **k):
    from vae_amd.losses import linear_cross_entropy
    leaf = {k: s[k].detach().requires_grad_() for k in ("x", "w", "bias") if s[k] is not None}
    loss = linear_cross_entropy(leaf["x"], leaf["w"], s["target"], bias=leaf.get("bias"), weight=s["weight"], reduction=reduction, **k)
    grads = torch.autograd.grad(loss, list(leaf.values()), up)
    return loss.detach(), dict(zip(leaf, grads))


SHAPES = [(1, 1, 1), (1, 8, 2), (3, 7, 5), (5, 30, 17), (64, 64, 64), (127, 33, 129), (129, 72, 255), (256, 256, 256), (257, 100, 300),
          (2048, 64, 64), (2049, 64, 64), (700, 33, 9), (1, 72, 65), (3, 65, 2), (5000, 16, 20), (256, 32, 65), (255, 65, 64),          (300, 520, 1000), (31, 1000, 4099), (1000, 40, 3), (512, 264, 6000)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v", SHAPES)
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("bias,weight,ignored", [(False, False, 0.0), (True, True, 0.3)])
def test_shapes(n, d, v, dtype, bias, weight, ignored):
    s = _inputs(n, d, v, dtype, bias, weight, ignored, seed=n + d + v)
    s["target"][0] = v - 1
    loss, grads = _run(s, "mean")
    _check(s, "mean", loss, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("reduction", ["none", "sum"])
@pytest.mark.parametrize("d,v", [(96, 700), (20, 12)])
def test_reductions_and_upstream_gradients(dtype, reduction, d, v):
    s = _inputs(200, d, v, dtype, True, True, 0.2, seed=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    up = torch.rand(200, generator=g, device="cuda") * 1e-3 if reduction == "none" else torch.tensor(0.25, device="cuda")
    loss, grads = _run(s, reduction, up)
    _check(s, reduction, loss, grads, up)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v", [(70, 3000, 10), (9, 2500, 3001), (600, 1700, 350), (2, 2000, 1025), (4096, 1565, 252), (1, 4096, 1)])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_few_tiles_over_many_features(n, d, v, dtype, reduction):
    """Logits of a few tiles and long sums, which are split."""
    s = _inputs(n, d, v, dtype, True, True, 0.2 if n > 9 else 0.0, seed=n + v)
    g = torch.Generator(device="cuda").manual_seed(2)
    up = torch.rand(n, generator=g, device="cuda") * 1e-3 if reduction == "none" else torch.tensor(0.5, device="cuda")
    loss, grads = _run(s, reduction, up)
    _check(s, reduction, loss, grads, up)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v", [(1, 70, 130), (2, 4099, 33), (16, 64, 5000), (17, 513, 1001), (33, 300, 2050), (64, 1030, 70), (64, 1030, 2100), (8, 1024, 40000)])
@pytest.mark.parametrize("off,bias,ignored", [(0, True, 0.0), (3, False, 0.4)])
def test_few_rows(n, d, v, off, bias, ignored):
    """fp32 rows in ones, sixteens and their neighbours, W read as it is, on and off 16-byte boundaries."""
    s = _inputs(n, d, v, "fp32", bias, not bias, ignored, seed=n + d, off=off)
    s["target"][n // 2] = v - 1
    loss, grads = _run(s, "mean")
    _check(s, "mean", loss, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v", [(4099, 700, 10), (2500, 1001, 33), (9000, 300, 64), (2049, 2050, 1), (40000, 65, 17)])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("off,bias,ignored,reduction", [(0, True, 0.0, "mean"), (3, False, 0.4, "none")])
def test_few_classes_of_many_rows(n, d, v, dtype, off, bias, ignored, reduction):
    """Heads whose loss reads x as it is, gathered by the rows that count, on and off 16-byte boundaries."""
    s = _inputs(n, d, v, dtype, bias, not bias, ignored, seed=n + d, off=off)
    g = torch.Generator(device="cuda").manual_seed(2)
    up = torch.rand(n, generator=g, device="cuda") * 1e-3 if reduction == "none" else None
    loss, grads = _run(s, reduction, up)
    _check(s, reduction, loss, grads, up)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v,dtype", [(40000, 72, 7000, "bf16"), (14000, 72, 6500, "fp32"), (8000, 520, 7100, "bf16"), (8200, 328, 7000, "fp16")])
def test_large_tiles_and_pieces(n, d, v, dtype):
    """Hundreds of tiles of 256 x 256, few and many steps of K, and (the longest batches) a vocabulary in two pieces."""
    s = _inputs(n, d, v, dtype, True, False, 0.4, seed=9)
    loss, grads = _run(s, "mean")
    _check(s, "mean", loss, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [1, 4, 8])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides_and_offsets(off, dtype):
    """Rows that are views into wider ones, at addresses that are not multiples of 16 bytes."""
    s = _inputs(70, 64, 300, dtype, False, False, 0.0, seed=off, off=off)
    assert s["w"].stride(0) == 64 + off and s["x"].stride(0) == 64 + off
    loss, grads = _run(s, "mean")
    _check(s, "mean", loss, grads)


@pytest.mark.gpu
def test_leading_dims_transposed_weights_and_broadcast_rows():
    from vae_amd.losses import linear_cross_entropy
    s = _inputs(60, 40, 90, "fp32", False, False, 0.0, seed=8)
    x3, t3 = s["x"].view(5, 12, 40), s["target"].view(5, 12)
    want = linear_cross_entropy(s["x"], s["w"], s["target"], reduction="none")
    got = linear_cross_entropy(x3, s["w"].t().contiguous().t(), t3, reduction="none")
    assert got.shape == (5, 12) and torch.equal(got.view(-1), want)
    one = s["x"][:1].detach().requires_grad_()
    linear_cross_entropy(one.expand(60, 40), s["w"], s["target"]).backward()
    s2 = {**s, "x": s["x"][:1].expand(60, 40)}
    val, mag, off = (t.sum(0, keepdim=True) for t in _oracle(s2, "mean")[1]["x"])
    assert bool(((one.grad.double() - val).abs() <= off + 64 * 2.0 ** -24 * mag).all())


@pytest.mark.gpu
@pytest.mark.parametrize("d,v", [(64, 500), (24, 10)])
def test_ignored_rows_cost_and_spoil_nothing(d, v):
    """Infinities and NaN in ignored rows reach nothing; a batch without rows that count; targets that are no class."""
    from vae_amd.losses import linear_cross_entropy
    s = _inputs(300, d, v, "bf16", True, False, 0.3, seed=4)
    loss, grads = _run(s, "mean")
    dirty = {**s, "x": s["x"].clone()}
    off = s["target"] == -100
    dirty["x"][off] = float("nan")
    dirty["x"][off.nonzero()[0, 0]] = float("inf")
    loss2, grads2 = _run(dirty, "mean")
    assert torch.equal(loss, loss2) and all(torch.equal(grads[k], grads2[k]) for k in grads)
    assert not bool(grads2["x"][off].any())
    none = {**s, "target": torch.full_like(s["target"], -100)}
    loss, grads = _run(none, "mean")
    assert bool(torch.isnan(loss)) and not any(bool(g.any()) for g in grads.values())
    loss, grads = _run(none, "none", torch.ones(300, device="cuda"))
    assert not bool(loss.any()) and not any(bool(g.any()) for g in grads.values())
    bad = {**s, "target": s["target"].clone()}
    bad["target"][5], bad["target"][7] = v, -1
    loss, grads = _run(bad, "none", torch.ones(300, device="cuda"))
    assert bool(torch.isnan(loss[[5, 7]]).all()) and int(torch.isnan(loss).sum()) == 2
    assert bool(torch.isnan(grads["x"][[5, 7]]).all()) and int(torch.isnan(grads["x"]).any(1).sum()) == 2 and bool(torch.isnan(grads["w"]).all())
    other = {**s, "target": torch.where(off, torch.full_like(s["target"], 3), s["target"])}
    a = linear_cross_entropy(other["x"], other["w"], other["target"], bias=s["bias"], ignore_index=3)
    assert bool(torch.isfinite(a))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("v", [600, 60])
def test_extreme_logits(dtype, v):
    """Logits of hundreds, classes masked by the type's lowest bias, and a row that holds a NaN."""
    s = _inputs(40, 64, v, dtype, True, False, 0.0, seed=6)
    s["x"].mul_(40)
    s["target"] = (s["x"].double() @ s["w"].double().t()).argmax(1)     # the likely class, so that the loss is of ordinary size
    s["bias"][v // 6:v // 2] = torch.finfo(DT[dtype]).min
    s["target"][(s["target"] >= v // 6) & (s["target"] < v // 2)] = 5
    loss, grads = _run(s, "none", torch.ones(40, device="cuda"))
    ref, _ = _oracle(s, "none")
    z = (s["x"].double() @ s["w"].double().t()).abs().amax()
    assert bool(((loss.double() - ref).abs() <= 64 * 2.0 ** -24 * (z + ref.abs())).all())
    assert all(bool(torch.isfinite(g).all()) for g in grads.values())
    assert not bool(grads["w"][v // 6:v // 2].any())                           # masked classes have no share at all
    s["x"][3, 9] = float("nan")
    loss, grads = _run(s, "none", torch.ones(40, device="cuda"))
    assert int(torch.isnan(loss).sum()) == 1 and bool(torch.isnan(loss[3])) and int(torch.isnan(grads["x"]).any(1).sum()) == 1


@pytest.mark.gpu
def test_differences():
    """Central differences of the forward pass in the direction of the gradient (fp32, steps of 2^-6: 1e-2 is wide)."""
    from vae_amd.losses import linear_cross_entropy
    s = _inputs(20, 24, 50, "fp32", True, True, 0.2, seed=5)
    _, grads = _run(s, "sum")
    for k, g in grads.items():
        step, dirn = 2.0 ** -6, g / g.norm()
        val = lambda e: float(linear_cross_entropy(**{k2: (s[k2] + e * dirn if k2 == k else s[k2]) for k2 in ("x", "w", "bias", "target")},  # noqa: E731
                                                   weight=s["weight"], reduction="sum"))
        assert abs((val(step) - val(-step)) / (2 * step) / float(g.norm()) - 1) < 1e-2, k


@pytest.mark.gpu
@pytest.mark.parametrize("d,v", [(136, 3000), (30, 17)])
def test_repeats_other_stream_and_graph(d, v):
    s = _inputs(700, d, v, "bf16", True, True, 0.2, seed=11)
    first = _run(s, "mean")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _run(s, "mean")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first[0], again[0]) and all(torch.equal(first[1][k], again[1][k]) for k in first[1])
    static = {k: v.clone() for k, v in s.items()}
    one, up = torch.tensor(1.0, device="cuda"), None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = _run(static, "mean", one)
    for seed in (12, 13, 14):                                            # another number of ignored rows every time
        new = _inputs(700, d, v, "bf16", True, True, 0.1 * (seed - 11), seed=seed)
        for k in static:
            static[k].copy_(new[k])
        graph.replay()
        torch.cuda.synchronize()
        want = _run(new, "mean", up)
        assert torch.equal(loss, want[0]) and all(torch.equal(grads[k], want[1][k]) for k in grads)


@pytest.mark.gpu
def test_partial_gradients_empty_and_module():
    from vae_amd.losses import LinearCrossEntropyLoss, linear_cross_entropy
    s = _inputs(50, 32, 40, "fp32", True, False, 0.0, seed=2)
    full = _run(s, "mean")[1]
    for k in ("x", "w", "bias"):
        leaf = s[k].detach().requires_grad_()
        args = {**s, k: leaf}
        linear_cross_entropy(args["x"], args["w"], s["target"], bias=args["bias"]).backward()
        assert torch.equal(leaf.grad, full[k])
    m = LinearCrossEntropyLoss(32, 40).cuda()
    with torch.no_grad():
        m.linear.weight.copy_(s["w"])
        m.linear.bias.copy_(s["bias"])
    m(s["x"], s["target"]).backward()
    assert torch.equal(m.linear.weight.grad, full["w"]) and torch.equal(m.linear.bias.grad, full["bias"])
    e = torch.zeros(0, 32, device="cuda", requires_grad=True)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    m.zero_grad()
    loss = linear_cross_entropy(e, m.linear.weight, none, bias=m.linear.bias, reduction="sum")
    loss.backward()
    assert float(loss.detach()) == 0 and e.grad.shape == (0, 32) and not bool(m.linear.weight.grad.any())
    assert bool(torch.isnan(m(e, none))) and linear_cross_entropy(e, m.linear.weight, none, reduction="none").shape == (0,)
    weighted = LinearCrossEntropyLoss(32, 40, weight=torch.rand(40, device="cuda")).cuda().bfloat16()    # takes the weights along
    weighted(s["x"].bfloat16(), s["target"]).backward()
    assert weighted.linear.weight.grad.dtype == torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("n,d,v", [(300, 64, 500), (300, 24, 10), (5000, 700, 12), (9, 2500, 3001)])
@pytest.mark.parametrize("weight", [False, True])
def test_a_target_that_is_no_class_spoils_its_row_alone(n, d, v, weight, reduction):
    """The other rows' gradients are those of the batch without it (fp32: sums may be split another way, see above)."""
    s = _inputs(n, d, v, "fp32", True, weight, 0.3 if n > 9 else 0.0, seed=n + d)
    bad = {**s, "target": s["target"].clone()}
    bad["target"][5], bad["target"][7], s["target"][[5, 7]] = v, -1, -100
    loss, grads = _run(bad, reduction)
    assert bool(torch.isnan(loss)) and all(bool(torch.isnan(grads[k]).all()) for k in ("w", "bias"))
    rows = torch.ones(n, dtype=torch.bool, device="cuda")
    rows[[5, 7]] = False
    assert bool(torch.isnan(grads["x"][~rows]).all())
    grads["x"][~rows] = 0
    loss, _ = _run(s, reduction)
    _check(s, reduction, loss, {"x": grads["x"]})


@pytest.mark.gpu
def test_strided_targets_biases_and_class_weights():
    from vae_amd.losses import linear_cross_entropy
    s = _inputs(60, 40, 90, "fp32", True, True, 0.2, seed=8)
    want, grads = _run(s, "mean")
    wide = {k: torch.stack((s[k], s[k]), 1) for k in ("bias", "weight", "target")}
    bias = wide["bias"].requires_grad_()
    got = linear_cross_entropy(s["x"], s["w"], wide["target"][:, 0], bias=bias[:, 1], weight=wide["weight"][:, 1])
    got.backward()
    assert torch.equal(got, want) and torch.equal(bias.grad[:, 1], grads["bias"]) and not bool(bias.grad[:, 0].any())
    one = torch.ones(1, 1, device="cuda", requires_grad=True)
    loss = linear_cross_entropy(s["x"][:, :1], one.expand(90, 1), s["target"])
    loss.backward()
    assert abs(float(loss) - math.log(90)) < 1e-5 and abs(float(one.grad)) < 1e-5           # all classes alike


def _check_uneven(s, reduction, up, grads):
    """fp16 gradients where the rows' factors g span many powers of two.  d is held in steps of 2^-24 times 2^s top / (2^14 2^s)
    (top: the largest |g|; s = 0 to 10 by how far a row is below it), so that besides the bounds of _check a row's d is off by half
    a step, 2^-25 2^-14 2^-s top; and dW takes x 2^-s, off by 2^-25 in those units."""
    _, ref = _oracle(s, reduction, up)
    kept = s["target"] != -100
    cw = kept.double() * (1 if s["weight"] is None else s["weight"].double()[s["target"].clamp(min=0)])
    g = cw * up.double() / (cw.sum() if reduction == "mean" else 1)
    top = g.abs().max()
    below = torch.where(g > 0, torch.log2(top / g.clamp(min=1e-300)).round(), torch.zeros_like(g))
    shift = (below - 6 - 1).clamp(0, 10)                # (an exponent's difference may be one less than the ratio's logarithm)
    step = torch.where(g > 0, 2.0 ** (-25 - 14 - shift) * top, torch.zeros_like(g))
    x, w = s["x"].double().abs(), s["w"].double().abs()
    x = torch.where(kept[:, None], x, torch.zeros_like(x))
    z = s["x"].double() @ s["w"].double().t() + (0 if s["bias"] is None else s["bias"].double())
    d = torch.softmax(z, 1)
    d.scatter_add_(1, s["target"].clamp(min=0)[:, None], -torch.ones_like(d[:, :1]))
    d = torch.where(kept[:, None], d.abs() * g[:, None], torch.zeros_like(d))
    shifted = (shift > 0).double() * 2.0 ** (-25 + (shift + 1).clamp(max=10))
    extra = {"x": step[:, None] * w.sum(0), "w": (step[:, None] * x).sum(0) + (d * shifted[:, None]).sum(0)[:, None], "bias": 0.0}
    eps = 2.0 ** -11
    for k, got in grads.items():
        val, mag, off = ref[k]
        k_len = s["w"].shape[0] if k == "x" else s["x"].shape[0]
        tol = off + max(32.0, 2 * (6 * k_len / 16) ** 0.5) * 2.0 ** -24 * mag + eps * mag + 1.01 * eps * val.abs() + extra[k] + 2.0 ** -25
        bad = (got.double() - val).abs() - tol
        assert float(bad.max()) <= 0, (k, float(bad.max()), float(val.abs().max()))


UNEVEN = [(128, 64, 30000), (300, 72, 5000), (64, 4000, 900), (2500, 136, 3001), (700, 1000, 40), (40000, 72, 7000)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v", UNEVEN)
@pytest.mark.parametrize("how", ["none", "mean"])
def test_fp16_factors_far_apart(n, d, v, how):
    """Upstream gradients, or class weights, over eight powers of ten; the weights have a common part, so that probabilities that
    are lost shift a row's gradient instead of averaging out."""
    s = _inputs(n, d, v, "fp16", True, how == "mean", 0.2, seed=n)
    s["x"].mul_(0.3)
    s["w"] = (s["w"].float() + 0.3).half()
    gen = torch.Generator(device="cuda").manual_seed(2)
    if how == "none":
        up = 512.0 * 10.0 ** (-8 * torch.rand(n, generator=gen, device="cuda"))
    else:
        s["weight"], up = 10.0 ** (-8 * torch.rand(v, generator=gen, device="cuda")), torch.tensor(512.0, device="cuda")
    _, grads = _run(s, how, up)
    _check_uneven(s, how, up, grads)


@pytest.mark.gpu
def test_fp16_rows_far_below_the_largest_keep_their_gradient():
    """At 1e-7 of the largest factor a row's gradient over 30000 classes was off by 30 % once: each of its 30000 probabilities is
    held to 2^-9 or better (8 bits and more), and so is the row."""
    s = _inputs(128, 64, 30000, "fp16", False, False, 0.0, seed=1)
    s["w"], s["x"] = (s["w"].float() + 0.3).half(), (0.1 * s["x"].float()).half()
    up = torch.full((128,), 2048.0, device="cuda")
    up[1::2] *= 1e-7
    _, grads = _run(s, "none", up)
    _, ref = _oracle(s, "none", up)
    off = (grads["x"].double() - ref["x"][0]).norm(dim=1) / ref["x"][0].norm(dim=1)
    assert float(off.max()) < 2.0 ** -8, float(off.max())


@pytest.mark.gpu
def test_fp16_factors_in_a_graph():
    """The factors' unevenness is found on the device: a captured pass follows new ones."""
    n, d, v = 700, 136, 3000
    static = _inputs(n, d, v, "fp16", True, False, 0.2, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(2)
    up = torch.ones(n, device="cuda")
    _run(static, "none", up)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = _run(static, "none", up)
    for k in range(3):
        up.copy_(10.0 ** (-2 * k * torch.rand(n, generator=gen, device="cuda")))
        graph.replay()
        torch.cuda.synchronize()
        want = _run(static, "none", up)
        assert torch.equal(loss, want[0]) and all(torch.equal(grads[name], want[1][name]) for name in grads)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v,dtype", [(2048, 512, 3000, "fp32"), (1000, 4096, 500, "fp32"), (64, 1024, 40000, "fp32"), (4096, 3000, 30, "fp32"),
                                         (2048, 512, 3000, "bf16"), (600, 2000, 900, "fp16"), (8192, 4000, 10, "bf16"), (3000, 1536, 9000, "fp16")])
def test_losses_are_as_exact_as_their_sums(n, d, v, dtype):
    """The mean error of the losses of many rows, where single ones are held to the bound of the largest (test_shapes).  A sum's
    steps: products of 32 of D, six of them for fp32; where fp32 goes into 32-bit instructions (few rows or classes) one for every
    feature, in two sums at least."""
    s = _inputs(n, d, v, dtype, False, False, 0.0, seed=n)
    z = s["x"].double() @ s["w"].double().t()
    lse, z_t = z.logsumexp(1), z.gather(1, s["target"][:, None])[:, 0]
    got, _ = _run(s, "none", torch.ones(n, device="cuda"))
    steps = d / 2 if dtype == "fp32" and min(n, v) <= 64 else 6 * d / 32 if dtype == "fp32" else d / 32
    assert _rms(got.double() - lse + z_t) <= _expected_loss_error(z_t, lse, lse - z_t, steps)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v", [(600, 512, 500), (2048, 256, 1500), (64, 1024, 4000)])
def test_fp32_gradients_are_as_exact_as_their_sums(n, d, v):
    """As above for dx and dW.  Their terms are products of d, whose p is off by the error of z - lse, its own in every class and one
    for the row, and which is held in 24 bits; a sum rounds at the size of its value or of its terms' root sum of squares; the
    result, its factors and d are rounded four times."""
    s = _inputs(n, d, v, "fp32", False, False, 0.0, seed=n)
    x, w, t = s["x"].double(), s["w"].double(), s["target"]
    z = x @ w.t()
    lse, z_t = z.logsumexp(1), z.gather(1, t[:, None])[:, 0]
    few = n <= 64
    off = _expected_loss_error(z_t, lse, lse - z_t, d / 2 if few else 6 * d / 32)
    p = torch.softmax(z, 1)
    dl = p.clone()
    dl[torch.arange(n), t] -= 1
    _, grads = _run(s, "sum")
    for name, a, b, pa, steps in (("x", dl, w, p, v / 2 if few else 6 * v / 32), ("w", dl.t(), x, p.t(), 6 * n / 32)):
        val = a @ b
        size = val.square() + a.square() @ b.square()
        bound = ((1.25 * 2.0 ** -25.2) ** 2 * steps + 4 * 2.0 ** -48 / 3) * size + off ** 2 * (pa.square() @ b.square() + (pa @ b).square())
        assert _rms(grads[name].double() - val) <= float(bound.mean().sqrt()), name


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,v", [(5000, 40, 30000), (4100, 64, 20000), (3000, 7, 9000), (130, 60, 70000), (100, 33, 80000), (9000, 1, 7000)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("ignored", [0.0, 0.6])
def test_one_step_of_features_and_many_tiles(n, d, v, dtype, ignored):
    """Workgroups that stay for several tiles of one step: both loads on the way belong to tiles other than the one in work."""
    s = _inputs(n, d, v, dtype, True, False, ignored, seed=n + d)
    s["target"][n // 2] = v - 1
    loss, grads = _run(s, "mean")
    _check(s, "mean", loss, grads)
    got, _ = _run(s, "none", torch.ones(n, device="cuda"))
    ref, _ = _oracle(s, "none")
    assert bool(((got.double() - ref).abs() <= 2e-6 * ref + 1e-6).all())
