"""AdamW over many separate tensors (vae_amd.optim.multi_tensor_adamw_, MultiTensorAdamW; C ABI vae_adamw_multi)
against one step in 64 bits; refusals on the CPU.

Tolerances.  fp32 arithmetic of one step rounds about ten times: 16 * 2^-24 of the terms' magnitudes.  A weight of 16 bits is
rounded once more, by finfo.eps / 2.  e4m3: nearest is off by at most 2^-4 of the value or 2^-10 (half the smallest step) of the
scaled range, rounding at random by at most a whole step, twice that; 1e-5 is added for the fp32 arithmetic ahead of it."""
import ctypes as C
import math

import pytest
import torch

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 256


# ---------------------------------------------------------------------------------------------------- on the CPU
def _args(lib_mod, tensors, bits=32, n_blocks=8, ptr=1 << 20, scales=None, master=None, step=1, lr=1e-3, clip=0.0, ws=None, wsb=0,
          wide=1 << 20):
    arr = (lib_mod.AdamWTensor * max(1, len(tensors)))(*tensors)
    return (arr, len(tensors), bits, C.c_void_p(ptr), C.c_void_p(ptr + wide), scales, n_blocks, master, lr, 0.9, 0.99, 1e-8, step,
            clip, 1.0, 0, ws, wsb, None, None)


def test_refusals_of_the_c_entry():
    """Every refusal is made before any launch, with a message."""
    from vae_amd import _lib
    lib = _lib.load()
    T = _lib.AdamWTensor
    base = 1 << 30
    ok = T(base, base + (1 << 20), 100, 0, 0.0, 0)

    def refused(msg, *a, **k):
        rc = lib.vae_adamw_multi(*_args(_lib, *a, **k))
        assert rc == 1 and msg in lib.vae_last_error().decode(), lib.vae_last_error()

    refused("state_bits", [ok], bits=16)
    refused("step counts from 1", [ok], step=0)
    refused("hyper-parameter", [ok], lr=float("nan"))
    refused("does not fit the state", [T(base, base + 4096, 2049, 0, 0.0, 0)])
    refused("does not fit the state", [T(base, base + 4096, 1, 8, 0.0, 0)])
    refused("does not fit the state", [T(base, base + 4096, 1, -1, 0.0, 0)])
    refused("a size", [T(base, base + 4096, -1, 0, 0.0, 0)])
    refused("null param", [T(None, base, 4, 0, 0.0, 0)])
    refused("dtype", [T(base, base + 4096, 4, 0, 0.0, 3)])
    refused("aligned to its element", [T(base + 2, base + 4096, 4, 0, 0.0, 0)])
    refused("weight decay", [T(base, base + 4096, 4, 0, -1.0, 0)])
    refused("overlap", [ok, T(base + 396, base + 8192, 4, 1, 0.0, 0)])          # the last element of the first one
    refused("overlap", [ok, ok])
    refused("overlap", [T((1 << 20) + 512, base, 4, 0, 0.0, 0)])                # a parameter inside exp_avg
    refused("share blocks", [ok, T(base + 4096, base, 4, 0, 0.0, 0)])
    refused("the gradient overlaps", [ok, T(base + 4096, base + 396, 4, 1, 0.0, 0)])      # a gradient inside another parameter
    refused("the gradient overlaps", [T(base, base, 4, 0, 0.0, 0)])
    refused("the gradient overlaps", [T(base, (1 << 20) + 8188, 4, 0, 0.0, 0)])           # ... or at the end of exp_avg
    refused("2^37", [T(base, base + (1 << 41), 1 << 38, 0, 0.0, 1)], n_blocks=1 << 30, ptr=1 << 43, wide=1 << 42)
    refused("scales", [ok], bits=8)
    refused("16-byte aligned", [ok], ptr=(1 << 20) + 4)
    refused("workspace", [ok], clip=1.0)
    refused("does not fit", [ok], n_blocks=0)
    assert lib.vae_adamw_multi(*_args(_lib, [])) == 0                           # nothing to do


def test_refusals_of_the_python_entry():
    from vae_amd.optim import MultiTensorAdamW, multi_tensor_adamw_
    p = torch.zeros(4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        multi_tensor_adamw_([p], [p], torch.zeros(256), torch.zeros(256), step=1, lr=1e-3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        MultiTensorAdamW([p])
    with pytest.raises(ValueError, match="twice"):
        MultiTensorAdamW([p, p])
    with pytest.raises(ValueError, match="no parameters"):
        MultiTensorAdamW([])
    with pytest.raises(ValueError, match="state_bits"):
        MultiTensorAdamW([p], state_bits=4)
    with pytest.raises(TypeError, match="float64"):
        MultiTensorAdamW([p.double()])


def test_refusals_of_the_counts_of_steps():
    from vae_amd import _lib
    lib = _lib.load()
    base = 1 << 30
    rc = lib.vae_adamw_multi(*_args(_lib, [_lib.AdamWTensor(base, base + (1 << 20), 100, 0, 0.0, 0, -1)]))
    assert rc == 1 and "step counts from 1" in lib.vae_last_error().decode()


# ---------------------------------------------------------------------------------------------------- on the GPU
SIZES = {"ragged": [1, 255, 256, 257, 7, 2047, 2048, 2049, 4100, 65537], "one": [1], "empty": [0, 5, 0, 300, 0],
         "many": [3 + 37 * k % 400 for k in range(230)], "long": [2 ** 20 + 3, 9]}


def _offset(n, dtype, k, gen, scale):
    """A contiguous tensor of n elements that starts k elements into its storage."""
    return (torch.randn(n + k, generator=gen, device="cuda") * scale).to(dtype)[k:]


def _step64(p, g, m, v, step, lr, wd, b1, b2, eps):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p * (1 - lr * wd) - lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps), m, v


def _close(got, ref, mag, dtype):
    tol = 16 * 2.0 ** -24 * mag + (torch.finfo(dtype).eps / 2 * ref.abs() if dtype != torch.float32 else 0)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25                                      # half the smallest subnormal
    assert bool(((got.double() - ref).abs() <= tol).all()), float(((got.double() - ref).abs() - tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("bits,master,clip", [(32, False, 0.0), (32, True, 0.3), (8, False, 0.0), (8, True, 0.0), (8, False, 0.3)])
def test_three_steps(sizes, dtype, bits, master, clip):
    from vae_amd.optim import MultiTensorAdamW
    gen = torch.Generator(device="cuda").manual_seed(5)
    t, sizes = DT[dtype], SIZES[sizes]
    params = [_offset(n, t, k % 3, gen, 0.3) for k, n in enumerate(sizes)]
    groups = [{"params": params[0::2], "weight_decay": 0.1}]
    if params[1::2]:
        groups.append({"params": params[1::2]})
    lr, b1, b2, eps = 1e-2, 0.9, 0.99, 1e-6
    opt = MultiTensorAdamW(groups, lr=lr, betas=(b1, b2), eps=eps, max_grad_norm=clip, state_bits=bits, master_weights=master, seed=3)
    order = params[0::2] + params[1::2]
    decay = [0.1] * len(params[0::2]) + [0.0] * len(params[1::2])
    for step in range(1, 4):
        for k, p in enumerate(order):
            p.grad = _offset(p.numel(), t, (k + step) % 2, gen, 10.0 ** (k % 4 - 2))
        before = [(opt.master[b:b + p.numel()] if master else p).double().clone() for p, b in zip(order, opt.starts)]
        state = [tuple(s.double() for s in opt.moments(k)) for k in range(len(order))]
        coef = 1.0
        total = math.sqrt(sum(float(p.grad.double().square().sum()) for p in order))
        if clip:
            coef = min(1.0, clip / (total + 1e-6))
        opt.step()
        if clip:
            assert abs(float(opt.grad_norm) - total) <= 2.0 ** -23 * total
        for k, (p, b) in enumerate(zip(order, opt.starts)):
            n = p.numel()
            g = p.grad.double() * coef
            ref, m, v = _step64(before[k], g, state[k][0], state[k][1], step, lr, decay[k], b1, b2, eps)
            mm = b1 * state[k][0].abs() + (1 - b1) * g.abs()
            # the update's error is that of its terms, which may cancel in m
            mag = before[k].abs() + lr * mm / (1 - b1 ** step) / ((v / (1 - b2 ** step)).sqrt() + eps)
            if master:
                _close(opt.master[b:b + n], ref, mag, torch.float32)
                assert torch.equal(p, opt.master[b:b + n].to(t))
            else:
                _close(p, ref, mag, t)
            m2, v2 = opt.moments(k)
            if bits == 32:
                _close(m2, m, mm, torch.float32)
                _close(v2, v, v, torch.float32)
            elif n:
                pad = (-n) % BLOCK
                z = torch.zeros(pad, dtype=torch.float64, device="cuda")
                blocks = lambda x: torch.cat((x, z)).view(-1, BLOCK)  # noqa: E731
                bm, bu = blocks(m), blocks(v.sqrt())
                sm, su = bm.abs().amax(1, keepdim=True) / 448, bu.amax(1, keepdim=True) / 448
                dm, du = blocks(m2.double()), blocks(v2.double().sqrt())
                assert bool(((dm - bm).abs() <= bm.abs() * 2.0 ** -4 + sm * (2.0 ** -10 + 448e-5)).all())
                assert bool(((du - bu).abs() <= bu * 2.0 ** -3 + su * (2.0 ** -9 + 448e-5)).all())
                assert bool((du[bu > 0] > 0).all())
                sc = opt.scales[:, b // BLOCK:b // BLOCK + bm.shape[0]].double()
                assert torch.allclose(sc[0], sm[:, 0], rtol=1e-5, atol=0) and torch.allclose(sc[1], su[:, 0], rtol=1e-5, atol=0)
                tail = opt.exp_avg[b + n:b + n + pad].view(torch.uint8), opt.exp_avg_sq[b + n:b + n + pad].view(torch.uint8)
                assert not any(bool(x.any()) for x in tail)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_random_rounding_keeps_the_decay():
    """beta2 = 0.998 moves the root by 0.1 % a step, a hundredth of a code: on average it has to fall all the same.  Over 200
    steps without gradients v falls by 0.998^200; the mean over n elements of a value that moves by whole steps (at most 1/8 of
    it) has a deviation of at most 1/8 * sqrt(200 * 0.016 / n) of it, and v twice that: 6 deviations are allowed, and the
    resolution of the random bits (2^-17 of a step, 200 times) is nothing beside that."""
    from vae_amd.optim import MultiTensorAdamW
    n = 1 << 18
    gen = torch.Generator(device="cuda").manual_seed(1)
    p = torch.zeros(n, device="cuda")
    opt = MultiTensorAdamW([p], lr=0.0, betas=(0.9, 0.998), state_bits=8)
    p.grad = 0.1 + torch.rand(n, generator=gen, device="cuda")
    opt.step()
    start = opt.moments(0)[1].double()
    p.grad = torch.zeros(n, device="cuda")
    # the largest of a block is its scale and falls exactly; the others fall on average
    for _ in range(200):
        opt.step()
    got = opt.moments(0)[1].double()
    want = 0.998 ** 200
    ratio = float((got.sqrt().sum() / start.sqrt().sum()) ** 2)
    assert abs(ratio / want - 1) < 6 * 2 / 8 * math.sqrt(200 * 0.016 / n) + 1e-4, ratio / want


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_none_gradients_are_left_alone_and_calls_repeat(bits):
    from vae_amd.optim import MultiTensorAdamW
    runs = []
    for _ in range(2):
        gen = torch.Generator(device="cuda").manual_seed(2)
        params = [torch.randn(n, generator=gen, device="cuda") for n in (300, 17, 5000)]
        opt = MultiTensorAdamW(params, state_bits=bits, seed=11)
        for step in range(3):
            for k, p in enumerate(params):
                p.grad = None if (k == 1 and step == 1) else torch.randn(p.shape, generator=gen, device="cuda")
            old = params[1].clone(), opt.moments(1)
            opt.step()
            if step == 1:
                assert torch.equal(old[0], params[1]) and all(torch.equal(a, b) for a, b in zip(old[1], opt.moments(1)))
        runs.append([*params, opt.exp_avg.view(torch.uint8), opt.exp_avg_sq.view(torch.uint8)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
def test_non_finite_gradients_are_loud():
    from vae_amd.optim import MultiTensorAdamW
    p = torch.ones(1000, device="cuda")
    opt = MultiTensorAdamW([p], state_bits=8)
    p.grad = torch.ones(1000, device="cuda")
    p.grad[300] = float("nan")
    p.grad[600] = float("inf")
    opt.step()
    assert torch.isnan(p[300]) and not bool(torch.isfinite(p[600]))
    m, v = opt.moments(0)
    assert bool(torch.isnan(m[256:512]).all()) and bool(torch.isfinite(m[:256]).all()) and bool(torch.isfinite(v[768:]).all())
    assert not bool(torch.isfinite(v[600]))
    q = torch.ones(1000, device="cuda")
    opt = MultiTensorAdamW([q], state_bits=32, max_grad_norm=1.0)
    q.grad = p.grad
    opt.step()
    assert bool(torch.isnan(q).all())                                   # as torch's clip_grad_norm_ spreads it


@pytest.mark.gpu
def test_state_dict_other_stream_and_capture():
    from vae_amd.optim import MultiTensorAdamW
    gen = torch.Generator(device="cuda").manual_seed(4)
    a = [torch.randn(n, generator=gen, device="cuda").bfloat16() for n in (513, 8)]
    b = [t.clone() for t in a]
    make = lambda ps: MultiTensorAdamW(ps, state_bits=8, master_weights=True, seed=9, lr_lambda=lambda s: 1.0 / (1 + s))  # noqa: E731
    one, two = make(a), make(b)
    grads = [[torch.randn(t.shape, generator=gen, device="cuda").bfloat16() for t in a] for _ in range(2)]
    for t, g in zip(a + b, grads[0] + grads[0]):
        t.grad = g
    one.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two.step()
    torch.cuda.current_stream().wait_stream(side)
    fresh = make(b)
    fresh.load_state_dict(two.state_dict())
    for t, g in zip(a + b, grads[1] + grads[1]):
        t.grad = g
    one.step()
    fresh.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(one.exp_avg_sq.view(torch.uint8), fresh.exp_avg_sq.view(torch.uint8))
    with pytest.raises(ValueError, match="does not fit"):
        MultiTensorAdamW(a, state_bits=32).load_state_dict(two.state_dict())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            one.step()


@pytest.mark.gpu
def test_every_e4m3_rounding():
    """The first moment's codes over a whole binade of every exponent are torch's (nearest even, subnormals included)."""
    from vae_amd.optim import multi_tensor_adamw_
    vals = torch.arange(0, 1 << 16, device="cuda", dtype=torch.int32) * (1 << 14)
    x = vals.view(torch.float32)                                        # every float with 9 upper mantissa bits, from 0 to 2
    x = (x[(x <= 1.75)] * 256).float()                                  # up to 448
    x = torch.cat((x, -x))
    per = BLOCK - 1                                                      # the last of each block pins its scale to 1
    x = x[:x.numel() // per * per].view(-1, per)
    g = torch.cat((x, torch.full((x.shape[0], 1), 448.0, device="cuda")), 1).reshape(-1).contiguous()
    n = g.numel()
    p = torch.zeros(n, device="cuda")
    m = torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    v, sc = m.clone(), torch.zeros(2, n // BLOCK, device="cuda")
    multi_tensor_adamw_([p], [g], m, v, step=1, lr=0.0, betas=(0.0, 0.99), scales=sc)
    inv = (torch.ones(1, device="cuda") * 448).reciprocal() * 448
    want = (g * inv).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(m.float(), want.float())


@pytest.mark.gpu
def test_a_step_shows_in_the_version_of_what_it_changed():
    """A backward pass that saved weights from before a step must not run on the new ones."""
    from vae_amd.optim import MultiTensorAdamW
    w, idle = (torch.ones(5, 5, device="cuda", requires_grad=True) for _ in range(2))
    x = torch.ones(2, 5, device="cuda", requires_grad=True)
    old = (x @ w + x @ idle).sum()
    w.grad = torch.ones_like(w)
    MultiTensorAdamW([w, idle], state_bits=32).step()
    assert idle._version == 0
    with pytest.raises(RuntimeError, match="inplace operation"):
        old.backward()


@pytest.mark.gpu
def test_two_parameters_may_share_a_gradient():
    from vae_amd.optim import MultiTensorAdamW
    a, b = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    a.grad = b.grad = torch.randn(300, device="cuda")
    MultiTensorAdamW([a, b], state_bits=32).step()
    assert torch.equal(a, b) and not bool((a == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [1e20, -1e20, math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_block_that_is_not_finite_decodes_as_nan(bad, dtype):
    """1e20 is finite and its square is not: m stays, the root is lost.  Zeros and ones beside it share the block's scale."""
    from vae_amd.optim import MultiTensorAdamW
    p = torch.ones(1000, device="cuda", dtype=DT[dtype])
    opt = MultiTensorAdamW([p], state_bits=8)
    p.grad = torch.ones_like(p)
    p.grad[300], p.grad[301:310] = bad, 0.0
    opt.step()
    m, v = opt.moments(0)
    inside = torch.zeros(1000, dtype=torch.bool, device="cuda")
    inside[256:512] = True
    assert bool(torch.isnan(v[inside]).all()) and bool(torch.isfinite(v[~inside]).all())
    assert bool((torch.isfinite(m) if math.isfinite(bad) else torch.isnan(m))[inside].all()) and bool(torch.isfinite(m[~inside]).all())
    p.grad = torch.ones_like(p)
    opt.step()
    assert bool(torch.isnan(p[inside]).all()) and bool(torch.isfinite(p[~inside]).all())


@pytest.mark.gpu
def test_an_infinite_norm_clips_to_nothing():
    """As torch's clip_grad_norm_: the coefficient is 0, finite gradients count as zeros and infinite ones become NaN."""
    from vae_amd.optim import MultiTensorAdamW
    p = torch.ones(600, device="cuda")
    opt = MultiTensorAdamW([p], lr=0.5, weight_decay=0.5, state_bits=32, max_grad_norm=1.0)
    p.grad = torch.ones(600, device="cuda")
    p.grad[3] = math.inf
    opt.step()
    assert float(opt.grad_norm) == math.inf and bool(torch.isnan(p[3]))
    p[3] = 0.75
    assert bool((p == 0.75).all())


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [0.0, 0.1])
@pytest.mark.parametrize("bits,master", [(32, False), (32, True), (8, False)])
def test_a_parameter_counts_its_own_steps(clip, bits, master):
    """Gradients that are absent now and then, 40 counts of steps among 120 tensors at the end: torch.optim.AdamW's weights, four
    steps of 16 roundings each, and in 8 bits no further than a step of the moments' codes takes them (a quarter of lr a step)."""
    from vae_amd.optim import MultiTensorAdamW
    gen = torch.Generator(device="cuda").manual_seed(6)
    lr, steps, n = 1e-2, 42, 120
    ours = [torch.randn(3 + 5 * k, generator=gen, device="cuda") for k in range(n)]
    ref = [t.double().requires_grad_() for t in ours]
    opt = MultiTensorAdamW(ours, lr=lr, state_bits=bits, master_weights=master, max_grad_norm=clip, weight_decay=0.1)
    torch_opt = torch.optim.AdamW(ref, lr=lr, betas=(0.9, 0.998), eps=1e-7, weight_decay=0.1)
    taken = [0] * n
    for step in range(1, steps + 1):
        for k in range(n):
            # the first third joins late, tensor by tensor; of the others every fifth misses one step in three
            absent = step <= k and k < 40 or (k >= 40 and k % 5 == 0 and step % 3 == 1)
            ours[k].grad = None if absent else torch.randn(ours[k].shape, generator=gen, device="cuda")
            ref[k].grad = None if absent else ours[k].grad.double()
            taken[k] += not absent
        if clip:
            torch.nn.utils.clip_grad_norm_(ref, clip)
        opt.step()
        torch_opt.step()
        if step == 40:                                                   # (the counts travel with the state)
            other = MultiTensorAdamW(ours, lr=lr, state_bits=bits, master_weights=master, max_grad_norm=clip, weight_decay=0.1)
            other.load_state_dict(opt.state_dict())
            opt = other
    assert opt.param_steps == taken and len(set(taken)) > 8 * 4 and opt.steps == steps
    for a, b, t in zip(ours, ref, taken):
        # an update is of at most 3 lr (its first ones: lr exactly); its error is 16 roundings of the moments' terms, in 8 bits
        # the codes': an eighth of the root (at random, both ways) and a sixteenth of the first moment
        tol = t * (16 * 2.0 ** -24 * (b.detach().abs().max() + 30 * lr) + (0.75 * lr if bits == 8 else 0))
        assert float((a.double() - b.detach()).abs().max()) <= float(tol)


@pytest.mark.gpu
def test_a_late_parameter_starts_with_a_full_step():
    """The first update of weights that had no gradient before is lr in the gradient's sign, not the 2.2 lr of three steps' bias."""
    from vae_amd.optim import MultiTensorAdamW, multi_tensor_adamw_
    a, b = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    opt = MultiTensorAdamW([a, b], lr=1.0, eps=0.0, state_bits=8)
    a.grad = torch.ones(300, device="cuda")
    opt.step()
    opt.step()
    b.grad = -torch.ones(300, device="cuda")
    opt.step()
    assert float((b - 1).abs().max()) <= 16 * 2.0 ** -24 and opt.param_steps == [3, 1]
    state = [torch.zeros(1024, device="cuda") for _ in range(2)]
    with pytest.raises(ValueError, match="counts of steps"):
        multi_tensor_adamw_([a, b], [a.grad, b.grad], *state, step=[1], lr=1.0)
    with pytest.raises(ValueError, match="counts from 1"):
        multi_tensor_adamw_([a, b], [a.grad, b.grad], *state, step=[1, 0], lr=1.0)
    with pytest.raises(ValueError, match="does not fit|counts"):
        opt.load_state_dict({**opt.state_dict(), "param_steps": [1]})


@pytest.mark.gpu
def test_moments_are_held_in_32_bits_unless_asked_otherwise():
    from vae_amd.optim import MultiTensorAdamW
    p = torch.ones(300, device="cuda")
    opt = MultiTensorAdamW([p])
    assert opt.exp_avg.dtype == opt.exp_avg_sq.dtype == torch.float32 and opt.scales is None
    assert MultiTensorAdamW([p], state_bits=8).exp_avg.dtype == torch.float8_e4m3fn
