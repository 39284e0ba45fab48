"""The gated residual norm, the linear cross entropy and the many-tensor AdamW step as one training step of a residual network
with a wide class head, on the framework's own linear layers, against the same network in 64 bits.

Tolerance of the gradients: every stage is held to some 1e-6 of its largest values by its own tests; five stages in a row, each
multiplying what comes in by a matrix or a norm of order one, stay within 1e-4 of a gradient tensor's largest element."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

pytestmark = pytest.mark.gpu


class Net(nn.Module):
    def __init__(self, n_in, width, classes, blocks, kind):
        from vae_amd.losses import LinearCrossEntropyLoss
        from vae_amd.modules import GatedResidualNorm
        super().__init__()
        self.kind = kind
        self.embed = nn.Linear(n_in, width)
        self.mid = nn.ModuleList(nn.Linear(width, width) for _ in range(blocks))
        self.gate = nn.ModuleList(nn.Linear(width, 1) for _ in range(blocks))
        self.norm = nn.ModuleList(GatedResidualNorm(width, kind=kind, residual_scale=0.5) for _ in range(blocks))
        weight = torch.linspace(0.5, 2.0, classes)
        self.head = LinearCrossEntropyLoss(width, classes, weight=weight)

    def forward(self, x, target):
        from vae_amd.modules import hip_linear
        y = h = hip_linear(self.embed, x)
        for mid, gate, norm in zip(self.mid, self.gate, self.norm):
            y, h = norm(y, F.gelu(hip_linear(mid, h)), hip_linear(gate, h))
        return self.head(h, target)

    def plain(self, p, x, target):
        """The same in the type of ``p`` (name -> tensor), with torch's own operations."""
        def norm(z, w, b):
            z = z - z.mean(-1, keepdim=True) if self.kind == "layer" else z
            return z / (z.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

        y = h = x @ p["embed.weight"].t() + p["embed.bias"]
        for k in range(len(self.mid)):
            b = F.gelu(h @ p[f"mid.{k}.weight"].t() + p[f"mid.{k}.bias"])
            g = torch.sigmoid(h @ p[f"gate.{k}.weight"].t() + p[f"gate.{k}.bias"])
            n = {name: p[f"norm.{k}.{name}"] for name in ("norm_weight", "norm_bias", "post_weight", "post_bias", "scale")}
            y = y + n["scale"] * g * norm(b, n["post_weight"], n["post_bias"])
            h = norm(y, n["norm_weight"], n["norm_bias"])
        z = h @ p["head.linear.weight"].t() + p["head.linear.bias"]
        return F.cross_entropy(z, target, weight=self.head.weight.to(z.dtype))


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("classes,width", [(17, 32), (1500, 96)])
def test_training_step(kind, classes, width):
    from vae_amd.optim import MultiTensorAdamW
    torch.manual_seed(3)
    net = Net(24, width, classes, 2, kind).cuda()
    x = torch.randn(130, 24, device="cuda")
    target = torch.randint(0, classes, (130,), device="cuda")
    target[::7] = -100
    lr, eps = 1e-3, 1e-7
    opt = MultiTensorAdamW([{"params": list(net.head.parameters()), "weight_decay": 0.1}, {"params": [p for n, p in net.named_parameters()
                           if not n.startswith("head")]}], lr=lr, eps=eps, state_bits=8, seed=5)
    for step in range(2):
        before = {k: p.detach().double().cpu() for k, p in net.named_parameters()}
        p64 = {k: p.clone().requires_grad_() for k, p in before.items()}
        net.head.weight = net.head.weight.cpu()
        ref = net.plain(p64, x.double().cpu(), target.cpu())
        net.head.weight = net.head.weight.cuda()
        grads = dict(zip(p64, torch.autograd.grad(ref, list(p64.values()))))
        opt.zero_grad()
        loss = net(x, target)
        loss.backward()
        assert abs(float(loss.detach()) - float(ref.detach())) < 1e-5 * float(ref.detach())
        for k, p in net.named_parameters():
            err = (p.grad.double().cpu() - grads[k]).abs().max()
            assert float(err) < 1e-4 * float(grads[k].abs().max()), (k, float(err), float(grads[k].abs().max()))
        used = {k: p.grad.double().cpu() for k, p in net.named_parameters()}
        opt.step()
        for k, p in net.named_parameters():
            if step:                                     # (later steps start from rounded moments: tested with the optimiser)
                assert bool(torch.isfinite(p).all()) and not torch.equal(p.detach().double().cpu(), before[k])
                continue
            # the first step: m / (1 - b1) = g, v / (1 - b2) = g^2, whatever the moments are held in afterwards
            wd = 0.1 if k.startswith("head") else 0.0
            want = before[k] * (1 - lr * wd) - lr * used[k] / (used[k].abs() + eps)
            assert float((p.detach().double().cpu() - want).abs().max()) < 16 * 2.0 ** -24 * float(before[k].abs().max() + lr)
