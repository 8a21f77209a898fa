"""optim.FusedMuon against its formula in 64 bits, under freeze patterns, gradient scaling and capture; and the whole tail of a training step --
linear_ce_loss, its gradients in the flat buffer, FusedMuon -- as it is used."""
import argparse

import numpy as np
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

from fedicra_amd import ops  # noqa: E402
from fedicra_amd.amp import GradScaler  # noqa: E402
from fedicra_amd.flat import FlatStoreMixin  # noqa: E402
from fedicra_amd.networks.unet import UNet, set_compute_dtype  # noqa: E402
from fedicra_amd.optim import FusedMuon  # noqa: E402

A, B, C = 3.4445, -4.7750, 2.0315


def _ns64(u):
    x = u.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.square().sum().sqrt() + 1e-7)
    for _ in range(5):
        g = x @ x.t()
        x = A * x + (B * g + C * (g @ g)) @ x
    return x.t() if tall else x


class _Reference:
    """The update in 64 bits on copies of the model's parameters, matrices as they lie in memory."""

    def __init__(self, net, lr, momentum=0.95, nesterov=True, wd=1e-2):
        self.lr, self.mu, self.nesterov, self.wd = lr, momentum, nesterov, wd
        self.p = {n: self._mat(p.detach()).double().clone() for n, p in net.named_parameters()}
        self.buf = {n: torch.zeros_like(p) for n, p in self.p.items()}
        self.v = {n: torch.zeros_like(p) for n, p in self.p.items()}
        self.t = 0

    @staticmethod
    def _mat(t):
        return t.permute(0, 2, 3, 1).reshape(t.shape[0], -1) if t.dim() == 4 else t.reshape(t.shape[0], -1) if t.dim() > 1 else t

    def step(self, grads, lr=None):
        lr = self.lr if lr is None else lr
        self.t += 1
        for n, g in grads.items():
            g, p, b = self._mat(g).double(), self.p[n], self.buf[n]
            if p.dim() == 1:                                           # AdamW
                b.mul_(0.9).add_(g, alpha=0.1)
                self.v[n].mul_(0.999).add_(g * g, alpha=0.001)
                p.mul_(1 - lr * self.wd)
                p.sub_(lr * (b / (1 - 0.9 ** self.t)) / ((self.v[n] / (1 - 0.999 ** self.t)).sqrt() + 1e-8))
                continue
            b.mul_(self.mu).add_(g, alpha=1 - self.mu)
            u = (1 - self.mu) * g + self.mu * b if self.nesterov else b
            p.mul_(1 - lr * self.wd).sub_(lr * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * _ns64(u))

    def check(self, net, steps):
        for n, q in net.named_parameters():
            got, want = self._mat(q.detach()).double(), self.p[n]
            if want.dim() == 1:
                tol = steps * self.lr * 2.0 ** -12 + 2.0 ** -20 * want.abs().max()      # (AdamW's sqrt and quotient in fp32)
            else:
                # a step leaves lr * scale times what the products may (4 * 3.4445^5 * 2^-22 of a unit matrix) and as much for the fp32 update itself
                tol = steps * self.lr * max(1.0, want.shape[0] / want.shape[1]) ** 0.5 * 8 * A ** 5 * 2.0 ** -22 + 2.0 ** -20 * want.abs().max()
            assert float((got - want).abs().max()) <= float(tol), (n, float((got - want).abs().max()), float(tol))


def _net(dtype="fp32"):
    torch.manual_seed(3)
    net = UNet(1, 2).cuda()
    set_compute_dtype(net, dtype)
    return net


def _set_grads(net, seed, names=None, scale=1.0):
    """Random gradients in the flat buffer, as a backward pass leaves them; returns them by name."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    net.zero_grad()
    out = {}
    for n, p in net.named_parameters():
        v = torch.randn(p.shape, generator=g, device="cuda") * 1e-3
        if names is None or n in names:
            p._fi_gview.copy_(v * scale)
            p.grad = p._fi_gview
            out[n] = v
    return out


@pytest.mark.parametrize("nesterov", [True, False])
def test_steps_equal_the_formula(nesterov):
    net = _net()
    opt = FusedMuon(net, lr=0.02, base_lr=0.02, max_iterations=100, nesterov=nesterov)
    ref = _Reference(net, 0.02, nesterov=nesterov)
    for k in range(3):
        grads = _set_grads(net, 10 + k)
        opt.step()
        ref.step(grads, lr=float(opt.lr_state))
        opt.advance_lr()
    ref.check(net, 3)
    assert float(opt.lr_state) < 0.02


def test_parameters_without_a_gradient_keep_value_and_momentum():
    net = _net()
    opt = FusedMuon(net, lr=0.02, base_lr=0.02, max_iterations=100)
    ref = _Reference(net, 0.02)
    names = [n for n, _ in net.named_parameters()]
    head, body = [n for n in names if "out_conv" in n], [n for n in names if "out_conv" not in n]
    before = net.flat_params.clone()
    for k in range(2):
        grads = _set_grads(net, 20 + k, head)
        opt.step()
        ref.step(grads)
    p = dict(net.named_parameters())
    for n in body:
        s, e = p[n]._fi_off, p[n]._fi_off + p[n].numel()
        assert torch.equal(net.flat_params[s:e], before[s:e]) and not opt.m[s:e].any()
    ref.t = 0                                                          # the body's own step counter
    grads = _set_grads(net, 30, body)
    opt.step()
    ref.step(grads)
    ref.check(net, 3)
    opt.reset_round()
    assert not opt.m.any() and not opt._groups


def test_gradient_scaling_steps_and_skips():
    net = _net()
    opt = FusedMuon(net, lr=0.02, base_lr=0.02, max_iterations=100)
    ref = _Reference(net, 0.02)
    sc = GradScaler(init_scale=1024.0)
    sc.scale(torch.ones((), device="cuda"))
    grads = _set_grads(net, 40, scale=1024.0)
    sc.step(opt)
    sc.update()
    ref.step(grads)
    ref.check(net, 1)
    keep, mom = net.flat_params.clone(), opt.m.clone()
    for bad in (float("inf"), float("nan")):
        _set_grads(net, 41, scale=1024.0)
        dict(net.named_parameters())["decoder.up2.conv1x1.weight"].grad[3, 5] = bad
        sc.step(opt)
        sc.update()
        assert torch.equal(net.flat_params, keep) and torch.equal(opt.m, mom)
    assert sc.get_scale() == 256.0


def test_refusals():
    net = _net()
    with pytest.raises(ValueError):
        FusedMuon(net, lr=0.02, frozen="torch1")
    with pytest.raises(ValueError):
        FusedMuon(net, lr=0.02, momentum=1.0)
    with pytest.raises(ValueError):
        FusedMuon(net, lr=0.02, ns_steps=0)


class _Head(FlatStoreMixin, nn.Module):
    def __init__(self, classes, width):
        super().__init__()
        self.weight = nn.Parameter(torch.randn(classes, width) / width ** 0.5)
        self.bias = nn.Parameter(torch.zeros(classes))
        self._fi_finish_init()


def _head_step(head, opt, x, lab):
    head.zero_grad()
    loss = ops.linear_ce_loss(x, head.weight, head.bias, lab, 255)
    loss.backward()
    opt.step()
    opt.advance_lr()
    return loss.detach()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_gradient_and_step_together(dtype):
    torch.manual_seed(5)
    head = _Head(105, 48).cuda()
    x = torch.randn(3, 20, 20, 48, device="cuda").to(dtype)
    lab = torch.randint(0, 105, (3, 20, 20), device="cuda")
    lab[torch.rand(lab.shape, device="cuda") < 0.5] = 255
    opt = FusedMuon(head, lr=0.02, base_lr=0.02, max_iterations=50)
    w0, b0 = head.weight.detach().clone().requires_grad_(True), head.bias.detach().clone().requires_grad_(True)
    loss = _head_step(head, opt, x, lab)
    # the gradients lie in the flat buffer and are the ones that plain leaves get
    want = ops.linear_ce_loss(x, w0, b0, lab, 255)
    gw, gb = torch.autograd.grad(want, (w0, b0))
    assert torch.equal(loss, want.detach()) and head.weight.grad.data_ptr() == head.weight._fi_gview.data_ptr()
    assert torch.equal(head.weight.grad, gw) and torch.equal(head.bias.grad, gb)
    ref = _Reference(argparse.Namespace(named_parameters=lambda: [("weight", w0), ("bias", b0)]), 0.02)
    ref.step({"weight": gw, "bias": gb})
    ref.check(head, 1)
    # two losses of one step add up in the buffer
    head.zero_grad()
    (ops.linear_ce_loss(x, head.weight, head.bias, lab, 255) + ops.linear_ce_loss(x, head.weight, None, lab, 255, "sum")).backward()
    one, two = (torch.autograd.grad(f, head_w) for f, head_w in (
        (lambda w: (ops.linear_ce_loss(x, w, head.bias.detach(), lab, 255), w))(head.weight.detach().clone().requires_grad_(True)),
        (lambda w: (ops.linear_ce_loss(x, w, None, lab, 255, "sum"), w))(head.weight.detach().clone().requires_grad_(True))))
    assert torch.allclose(head.weight.grad, one[0] + two[0], rtol=0, atol=2.0 ** -22 * float(two[0].abs().max()))


def test_captured_steps_equal_eager_steps():
    torch.manual_seed(6)
    heads = [_Head(300, 64).cuda() for _ in range(2)]
    heads[1].load_state_dict(heads[0].state_dict())
    x = torch.randn(2000, 64, device="cuda").bfloat16()
    lab = torch.randint(0, 300, (2000,), device="cuda")
    opts = [FusedMuon(h, lr=0.02, base_lr=0.02, max_iterations=50) for h in heads]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _head_step(heads[0], opts[0], x, lab)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = _head_step(heads[0], opts[0], x, lab)
    want = _head_step(heads[1], opts[1], x, lab)
    for k in range(4):
        x.copy_(torch.randn(2000, 64, device="cuda"))
        lab.copy_(torch.randint(0, 300, (2000,), device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        want = _head_step(heads[1], opts[1], x, lab)
        assert torch.equal(got, want) and torch.equal(heads[0].flat_params, heads[1].flat_params), k
        torch.cuda.synchronize()


@pytest.mark.parametrize("use_graph", [False, True])
def test_a_client_trains_with_it(use_graph):
    """args.optimizer = "muon": the federated client's round, eager and captured, FedICRA's freeze schedule included."""
    from fedicra_amd.flower_common import MyModel
    from fedicra_amd.flower_pCE_2D import MyClient
    from fedicra_amd.networks.unet import UNet_LC
    from helpers import loader
    K, cid = 3, 1
    args = argparse.Namespace(strategy="FedICRA", amp=0, model="unet_lc", cid=cid, min_num_clients=K, num_classes=2, img_class="odoc", base_lr=0.02,
                              max_iterations=100, iters=6, rep_iters=3, alpha=1.0, use_graph=use_graph, optimizer="muon", in_chns=1)
    ops.manual_seed(5)
    torch.manual_seed(2)
    net = UNet_LC(1, 2, 1, K, K, cid).cuda()
    set_compute_dtype(net, "fp32")
    batches = loader(2, 2, 32, cid=cid)
    for b in batches:
        b["image"] = b["image"].unsqueeze(1) if b["image"].dim() == 3 else b["image"]
    client = MyClient(args, MyModel(args, net, batches, batches), batches, batches)
    before = net.flat_params.clone()
    for r in range(2):
        client._train({"iter_global": 6 * (r + 1), "iters": 6, "eval_iters": 6, "batch_size": 2, "stage": "fit"})
        assert np.isfinite(np.array([v for row in [client.last_losses] for v in np.ravel(row)], dtype=np.float64)).all()
    assert isinstance(client.optimizer, FusedMuon) and torch.isfinite(net.flat_state).all()
    p = dict(net.named_parameters())
    moved = [n for n in p if not torch.equal(net.flat_params[p[n]._fi_off:p[n]._fi_off + p[n].numel()], before[p[n]._fi_off:p[n]._fi_off + p[n].numel()])]
    assert "decoder.out_conv.weight" in moved and "encoder.down4.maxpool_conv.1.conv_conv.4.weight" in moved
    if use_graph:
        assert any(st.graph is not None for st in client._steps.values())
