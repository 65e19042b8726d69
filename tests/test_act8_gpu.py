"""GPU: layers that keep their input in 8 bits (quant.act8_linear, quant.act8_norm_relu) against their definition evaluated in
64 bits on the CPU.  What is kept -- codes, scales, the ReLU's bits, mean and 1/deviation -- is fixed bit by bit.  A sum of n
float32 roundings, each at most 2^-24 of the sum of magnitudes and of either sign, is off by at most 8 sqrt(n) 2^-24 of it
(eight standard deviations: the largest of some 10^6 values stays below six).  n counts six part products a multiply-add."""
import copy

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
GROUP = 128


def close(got, want, size, n, what=""):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = 8 * n ** 0.5 * E32 * size.double().cpu() + 1e-35
    err = (got - want).abs()
    worst = float((err / tol).max())
    print(f"{what}: {worst:.3f} of the tolerance")
    assert worst <= 1.0, f"{what}: {worst}"


def rule64(v):
    """codes and scales of groups of 128 along the last dimension; returns codes padded to whole groups, scales"""
    B, C, L = v.shape
    pad = -L % GROUP
    g = torch.nn.functional.pad(v.double(), (0, pad)).view(B, C, -1, GROUP)
    s = (g.abs().amax(3, keepdim=True) / 127).float().double()
    q = (g / torch.where(s > 0, s, torch.ones_like(s))).round().clamp(-127, 127) * (s > 0)
    return q, s


class Definition:
    """forward and backward of one layer, in 64 bits apart from what is a float32 number by definition; CPU"""

    def __init__(self, x, W, b, norm):
        self.x, self.W, self.b, self.norm = x.detach().cpu().double(), None if W is None else W.detach().cpu().double(), b, norm
        if b is not None:
            self.b = b.detach().cpu().double()
        B, C, L = x.shape
        self.P = B * L
        if norm is None:
            self.u = self.a = self.x
            self.asize = self.x.abs()
        else:
            self.frozen = not norm.training and norm.running_mean is not None
            self.gamma, self.beta = norm.weight.detach().cpu().double()[:, None], norm.bias.detach().cpu().double()[:, None]
            if self.frozen:
                mean, var = norm.running_mean.cpu().double()[:, None], norm.running_var.cpu().double()[:, None]
            else:
                mean = self.x.mean((0, 2))[:, None]
                var = (self.x - mean).square().mean((0, 2))[:, None]
            self.var = var
            self.mu, self.r = mean.float(), (1 / (var + norm.eps).sqrt()).float()
            self.u = ((self.x.float() - self.mu) * self.r).double()
            y = self.gamma * self.u + self.beta
            self.m = (y > 0).double()
            self.a = y.clamp_min(0)
            self.asize = (self.gamma * self.u).abs() + self.beta.abs()
        q, s = rule64(self.u)
        self.q, self.s = q, s
        self.uh = (q * s).reshape(B, C, -1)[:, :, :L]
        self.step = s.expand_as(q).reshape(B, C, -1)[:, :, :L] / 2        # a code is off by at most half a step
        self.ah = self.uh if norm is None else self.m * (self.gamma * self.uh + self.beta).clamp_min(0)
        self.ahsize = self.uh.abs() if norm is None else (self.gamma * self.uh).abs() + self.beta.abs()

    def forward(self):
        h = torch.matmul(self.W, self.a)
        size = torch.matmul(self.W.abs(), self.asize)
        if self.b is not None:
            h, size = h + self.b[:, None], size + self.b.abs()[:, None]
        return h, size

    def through_norm(self, da, dasize):
        """(dx, size), (dgamma, size), (dbeta, size) of a gradient da of a"""
        dy, dysize = self.m * da, self.m * dasize
        dbeta, dgamma = dy.sum((0, 2)), (dy * self.uh).sum((0, 2))
        sb, sg = dysize.sum((0, 2)), (dysize * self.uh.abs()).sum((0, 2))
        k = self.gamma * self.r.double()
        if self.frozen:
            return (k * dy, k.abs() * dysize), (dgamma, sg), (dbeta, sb)
        dx = k * (dy - dbeta[:, None] / self.P - self.uh * dgamma[:, None] / self.P)
        size = k.abs() * (dysize + sb[:, None] / self.P + self.uh.abs() * sg[:, None] / self.P)
        return (dx, size), (dgamma, sg), (dbeta, sb)

    def backward(self, g):
        g = g.detach().cpu().double()
        dW = torch.einsum("bnl,bkl->nk", g, self.ah)
        dWsize = torch.einsum("bnl,bkl->nk", g.abs(), self.ahsize)
        da, dasize = torch.matmul(self.W.t(), g), torch.matmul(self.W.abs().t(), g.abs())
        out = {"dW": (dW, dWsize), "db": (g.sum((0, 2)), g.abs().sum((0, 2)))}
        if self.norm is None:
            out["dx"] = (da, dasize)
        else:
            out["dx"], out["dgamma"], out["dbeta"] = self.through_norm(da, dasize)
        return out


def make(B, K, L, N, norm, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed + 7 * B + 11 * K + L + 13 * N)
    x = torch.randn(B, K, L, generator=g) * (0.3 + torch.rand(K, 1, generator=g)) + torch.randn(K, 1, generator=g) * 0.5
    W = torch.randn(N, K, generator=g) / K ** 0.5
    b = torch.randn(N, generator=g) * 0.1 if bias else None
    go = torch.randn(B, N, L, generator=g)
    bn = None
    if norm:
        bn = nn.BatchNorm1d(K)
        with torch.no_grad():
            bn.weight.copy_(torch.rand(K, generator=g) + 0.5)
            bn.bias.copy_(torch.randn(K, generator=g) * 0.3)
            bn.running_mean.copy_(torch.randn(K, generator=g) * 0.5)
            bn.running_var.copy_(torch.rand(K, generator=g) + 0.3)
            if K > 2:
                bn.weight[1] = 0          # a channel that the norm switches off still has a gradient for its weight
                bn.weight[2] *= -1
        bn = bn.cuda()
    cuda = [t if t is None else t.cuda() for t in (x, W, b, go)]
    for t in cuda[:3]:
        if t is not None:
            t.requires_grad_()
    return (*cuda, bn)


SHAPES = [(1, 1, 2, 1), (1, 3, 1, 5), (2, 6, 33, 32), (1, 32, 128, 64), (3, 67, 129, 64), (2, 64, 1000, 128), (2, 131, 300, 128), (1, 384, 515, 256),
          (4, 40, 31, 7), (1, 16, 2050, 33), (2, 256, 260, 256), (1, 1000, 70, 20), (1, 20, 70, 1000), (1, 300, 257, 300), (5, 130, 127, 129)]


@pytest.mark.parametrize("mode", ["plain", "batch", "frozen"])
@pytest.mark.parametrize("B,K,L,N", SHAPES)
def test_layer_against_its_definition(B, K, L, N, mode):
    from pointcloudsegmentation_amd import quant
    if mode == "batch" and B * L < 2:
        pytest.skip("batch statistics need two values")
    x, W, b, g, norm = make(B, K, L, N, mode != "plain", bias=(K + N) % 3 != 0)
    if norm is not None:
        norm.train(mode == "batch")
    ref = Definition(x, W, b, norm)
    rm = None if norm is None else (norm.running_mean.clone(), norm.running_var.clone())
    h = quant.act8_linear(x, W, b, norm=norm)
    want, size = ref.forward()
    close(h, want, size, 6 * K + 8, "h")
    leaves = [t for t in (x, W, b) if t is not None] + ([norm.weight, norm.bias] if norm is not None else [])
    names = ["dx", "dW"] + (["db"] if b is not None else []) + (["dgamma", "dbeta"] if norm is not None else [])
    grads = torch.autograd.grad(h, leaves, g)
    P = B * L
    n = {"dx": 6 * N + P + 16, "dW": 6 * P + 16, "db": P, "dgamma": P + 6 * N + 8, "dbeta": P + 6 * N}
    exp = ref.backward(g)
    for name, got in zip(names, grads):
        close(got, exp[name][0], exp[name][1], n[name], name)
    if norm is not None:
        if mode == "batch":
            m = norm.momentum
            P = B * L
            close(norm.running_mean, (1 - m) * rm[0].cpu().double() + m * ref.x.mean((0, 2)), rm[0].abs().cpu() + 1, 4, "running mean")
            close(norm.running_var, (1 - m) * rm[1].cpu().double() + m * ref.var[:, 0] * P / (P - 1), rm[1].cpu() + ref.var[:, 0] * 2, 4, "running var")
            assert int(norm.num_batches_tracked) == 1
        else:
            assert torch.equal(norm.running_mean, rm[0]) and torch.equal(norm.running_var, rm[1])
            assert int(norm.num_batches_tracked) == 0


@pytest.mark.parametrize("L,offset", [(4100, 0), (4099, 0), (4160, 0), (4100, 1), (4160, 3)])
def test_wide_weight_gradient_with_part_of_a_block_at_the_end(L, offset):
    """long enough for 128 x 128 tiles of dW; the last block of a cloud ends in its first, its third piece of 32 points, rows start on 16
    bytes or not (by their length, by where g begins), and the last tile holds 72 of 128 rows: what lies behind a cloud's last point
    is neither read nor added"""
    from pointcloudsegmentation_amd import quant
    B, K, N = 17, 130, 200
    x, W, b, g, _ = make(B, K, L, N, False)
    room = torch.full((B * N * L + 4096,), float("nan"), device="cuda")
    room[offset:offset + B * N * L] = g.reshape(-1)
    g = room[offset:offset + B * N * L].view(B, N, L)
    ref = Definition(x, W, b, None).backward(g)
    h = quant.act8_linear(x, W, b)
    dW, db = torch.autograd.grad(h, [W, b], g)
    close(dW, *ref["dW"], 6 * B * L + 16, "dW")
    close(db, *ref["db"], B * L, "db")


@pytest.mark.parametrize("mode", ["batch", "frozen", "untracked"])
@pytest.mark.parametrize("B,C,L", [(1, 1, 2), (3, 5, 1), (2, 64, 130), (1, 100, 1025), (3, 33, 257), (2, 256, 64)])
def test_norm_relu_against_its_definition(B, C, L, mode):
    from pointcloudsegmentation_amd import quant
    x, _, _, _, norm = make(B, C, L, 1, True)
    if mode == "untracked":
        n2 = nn.BatchNorm1d(C, track_running_stats=False).cuda()
        n2.load_state_dict({"weight": norm.weight, "bias": norm.bias})
        norm = n2.eval()
    norm.train(mode == "batch")
    ref = Definition(x, None, None, norm)
    y = quant.act8_norm_relu(x, norm)
    close(y, ref.a, ref.asize, 8, "y")
    g = torch.randn(B, C, L, generator=torch.Generator().manual_seed(3)).cuda()
    dx, dgamma, dbeta = torch.autograd.grad(y, [x, norm.weight, norm.bias], g)
    gd = g.cpu().double()
    want = ref.through_norm(gd, gd.abs())
    P = B * L
    for name, got, (w, size) in zip(("dx", "dgamma", "dbeta"), (dx, dgamma, dbeta), want):
        close(got, w, size, P + 16, name)


@pytest.mark.parametrize("B,K,L", [(1, 1, 1), (2, 5, 127), (3, 40, 300), (1, 64, 1024)])
@pytest.mark.parametrize("norm", [False, True])
def test_what_is_kept(B, K, L, norm):
    """codes, scales, bits, mean and 1/deviation, bit by bit, and nothing behind them"""
    from pointcloudsegmentation_amd import _lib, runtime as rt
    if norm and B * L < 2:
        pytest.skip("batch statistics need two values")
    N = 8
    x, W, b, _, bn = make(B, K, L, N, norm)
    with torch.no_grad():
        x[:, 0, : L // 2] = 0
    ref = Definition(x, W, b, bn)
    lib = _lib.lib()
    nk, nw = lib.p2n_act8_kept_bytes(B, K, L, int(norm)), lib.p2n_act8_workspace_bytes(B, K, L, N)
    kept = torch.full((nk + 256,), 0x5A, dtype=torch.uint8, device="cuda")
    ws, h = torch.empty(nw, dtype=torch.uint8, device="cuda"), torch.empty(B, N, L, device="cuda")
    q = rt.ptr
    _lib.check(lib.p2n_act8_forward(x.data_ptr(), B, K, L, W.data_ptr(), b.data_ptr(), N, q(bn.weight) if norm else None, q(bn.bias) if norm else None,
                                    None, None, None, 0.0, 1e-5, h.data_ptr(), kept.data_ptr(), nk, ws.data_ptr(), nw, rt.stream_handle(x.device)), "fwd")
    assert bool((kept[nk:] == 0x5A).all())
    NB, K4 = (L + 127) // 128, (K + 3) // 4 * 4
    up = lambda n: (n + 255) // 256 * 256                                             # noqa: E731
    codes = kept[:B * NB * K * 128].view(torch.int8).view(B, NB, K, 128).transpose(1, 2)
    assert torch.equal(codes.cpu().double(), ref.q)
    off = up(B * NB * K * 128)
    scale = kept[off:off + B * NB * K4 * 4].view(torch.float32).view(B, NB, K4)
    assert torch.equal(scale[:, :, :K].transpose(1, 2).unsqueeze(3).cpu().double(), ref.s) and float(scale[:, :, K:].abs().sum()) == 0
    if norm:
        off += up(B * NB * K4 * 4)
        words = kept[off:off + B * NB * 4 * K4 * 4].view(torch.int32).view(B, NB, 4, K4).cpu()
        p = torch.arange(32, dtype=torch.int32)
        bits = (words.unsqueeze(4) >> ((p >> 1) + 16 * (p & 1))) & 1                  # (B, NB, 4, K4, 32)
        bits = bits.permute(0, 3, 1, 2, 4).reshape(B, K4, -1)
        assert torch.equal(bits[:, :K, :L].double(), ref.m) and int(bits[:, :K, L:].sum()) == 0 and int(bits[:, K:].sum()) == 0
        off += up(B * NB * 4 * K4 * 4)
        stat = kept[off:off + 8 * K].view(torch.float32).cpu()
        assert torch.equal(stat[:K], ref.mu[:, 0]) and torch.equal(stat[K:], ref.r[:, 0])


def true_gradients(x, W, b, norm, g):
    """stock torch in float64: the gradients of the layer itself, nothing in 8 bits"""
    xd, Wd = x.detach().cpu().double().requires_grad_(), W.detach().cpu().double().requires_grad_()
    n = copy.deepcopy(norm).cpu().double()
    h = nn.functional.conv1d(torch.relu(n(xd)), Wd.unsqueeze(2), b.detach().cpu().double())
    return torch.autograd.grad(h, [xd, Wd, n.weight, n.bias], g.cpu().double())


@pytest.mark.parametrize("mode", ["batch", "frozen"])
def test_gradients_are_the_layers_up_to_half_a_step(mode):
    """against the float64 gradients of the layer without any 8 bits: what the codes can move them by is at most half a
    step of each kept value, carried through the formulas"""
    from pointcloudsegmentation_amd import quant
    B, K, L, N = 3, 64, 500, 48
    x, W, b, g, norm = make(B, K, L, N, True)
    norm.train(mode == "batch")
    n2 = copy.deepcopy(norm)
    ref = Definition(x, W, b, norm)
    h = quant.act8_linear(x, W, b, norm=norm)
    dx, dW, dgamma, dbeta = torch.autograd.grad(h, [x, W, norm.weight, norm.bias], g)
    tx, tW, tg, tb = true_gradients(x, W, b, n2, g)
    gd, P = g.cpu().double().abs(), B * L
    slack = 1e-5                                                       # float32 roundings (test above), of the sums of magnitudes
    e = ref.backward(g)
    dW_bound = torch.einsum("bnl,bkl->nk", gd, ref.gamma.abs() * ref.step) + slack * e["dW"][1]
    assert bool(((dW.cpu().double() - tW).abs() <= dW_bound).all())
    dy = (ref.m * torch.matmul(ref.W.t(), g.cpu().double())).abs()
    dg_bound = (dy * ref.step).sum((0, 2)) + slack * e["dgamma"][1]
    assert bool(((dgamma.cpu().double() - tg).abs() <= dg_bound).all())
    assert bool(((dbeta.cpu().double() - tb).abs() <= slack * e["dbeta"][1]).all())
    k = (ref.gamma * ref.r.double()).abs()
    dx_bound = slack * e["dx"][1]
    if mode == "batch":
        dx_bound = dx_bound + k * (ref.step * tg.abs()[:, None] + (ref.u.abs() + ref.step) * dg_bound[:, None]) / P
    assert bool(((dx.cpu().double() - tx).abs() <= dx_bound).all())


def test_gradients_against_differences():
    """directional differences of the float64 layer, along random directions of every input"""
    from pointcloudsegmentation_amd import quant
    B, K, L, N = 2, 24, 400, 16
    x, W, b, g, norm = make(B, K, L, N, True)
    h = quant.act8_linear(x, W, b, norm=norm)
    leaves = [x, W, b, norm.weight, norm.bias]
    grads = [t.cpu().double() for t in torch.autograd.grad(h, leaves, g)]
    base = [t.detach().cpu().double() for t in leaves]
    gd = g.cpu().double()

    def loss(v):
        xx, WW, bb, ga, be = v
        mean = xx.mean((0, 2), keepdim=True)
        u = (xx - mean) / ((xx - mean).square().mean((0, 2), keepdim=True) + norm.eps).sqrt()
        return float((gd * (torch.matmul(WW, (ga[:, None] * u + be[:, None]).clamp_min(0)) + bb[:, None])).sum())

    gen = torch.Generator().manual_seed(11)
    for i in range(5):
        d = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        eps = 1e-6
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + eps * d, base[i] - eps * d
        diff = (loss(up) - loss(down)) / (2 * eps)
        size = float((grads[i].abs() * d.abs()).sum())
        # half a step of 8 bits is 1/254 of a group's largest value, some 1/70 of a typical one; signs are random: 1 % of the
        # magnitudes bounds the sum with room (the exact bound is the test above)
        assert abs(float((grads[i] * d).sum()) - diff) <= 0.01 * size, i


@pytest.mark.parametrize("B,K,L,N", [(2, 40, 200, 24), (2, 70, 200, 24), (2, 40, 200, 100), (17, 130, 4100, 200)])
def test_only_what_is_asked_for(B, K, L, N):
    from pointcloudsegmentation_amd import quant
    x, W, b, g, norm = make(B, K, L, N, True)
    full = torch.autograd.grad(quant.act8_linear(x, W, b, norm=norm), [x, W, b, norm.weight, norm.bias], g)
    for wanted in ([0], [1], [2], [3], [4], [1, 2], [0, 3]):
        ts = [x, W, b, norm.weight, norm.bias]
        for i, t in enumerate(ts):
            t.requires_grad_(i in wanted)
        got = torch.autograd.grad(quant.act8_linear(x, W, b, norm=norm), [ts[i] for i in wanted], g)
        for i, t in zip(wanted, got):
            assert torch.equal(t, full[i]), (wanted, i)
        for t in ts:
            t.requires_grad_(True)
    for wanted in ([0], [1], [2]):
        ts = [x, W, b]
        ref = torch.autograd.grad(quant.act8_linear(x, W, b), ts, g)
        for i, t in enumerate(ts):
            t.requires_grad_(i in wanted)
        got = torch.autograd.grad(quant.act8_linear(x, W, b), [ts[i] for i in wanted], g)
        assert torch.equal(got[0], ref[wanted[0]])
        for t in ts:
            t.requires_grad_(True)


@pytest.mark.parametrize("B,K,L,N", [(2, 33, 131, 31), (1, 70, 45, 67), (3, 5, 129, 130), (17, 130, 4100, 200)])
def test_memory_behind_the_results_is_left_as_it_was(B, K, L, N):
    from pointcloudsegmentation_amd import _lib, runtime as rt
    lib = _lib.lib()
    x, W, b, g, bn = make(B, K, L, N, True)
    nk, nw = lib.p2n_act8_kept_bytes(B, K, L, 1), lib.p2n_act8_workspace_bytes(B, K, L, N)
    sizes = {"h": B * N * L, "dx": B * K * L, "dW": N * K, "db": N, "dgamma": K, "dbeta": K, "kept": nk // 4, "ws": (nw + 3) // 4}
    room = {k: torch.full((n + 1024,), 7.0, device="cuda") for k, n in sizes.items()}
    p = {k: t.data_ptr() for k, t in room.items()}
    s = rt.stream_handle(x.device)
    _lib.check(lib.p2n_act8_forward(x.data_ptr(), B, K, L, W.data_ptr(), rt.ptr(b), N, bn.weight.data_ptr(), bn.bias.data_ptr(), None, None, None, 0.0,
                                    1e-5, p["h"], p["kept"], nk, p["ws"], nw, s), "forward")
    _lib.check(lib.p2n_act8_backward(g.data_ptr(), B, K, L, W.data_ptr(), N, bn.weight.data_ptr(), bn.bias.data_ptr(), 0, p["kept"], nk, p["dx"], p["dW"],
                                     p["db"], p["dgamma"], p["dbeta"], p["ws"], nw, s), "backward")
    for k, n in sizes.items():
        assert bool((room[k][n:] == 7.0).all()), k
        if k not in ("kept", "ws"):
            assert not bool((room[k][:n] == 7.0).any()), k


def test_strides_expanded_gradients_and_second_backward():
    from pointcloudsegmentation_amd import quant
    x, W, b, g, norm = make(2, 40, 200, 24, True)
    h = quant.act8_linear(x, W, b, norm=norm)
    a1 = torch.autograd.grad(h, [x, W, b], g, retain_graph=True)
    a2 = torch.autograd.grad(h, [x, W, b], g, retain_graph=True)            # what is kept is only read
    a3 = torch.autograd.grad(h, [x, W, b], g.transpose(1, 2).contiguous().transpose(1, 2))
    for p, q, r in zip(a1, a2, a3):
        assert torch.equal(p, q) and torch.equal(p, r)
    xt = x.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    ht = quant.act8_linear(xt, W.unsqueeze(2), b, norm=norm)
    assert torch.equal(ht, h)
    s1 = torch.autograd.grad(quant.act8_linear(x, W, b, norm=norm).sum(), [x, W, b])
    s2 = torch.autograd.grad(quant.act8_linear(x, W, b, norm=norm), [x, W, b], torch.ones_like(g))
    for p, q in zip(s1, s2):
        assert torch.equal(p, q)
    one = x.detach()[:1].clone().requires_grad_()
    gx, = torch.autograd.grad(quant.act8_linear(one.expand(2, 40, 200), W, b), [one], g)
    two = one.detach().expand(2, 40, 200).contiguous().requires_grad_()
    gt, = torch.autograd.grad(quant.act8_linear(two, W, b), [two], g)
    assert torch.equal(gx, gt.sum(0, keepdim=True))
    with pytest.raises(RuntimeError):
        q = torch.autograd.grad(quant.act8_linear(x, W, b), [x], g, create_graph=True)[0]
        torch.autograd.grad(q.sum(), [W])


def test_no_second_derivative():
    """under create_graph the gradients are the same, and differentiating them is refused instead of answered with nothing"""
    from pointcloudsegmentation_amd import quant
    x, W, b, g, norm = make(2, 20, 150, 12, True)
    plain = torch.autograd.grad(quant.act8_linear(x, W, b, norm=norm), [x, W], g)
    g.requires_grad_()
    again = torch.autograd.grad(quant.act8_linear(x, W, b, norm=norm), [x, W], g, create_graph=True)
    for p, q in zip(plain, again):
        assert torch.equal(p, q)
        with pytest.raises(RuntimeError):
            q.sum().backward(retain_graph=True)
    go = torch.randn(2, 20, 150, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(quant.act8_norm_relu(x, norm), [x], go, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_buffers_show_that_they_changed():
    """the running statistics and the count of batches are written by the kernels: their versions move, as BatchNorm1d moves them"""
    from pointcloudsegmentation_amd import quant
    x, W, b, g, norm = make(2, 20, 150, 12, True)
    norm.train()
    for call in (lambda: quant.act8_linear(x, W, b, norm=norm), lambda: quant.act8_norm_relu(x, norm)):
        before = [t._version for t in norm.buffers()]
        n = int(norm.num_batches_tracked)
        call()
        assert int(norm.num_batches_tracked) == n + 1
        assert all(t._version > v for t, v in zip(norm.buffers(), before))
    norm.eval()
    before = [t._version for t in norm.buffers()]
    quant.act8_linear(x, W, b, norm=norm)
    assert [t._version for t in norm.buffers()] == before
    norm.train()
    norm.num_batches_tracked = norm.num_batches_tracked.cpu()
    with pytest.raises(ValueError):
        quant.act8_linear(x, W, b, norm=norm)


def test_repeats_are_identical():
    """every sum has a fixed order: the same call gives the same bits"""
    from pointcloudsegmentation_amd import quant
    x, W, b, g, norm = make(4, 96, 3000, 80, True)
    leaves = [x, W, b, norm.weight, norm.bias]
    first = None
    for _ in range(3):
        h = quant.act8_linear(x, W, b, norm=norm)
        got = [h.detach()] + list(torch.autograd.grad(h, leaves, g))
        if first is not None:
            assert all(torch.equal(p, q) for p, q in zip(first, got))
        first = got


def test_kept_bytes_and_peak_memory():
    from pointcloudsegmentation_amd import _lib, quant
    B, K, L, N = 4, 128, 8192, 64
    x, W, b, g, norm = make(B, K, L, N, True)
    n = _lib.lib().p2n_act8_kept_bytes(B, K, L, 1)
    assert n <= B * K * L * 1.16 + 8 * K + 1024
    del g
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    h = quant.act8_linear(x, W, b, norm=norm)
    held = torch.cuda.memory_allocated() - before - h.numel() * 4
    assert held <= n + 8192, (held, n)


@pytest.mark.parametrize("B,K,L,N,normed", [(1, 72, 2 ** 24, 72, False), (3, 40, 2 ** 23 - 57, 130, True)])
def test_offsets_past_32_bits(B, K, L, N, normed):
    """x and h are over 4 GiB: outputs and dx at columns from everywhere, and the sums over all columns, which are formed here from the
    rule's codes in 64 bits, 2^20 columns (a multiple of 128) at a time"""
    from pointcloudsegmentation_amd import quant
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(B, K, L, device="cuda", generator=gen)
    W = torch.randn(N, K, device="cuda", generator=gen) / K ** 0.5
    norm = None
    if normed:
        norm = nn.BatchNorm1d(K).cuda().eval()
        with torch.no_grad():
            norm.weight.uniform_(0.5, 1.5, generator=gen)
            norm.bias.uniform_(-0.3, 0.3, generator=gen)
    leaves = [x.requires_grad_(), W.requires_grad_()] + ([norm.weight, norm.bias] if normed else [])
    h = quant.act8_linear(x, W, None, norm=norm)
    g = torch.randn(B, N, L, device="cuda", generator=gen)
    grads = [t.detach() for t in torch.autograd.grad(h, leaves, g)]
    h, x, Wd = h.detach(), x.detach(), W.detach().double()
    sums = [torch.zeros(2, N, K, device="cuda", dtype=torch.float64)] + [torch.zeros(2, K, device="cuda", dtype=torch.float64) for _ in range(2)]
    for b in range(B):
        for l in range(0, L, 2 ** 20):
            n = min(2 ** 20, L - l)
            v, gg = x[b, :, l:l + n], g[b, :, l:l + n].double()
            mask = torch.ones((), device="cuda", dtype=torch.float64)
            u = v
            if normed:
                r = (1 / (norm.running_var.double() + norm.eps).sqrt()).float()[:, None]
                u = (v - norm.running_mean[:, None]) * r
            s = (torch.nn.functional.pad(u.double(), (0, -n % GROUP)).view(K, -1, GROUP).abs().amax(2, keepdim=True) / 127).float().double()
            uh = ((torch.nn.functional.pad(u.double(), (0, -n % GROUP)).view(K, -1, GROUP) / s.clamp_min(1e-300)).round().clamp(-127, 127) * s).reshape(K, -1)[:, :n]
            a, ah, asize = u.double(), uh, uh.abs()
            if normed:
                ga, be = norm.weight.detach().double()[:, None], norm.bias.detach().double()[:, None]
                y = ga * u.double() + be
                mask = (y > 0).double()
                a, ah, asize = y.clamp_min(0), mask * (ga * uh + be).clamp_min(0), (ga * uh).abs() + be.abs()
            sums[0] += torch.stack([torch.matmul(gg, ah.t().contiguous()), torch.matmul(gg.abs(), asize.t().contiguous())])
            da, dasize = torch.matmul(Wd.t().contiguous(), gg), torch.matmul(Wd.abs().t().contiguous(), gg.abs())
            dy, dysize = mask * da, mask * dasize
            sums[1] += torch.stack([(dy * uh).sum(1), (dysize * uh.abs()).sum(1)])
            sums[2] += torch.stack([dy.sum(1), dysize.sum(1)])
            if l in (0, L // 2 ** 21 * 2 ** 20) or l + n == L:
                k = (ga * r.double()) if normed else torch.ones((), device="cuda", dtype=torch.float64)
                for c in (slice(0, 2000), slice(n - 2000, n)):
                    close(h[b, :, l:l + n][:, c], torch.matmul(Wd, a[:, c]), torch.matmul(Wd.abs(), a[:, c].abs() + (be.abs() if normed else 0)), 6 * K + 8, "h")
                    close(grads[0][b, :, l:l + n][:, c], k * dy[:, c], k.abs() * dysize[:, c], 6 * N + 16, "dx")
    # terms of either sign: a sum of k of them stays within 6 sqrt(k) of their deviation d, its rounding within 2^-24 of that; 6 P
    # such roundings of either sign stay within 8 * 6 d sqrt(6 P P / 2) 2^-24 = 83 P d 2^-24, and the sum of magnitudes is 0.8 P d:
    # 104 = 8 sqrt(169)
    for name, got, want in zip(("dW", "dgamma", "dbeta"), grads[1:], sums):
        close(got, want[0], want[1], 169, name)


def test_wide_weight_gradient_of_the_longest_rows():
    """128 rows of over 4 GiB whose last 32 points are not all there: nothing behind a row's end is added.  g holds whole numbers, so the
    sums of its rows are exact, and dW is a sum of whole numbers times scales"""
    from pointcloudsegmentation_amd import quant
    L = 2 ** 24 - 12
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.ones(1, 128, L, device="cuda")
    W = torch.zeros(140, 128, device="cuda", requires_grad=True)
    b = torch.zeros(140, device="cuda", requires_grad=True)
    h = quant.act8_linear(x, W, b)
    g = torch.randint(0, 2, (1, 140, L), device="cuda", generator=gen).float()
    dW, db = torch.autograd.grad(h, [W, b], g)
    want = g[0].sum(1, dtype=torch.float64)
    assert bool((want < 2 ** 24).all())
    assert torch.equal(db.double(), want)
    # every code is 127 and its scale the float32 next to 1/127; a share's sum is rounded 6 times a step at most (as above, of one sign)
    uh = 127 * float(torch.tensor(1.0).div(127))
    assert bool(((dW.double() - want[:, None] * uh).abs() <= want[:, None] * 2.0 ** -24 * 8 * 169 ** 0.5).all())


def test_two_streams_at_once():
    """steps on two streams share nothing: each gives what it gives alone"""
    from pointcloudsegmentation_amd import quant
    def step(x, W, b, g, norm):
        h = quant.act8_linear(x, W, b, norm=norm)
        return (h.detach(),) + torch.autograd.grad(h, [x, W, b, norm.weight, norm.bias], g)
    data = [make(2, 64, 3000, 128, True, seed=s, bias=True) for s in (0, 1)]
    for d in data:
        d[4].momentum = 0.0          # running statistics stay as they are
    want = [step(*d) for d in data]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        for d, s in zip(data, streams):
            with torch.cuda.stream(s):
                got.append(step(*d))
    torch.cuda.synchronize()
    for i, ts in enumerate(got):
        for a, b in zip(ts, want[i % 2]):
            assert torch.equal(a, b), i


def test_captured_step_replays():
    from pointcloudsegmentation_amd import quant
    x, W, b, g, norm = make(2, 64, 700, 96, True)
    leaves = [x, W, b, norm.weight, norm.bias]

    def step():
        h = quant.act8_linear(x, W, b, norm=norm)
        return [h.detach()] + list(torch.autograd.grad(h, leaves, g))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(4):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            g.copy_(torch.randn_like(g))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q), rep


def test_nonfinite_values_show():
    """a NaN reaches the outputs and gradients of its channel; without a norm it stays in its cloud's point on the way forward"""
    from pointcloudsegmentation_amd import quant
    x, W, b, g, _ = make(2, 20, 300, 12, False)
    clean = quant.act8_linear(x, W, b).detach()
    with torch.no_grad():
        x[1, 3, 200] = float("nan")
    h = quant.act8_linear(x, W, b)
    assert bool(torch.isnan(h[1, :, 200]).all())
    keep = torch.ones(2, 300, dtype=torch.bool)
    keep[1, 200] = False
    assert torch.equal(h.detach().transpose(1, 2)[keep], clean.transpose(1, 2)[keep])
    dx, dW = torch.autograd.grad(h, [x, W], g)
    assert bool(torch.isnan(dW[:, 3]).all()) and not bool(torch.isnan(dW[:, :3]).any()) and not bool(torch.isnan(dx).any())
    x, W, b, g, norm = make(2, 20, 300, 12, True)
    with torch.no_grad():
        x[1, 3, 200] = float("inf")
    h = quant.act8_linear(x, W, b, norm=norm)
    assert bool(torch.isnan(h).all())           # the channel's mean is infinite
    dx, dW, dgamma = torch.autograd.grad(h, [x, W, norm.weight], g)
    assert bool(torch.isnan(dW[:, 3]).all()) and not bool(torch.isnan(dW[:, :3]).any())
    assert bool(torch.isnan(dx[:, 3]).all()) and not bool(torch.isnan(dx[:, 4:]).any())
    assert bool(torch.isnan(dgamma[3])) and not bool(torch.isnan(dgamma[4:]).any())
    y = quant.act8_norm_relu(x, norm)
    assert bool(torch.isnan(y[:, 3]).all()) and not bool(torch.isnan(y[:, 4:]).any())


def test_refusals():
    from pointcloudsegmentation_amd import quant
    x, W, b, _, norm = make(2, 16, 30, 8, True)
    for bad in (x.bfloat16(), x.double()):
        with pytest.raises(TypeError):
            quant.act8_linear(bad, W, b)
    for bad in (x.cpu(), x[0], x[:, :, :0], x[:, :15]):
        with pytest.raises(ValueError):
            quant.act8_linear(bad, W, b)
    with pytest.raises(ValueError):
        quant.act8_linear(x, W.cpu(), b)
    with pytest.raises(ValueError):
        quant.act8_linear(x, W, b[:3])
    with pytest.raises(ValueError):
        quant.act8_linear(x, W, b, norm=nn.BatchNorm1d(17).cuda())
    with pytest.raises(ValueError):
        quant.act8_linear(x, W, b, norm=nn.BatchNorm1d(16))
    with pytest.raises(TypeError):
        quant.act8_linear(x, W, b, norm=nn.LayerNorm(16).cuda())
    with pytest.raises(NotImplementedError):
        quant.act8_linear(x, W, b, norm=nn.BatchNorm1d(16, affine=False).cuda())
    with pytest.raises(NotImplementedError):
        quant.act8_linear(x, W, b, norm=nn.BatchNorm1d(16, momentum=None).cuda())
    with pytest.raises(ValueError):
        quant.act8_linear(x[:1, :, :1], W, b, norm=norm.train())
    with pytest.raises(ValueError):
        quant.act8_linear(torch.randn(1, 1025, 4, device="cuda"), torch.randn(3, 1025, device="cuda"))
    with pytest.raises(TypeError):
        quant.act8_norm_relu(x, None)
    with pytest.raises(ValueError):
        quant.act8_norm_relu(x[0], norm)
