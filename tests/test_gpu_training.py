"""The training step and its parts: autograd functions against torch's in 64
bits, the optimizer against torch's, whole steps of HiveFNN, graph replays."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _randn(shape, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _near(got, want, rel, what):
    """Within rel of the largest value: float32 sums of up to a few thousand terms are about 1e-6 of it off, and
    chains of five layers under 20 times that."""
    want = want.double()
    assert float((got.double() - want).abs().max()) <= rel * float(want.abs().max()) + 1e-30, what


def test_layer_norm_autograd():
    from hive_neuralnet_amd.training import layer_norm
    x, w, b, g = _randn((4, 33, 64), 1), _randn((64,), 2), _randn((64,), 3), _randn((4, 33, 64), 4)
    for act in (None, "sigmoid"):
        ins = [t.clone().requires_grad_() for t in (x, w, b)]
        ref = [t.double().requires_grad_() for t in (x, w, b)]
        y = layer_norm(*ins, activation=act)
        a = torch.sigmoid(ref[0]) if act else ref[0]
        z = F.layer_norm(a, (64,), ref[1], ref[2], 1e-5)
        _near(y.detach(), z.detach(), 1e-6, act)
        for p, q in zip(torch.autograd.grad(y, ins, g), torch.autograd.grad(z, ref, g.double())):
            _near(p, q, 1e-5, act)
    x = x.clone().requires_grad_()  # a broadcast gradient, no parameters, a frozen input
    layer_norm(x).sum().backward()
    assert float(x.grad.abs().max()) < 1e-4
    w = w.clone().requires_grad_()
    layer_norm(x.detach(), w, None).sum().backward()
    assert w.grad.shape == (64,)


def test_loss_autograd():
    from hive_neuralnet_amd.training import policy_value_loss
    n = torch.tensor([5, 0, 130, 1, 77], device="cuda")
    B, N = 5, int(n.sum())
    logits, values = _randn((N,), 1), torch.tanh(_randn((B, 1), 2))
    targets = torch.rand((B, 256), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    live = torch.arange(256, device="cuda") < n.unsqueeze(1)
    targets = targets * live / (targets * live).sum(1, keepdim=True).clamp(min=1e-9)
    pw, vt, vw = torch.tensor([1.0, 1, 1, 0, 1], device="cuda"), _randn((B, 1), 4), torch.full((B, 1), 2.0, device="cuda")
    ins = [t.clone().requires_grad_() for t in (logits, values)]
    total, policy, value = policy_value_loss(*ins, n, targets, pw, vt, vw, 0.3)
    assert not policy.requires_grad and not value.requires_grad
    ref = [t.double().requires_grad_() for t in (logits, values)]
    dense = torch.full((B, 256), -1e30, dtype=torch.float64, device="cuda")
    dense[live] = ref[0]
    ce = -(targets.double() * torch.log_softmax(dense, 1) * live).sum(1)
    want = (pw * ce).sum() / pw.sum() + 0.3 * (ref[1] - vt.double()).square().mean()
    _near(total.detach(), want.detach(), 1e-6, "total")
    for p, q in zip(torch.autograd.grad(3.0 * total, ins), torch.autograd.grad(3.0 * want, ref)):
        _near(p, q, 1e-5, "gradient")


def _plain_step(net, batch, value_coef):
    """The losses and gradients of a step, from a double copy of the network and torch's operators on the host."""
    from hive_neuralnet_amd import hive_gpu
    from hive_neuralnet_amd.fnn import HiveFNN
    from hive_neuralnet_amd.replay import build_forward_batch
    twin = HiveFNN(net.config)
    twin.load_state_dict(net.state_dict())
    twin = twin.double()
    ext = hive_gpu.load_extension()
    B = batch.num_actions.shape[0]
    root, succ, a2r, n = build_forward_batch(ext, batch.state_bytes, B, batch.num_actions, batch.root_features,
                                             batch.legal_moves)
    host = lambda t: t.cpu().double() if t.is_floating_point() else t.cpu()  # noqa: E731
    logits, values = twin(host(root), host(succ), host(a2r), host(n))
    logits.retain_grad()
    live = torch.arange(256) < host(n).unsqueeze(1)
    dense = torch.full((B, 256), -1e30, dtype=torch.float64)
    dense[live] = logits
    ce = -(host(batch.policy_targets) * torch.log_softmax(dense, 1) * live).sum(1, keepdim=True)
    pw, vw = host(batch.policy_mask), host(batch.value_mask * batch.value_weights)
    policy = (pw * ce).sum() / pw.sum()
    value = (vw * (values - host(batch.value_targets)).square()).sum() / vw.sum()
    total = policy + value_coef * value
    total.backward()
    # a position's logit gradients add up to zero, so the action tower's biases get sums that cancel: what counts
    # there is the size of the terms, |dlogit| and |dlogit w2 sigmoid'|
    terms = {"action_fc2.bias": float(logits.grad.abs().sum())}
    terms["action_fc1.bias"] = 0.25 * terms["action_fc2.bias"] * float(twin.action_fc2.weight.detach().abs().max())
    return torch.stack([total, policy, value]).detach(), {k: p.grad for k, p in twin.named_parameters()}, terms


@pytest.mark.parametrize("config,mask", [("large", 0), ("medium", 7), ("small", 0)])
def test_train_batch_gradients_match_torch(config, mask):
    from hive_neuralnet_amd.fnn import FNNConfig, HiveFNN
    from hive_neuralnet_amd.training import synthetic_batch, train_batch
    torch.manual_seed(3)
    net = HiveFNN(getattr(FNNConfig, config)()).cuda()
    batch = synthetic_batch(96, mask, 80, 5)
    batch.policy_mask = (torch.arange(96, device="cuda") % 5 != 0).float().unsqueeze(1)
    batch.value_weights = 1.0 + torch.arange(96, device="cuda").float().unsqueeze(1) % 3
    want, grads, terms = _plain_step(net, batch, 0.6)

    class Keep:  # the gradients as the optimizer would see them
        def zero_grad(self, set_to_none):
            net.zero_grad(set_to_none=True)

        def step(self):
            self.grads = {k: p.grad.clone() for k, p in net.named_parameters()}

    keep = Keep()
    losses = train_batch(net, keep, batch, 0.6)
    _near(losses.cpu(), want, 1e-6, "losses")
    for k, g in grads.items():
        if k in terms:  # a term 8 u off, a sum of thousands in a tree 16 u
            assert float((keep.grads[k].cpu().double() - g).abs().max()) <= 24 * U * terms[k], k
        else:
            _near(keep.grads[k].cpu(), g, 5e-5, k)


def test_training_goes_as_torch_does():
    """Fifty steps on one batch against the same network under torch's operators and torch.optim.AdamW in 64 bits
    on the host: the losses stay together (float32 noise of 1e-6 a step, at most 50 of them, each passed on), and
    moments in 8 bits give up less than a tenth of what the steps gain."""
    from hive_neuralnet_amd import hive_gpu
    from hive_neuralnet_amd.fnn import FNNConfig, HiveFNN
    from hive_neuralnet_amd.replay import build_forward_batch
    from hive_neuralnet_amd.training import AdamW, synthetic_batch, train_batch
    batch = synthetic_batch(64, 0, 100, 9)

    def ours(bits):
        torch.manual_seed(1)
        net = HiveFNN(FNNConfig.medium()).cuda()
        optimizer = AdamW(net.parameters(), lr=1e-2, state_bits=bits)
        return torch.stack([train_batch(net, optimizer, batch)[0] for _ in range(50)]).cpu().double()

    torch.manual_seed(1)
    twin = HiveFNN(FNNConfig.medium()).double()
    optimizer = torch.optim.AdamW(twin.parameters(), lr=1e-2)
    root, succ, a2r, n = [t.cpu() for t in build_forward_batch(
        hive_gpu.load_extension(), batch.state_bytes, 64, batch.num_actions, batch.root_features, batch.legal_moves)]
    live = torch.arange(256) < n.unsqueeze(1)
    theirs = []
    for _ in range(50):
        logits, values = twin(root.double(), succ.double(), a2r, n)
        dense = torch.full((64, 256), -1e30, dtype=torch.float64)
        dense[live] = logits
        ce = -(batch.policy_targets.cpu().double() * torch.log_softmax(dense, 1) * live).sum(1)
        total = ce.mean() + (values - batch.value_targets.cpu().double()).square().mean()
        theirs.append(float(total.detach()))
        optimizer.zero_grad()
        total.backward()
        optimizer.step()
    theirs = torch.tensor(theirs, dtype=torch.float64)
    wide, narrow = ours(32), ours(8)
    assert float((wide - theirs).abs().max()) < 50 * 50 * 1e-6 * float(theirs.max())
    assert float(theirs[0] - narrow[-1]) > 0.9 * float(theirs[0] - theirs[-1]) > 0.0


def test_optimizer_matches_torch():
    """Ten steps of two groups against torch.optim.AdamW in 64 bits: each step moves a weight by at most lr, 16 u
    of that and 4 u of the weight off."""
    from hive_neuralnet_amd.training import AdamW
    shapes = [(64, 122), (64,), (1,), (33, 5)]
    a = [torch.nn.Parameter(_randn(s, i)) for i, s in enumerate(shapes)]
    b = [torch.nn.Parameter(p.detach().double()) for p in a]
    groups = lambda ps: [{"params": ps[:2], "weight_decay": 0.2}, {"params": ps[2:], "lr": 3e-3}]  # noqa: E731
    ours = AdamW(groups(a), lr=1e-2, betas=(0.8, 0.95))
    theirs = torch.optim.AdamW(groups(b), lr=1e-2, betas=(0.8, 0.95))
    for k in range(10):
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad = _randn(p.shape, 100 * k + i)
            q.grad = p.grad.double()
        ours.step()
        theirs.step()
    for p, q in zip(a, b):
        bound = 10 * (16 * U * 1e-2 + 4 * U * float(q.detach().abs().max()))
        assert float((p.detach().double() - q.detach()).abs().max()) < bound


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_and_missing_gradients(bits):
    from hive_neuralnet_amd.training import AdamW

    def make():
        ps = [torch.nn.Parameter(_randn(s, i)) for i, s in enumerate([(40, 9), (300,)])]
        ps.append(torch.nn.Parameter(_randn((70,), 7).bfloat16()))
        return ps, AdamW(ps, lr=1e-2, state_bits=bits, seed=5)

    def steps(ps, opt, ks):
        for k in ks:
            for i, p in enumerate(ps):
                p.grad = _randn(p.shape, 50 * k + i).to(p.dtype)
            opt.step()

    a, opt_a = make()
    steps(a, opt_a, range(6))
    b, opt_b = make()
    steps(b, opt_b, range(3))
    c, opt_c = make()
    for p, q in zip(c, b):
        p.data.copy_(q.data)
    saved = {k: v for k, v in opt_b.state_dict().items()}
    opt_c.load_state_dict(saved)
    steps(c, opt_c, range(3, 6))
    for p, q in zip(a, c):
        assert torch.equal(p, q)
    held = [t.clone() for t in opt_c._plans[0][1].state.values()]
    before = [p.detach().clone() for p in c]
    c[0].grad = None
    c[1].grad, c[2].grad = torch.ones_like(c[1]), torch.ones_like(c[2])
    opt_c.step()
    assert torch.equal(c[0], before[0]) and not torch.equal(c[1], before[1]) and not torch.equal(c[2], before[2])
    for t, u in zip(opt_c._plans[0][1].state.values(), held):
        n = 512 if t.shape[0] >= 512 else 2  # the first parameter's two blocks
        assert torch.equal(t[:n].view(torch.uint8), u[:n].view(torch.uint8))
    with pytest.raises(ValueError, match="bits"):
        make_other = AdamW(c, state_bits=40 - bits)
        make_other.load_state_dict(saved)
    with pytest.raises(ValueError, match="fixed"):
        opt_c.add_param_group({"params": [torch.nn.Parameter(_randn((3,), 1))]})


def test_a_step_invalidates_what_autograd_saved():
    from hive_neuralnet_amd.training import AdamW
    w = torch.nn.Parameter(_randn((8, 8), 1))
    optimizer = AdamW([w])
    x = _randn((8, 8), 2).requires_grad_()
    y = (x @ w).sum()
    w.grad = torch.ones_like(w)
    optimizer.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_graph_replays_match_eager():
    """Layer norm both ways and the loss captured in a graph, replayed with other inputs and eager work between."""
    from hive_neuralnet_amd import hive_gpu
    ext = hive_gpu.load_extension()
    w = _randn((64,), 1)
    x, dy = _randn((5000, 64), 2), _randn((5000, 64), 3)
    n = torch.randint(0, 60, (5000,), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    N = int(n.sum())
    logits, values, vt = _randn((N,), 5), _randn((5000,), 6), _randn((5000,), 7)
    targets = torch.softmax(_randn((5000, 64), 8), 1)
    ones = torch.ones((5000,), device="cuda")

    def work():
        y, mean, rstd = ext.layer_norm_forward(x, w, w, activation="sigmoid")
        return (y, *ext.layer_norm_backward(dy, x, mean, rstd, w, w, "sigmoid"),
                *ext.policy_value_loss(logits, values, n, targets, ones, vt, ones))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for k in range(4):
        for t, seed in ((x, 20), (dy, 30), (logits, 40), (values, 50)):
            t.copy_(_randn(t.shape, seed + k))
        torch.cuda.synchronize()
        want = [t.clone() for t in work()]
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q), k


def test_training_command(capsys, monkeypatch):
    import sys

    from hive_neuralnet_amd import training
    monkeypatch.setattr(sys, "argv", ["training", "--steps", "3", "--batch", "32", "--state-bits", "8"])
    training.main()
    lines = capsys.readouterr().out.strip().splitlines()
    assert len(lines) == 3 and "policy" in lines[0]


def test_optimizer_refuses_a_weight_twice():
    """A weight that is listed twice would be stepped by two blocks at once."""
    from hive_neuralnet_amd.training import AdamW
    p = torch.nn.Parameter(_randn((9,), 1))
    with pytest.warns(UserWarning, match="duplicate"), pytest.raises(ValueError, match="share memory"):
        AdamW([p, p])


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_counts_each_parameters_steps(bits):
    """Parameters whose gradients come late or now and then: the bias correction is that of a parameter's own steps.
    A first step moves a weight by lr and its decay whenever it comes (m / sqrt(v) is the gradient's sign); in 32 bits
    all steps are compared with torch.optim.AdamW in 64 (16 u of lr and 4 u of the weight a step)."""
    from hive_neuralnet_amd.training import AdamW
    shapes, every = [(64, 3), (300,), (1,), (33,)], [1, 7, 3, 1]
    a = [torch.nn.Parameter(_randn(s, i)) for i, s in enumerate(shapes)]
    b = [torch.nn.Parameter(p.detach().double()) for p in a]
    ours, theirs = AdamW(a, lr=1e-2, state_bits=bits), torch.optim.AdamW(b, lr=1e-2)
    for k in range(1, 22):
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad = _randn(p.shape, 100 * k + i) if k % every[i] == 0 else None
            q.grad = None if p.grad is None else p.grad.double()
        before = a[1].detach().clone()
        ours.step()
        theirs.step()
        if k == 7:
            want = before.double() * (1.0 - 1e-4) - 1e-2 * torch.sign(a[1].grad.double())
            bound = 16 * U * 1e-2 + 4 * U * before.double().abs() + 1e-2 * 1e-8 / a[1].grad.double().abs()
            assert ((a[1].detach().double() - want).abs() <= bound).all()
    if bits == 32:
        for p, q in zip(a, b):
            bound = 21 * (16 * U * 1e-2 + 4 * U * float(q.detach().abs().max()))
            assert float((p.detach().double() - q.detach()).abs().max()) < bound


def test_optimizer_state_holds_each_parameters_steps():
    """Saved and loaded, the counts go on; a state without them (one count for all) still loads."""
    from hive_neuralnet_amd.training import AdamW

    def make():
        ps = [torch.nn.Parameter(_randn(s, i)) for i, s in enumerate([(40, 9), (300,)])]
        return ps, AdamW(ps, lr=1e-2)

    def steps(ps, opt, ks):
        for k in ks:
            ps[0].grad = _randn(ps[0].shape, 50 * k)
            ps[1].grad = _randn(ps[1].shape, 50 * k + 1) if k >= 2 else None
            opt.step()

    a, opt_a = make()
    steps(a, opt_a, range(6))
    b, opt_b = make()
    steps(b, opt_b, range(3))
    saved = opt_b.state_dict()
    c, opt_c = make()
    for p, q in zip(c, b):
        p.data.copy_(q.data)
    opt_c.load_state_dict(saved)
    steps(c, opt_c, range(3, 6))
    for p, q in zip(a, c):
        assert torch.equal(p, q)
    d, opt_d = make()
    opt_d.load_state_dict({k: saved[k] for k in ("state_bits", "seed", "steps", "states", "param_groups")})
    assert opt_d.steps == 3
    steps(d, opt_d, range(3, 4))


def test_optimizer_does_not_count_a_refused_step():
    from hive_neuralnet_amd.training import AdamW
    p = [torch.nn.Parameter(_randn((9,), 1)), torch.nn.Parameter(_randn((4,), 2))]
    opt = AdamW(p, lr=1e-2)
    for t in p:
        t.grad = torch.ones_like(t)
    before = [t.detach().clone() for t in p]
    with pytest.raises(ValueError, match="grad_scale"):
        opt.step(grad_scale=torch.ones((2,), device="cuda"))
    assert opt.steps == 0
    opt.step()
    for t, q in zip(p, before):  # a first step: lr and the decay
        want = q.double() * (1.0 - 1e-4) - 1e-2
        assert ((t.detach().double() - want).abs() <= 16 * U * 1e-2 + 4 * U * q.double().abs() + 1e-10).all()


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16], ids=str)
def test_loss_autograd_in_16_bits_is_rounded_once(t):
    """The gradient times what comes in, a scaler's factor, rounded to the logits' type once: 2,048 positions' shares
    of small probabilities are below half precision's smallest numbers before the factor.  Off by half a unit of the
    type and by what the float32 gradient is: (longest / 64 + 64) 4 u of a position's share, 8 u of a value's."""
    from hive_neuralnet_amd.training import policy_value_loss
    B, K, coming = 2048, 64, 3.0 * 2.0 ** 12
    half, tiny = (2.0 ** -11, 2.0 ** -25) if t == torch.float16 else (2.0 ** -8, 2.0 ** -134)
    n = torch.full((B,), K, device="cuda")
    logits, values = (3.0 * _randn((B * K,), 1)).to(t).requires_grad_(), torch.tanh(_randn((B, 1), 2)).to(t).requires_grad_()
    targets = torch.softmax(4.0 * _randn((B, K), 3), 1)
    ones, vt = torch.ones((B,), device="cuda"), _randn((B,), 4)
    total, _, _ = policy_value_loss(logits, values, n, targets, ones, vt, ones, 0.5)
    dx, dv = torch.autograd.grad(coming * total, (logits, values))
    assert dx.dtype == t and dv.dtype == t
    x, v = logits.detach().double().view(B, K), values.detach().double().view(-1)
    q = targets.double()
    want = coming / B * (torch.softmax(x, 1) * q.sum(1, keepdim=True) - q).view(-1)
    want_v = (coming / B * (v - vt.double())).view(-1, 1)
    for got, exact, bound in ((dx, want, coming / B * (K / 64 + 64) * 4 * U), (dv, want_v, 8 * U * want_v.abs())):
        over = (got.double() - exact).abs() - half * exact.abs() - tiny - bound
        assert float(over.max()) <= 0.0, float(over.max())


def test_train_batch_runs_the_layers_hooks():
    """fc1 under a weight norm that a forward hook puts together, hooks on fc1 and on ln1: they take part, and the
    gradients are those of the module's own forward pass."""
    from hive_neuralnet_amd import hive_gpu
    from hive_neuralnet_amd.fnn import FNNConfig, HiveFNN
    from hive_neuralnet_amd.training import encode, synthetic_batch, train_batch
    torch.manual_seed(3)
    net = HiveFNN(FNNConfig.medium()).cuda()
    net.fc1 = torch.nn.utils.weight_norm(net.fc1)
    batch = synthetic_batch(48, 0, 80, 5)
    optimizer = torch.optim.SGD(net.parameters(), lr=1e-2)
    for _ in range(2):  # the weight is put together again for every step
        train_batch(net, optimizer, batch)
    assert all(p.grad is not None for p in net.parameters())
    x = _randn((33, 122), 1)
    seen = []
    handles = [m.register_forward_hook(lambda m, i, o, k=k: seen.append(k) or 2.0 * o)
               for k, m in (("fc1", net.fc1), ("ln1", net.ln1))]
    got = encode(net, x)
    assert seen == ["fc1", "ln1"]
    _near(got.detach(), net.encode(x).detach(), 1e-5, "hooks")
    handles[1].remove()
    _near(encode(net, x).detach(), net.encode(x).detach(), 1e-5, "fc1's hook")
    handles[0].remove()
    net.ln1 = torch.nn.RMSNorm(32).cuda()  # another layer in its place
    _near(encode(net, x).detach(), net.encode(x).detach(), 1e-5, "another norm")


@pytest.mark.parametrize("trained", [("action_fc1", "action_fc2"), ("value_fc",), ("ln1",)], ids=lambda t: t[0])
def test_train_batch_of_a_part_of_the_network(trained):
    """Only some layers trained: the heads that depend on them give their gradients, the others none."""
    from hive_neuralnet_amd.fnn import FNNConfig, HiveFNN
    from hive_neuralnet_amd.training import synthetic_batch, train_batch
    torch.manual_seed(3)
    batch = synthetic_batch(48, 0, 80, 5)
    torch.manual_seed(4)
    net = HiveFNN(FNNConfig.medium()).cuda()
    _, want, terms = _plain_step(net, batch, 1.0)
    for k, p in net.named_parameters():
        p.requires_grad_(k.split(".")[0] in trained)
    train_batch(net, torch.optim.SGD(net.parameters(), lr=0.0), batch)
    for k, p in net.named_parameters():
        if not p.requires_grad:
            assert p.grad is None, k
        elif k in terms:
            assert float((p.grad.cpu().double() - want[k]).abs().max()) <= 24 * U * terms[k], k
        else:
            _near(p.grad.cpu(), want[k], 5e-5, k)


def test_train_batch_under_autocast():
    """bfloat16 products, also where no position has a move: logits and values have one type."""
    from hive_neuralnet_amd.fnn import FNNConfig, HiveFNN
    from hive_neuralnet_amd.training import synthetic_batch, train_batch
    torch.manual_seed(3)
    net = HiveFNN(FNNConfig.medium()).cuda()
    batch = synthetic_batch(16, 0, 60, 5)
    optimizer = torch.optim.SGD(net.parameters(), lr=1e-2)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        losses = train_batch(net, optimizer, batch)
        assert torch.isfinite(losses).all() and float(losses[1]) > 0.0
        batch.num_actions = torch.zeros_like(batch.num_actions)
        losses = train_batch(net, optimizer, batch)
    assert torch.isfinite(losses).all() and float(losses[1]) == 0.0


def test_optimizer_refuses_another_networks_state():
    """Parameters of other sizes in as many blocks of 256."""
    from hive_neuralnet_amd.training import AdamW
    make = lambda shapes: AdamW([torch.nn.Parameter(_randn(s, 1)) for s in shapes])  # noqa: E731
    saved = make([(300,), (200,)]).state_dict()
    for shapes in ([(200,), (300,)], [(301,), (200,)], [(300,), (100,), (100,)], [(300,)]):
        with pytest.raises(ValueError, match="sizes"):
            make(shapes).load_state_dict(saved)
    make([(30, 10), (200,)]).load_state_dict(saved)  # the same numbers of elements


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_optimizer_copies_go_on_alike(bits, how):
    import copy
    import pickle

    from hive_neuralnet_amd.training import AdamW

    ps = [torch.nn.Parameter(_randn(s, i)) for i, s in enumerate([(40, 9), (300,)])]
    opt = AdamW([{"params": ps[:1], "weight_decay": 0.2}, {"params": ps[1:], "lr": 3e-3}], lr=1e-2, state_bits=bits, seed=5)

    def steps(ps, opt, ks):
        for k in ks:
            for i, p in enumerate(ps):
                p.grad = _randn(p.shape, 50 * k + i)
            opt.step()

    steps(ps, opt, range(3))
    if how == "deepcopy":
        twin_ps, twin = copy.deepcopy((ps, opt))
    else:
        twin_ps, twin = pickle.loads(pickle.dumps((ps, opt)))
    steps(twin_ps, twin, range(3, 5))
    held = [p.detach().clone() for p in ps]
    steps(ps, opt, range(3, 5))
    for p, q, h in zip(ps, twin_ps, held):
        assert torch.equal(p, q) and not torch.equal(p, h)
    assert twin.steps == opt.steps == 5 and twin.param_groups[0]["weight_decay"] == 0.2


def test_optimizer_runs_the_state_dicts_hooks():
    from hive_neuralnet_amd.training import AdamW
    p = torch.nn.Parameter(_randn((9,), 1))
    opt, calls = AdamW([p]), []
    opt.register_state_dict_pre_hook(lambda o: calls.append("pre"))
    opt.register_state_dict_post_hook(lambda o, d: calls.append("post") or {**d, "note": 7})
    opt.register_load_state_dict_pre_hook(lambda o, d: calls.append("load") or {**d, "steps": 41})
    opt.register_load_state_dict_post_hook(lambda o: calls.append("loaded"))
    saved = opt.state_dict()
    assert calls == ["pre", "post"] and saved["note"] == 7
    opt.load_state_dict(saved)
    assert calls[2:] == ["load", "loaded"] and opt.steps == 41


def test_optimizer_refuses_settings_out_of_range():
    from hive_neuralnet_amd.training import AdamW
    p = torch.nn.Parameter(_randn((9,), 1))
    nan = float("nan")
    for bad, word in ((dict(lr=-1e-3), "lr"), (dict(lr=nan), "lr"), (dict(weight_decay=-0.1), "weight_decay"),
                      (dict(weight_decay=nan), "weight_decay"), (dict(betas=(1.0, 0.9)), "betas"),
                      (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=-1e-8), "eps"), (dict(eps=nan), "eps")):
        with pytest.raises(ValueError, match=word):
            AdamW([p], **bad)
        with pytest.raises(ValueError, match=word):
            AdamW([{"params": [p], **bad}])
    AdamW([p], lr=0.0, weight_decay=0.0, betas=(0.0, 0.0), eps=0.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_graph_replays_of_a_step_and_of_long_lists_match_eager(bits):
    """An AdamW step (the step's number as captured, gradients and their scale as they are at the replay) and the loss
    over lists in slices, by each way to a position's first logit."""
    from hive_neuralnet_amd import hive_gpu
    ext = hive_gpu.load_extension()
    shapes = [(64, 122), (64,), (5000,), (1,)]
    a = [_randn(s, i) for i, s in enumerate(shapes)]
    b = [t.clone() for t in a]
    grads, scale = [_randn(s, 10 + i) for i, s in enumerate(shapes)], torch.ones((1,), device="cuda")
    plan, twin = ext.prepare_adamw(a, bits), ext.prepare_adamw(b, bits)
    lists = []
    for B, width in ((5, 9001), (300, 4096), (4200, 1100)):
        n = torch.randint(0, width + 1, (B,), generator=torch.Generator(device="cuda").manual_seed(B), device="cuda")
        n = n if B < 4000 else n % 20
        ones = torch.ones((B,), device="cuda")
        lists.append([_randn((int(n.sum()),), 5), _randn((B,), 6), n, torch.softmax(_randn((B, width), 8), 1), ones,
                      _randn((B,), 7), ones])

    def work(plan):
        plan.step(grads, 3, 1e-2, grad_scale=scale, seed=11)
        return [t for args in lists for t in ext.policy_value_loss(*args)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(plan)
    torch.cuda.current_stream().wait_stream(side)
    work(twin)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(plan)
    for k in range(4):
        for i, t in enumerate([*grads, *[args[0] for args in lists], *[args[1] for args in lists]]):
            t.copy_(_randn(t.shape, 20 + 10 * k + i))
        scale.fill_(0.5 ** k)
        torch.cuda.synchronize()
        want = [t.clone() for t in work(twin)]
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q), k
        for p, q in zip([*a, *plan.state.values()], [*b, *twin.state.values()]):
            assert torch.equal(p.view(torch.uint8), q.view(torch.uint8)), k


def test_train_batch_of_a_frozen_network_is_refused():
    from hive_neuralnet_amd.fnn import FNNConfig, HiveFNN
    from hive_neuralnet_amd.training import synthetic_batch, train_batch
    net = HiveFNN(FNNConfig.small()).cuda()
    optimizer = torch.optim.SGD(net.parameters(), lr=0.1)
    net.requires_grad_(False)
    with pytest.raises(RuntimeError, match="gradient"):
        train_batch(net, optimizer, synthetic_batch(8, 0, 40, 5))
