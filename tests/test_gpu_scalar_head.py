"""The scalar head's operators run together: NodewiseMLP in the energy model, its gradients and the forces' gradients against the same
model with the head in plain torch operations in 64 bits, and training steps with optim.AdamW, launch by launch and captured."""
import copy
import math

import pytest
import torch

from tests import models as M

U = 2.0**-24
HEAD = {"hidden": 40, "num_blocks": 2, "activation": "silu"}


@pytest.fixture(scope="module")
def dataset():
    return M.load_dataset()


def _model(hp, head=HEAD):
    from matten_amd import model_factory

    torch.manual_seed(35)
    return model_factory.create_energy_model(dict(M.MINIMAL, output_mlp=head), hp)


def test_structure_and_refusals(dataset):
    from matten_amd import keys as K
    from matten_amd import nn

    _, _, hp = dataset
    m, plain = _model(hp), M.build("hip", "energy", hp)
    names = [n for n, _ in m.named_children()]
    assert names[6:9] == ["conv_to_output_hidden", "output_mlp", "output_hidden_to_scalar"]
    assert {k for k in m.state_dict() if not k.startswith("output_mlp.")} == set(plain.state_dict())
    assert tuple(m.output_mlp.blocks[1]["up"].weight.shape) == (16, 40) and m.output_mlp.out is None
    assert nn.NodewiseMLP({K.NODE_FEATURES: "8x0e"}, "3x0e").out["linear"].weight.shape == (8, 3)
    for irreps, kw in (("8x0e + 4x1o", {}), ("8x0o", {}), ("8x0e", {"irreps_out": "2x1o"}), ("8x0e", {"num_blocks": 0}),
                       ("8x0e", {"hidden": -1}), ("8x0e", {"activation": "relu6"})):
        with pytest.raises(ValueError):
            nn.NodewiseMLP({K.NODE_FEATURES: irreps}, **kw)


class _Plain(torch.nn.Module):
    """The head in torch operations, with the parameters of a NodewiseMLP, in 64 bits."""

    def __init__(self, mlp):
        super().__init__()
        self.mlp = mlp

    def forward(self, x):
        def dense(layer, v):
            z = v @ layer.weight / math.sqrt(layer.weight.shape[0]) + layer.bias
            return torch.nn.functional.silu(z) * layer.act_cst if layer.act == "silu" else z

        norm = lambda layer, v: torch.nn.functional.layer_norm(v, v.shape[-1:], layer.weight, layer.bias, layer.eps)  # noqa: E731
        for b in self.mlp.blocks:
            x = x + dense(b["down"], dense(b["up"], norm(b["norm"], x)))
        return x if self.mlp.out is None else dense(self.mlp.out["linear"], norm(self.mlp.out["norm"], x))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d,d_out", [(1, 16, 16), (37, 16, 3), (600, 64, 64), (2048, 130, 1)])
def test_head_and_its_gradients(device, rows, d, d_out):
    """Elementwise errors are bounded where the operators are tested; here the sum of the blocks: 2-norms, 64 roundings of 2^-24 for each
    of the nine operators in a row, forward and again backward."""
    from matten_amd import keys as K
    from matten_amd import nn

    torch.manual_seed(1)
    mlp = nn.NodewiseMLP({K.NODE_FEATURES: f"{d}x0e"}, f"{d_out}x0e", hidden=96, num_blocks=2).to(device)
    with torch.no_grad():
        for p in mlp.parameters():
            p.add_(0.1 * torch.randn_like(p))
    x = torch.randn(rows, d, device=device, requires_grad=True)
    y = mlp({K.NODE_FEATURES: x})[K.NODE_FEATURES]
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, [x, *mlp.parameters()], dy)
    twin = _Plain(copy.deepcopy(mlp).double())
    x64 = x.detach().double().requires_grad_(True)
    y64 = twin(x64)
    want = torch.autograd.grad(y64, [x64, *twin.parameters()], dy.double())
    assert y.shape == (rows, d_out)
    for a, b in zip((y, *got), (y64, *want)):
        assert (a.double() - b).norm() <= 9 * 64 * U * b.norm() + 1e-30


@pytest.mark.gpu
def test_forces_and_their_gradients(device, dataset):
    """d(force loss)/d(parameters) goes through the second derivatives of the head: against differences of the loss along the
    gradient's own direction, in the head's parameters.  Step 2^-9 of the parameters' norm; allowed: the difference between the
    slopes at two steps (what the cut series leaves), and the loss's own noise, 2^-16 of it, over the step."""
    from matten_amd import keys as K

    graphs, _, hp = dataset
    m = _model(hp).to(device)
    b = M.make_batch(graphs, [0, 1, 2], device, torch.float32)
    head = list(m.output_mlp.parameters())

    def loss():
        pos = b[K.POSITIONS].detach().clone().requires_grad_(True)
        e = m(dict(b, **{K.POSITIONS: pos}))["total_energy"]
        f = torch.autograd.grad(e.sum(), pos, create_graph=True)[0]
        return (f * f).sum()

    value = loss()
    grads = torch.autograd.grad(value, head)
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert norm > 0 and all(torch.isfinite(g).all() for g in grads)
    size = math.sqrt(sum(float(p.detach().double().square().sum()) for p in head))
    way = [g / norm for g in grads]

    def slope(t):
        at = []
        for s in (1, -2):
            with torch.no_grad():
                for p, w in zip(head, way):
                    p.add_(w, alpha=s * t)
            at.append(float(loss()))
        with torch.no_grad():
            for p, w in zip(head, way):
                p.add_(w, alpha=t)
        return (at[0] - at[1]) / (2 * t)

    t = size * 2.0**-9
    near, far = slope(t), slope(2 * t)
    assert abs(near - norm) <= abs(far - near) + 2.0**-16 * float(value) / t


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_energy_model_steps(device, dataset, bits):
    """The energy model with its head under the optimizer: every parameter moves, nothing is left that is no number, and the same
    steps from the same start give the same bits."""
    from matten_amd import optim

    graphs, targets, hp = dataset
    models = [_model(hp).to(device) for _ in range(2)]
    start = [p.detach().clone() for p in models[0].parameters()]
    batch = M.make_batch(graphs, [0, 1, 2, 3], device, torch.float32)
    want = targets[:4].to(device=device, dtype=torch.float32)
    for m in models:
        opt = optim.AdamW(m.parameters(), lr=1e-3, weight_decay=0.01, state_bits=bits, max_grad_norm=1.0)
        for _ in range(3):
            opt.zero_grad()
            torch.nn.functional.l1_loss(m(dict(batch))["total_energy"].reshape(-1), want).backward()
            opt.step()
            assert float(opt.grad_norm) > 0
    for p, q, s in zip(models[0].parameters(), models[1].parameters(), start):
        assert torch.equal(p, q) and torch.isfinite(p).all() and not torch.equal(p, s)


class _Net(torch.nn.Module):
    """Convolution stack with a perceptron on its even scalars."""

    def __init__(self, cfg):
        from matten_amd import keys as K
        from matten_amd import nn
        from matten_amd.irreps import Irreps
        from tests.parity import Stack

        super().__init__()
        self.stack = Stack("hip", cfg)
        irreps = Irreps(str(self.stack.convs[-1].irreps_out[K.NODE_FEATURES]))
        self.at, self.width = next((o, m.mul) for o, m in zip(irreps.offsets(), irreps) if m.ir.l == 0 and m.ir.p == 1)
        self.head = nn.NodewiseMLP({K.NODE_FEATURES: f"{self.width}x0e"}, "1x0e", hidden=48, num_blocks=2, activation="gelu")

    def forward(self, batch, n_graphs):
        from matten_amd import keys as K

        feats, energy, _ = self.stack(batch, n_graphs)
        x = feats[:, self.at : self.at + self.width]
        return energy.sum() + self.head({K.NODE_FEATURES: x})[K.NODE_FEATURES].sum()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps_together(device, bits):
    """Stack, head, backward and optimizer step: what a captured step does is what the launch-by-launch steps do, bit for bit, over
    several replays with the program's own work in between."""
    from matten_amd import keys as K
    from matten_amd import optim
    from matten_amd.graphs import GraphedStep
    from tests.parity import CONFIGS, _prep, make_batch

    cfg = CONFIGS["minimal"]
    torch.manual_seed(35)
    a = _Net(cfg).to(device)
    b = copy.deepcopy(a)
    batch = _prep(make_batch(cfg), str(device), torch.float32)
    # (no leaf of the batch collects gradients: one that outlives the steps would be accumulated into on the stream of an earlier
    # step's graph, inside the capture)
    batch[K.POSITIONS] = batch[K.POSITIONS].detach()

    def trainer(model):
        opt = optim.AdamW(model.parameters(), lr=1e-3, weight_decay=0.01, state_bits=bits, max_grad_norm=1.0)

        def step():
            for p in model.parameters():
                p.grad = None
            loss = model(dict(batch), cfg["graphs"]) ** 2
            loss.backward()
            opt.step()
            return loss.detach(), opt.grad_norm

        return opt, step

    (oa, sa), (ob, sb) = trainer(a), trainer(b)
    for _ in range(3):  # the warm-up of the captured step steps three times
        sb()
    replay = GraphedStep(sa, warmup=3)
    start = [p.detach().clone() for p in b.parameters()]
    for k in range(4):
        (la, na), (lb, nb) = replay(), sb()
        torch.cuda.synchronize()
        assert torch.equal(la, lb) and torch.equal(na, nb) and float(na) > 0
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
        torch.randn(1000, device=device).sum().item()  # eager work and a wait between the replays
    assert all(not torch.equal(p, q) for p, q in zip(b.parameters(), start))
    for p, q in zip(a.parameters(), b.parameters()):
        assert int(oa.state[p]["step"]) == int(ob.state[q]["step"]) == 7


@pytest.mark.gpu
def test_two_threads_at_once(device):
    """The operators from two host threads, each on its own stream, give the bits they give one after the other."""
    import threading

    from matten_amd import ops, optim

    def work(seed, out):
        g = torch.Generator(device=device).manual_seed(seed)
        w, v = (torch.nn.Parameter(torch.randn(130, 130, generator=g, device=device)) for _ in range(2))
        n = torch.nn.Parameter(torch.ones(130, device=device))
        opt = optim.AdamW([w, v, n], lr=1e-2, state_bits=8, max_grad_norm=1.0, seed=seed)
        x = torch.randn(1500 + seed, 130, generator=g, device=device)
        for _ in range(15):
            opt.zero_grad()
            y = ops.dense(ops.dense(ops.layer_norm(x, n), w, act="gelu", alpha=0.09), v, residual=x, alpha=0.09)
            (y * y).mean().backward()
            opt.step()
        out[seed] = [t.detach().clone() for t in (w, v, n, y)]

    alone, together = {}, {}
    for seed in (1, 2):
        work(seed, alone)
    torch.cuda.synchronize()

    def on_its_own_stream(seed):
        with torch.cuda.stream(torch.cuda.Stream()):
            work(seed, together)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=on_its_own_stream, args=(seed,)) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for seed in (1, 2):
        assert all(torch.equal(p, q) for p, q in zip(alone[seed], together[seed]))
