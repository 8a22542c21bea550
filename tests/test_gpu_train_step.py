"""The operators of a training step together, as a small language model uses them: block norms, fused linear layers, the cross
entropy of the output projection, AdamW.  Each operator is held to 64-bit references in its own file; here the whole step has to be
the chain of those calls bit for bit, to repeat, and to give the same bits when it is captured into a CUDA graph."""
import pytest
import torch

from bit_reproducible_training_b200 import layers, repro_optim
from bit_reproducible_training_b200 import repro_gemm as rg
from bit_reproducible_training_b200 import repro_loss as rl
from bit_reproducible_training_b200 import repro_norm as rn

pytestmark = pytest.mark.gpu

DIM, HIDDEN, VOCAB, BATCH, LENGTH = 96, 160, 331, 3, 37


class Model(torch.nn.Module):
    def __init__(self, blocks=2):
        super().__init__()
        self.head = layers.LinearCrossEntropy(DIM, VOCAB)
        self.norms = torch.nn.ModuleList([layers.BlockNorm(DIM, post=i > 0, gate=i > 0, residual_scale=0.9) for i in range(blocks + 1)])
        self.up = torch.nn.ModuleList([layers.FusedLinear(DIM, HIDDEN, activation="gelu_tanh") for _ in range(blocks)])
        self.down = torch.nn.ModuleList([layers.FusedLinear(HIDDEN, DIM) for _ in range(blocks)])

    def forward(self, x, target):
        r, h = self.norms[0](x)
        for norm, up, down in zip(self.norms[1:], self.up, self.down):
            r, h = norm(r, down(up(h)))
        return self.head(h, target)


def build(seed=0, state_bits=32, capturable=False):
    torch.manual_seed(seed)
    model = Model().cuda()
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(BATCH, LENGTH, DIM, device="cuda", generator=g)
    t = torch.randint(0, VOCAB, (BATCH, LENGTH), device="cuda", generator=g)
    t[:, :5] = -100
    return model, x, t, repro_optim.AdamW(model.parameters(), lr=1e-2, state_bits=state_bits, capturable=capturable)


def train(steps, **kw):
    model, x, t, opt = build(**kw)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = model(x, t)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return model, torch.stack(losses)


@pytest.mark.parametrize("state_bits", [32, 8])
def test_training_repeats_bit_for_bit(state_bits):
    a, la = train(4, state_bits=state_bits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, lb = train(4, state_bits=state_bits)
    torch.cuda.synchronize()
    assert torch.equal(la, lb) and torch.isfinite(la).all()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)


def test_gradients_are_the_chain_of_the_calls():
    model, x, t, _ = build(seed=3)
    x.requires_grad_()
    loss = model(x, t)
    names, params = zip(*model.named_parameters())
    grads = dict(zip(names + ("x",), torch.autograd.grad(loss, list(params) + [x])))

    with torch.no_grad():
        flat, n = x.view(-1, DIM), BATCH * LENGTH
        norm_args = [dict(weight=m.weight, post_weight=m.post_weight, gate=m.gate, residual_scale=m.residual_scale) for m in model.norms]
        norm_args[0].update(post_weight=None, gate=None)
        r, h, st = rn.block_norm(flat, keep_stats=True, **norm_args[0])
        kept = [(r, None, st)]
        hs, zs, ups = [], [], []
        for i, (up, down) in enumerate(zip(model.up, model.down)):
            hs.append(h)
            u, z = rg.gemm_epilogue(h, up.weight, n, HIDDEN, DIM, False, True, 3, up.bias, "gelu_tanh", None, True)
            y = rg.gemm_epilogue(u, down.weight, n, DIM, HIDDEN, False, True, 3, down.bias)
            zs.append(z)
            ups.append(u)
            r, h, st = rn.block_norm(r, y, keep_stats=True, **norm_args[i + 1])
            kept.append((r, y, st))
        want_loss, stats = rl.linear_cross_entropy(h, model.head.weight, t.view(-1))
        assert torch.equal(want_loss, loss)
        one = torch.ones((), device="cuda")
        dh, want = None, {}
        dh, want["head.weight"] = rl.linear_cross_entropy_backward(one, h, model.head.weight, t.view(-1), stats)
        dr = None
        for i in reversed(range(2)):
            g = rn.block_norm_backward(dh, dr, *kept[i + 1], **norm_args[i + 1])
            want.update({"norms.%d.%s" % (i + 1, k): getattr(g, k) for k in ("weight", "post_weight", "gate")})
            dr = g.x
            du, want["down.%d.weight" % i], want["down.%d.bias" % i] = rg.linear_backward(g.y, None, ups[i], model.down[i].weight, n, DIM, HIDDEN, None, 3, True, True, True)
            dh, want["up.%d.weight" % i], want["up.%d.bias" % i] = rg.linear_backward(du, zs[i], hs[i], model.up[i].weight, n, HIDDEN, DIM, "gelu_tanh", 3, True, True, True)
        g = rn.block_norm_backward(dh, None, *kept[0], **norm_args[0])
        want["norms.0.weight"] = g.weight
        want["x"] = (dr + g.x).view(x.shape)
    for k, v in want.items():
        assert torch.equal(grads[k], v), k
    assert set(want) == {k for k, v in grads.items()}


def test_a_captured_step_gives_the_same_bits():
    eager, _ = train(4, seed=5)
    model, x, t, opt = build(seed=5, capturable=True)

    def step():
        opt.zero_grad(set_to_none=True)
        model(x, t).backward()
        opt.step()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    opt.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(model.parameters(), eager.parameters()):
        assert torch.equal(p, q)
