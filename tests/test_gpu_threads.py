"""Two threads that call the operators on one stream: each call's workspace is its own, so the kernels of the two may interleave."""
import threading

import pytest
import torch

from bit_reproducible_training_b200 import layers
from bit_reproducible_training_b200 import repro_gemm as rg
from bit_reproducible_training_b200 import repro_loss as rl
from bit_reproducible_training_b200 import repro_norm as rn

pytestmark = pytest.mark.gpu


def work(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    m, n, k, v = 200 + seed, 130, 96, 3000
    x, w, z, dy = (torch.randn(*s, device="cuda", generator=g) for s in ((m, k), (n, k), (m, n), (m, n)))
    b, gate, words = torch.randn(n, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g), torch.randn(v, n, device="cuda", generator=g) / 10
    t = torch.randint(0, v, (m,), device="cuda", generator=g)

    def once():
        y = rg.gemm_epilogue(x, w, m, n, k, False, True, bias=b, activation="gelu")
        out = [y, *rg.linear_backward(dy, z, x, w, m, n, k, "gelu", 3, True, True, True)]
        how = dict(weight=b, gate=gate, kind="layer")
        r, h, stats = rn.block_norm(z, y, keep_stats=True, **how)
        grads = rn.block_norm_backward(dy, z, r, y, stats, **how)
        loss, st = rl.linear_cross_entropy(h, words, t)
        return out + [r, h, grads.x, grads.y, grads.weight, grads.gate, loss, *rl.linear_cross_entropy_backward(torch.ones((), device="cuda"), h, words, t, st)]

    return once


@pytest.mark.parametrize("shared", [True, False], ids=["one stream", "two streams"])
def test_two_threads(shared):
    jobs = [work(1), work(2)]
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    bad, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]

    def run(i):
        try:
            with torch.cuda.stream(streams[0 if shared else i]):
                for _ in range(25):
                    got = jobs[i]()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        bad.append(i)
        except Exception as e:                       # an assertion in a thread would be lost
            bad.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad


def test_layers_in_threads():
    """The same through autograd: each thread's backward pass runs on the device's autograd thread, between the other's calls."""
    def job(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(150, 64, device="cuda", generator=g)
        w, words = torch.randn(64, 64, device="cuda", generator=g) / 8, torch.randn(500, 64, device="cuda", generator=g)
        t = torch.randint(0, 500, (150,), device="cuda", generator=g)

        def once():
            a = [q.clone().requires_grad_() for q in (x, w, words)]
            r, h = layers.block_norm(a[0], layers.linear(a[0], a[1], activation="silu"), weight=w[0])
            return torch.autograd.grad(layers.linear_cross_entropy(h, a[2], t), a)

        return once

    jobs = [job(1), job(2)]
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        try:
            for _ in range(15):
                got = jobs[i]()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
        except Exception as e:
            bad.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad
