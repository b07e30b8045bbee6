"""The operators called from two threads at once, each on its own stream, over the same kernels with other data: the results of every
round are those of the call alone."""
import threading

import pytest
import torch

from spherical_distortion import functional as F
from sphmap import optim

pytestmark = pytest.mark.gpu
ROUNDS = 30


def values(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def norm(shape, dim, dtype):
    def call(seed):
        x, r, w = (values(s, 10 * seed + i, dtype).requires_grad_() for i, s in enumerate((shape, shape, shape[dim:dim + 1])))
        g = values(shape, 10 * seed + 4, dtype)

        def run():
            out = F.rms_norm(x, w, r, dim=dim)
            return [*out, *torch.autograd.grad(out, (x, w, r), (g, g)), *F.rms_norm_quantized(x.detach(), w.detach(), dim=dim)]
        return run
    return call


def log_probs(shape, dim, k):
    def call(seed):
        x = values(shape, 10 * seed).requires_grad_()
        target = torch.randint(shape[dim], [s for i, s in enumerate(shape) if i != dim], generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")

        def run():
            p = F.token_log_probs(x, target, dim, k)
            return [t for t in p if t is not None] + [*torch.autograd.grad(p.log_probs.sum() + p.entropy.sum(), x)]
        return run
    return call


def adamw(bits):
    def call(seed):
        sizes = [70001, 256, 5000, 33]
        p, g = ([values((n,), 10 * seed + i + j) for i, n in enumerate(sizes)] for j in (0, 5))

        def run():
            params = [t.clone().requires_grad_() for t in p]
            o = optim.AdamW(params, state_bits=bits)
            for q, t in zip(params, g):
                q.grad = t
            for _ in range(2):
                o.step()
            return [t for q in params for t in (q.detach(), o.state[q]["exp_avg"], o.state[q]["exp_avg_sq"])]
        return run
    return call


CALLS = {"planes": norm((16, 40, 9, 16), 1, torch.float32), "odd planes": norm((8, 96, 31, 33), 1, torch.bfloat16), "rows": norm((700, 1024), 1, torch.bfloat16),
         "block rows": norm((1200, 4096), 1, torch.bfloat16), "odd rows": norm((400, 333), 1, torch.float32), "long rows": norm((40, 20000), 1, torch.float32),
         "deep planes": norm((2, 700, 5, 9), 1, torch.float32), "cluster": log_probs((3, 50000), 1, 0), "cluster, best": log_probs((3, 50000), 1, 8),
         "stream": log_probs((400, 5000), 1, 0), "many best": log_probs((5, 3000), 1, 40), "short rows": log_probs((900, 100), 1, 3),
         "pixels": log_probs((2, 13, 40, 64), 1, 2), "adamw": adamw(32), "adamw 8 bit": adamw(8)}


@pytest.mark.parametrize("name", CALLS)
def test_two_threads(name):
    runs = [CALLS[name](seed) for seed in (1, 2)]
    alone = [[t.detach().clone() for t in run()] for run in runs]
    torch.cuda.synchronize()
    together, errors, start = [[], []], [], threading.Barrier(2, timeout=60)

    def worker(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(ROUNDS):
                    start.wait()
                    together[i].append([t.detach() for t in runs[i]()])
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            errors.append(e)
            start.abort()

    threads = [threading.Thread(target=worker, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for rounds, want in zip(together, alone):
        assert len(rounds) == ROUNDS
        for got in rounds:
            assert all(torch.equal(a.float().nan_to_num(5e30), b.float().nan_to_num(5e30)) for a, b in zip(got, want))
