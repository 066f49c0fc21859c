"""An adapted projection behind a layer norm, as a fine-tune and a server use it: the calls one after the other, against the
same chain in 64 bits from the same inputs."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import caif_oracle as orc
from caif_b200 import native as nv
from gpu_util import make_weight

pytestmark = pytest.mark.gpu

HALF = torch.finfo(torch.bfloat16).eps / 2


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


def norm_64(x, gamma, beta):
    x = x.double()
    off = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(off.square().mean(1, keepdim=True) + 1e-5)
    return off * rstd, rstd, off * rstd * gamma.double() + beta.double()


def setup(seed, storage, hidden, out, m):
    g = torch.Generator(device="cuda").manual_seed(seed)
    weight, _, _ = make_weight(np.random.default_rng(seed), out, hidden, storage)
    x = (torch.randn(m, hidden, generator=g, device="cuda") + 0.3).to(torch.bfloat16)
    gamma = 1.0 + 0.1 * torch.randn(hidden, generator=g, device="cuda")
    beta = 0.1 * torch.randn(hidden, generator=g, device="cuda")

    def lora(rank):
        a = (torch.randn(rank, hidden, generator=g, device="cuda") / hidden ** 0.5).to(torch.bfloat16)
        return nv.Lora(a, (torch.randn(out, rank, generator=g, device="cuda") * 0.02).to(torch.bfloat16), 2.0 * rank)

    return g, weight, x, gamma, beta, lora


@pytest.mark.parametrize("storage,compute", [(orc.I8, nv.F32), (orc.I4, nv.BF16)])
@pytest.mark.parametrize("m", [40, 1111])
def test_training_step_with_the_input_kept_in_8_bits(storage, compute, m):
    """Every stage rounds to bf16 once or twice (HALF relative at most each), an int4 weight once more; the input kept in 8 bits
    is off by max|x| / 126 of its block at most, which a normal row's 32 values have at 2.7 of their deviation: 2.2 % of it at most,
    1.3 % as a 2-norm (a uniform error), in dA alone."""
    hidden, out = 512, 768
    g, weight, x, gamma, beta, make = setup(m, storage, hidden, out, m)
    lora = make(16)
    dy = torch.randn(m, out, generator=g, device="cuda").to(torch.bfloat16)

    normed, mean, rstd = nv.layernorm_fwd(x, gamma, beta)
    kept = nv.act_pack(normed)
    y, h = nv.lora_linear_fwd(weight, lora, normed, compute, expanded=True)
    dn, d_a, d_b = nv.lora_linear_bwd_packed(weight, lora, dy, kept, h, compute)
    dx, d_gamma, d_beta = nv.layernorm_bwd(dn, x, mean, rstd, gamma)

    xh, r, n64 = norm_64(x, gamma, beta)
    w, a, b, s = nv.weight_materialize(weight).double(), lora.a.double(), lora.b.double(), lora.alpha / lora.rank
    d = dy.double()
    h64 = n64 @ a.t()
    assert rel(y, n64 @ w.t() + s * h64 @ b.t()) <= 5 * HALF
    dn64 = d @ w + s * (d @ b) @ a
    assert rel(dn, dn64) <= 5 * HALF
    assert rel(d_b, s * d.t() @ h64) <= 4 * HALF
    assert rel(d_a, s * (d @ b).t() @ n64) <= 0.013 + 4 * HALF
    # the gradient through the norm, from dn as it was rounded
    g64 = dn64 * gamma.double()
    dx64 = r * (g64 - g64.mean(1, keepdim=True) - xh * (g64 * xh).mean(1, keepdim=True))
    assert rel(dx, dx64) <= 7 * HALF
    assert rel(d_gamma, (dn64 * xh).sum(0)) <= 6 * HALF
    assert rel(d_beta, dn64.sum(0)) <= 6 * HALF
    assert nv.lib().caifq_device_status() == 0


@pytest.mark.parametrize("m", [1, 7, 64, 300])
def test_serving_step_of_requests_with_adapters_of_their_own(m):
    """One captured step over q and k projections; the next batch of rows, with other adapters, through the same graph."""
    hidden, out = 512, 384
    g, weight, x, gamma, beta, make = setup(m, orc.I4, hidden, out, m)
    second, _, _ = make_weight(np.random.default_rng(m + 1), out, hidden, orc.I4)
    banks = [nv.LoraBank([make(r) for r in (16, 8, 64, 16)]) for _ in range(2)]
    idx = torch.randint(-1, 4, (m,), generator=g, device="cuda", dtype=torch.int32)

    def step():
        n, _, _ = nv.layernorm_fwd(x, gamma, beta)
        return [nv.lora_bank_linear_fwd(w, b, idx, n, nv.BF16) for w, b in zip((weight, second), banks)]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(2):
        graph.replay()
        n64 = norm_64(x, gamma, beta)[2]
        for y, w, bank in zip(got, (weight, second), banks):
            want = n64 @ nv.weight_materialize(w).double().t()
            for i, l in enumerate(bank.loras):
                rows = torch.nonzero(idx == i)[:, 0]
                want[rows] += l.alpha / l.rank * (n64[rows] @ l.a.double().t()) @ l.b.double().t()
            assert rel(y, want) <= 5 * HALF
        x.copy_((torch.randn(m, hidden, generator=g, device="cuda") - 1.0).to(torch.bfloat16))
        idx.copy_(torch.randint(-1, 4, (m,), generator=g, device="cuda", dtype=torch.int32))
    assert nv.lib().caifq_device_status() == 0


def test_calls_on_two_streams_at_once():
    """Each stream's calls have scratch of their own: the results are those of one stream."""
    g, weight, x, gamma, beta, make = setup(5, orc.I4, 512, 384, 200)
    bank = nv.LoraBank([make(r) for r in (16, 8, 64, 16)])
    lora = make(16)
    idx = torch.randint(-1, 4, (200,), generator=g, device="cuda", dtype=torch.int32)
    dy = torch.randn(200, 384, generator=g, device="cuda").bfloat16()

    def step():
        n, mean, rstd = nv.layernorm_fwd(x, gamma, beta)
        y = nv.lora_bank_linear_fwd(weight, bank, idx, n, nv.BF16)
        few = nv.lora_bank_linear_fwd(weight, bank, idx[:7], n[:7], nv.BF16)
        h = (n.float() @ lora.a.float().t()).bfloat16()
        dn, d_a, d_b = nv.lora_linear_bwd_packed(weight, lora, dy, nv.act_pack(n), h, nv.BF16)
        return (y, few, d_a, d_b) + nv.layernorm_bwd(dn, x, mean, rstd, gamma)

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step())
    torch.cuda.synchronize()
    for results in got:
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, want))


def test_without_dependent_launches():
    """Launches that wait for one another as a stream's do give the same numbers (the switch is read once a process)."""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, CAIFQ_PDL="0")
    tests = [os.path.join(here, "test_gpu_adapted_block.py") + "::" + name for name in
             ("test_training_step_with_the_input_kept_in_8_bits", "test_serving_step_of_requests_with_adapters_of_their_own")]
    done = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider"] + tests, env=env, cwd=os.path.dirname(here),
                          capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stdout[-2000:]
