"""Where the operators around an adapted projection round (caif_b200/csrc/lora_bank.cu): once, to the result's type.

Tolerances, element by element, as in the operators' other tests: `half` is half a step of the result's type; a sum of n products in
fp32 is off by at most (n / 32 + 64) 2^-23 times the sum of the products' magnitudes; a sum that enters the tensor core a second time
does so as two bf16 terms (2^-16 relative).
"""
import pytest
import torch

from caif_b200 import native as nv

pytestmark = pytest.mark.gpu

S = 2.0 ** -23


def half(t):
    return torch.finfo(t).eps / 2


def chain(n):
    return (n / 32 + 64) * S


# one launch after the product; one before and one after; rows placed by a launch ahead; many rows; multiply-adds
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,in_dim,out_dim,rank,count", [(1, 128, 256, 8, 1), (16, 128, 256, 8, 2), (16, 128, 14336, 8, 12), (128, 256, 4096, 16, 9),
                                                         (300, 128, 256, 8, 2), (1500, 256, 640, 16, 3), (20, 128, 256, 5, 2), (9, 136, 72, 8, 2),
                                                         (200, 128, 384, 72, 2)])
def test_bank_rounds_where_it_adds(m, in_dim, out_dim, rank, count, dtype):
    """The adapters take back all but a 64th of the frozen product: either of them rounded by itself would show."""
    g = torch.Generator(device="cuda").manual_seed(m + out_dim)
    top = min(rank, 40)      # (factors of -1, 0, 1, whose product the weight's codes hold)
    a = torch.zeros(rank, in_dim, device="cuda")
    b = torch.zeros(out_dim, rank, device="cuda")
    a[:top] = torch.randint(-1, 2, (top, in_dim), generator=g, device="cuda").float()
    b[:, :top] = torch.randint(-1, 2, (out_dim, top), generator=g, device="cuda").float()
    codes = b @ a
    assert float(codes.abs().max()) <= 127
    scale = 2.0 ** -6
    weight = nv.Weight(codes.to(torch.int8), nv.I8, in_dim, out_dim, torch.full((1,), scale, device="cuda"))
    back = scale * (1 - 2.0 ** -6)
    bank = nv.LoraBank([nv.Lora(a.to(dtype), b.to(dtype), -back * rank) for _ in range(count)])
    x = torch.randn(m, in_dim, generator=g, device="cuda").to(dtype)
    idx = torch.randint(-1 if m > 1 else 0, count, (m,), generator=g, device="cuda", dtype=torch.int32)
    y = nv.lora_bank_linear_fwd(weight, bank, idx, x)
    xd, a, b, codes = x.double(), a.double(), b.double(), codes.double()
    mine = (idx >= 0).double()[:, None]
    h = xd @ a.t()
    want = scale * (xd @ codes.t()) - mine * back * (h @ b.t())
    tol = scale * chain(in_dim) * (xd.abs() @ codes.abs().t())
    tol = tol + mine * back * ((chain(in_dim) * (xd.abs() @ a.abs().t()) + (2.0 ** -16 + (rank / 32 + 70) * S) * h.abs()) @ b.abs().t())
    # (s * sum, the addition: two roundings of fp32)
    tol = tol + 2 * S * (scale * (xd @ codes.t()).abs() + mine * back * (h @ b.t()).abs())
    tol = tol + half(dtype) * (want.abs() + tol) + (2.0 ** -24 if dtype == torch.float16 else 0.0)
    assert bool(((y.double() - want).abs() <= tol).all())
