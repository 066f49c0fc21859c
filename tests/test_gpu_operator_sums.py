"""Long sums of the operators around an adapted projection (caif_b200/csrc/act8.cu, lora_bank.cu) in fp32, where the order of the
additions shows.

In a sum of n products the longest chain of additions is at most n / 32 + 64 long, so it is off by at most that many times
2^-24 times the sum of the products' magnitudes, and the result is stored in fp32: one more 2^-24, and one for alpha / rank.
The terms here are one large one and small ones that a chain which already holds the large one loses whole (2^-25 or 2^-24
beside 1, ties to even): a chain longer than the bound loses more than the bound.  Every product is a power of two, so that nothing but the additions
rounds.
"""
import pytest
import torch

from caif_b200 import native as nv

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def bound(n):
    return (n / 32 + 64 + 2) * U


def zeros(in_dim, out_dim):
    return nv.Weight(torch.zeros(out_dim, in_dim, dtype=torch.int8, device="cuda"), nv.I8, in_dim, out_dim,
                     torch.ones(1, device="cuda"))


def near(got, n, first, rest, terms):
    """every element of `got` is the sum of `terms` terms, `first` and as often `rest`, within the bound"""
    want = first + (terms - 1) * rest
    assert float((got.double() - want).abs().max()) <= bound(n) * (abs(first) + (terms - 1) * abs(rest))


# few slices of many tokens (wide layers), one slice, many slices
@pytest.mark.parametrize("in_dim,out_dim,rank,m", [(4096, 4096, 64, 8192), (2048, 2048, 64, 8192), (7168, 7168, 40, 3001), (1024, 512, 16, 9000),
                                                   (2048, 2048, 64, 64)])
def test_gradients_over_many_tokens(in_dim, out_dim, rank, m):
    """Token 0 gives 1 to every sum, the others 2^-25."""
    dy = torch.full((m, out_dim), 2.0 ** -25, device="cuda")
    dy[0] = 1.0
    b = torch.zeros(out_dim, rank, device="cuda")
    b[0] = 1.0                                         # dH[t, :] = dy[t, 0]
    lora = nv.Lora(torch.zeros(rank, in_dim, device="cuda"), b, float(rank))
    packed = nv.act_pack(torch.ones(m, in_dim, device="cuda"))
    dx, d_a, d_b = nv.lora_linear_bwd_packed(zeros(in_dim, out_dim), lora, dy, packed, torch.ones(m, rank, device="cuda"))
    near(d_b, m, 1.0, 2.0 ** -25, m)
    near(d_a, m, 1.0, 2.0 ** -25, m)
    assert not bool(dx.any())

@pytest.mark.parametrize("in_dim,m", [(64, 20), (64, 100), (300, 700), (512, 2000)])
def test_dx_of_a_large_rank(in_dim, m):
    """The adapter's part of dx is a sum over 1024 ranks."""
    rank, out_dim = 1024, 64
    dy = torch.zeros(m, out_dim, device="cuda")
    dy[:, 3] = 1.0
    b = torch.zeros(out_dim, rank, device="cuda")
    b[3] = 2.0 ** -25
    b[3, 0] = 1.0                                      # dH[t, :] = 1, 2^-25, 2^-25, ...
    lora = nv.Lora(torch.ones(rank, in_dim, device="cuda"), b, float(rank))
    packed = nv.act_pack(torch.ones(m, in_dim, device="cuda"))
    dx, _, _ = nv.lora_linear_bwd_packed(zeros(in_dim, out_dim), lora, dy, packed, torch.zeros(m, rank, device="cuda"))
    near(dx, rank, 1.0, 2.0 ** -25, rank)


# a block several rows and the whole of B; a cluster; a block a row
@pytest.mark.parametrize("out_dim,rank,m,small", [(14336, 256, 4736, 2.0 ** -25), (14336, 300, 4800, 2.0 ** -25), (14336, 256, 200, 2.0 ** -25),
                                                  (1024, 1, 5, 2.0 ** -24), (1000, 16, 40, 2.0 ** -24), (20000, 1, 300, 2.0 ** -24)])
def test_hidden_gradient_of_a_wide_layer(out_dim, rank, m, small):
    """dH = dy . B, seen through dA: token 1 alone is not zero."""
    in_dim = 64
    b = torch.full((out_dim, rank), small, device="cuda")
    b[0] = 1.0
    dy = torch.zeros(m, out_dim, device="cuda")
    dy[1] = 1.0
    lora = nv.Lora(torch.zeros(rank, in_dim, device="cuda"), b, float(rank))
    packed = nv.act_pack(torch.ones(m, in_dim, device="cuda"))
    _, d_a, _ = nv.lora_linear_bwd_packed(zeros(in_dim, out_dim), lora, dy, packed, torch.zeros(m, rank, device="cuda"))
    near(d_a, out_dim, 1.0, small, out_dim)
    # every 32nd value of it the large one: the partial sums of threads that share a sum
    b[:] = small / 4
    b[0] = 1.0
    _, d_a, _ = nv.lora_linear_bwd_packed(zeros(in_dim, out_dim), lora, dy, packed, torch.zeros(m, rank, device="cuda"))
    near(d_a, out_dim, 1.0, small / 4, out_dim)


@pytest.mark.parametrize("rank,out_dim,m", [(1024, 100, 3), (1024, 64, 200), (520, 33, 40)])
def test_bank_of_a_large_rank(rank, out_dim, m):
    """h . B^T is a sum over the ranks: four large terms, one for each of the threads that share a column."""
    in_dim = 64
    a = torch.full((rank, in_dim), 2.0 ** -24, device="cuda")
    a[:4] = 1.0
    bank = nv.LoraBank([nv.Lora(a, torch.ones(out_dim, rank, device="cuda"), float(rank))])
    x = torch.zeros(m, in_dim, device="cuda")
    x[:, 5] = 1.0
    y = nv.lora_bank_linear_fwd(zeros(in_dim, out_dim), bank, torch.zeros(m, dtype=torch.int32, device="cuda"), x)
    want = 4.0 + (rank - 4) * U
    assert float((y.double() - want).abs().max()) <= bound(rank) * want


@pytest.mark.parametrize("storage,compute", [(nv.I8, nv.F32), (nv.I4, nv.BF16)])
@pytest.mark.parametrize("in_dim,out_dim,m,rank", [(256, 384, 32, 16), (384, 256, 100, 8), (512, 128, 128, 64), (256, 640, 333, 16), (1024, 1024, 700, 32),
                                                   (256, 1024, 2049, 8), (128, 1408, 3000, 16), (256, 896, 2500, 64), (256, 1024, 4097, 32)])
@pytest.mark.parametrize("aligned", [True, False])
def test_gradient_of_a_has_the_whole_hidden_gradient(storage, compute, in_dim, out_dim, m, rank, aligned):
    """bf16 rows: dH is a sum of eight whole numbers up to 127, which bf16 does not hold, and every sum is below 2^24: dA is exact but for
    its own rounding."""
    g = torch.Generator(device="cuda").manual_seed(m + rank)
    if storage == nv.I8:
        weight = zeros(in_dim, out_dim)
    else:
        weight = nv.Weight(torch.zeros(out_dim * in_dim // 2, dtype=torch.uint8, device="cuda"), nv.I4, in_dim, out_dim,
                           torch.ones(out_dim * in_dim // 128, dtype=torch.float16, device="cuda"))
    b = torch.randint(-127, 128, (out_dim, rank), generator=g, device="cuda").bfloat16()
    lora = nv.Lora(torch.zeros(rank, in_dim, dtype=torch.bfloat16, device="cuda"), b, float(rank))
    dy = torch.zeros(m, out_dim, dtype=torch.bfloat16, device="cuda")
    at = torch.rand(m, out_dim, generator=g, device="cuda").topk(8, dim=1).indices
    dy.scatter_(1, at, (torch.randint(0, 2, (m, 8), generator=g, device="cuda") * 2 - 1).bfloat16())
    x = torch.randint(-3, 4, (m, in_dim), generator=g, device="cuda").bfloat16()
    packed = nv.act_pack(x)
    hidden = torch.randint(-3, 4, (m, rank), generator=g, device="cuda").bfloat16()
    if not aligned:
        flat = torch.empty(hidden.numel() + 1, dtype=torch.bfloat16, device="cuda")
        flat[1:] = hidden.view(-1)
        hidden = flat[1:].view(m, rank)
    dx, d_a, d_b = nv.lora_linear_bwd_packed(weight, lora, dy, packed, hidden, compute)
    dh = dy.double() @ b.double()
    assert torch.equal(d_a, (dh.t() @ x.double()).bfloat16())
    assert torch.equal(d_b, (dy.double().t() @ hidden.double()).bfloat16())
    assert not bool(dx.any())


# (slices: the blocks or clusters that walk over the rows, and the slices of rows of the form for any width)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,dim,slices", [(3000, 4096, 148), (3000, 12288, 74), (3000, 20480, 32), (3000, 40000, 16), (5000, 33003, 16), (4000, 70000, 62),
                                             (9000, 9001, 72)])
def test_layernorm_gradients_over_many_wide_rows(rows, dim, slices, dtype):
    """A column's sum is a chain of rows / slices and the slices' sums, 32 of them side by side: row 0 gives 1, the others 2^-25."""
    dy = torch.full((rows, dim), 2.0 ** -25, dtype=dtype, device="cuda")
    dy[0] = 1.0
    x = torch.ones(rows, dim, dtype=dtype, device="cuda")
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    _, d_gamma, d_beta = nv.layernorm_bwd(dy, x, mean, rstd)
    want = 1.0 + (rows - 1) * 2.0 ** -25
    for got in (d_gamma, d_beta):
        assert float((got.double() - want).abs().max()) <= (rows / slices + slices / 32 + 16) * U * want
