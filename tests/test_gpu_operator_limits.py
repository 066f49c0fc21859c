"""The operators around an adapted projection at the ends of what their entry points take."""
import pytest
import torch

from caif_b200 import native as nv

pytestmark = pytest.mark.gpu


def test_layernorm_of_the_most_rows():
    """2^31 - 1 rows of one column off a 16-byte boundary: the form that walks over the rows counts them past 2^31.  One value's mean is
    the value, its distance from it 0."""
    rows = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    x = torch.zeros(rows + 1, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 1183, 1184, rows // 2, rows - 1185, rows - 1184, rows - 2, rows - 1], device="cuda")
    x[1:][at] = torch.arange(1.0, 10.0, device="cuda").bfloat16()
    x = x[1:].view(rows, 1)
    y = torch.empty(rows + 2, dtype=torch.bfloat16, device="cuda")
    y[-1] = 7.0                                        # behind the last row
    mean = torch.empty(rows + 1, device="cuda")
    rstd = torch.empty(rows + 1, device="cuda")
    mean[-1] = rstd[-1] = 7.0
    beta = torch.full((1,), 0.5, device="cuda")
    lib, s = nv.lib(), torch.cuda.current_stream().cuda_stream
    out = y[1:]
    nv._check(lib.caifq_layernorm_fwd(x.data_ptr(), None, beta.data_ptr(), out.data_ptr(), mean.data_ptr(), rstd.data_ptr(), 0.25, nv.BF16, rows, 1, s),
              "layernorm_fwd")
    assert float(y[-1]) == 7.0 and float(mean[-1]) == 7.0 and float(rstd[-1]) == 7.0
    step = 1 << 28
    for i in range(0, rows, step):
        end = min(rows, i + step)
        assert bool((mean[i:end] == x[i:end, 0]).all()) and bool((out[i:end] == 0.5).all()) and bool((rstd[i:end] == 2.0).all())
    # dx over dy, without the columns' sums: a row of one value has no gradient
    out.fill_(1.0)
    y[-1] = 7.0
    nv._check(lib.caifq_layernorm_bwd(out.data_ptr(), x.data_ptr(), None, mean.data_ptr(), rstd.data_ptr(), out.data_ptr(), None, None, 0, None, nv.BF16,
                                      rows, 1, s), "layernorm_bwd")
    assert float(y[-1]) == 7.0
    for i in range(0, rows, step):
        assert not bool(out[i:min(rows, i + step)].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 45])
def test_pack_error_down_to_the_least_scale(dtype, dim):
    """Half a step of error everywhere; less than a 127th of the block's largest value above the least scale, and at it as much as that value."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    tops = torch.tensor([2.0 ** e for e in (-133, -128, -127, -126, -121, -120, -119, -100, 0, 100, 127)], device="cuda", dtype=torch.float64)
    x = (torch.rand(len(tops), dim, generator=g, device="cuda", dtype=torch.float64) * 2 - 1) * tops[:, None]
    x[:, 3::32] = tops[:, None]
    x = x.to(dtype)
    p = nv.act_pack(x)
    s = torch.exp2(p.scales.double() - 127).repeat_interleave(32, 1)[:, :dim]
    error = (x.double() - p.codes.double() * s).abs()
    assert bool((error <= s / 2).all()) and bool((p.scales >= 1).all())
    assert torch.equal(p.scales.min(1).values == 1, tops <= 127 * 2.0 ** -126) and torch.equal(p.scales.max(1).values == 1, tops <= 127 * 2.0 ** -126)
    above = tops > 127 * 2.0 ** -126
    assert bool((s[above] / 2 < tops[above][:, None] / 127).all())
    lost = p.codes[tops == 2.0 ** -127]
    assert not bool(lost.any()) and float(error[tops == 2.0 ** -127].max()) == 2.0 ** -127


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("storage", [nv.I8, nv.I4])
@pytest.mark.parametrize("out_dim,m,few_32,few_16", [(14344, 32, True, True), (14344, 48, False, True), (14344, 64, False, False), (14344, 128, False, False),
                                                     (4104, 96, True, True), (1776, 128, True, True), (60008, 8, True, True), (60008, 33, False, True),
                                                     (60008, 64, False, False)])
def test_bank_takes_the_product_of_odd_widths_by_its_size(out_dim, m, few_32, few_16, storage, dtype):
    """Few rows of few columns by the kernel that reads the codes once for eight rows, others by the one for any cell: the same sums."""
    in_dim = 136
    few = few_32 if dtype == torch.float32 else few_16
    g = torch.Generator(device="cuda").manual_seed(out_dim + m)
    if storage == nv.I8:
        codes = torch.randint(-127, 128, (out_dim, in_dim), generator=g, device="cuda", dtype=torch.int8)
        weight = nv.Weight(codes, nv.I8, in_dim, out_dim, torch.full((1,), 0.25, device="cuda"))
    else:
        codes = torch.randint(0, 256, (out_dim * in_dim // 2,), generator=g, device="cuda", dtype=torch.uint8)
        weight = nv.Weight(codes, nv.I4, in_dim, out_dim, torch.full((out_dim * in_dim // 8,), 0.25, device="cuda", dtype=torch.float16), 0, 8)
    bank = nv.LoraBank([nv.Lora(torch.zeros(8, in_dim, device="cuda", dtype=dtype), torch.zeros(out_dim, 8, device="cuda", dtype=dtype), 8.0)])
    x = torch.randint(-2, 3, (m, in_dim), generator=g, device="cuda").to(dtype)     # (whole numbers: sums without rounding)
    rows = torch.zeros(m, dtype=torch.int32, device="cuda")
    other = nv.Weight(torch.zeros(128, 128, dtype=torch.int8, device="cuda"), nv.I8, 128, 128, torch.ones(1, device="cuda"))
    nv.linear_fwd(other, torch.zeros(200, 128, dtype=torch.bfloat16, device="cuda"))
    assert nv.last_path() == "umma"
    got = nv.lora_bank_linear_fwd(weight, bank, rows, x)
    assert nv.last_path() == ("decode" if few else "generic")
    want = x.double() @ nv.weight_materialize(weight).double().t()
    assert torch.equal(got, want.to(dtype))
