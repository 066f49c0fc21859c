"""Adapters of many requests beside one frozen linear (caif_b200/csrc/lora_bank.cu) against the formula in 64 bits.

Tolerances, element by element: `half` is half a step of the result's type; a sum of n products in fp32, whose chain of
additions is at most n / 32 + 64 long in any kernel, is off by at most that many times 2^-23 times the sum of the products'
magnitudes (2^-23: the tensor core truncates where it adds).  x . A^T enters the second product in fp32 or as two bf16 terms
(2^-16 relative).  The result is rounded where the adapters' part is stored and where the frozen product is added to it, and
the frozen product by itself before that at most once more.
"""
import numpy as np
import pytest
import torch

import caif_oracle as orc
from caif_b200 import native as nv
from gpu_util import make_weight

pytestmark = pytest.mark.gpu

S = 2.0 ** -23


def half(t):
    return torch.finfo(t).eps / 2


def make_bank(seed, in_dim, out_dim, ranks, dtype, std_b=0.05):
    g = torch.Generator(device="cuda").manual_seed(seed)
    loras = []
    for i, r in enumerate(ranks):
        a = (torch.randn(r, in_dim, generator=g, device="cuda") / in_dim ** 0.5).to(dtype)
        b = (torch.randn(out_dim, r, generator=g, device="cuda") * std_b).to(dtype)
        loras.append(nv.Lora(a, b, 2.0 * r + i))
    return nv.LoraBank(loras)


def make_rows(seed, m, in_dim, count, dtype, kind="any"):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    x = torch.randn(m, in_dim, generator=g, device="cuda").to(dtype)
    if kind == "any":
        idx = torch.randint(-1, count + 1, (m,), generator=g, device="cuda", dtype=torch.int32)
    elif kind == "one":
        idx = torch.full((m,), count - 1, dtype=torch.int32, device="cuda")
    elif kind == "none":
        idx = torch.full((m,), -1, dtype=torch.int32, device="cuda")
    else:   # runs of rows, as prompts are
        idx = (torch.arange(m, device="cuda", dtype=torch.int32) * count // max(m, 1)).to(torch.int32)
    return x, idx


def zero_weight(in_dim, out_dim, storage=nv.I8):
    if storage == nv.I8:
        return nv.Weight(torch.zeros(out_dim, in_dim, dtype=torch.int8, device="cuda"), nv.I8, in_dim, out_dim,
                         torch.ones(1, device="cuda"))
    return nv.Weight(torch.zeros(out_dim, in_dim, device="cuda"), nv.F32, in_dim, out_dim)


def adapters_64(bank, idx, x, out_dim):
    """the adapters' part and the bound of its error before any rounding to the result's type"""
    xd = x.double()
    y = torch.zeros(x.shape[0], out_dim, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(y)
    for i, l in enumerate(bank.loras):
        rows = torch.nonzero(idx == i)[:, 0]
        a, b, s = l.a.double(), l.b.double(), l.alpha / l.rank
        h = xd[rows] @ a.t()
        y[rows] = s * (h @ b.t())
        eh = (x.shape[1] / 32 + 64) * S * (xd[rows].abs() @ a.abs().t())
        tol[rows] = s * ((eh + (2.0 ** -16 + (l.rank / 32 + 70) * S) * h.abs()) @ b.abs().t())
    return y, tol


def tiny(t):
    return 2.0 ** -24 if t == torch.float16 else 0.0


DTYPES = [torch.bfloat16, torch.float32, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,in_dim,out_dim,ranks,kind", [
    (1, 128, 128, [16], "one"), (1, 1024, 512, [8, 16, 64], "any"), (3, 96, 40, [16, 8], "any"),
    (16, 256, 264, [16] * 5, "any"), (17, 512, 128, [8, 32, 16], "any"), (33, 4096, 136, [64, 24, 8, 40], "any"),
    (64, 1024, 1024, [16] * 70, "any"), (300, 256, 384, [16, 32], "runs"), (129, 160, 8, [8], "none"),
    (1000, 128, 256, [16, 8, 64, 32, 48], "runs"), (5, 14336, 128, [16, 16], "any"),
    # few rows into many columns
    (16, 512, 14336, [32] * 12, "any"), (100, 256, 2056, [16, 8, 64] * 30, "any"), (60, 1024, 8192, [64, 8] * 10, "any"),
    (1, 64, 14336, [8], "one"), (128, 128, 4096, [16], "runs"), (128, 128, 4096, [16] * 16, "runs"),
    # general forms: ranks, widths and rows that no 16-byte piece fits
    (7, 100, 36, [5, 1, 17], "any"), (50, 33, 77, [3, 200], "any"), (2, 64, 64, [1024], "one"), (40, 130, 9, [16], "any"),
    (20, 1, 1, [1], "any"),
])
def test_adapters_part(dtype, m, in_dim, out_dim, ranks, kind):
    """A frozen weight of zeros: the result is the adapters' part."""
    bank = make_bank(m + in_dim, in_dim, out_dim, ranks, dtype)
    x, idx = make_rows(m, m, in_dim, len(ranks), dtype, kind)
    y = nv.lora_bank_linear_fwd(zero_weight(in_dim, out_dim), bank, idx, x)
    want, tol = adapters_64(bank, idx, x, out_dim)
    tol = tol + 2 * half(dtype) * (want.abs() + tol) + tiny(dtype)
    assert y.dtype == dtype and y.shape == (m, out_dim)
    assert bool(((y.double() - want).abs() <= tol).all())
    none = (idx < 0) | (idx >= len(ranks))
    assert not bool(y[none].any())


@pytest.mark.parametrize("storage,compute", [(orc.I8, orc.F32), (orc.I8, orc.BF16), (orc.I4, orc.BF16), (orc.I4, orc.F32),
                                             (orc.BF16, orc.BF16), (orc.F32, orc.F32)])
@pytest.mark.parametrize("m", [1, 5, 16, 17, 100, 769, 1500])
def test_beside_a_frozen_weight(storage, compute, m):
    in_dim, out_dim = 512, 640
    rng = np.random.default_rng(m)
    weight, codes, scales = make_weight(rng, out_dim, in_dim, storage)
    w64 = nv.weight_materialize(weight).double()
    bank = make_bank(m, in_dim, out_dim, [16, 8, 32], torch.bfloat16)
    x, idx = make_rows(m, m, in_dim, 3, torch.bfloat16)
    y = nv.lora_bank_linear_fwd(weight, bank, idx, x, compute)
    part, tol = adapters_64(bank, idx, x, out_dim)
    xd = x.double()
    base = xd @ w64.t()
    terms = xd.abs() @ w64.abs().t()
    # int4 under bf16 compute: the scale, or code times scale, is rounded to bf16; as two bf16 terms under fp32
    once = half(torch.bfloat16) * 1.01 if storage in (orc.I4, orc.F32) and compute == orc.BF16 else (2.0 ** -16 if storage == orc.I4 else 0.0)
    tol = tol + (once + (in_dim / 32 + 64) * S) * terms
    tol = tol + half(torch.bfloat16) * (base.abs() + part.abs() + (base + part).abs() + 3 * tol)
    assert bool(((y.double() - (base + part)).abs() <= tol).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("storage", [orc.I8, orc.I4])
@pytest.mark.parametrize("in_dim,out_dim,m", [(128, 1, 1), (384, 40, 8), (640, 880, 2), (1408, 1776, 9), (256, 136, 128), (256, 136, 129)])
def test_beside_a_weight_of_another_width(storage, dtype, in_dim, out_dim, m):
    weight, _, _ = make_weight(np.random.default_rng(m), out_dim, in_dim, storage)
    w64 = nv.weight_materialize(weight).double()
    bank = make_bank(m, in_dim, out_dim, [16, 5], dtype)
    x, idx = make_rows(m, m, in_dim, 2, dtype)
    y = nv.lora_bank_linear_fwd(weight, bank, idx, x, orc.F32)
    part, tol = adapters_64(bank, idx, x, out_dim)
    base, terms = x.double() @ w64.t(), x.double().abs() @ w64.abs().t()
    tol = tol + (S + (in_dim / 32 + 64) * S + (2.0 ** -16 if storage == orc.I4 and dtype == torch.bfloat16 else 0.0)) * terms
    tol = tol + half(dtype) * (base.abs() + part.abs() + (base + part).abs() + 3 * tol) + tiny(dtype)
    assert bool(((y.double() - (base + part)).abs() <= tol).all())


@pytest.mark.parametrize("m", [1, 16, 17, 48, 128, 129, 500, 768, 1500])
def test_int4_weight_is_rounded_once(m):
    """Rows of one 1 pick columns of the weight: code times scale as bf16, with no rounding of the scale before that."""
    in_dim, out_dim = 256, 640
    weight, _, _ = make_weight(np.random.default_rng(m), out_dim, in_dim, orc.I4)
    bank = make_bank(m, in_dim, out_dim, [16, 8], torch.bfloat16)
    pick = torch.randint(0, in_dim, (m,), generator=torch.Generator(device="cuda").manual_seed(m), device="cuda")
    x = torch.zeros(m, in_dim, dtype=torch.bfloat16, device="cuda")
    x[torch.arange(m, device="cuda"), pick] = 1.0
    none = torch.full((m,), -1, dtype=torch.int32, device="cuda")
    y = nv.lora_bank_linear_fwd(weight, bank, none, x, nv.BF16)
    assert torch.equal(y, nv.weight_materialize(weight).float().t()[pick].bfloat16())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_beside_a_frozen_weight_other_types(dtype):
    in_dim, out_dim, m = 256, 384, 30
    weight, _, _ = make_weight(np.random.default_rng(3), out_dim, in_dim, orc.I8)
    w64 = nv.weight_materialize(weight).double()
    bank = make_bank(3, in_dim, out_dim, [16, 8], dtype)
    x, idx = make_rows(3, m, in_dim, 2, dtype)
    y = nv.lora_bank_linear_fwd(weight, bank, idx, x, orc.F32)
    part, tol = adapters_64(bank, idx, x, out_dim)
    base, terms = x.double() @ w64.t(), x.double().abs() @ w64.abs().t()
    # (fp32 rows enter the tensor core as three bf16 terms: 2^-23 relative)
    tol = tol + (S + (in_dim / 32 + 64) * S) * terms
    tol = tol + half(dtype) * (base.abs() + part.abs() + (base + part).abs() + 3 * tol) + tiny(dtype)
    assert bool(((y.double() - (base + part)).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bad_values_stay_with_their_rows(dtype):
    """An adapter full of NaN and infinities, and a row of them, reach their own rows alone, bit for bit."""
    in_dim, out_dim, m = 512, 256, 48
    bank = make_bank(5, in_dim, out_dim, [16, 16, 8, 16], dtype)
    x, idx = make_rows(5, m, in_dim, 4, dtype)
    idx[7], idx[8] = 2, 0
    w = zero_weight(in_dim, out_dim)
    clean = nv.lora_bank_linear_fwd(w, bank, idx, x)
    bank.loras[2].a.fill_(float("nan"))
    bank.loras[2].b.fill_(float("inf"))
    x[8].fill_(float("nan"))
    got = nv.lora_bank_linear_fwd(w, bank, idx, x)
    rest = torch.nonzero((idx != 2) & (torch.arange(m, device="cuda") != 8))[:, 0]
    assert torch.equal(got[rest], clean[rest])
    assert bool(torch.isnan(got[8]).all()) and bool(torch.isnan(got[7]).all())


@pytest.mark.parametrize("m,out_dim", [(16, 384), (50, 384), (400, 384), (100, 8192), (16, 28800)])
def test_rows_in_any_order_give_the_same_bits(m, out_dim):
    in_dim = 1024
    bank = make_bank(6, in_dim, out_dim, [16, 32, 8, 16, 64], torch.bfloat16)
    x, idx = make_rows(6, m, in_dim, 5, torch.bfloat16)
    w = zero_weight(in_dim, out_dim)
    y = nv.lora_bank_linear_fwd(w, bank, idx, x)
    order = torch.randperm(m, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    assert torch.equal(nv.lora_bank_linear_fwd(w, bank, idx[order].contiguous(), x[order].contiguous()), y[order])
    assert torch.equal(nv.lora_bank_linear_fwd(w, bank, idx, x), y)


@pytest.mark.parametrize("m", [127, 128, 129, 5000])
@pytest.mark.parametrize("count", [1, 4096, 4097])
def test_many_adapters_and_the_ends_of_the_forms(m, count):
    """Every row's adapter its own where there are so many; scratch full of NaN is not read before it is written."""
    in_dim, out_dim, r = 64, 72, 8
    g = torch.Generator(device="cuda").manual_seed(count + m)
    a = (torch.randn(count, r, in_dim, generator=g, device="cuda") / 8).bfloat16()
    b = (torch.randn(count, out_dim, r, generator=g, device="cuda") * 0.05).bfloat16()
    bank = nv.LoraBank([nv.Lora(a[i], b[i], 16.0) for i in range(count)])
    w = zero_weight(in_dim, out_dim)
    x = torch.randn(m, in_dim, generator=g, device="cuda").bfloat16()
    idx = torch.randint(-1, count + 1, (m,), generator=g, device="cuda", dtype=torch.int32)
    idx[0], idx[-1] = count - 1, 2 ** 31 - 1
    ws = torch.full((nv.lora_bank_workspace_bytes(w, bank, m),), 255, dtype=torch.uint8, device="cuda")
    y = nv.lora_bank_linear_fwd(w, bank, idx, x, workspace=ws)
    mine = (idx >= 0) & (idx < count)
    at = idx.clamp(0, count - 1).long()
    xd = x.double()
    h = torch.einsum("mi,mri->mr", xd, a[at].double())
    eh = (in_dim / 32 + 64) * S * torch.einsum("mi,mri->mr", xd.abs(), a[at].double().abs())
    want = 2.0 * torch.einsum("mr,mor->mo", h, b[at].double()) * mine[:, None]
    tol = 2.0 * torch.einsum("mr,mor->mo", eh + (2.0 ** -16 + (r / 32 + 70) * S) * h.abs(), b[at].double().abs())
    tol = tol + 2 * half(torch.bfloat16) * (want.abs() + tol)
    assert bool(((y.double() - want).abs() <= tol).all())
    assert not bool(y[~mine].any())


def test_operands_off_a_16_byte_boundary():
    in_dim, out_dim, m = 256, 128, 20
    bank = make_bank(7, in_dim, out_dim, [16, 8], torch.bfloat16)
    x, idx = make_rows(7, m, in_dim, 2, torch.bfloat16)
    w = zero_weight(in_dim, out_dim)
    want, tol = adapters_64(bank, idx, x, out_dim)
    tol = tol + 2 * half(torch.bfloat16) * (want.abs() + tol)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    other = nv.LoraBank([nv.Lora(shifted(l.a), l.b, l.alpha) for l in bank.loras])
    third = nv.LoraBank([nv.Lora(l.a, shifted(l.b), l.alpha) for l in bank.loras])
    out = shifted(torch.empty(m, out_dim, dtype=torch.bfloat16, device="cuda"))
    for b, xs, o in ((bank, shifted(x), None), (other, x, None), (third, x, None), (bank, x, out)):
        y = nv.lora_bank_linear_fwd(w, b, idx, xs, out=o)
        assert bool(((y.double() - want).abs() <= tol).all())
    assert y.data_ptr() == out.data_ptr()


def test_given_result_and_scratch_and_no_rows():
    in_dim, out_dim, m = 512, 256, 40
    bank = make_bank(8, in_dim, out_dim, [16, 8], torch.bfloat16)
    x, idx = make_rows(8, m, in_dim, 2, torch.bfloat16)
    weight, _, _ = make_weight(np.random.default_rng(8), out_dim, in_dim, orc.I4)
    want = nv.lora_bank_linear_fwd(weight, bank, idx, x, nv.BF16)
    ws = torch.empty(nv.lora_bank_workspace_bytes(weight, bank, m, nv.BF16) + 512, dtype=torch.uint8, device="cuda")
    out = torch.empty(m + 2, out_dim, dtype=torch.bfloat16, device="cuda")
    out.fill_(7.0)
    got = nv.lora_bank_linear_fwd(weight, bank, idx, x, nv.BF16, out=out[:m], workspace=ws)
    assert torch.equal(got, want) and bool((out[m:] == 7.0).all())
    # rows in more than two dimensions
    got = nv.lora_bank_linear_fwd(weight, bank, idx.view(4, 10), x.view(4, 10, in_dim), nv.BF16)
    assert got.shape == (4, 10, out_dim) and torch.equal(got.view(m, out_dim), want)
    empty = nv.lora_bank_linear_fwd(weight, bank, idx[:0], x[:0], nv.BF16)
    assert empty.shape == (0, out_dim)


def test_captured_with_other_rows_and_on_another_stream():
    in_dim, out_dim, m = 512, 256, 24
    bank = make_bank(9, in_dim, out_dim, [16, 8, 32], torch.bfloat16)
    weight, _, _ = make_weight(np.random.default_rng(9), out_dim, in_dim, orc.I4)
    x, idx = make_rows(9, m, in_dim, 3, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = nv.lora_bank_linear_fwd(weight, bank, idx, x, nv.BF16)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):      # two captured calls, each with scratch of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(nv.lora_bank_linear_fwd(weight, bank, idx, x, nv.BF16))
        graphs.append(graph)
    for g, o in zip(graphs, outs):
        g.replay()
        assert torch.equal(o, y)
    x2, idx2 = make_rows(10, m, in_dim, 3, torch.bfloat16)
    want = nv.lora_bank_linear_fwd(weight, bank, idx2, x2, nv.BF16)
    x.copy_(x2)
    idx.copy_(idx2)
    for g, o in zip(graphs, outs):
        g.replay()
        assert torch.equal(o, want)


def test_refusals():
    in_dim, out_dim, m = 128, 256, 4
    bank = make_bank(11, in_dim, out_dim, [16, 8], torch.bfloat16)
    x, idx = make_rows(11, m, in_dim, 2, torch.bfloat16)
    w = zero_weight(in_dim, out_dim)
    call = nv.lora_bank_linear_fwd
    with pytest.raises(nv.CaifqError, match="must be"):
        call(w, bank, idx.long(), x)
    with pytest.raises(nv.CaifqError, match="adapter_of_row has"):
        call(w, bank, idx[:3], x)
    with pytest.raises(nv.CaifqError, match="dtype"):
        call(w, bank, idx, x.float())
    with pytest.raises(nv.CaifqError, match="last dimension"):
        call(w, bank, idx, x[:, :64].contiguous())
    with pytest.raises(nv.CaifqError, match="contiguous"):
        call(w, bank, idx, x.t().contiguous().t())
    with pytest.raises(nv.CaifqError, match="out has"):
        call(w, bank, idx, x, out=torch.empty(3, out_dim, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(nv.CaifqError, match="workspace"):
        call(w, bank, idx, x, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(nv.CaifqError, match="the weight has"):
        call(zero_weight(in_dim, 128), bank, idx, x)
    square = make_bank(12, in_dim, in_dim, [8], torch.bfloat16)
    with pytest.raises(nv.CaifqError, match="overlap"):
        call(zero_weight(in_dim, in_dim), square, idx, x, out=x)
    with pytest.raises(nv.CaifqError, match="no adapters"):
        nv.LoraBank([])
    a, b = bank.loras[0].a, bank.loras[0].b
    with pytest.raises(nv.CaifqError, match="factors"):
        nv.LoraBank([nv.Lora(a, b, 1.0), nv.Lora(a, b[:128], 1.0)])
    with pytest.raises(nv.CaifqError, match="two types"):
        nv.LoraBank([nv.Lora(a, b.float(), 1.0)])
    with pytest.raises(nv.CaifqError, match="dtype"):
        nv.LoraBank([nv.Lora(a, b, 1.0), nv.Lora(a.float(), b.float(), 1.0)])
