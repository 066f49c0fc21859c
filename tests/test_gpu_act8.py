"""Activations kept in 8 bits (caif_b200/csrc/act8.cu) and an adapter's backward pass on them.

Packing is defined without rounding but the code's own, so codes and scales are compared for equality with the definition in
64 bits.  The gradients' tolerances, element by element: `half` is half a step of the storage type, and a sum of n products in
fp32, whose chain of additions is at most n / 32 + 64 long in any kernel, is off by at most that many times 2^-23 times the
sum of the products' magnitudes.
"""
import numpy as np
import pytest
import torch

import caif_oracle as orc
from caif_b200 import native as nv
from gpu_util import make_weight

pytestmark = pytest.mark.gpu

S = 2.0 ** -23
DTYPES = [torch.bfloat16, torch.float32, torch.float16]


def half(t):
    return torch.finfo(t).eps / 2


def define(x):
    """codes and scale bytes of the definition, in 64 bits"""
    rows, dim = x.shape
    blocks = (dim + 31) // 32
    b = torch.zeros(rows, blocks * 32, dtype=torch.float64, device=x.device)
    b[:, :dim] = x.double()
    b = b.view(rows, blocks, 32)
    bad = ~torch.isfinite(b).all(2)
    b = torch.where(bad[:, :, None], 0.0, b)
    most = b.abs().amax(2)
    e = torch.full_like(most, -126)
    for step in range(-126, 128):     # the smallest power of two that holds the block
        e = torch.where((most > 127 * 2.0 ** (step - 1)) & (step - 1 >= -126), float(step), e)
    q = torch.round(b / torch.exp2(e)[:, :, None])
    byte = torch.where(bad, 255.0, e + 127)
    return q.view(rows, -1)[:, :dim].to(torch.int8), byte.to(torch.uint8)


def check_pack(x):
    p = nv.act_pack(x)
    codes, scales = define(x)
    assert torch.equal(p.scales, scales)
    assert torch.equal(p.codes, codes)
    return p


def rows_of(rows, dim, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + dim)
    x = torch.randn(rows, dim, generator=g, device="cuda")
    x[:, ::17] *= 30.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 64), (7, 100), (16, 1001), (9, 1024), (33, 4096),
                                      (130, 160), (4, 14336), (1, 40000)])
def test_pack_and_unpack(rows, dim, dtype):
    x = rows_of(rows, dim, dtype)
    p = check_pack(x)
    scale = torch.exp2(p.scales.double() - 127).repeat_interleave(32, 1)[:, :dim]
    value = p.codes.double() * scale
    assert bool(((x.double() - value).abs() <= scale / 2).all())
    for t in DTYPES:
        back = nv.act_unpack(p, t)
        assert back.dtype == t and torch.equal(back, value.to(t))
    assert torch.equal(nv.act_unpack(p, torch.float32).double(), value)


def test_pack_of_other_shapes():
    x = rows_of(24, 96, torch.bfloat16)
    p = nv.act_pack(x)
    q = nv.act_pack(x.view(2, 3, 4, 96))
    assert q.codes.shape == (2, 3, 4, 96) and q.scales.shape == (2, 3, 4, 3)
    assert torch.equal(q.codes.view(24, 96), p.codes) and torch.equal(q.scales.view(24, 3), p.scales)
    assert nv.act_unpack(q, torch.float32).shape == (2, 3, 4, 96)
    v = nv.act_pack(x[0])
    assert torch.equal(v.codes, p.codes[0]) and torch.equal(v.scales, p.scales[0])
    e = nv.act_pack(x[:0])
    assert e.codes.shape == (0, 96) and e.scales.shape == (0, 3) and nv.act_unpack(e).shape == (0, 96)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 45])
def test_pack_at_the_ends_of_the_format(dtype, dim):
    """Zeros, the largest and smallest values, blocks that just fit 127 steps and that just do not, ties."""
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    one_up = 1 + torch.finfo(dtype).eps
    tops = [0.0, -0.0, big, -big, small, -small, torch.finfo(dtype).tiny * torch.finfo(dtype).eps, 127.0, 127.0 * one_up, 63.5,
            128.0, 1.0, one_up, 126.5, 2.0 ** -14, -127.0 * 2.0 ** 7]
    x = torch.zeros(len(tops), dim, device="cuda", dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(dim)
    x[:, :] = (torch.randint(-254, 255, x.shape, generator=g, device="cuda") / 254.0).to(dtype)    # halves of a step: ties
    x = x * torch.tensor(tops, device="cuda", dtype=torch.float64).abs()[:, None]
    x[:, 3] = torch.tensor(tops, device="cuda", dtype=torch.float64)
    x = x.to(dtype)
    assert bool(torch.isfinite(x).all())
    check_pack(x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 77])
def test_pack_of_values_that_are_not_finite(dtype, dim):
    x = rows_of(6, dim, dtype)
    clean = nv.act_unpack(nv.act_pack(x), dtype)
    x[1, 5], x[2, 40], x[4, 70] = float("nan"), float("inf"), float("-inf")
    p = check_pack(x)
    back = nv.act_unpack(p, dtype)
    blocks = {(1, 0), (2, 1), (4, 2)}
    for r in range(6):
        for b in range((dim + 31) // 32):
            got = back[r, 32 * b:32 * b + 32]
            if (r, b) in blocks:
                assert bool(torch.isnan(got).all())
            else:
                assert torch.equal(got, clean[r, 32 * b:32 * b + 32])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 1001, 4096])
def test_pack_off_a_16_byte_boundary(dtype, dim):
    x = rows_of(5, dim, dtype)
    p = check_pack(x)
    flat = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")
    flat[1:] = x.reshape(-1)
    q = nv.act_pack(flat[1:].view(5, dim))
    assert torch.equal(q.codes, p.codes) and torch.equal(q.scales, p.scales)
    # codes, scales and results that start anywhere, through the C call
    codes = torch.empty(x.numel() + 1, dtype=torch.int8, device="cuda")[1:]
    scales = torch.empty(p.scales.numel() + 1, dtype=torch.uint8, device="cuda")[1:]
    code = nv.dtype_code(x)
    nv._check(nv.lib().caifq_act_pack(nv._ptr(x), code, nv._ptr(codes), nv._ptr(scales), 5, dim, nv._stream()), "pack")
    assert torch.equal(codes.view(5, dim), p.codes) and torch.equal(scales.view(5, -1), p.scales)
    back = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:]
    nv._check(nv.lib().caifq_act_unpack(nv._ptr(codes), nv._ptr(scales), nv._ptr(back), code, 5, dim, nv._stream()), "unpack")
    assert torch.equal(back.view(5, dim), nv.act_unpack(p, dtype))


def test_pack_past_32_bits_of_elements():
    rows, dim = 33000, 65568      # 2.16e9 elements
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    tail = rows_of(40, dim, torch.bfloat16)
    x[-40:] = tail
    p = nv.act_pack(x)
    codes, scales = define(tail)
    assert torch.equal(p.codes[-40:], codes) and torch.equal(p.scales[-40:], scales)
    assert not bool(p.codes[:40].any()) and bool((p.scales[:40] == 1).all())
    back = nv.act_unpack(p, torch.bfloat16)
    assert torch.equal(back[-40:], nv.act_unpack(nv.PackedRows(codes, scales))) and not bool(back[:40].any())


# ---- the adapter's backward pass ----

def make_case(seed, storage, dtype, in_dim, out_dim, m, rank, alpha=None):
    weight, _, _ = make_weight(np.random.default_rng(seed), out_dim, in_dim, storage)
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = (torch.randn(rank, in_dim, generator=g, device="cuda") / in_dim ** 0.5).to(dtype)
    b = (torch.randn(out_dim, rank, generator=g, device="cuda") * 0.05).to(dtype)
    lora = nv.Lora(a, b, 1.3 * rank if alpha is None else alpha)
    packed = nv.act_pack(torch.randn(m, in_dim, generator=g, device="cuda").to(dtype))
    hidden = torch.randn(m, rank, generator=g, device="cuda").to(dtype)
    dy = torch.randn(m, out_dim, generator=g, device="cuda").to(dtype)
    return weight, lora, packed, hidden, dy


def check_grads(weight, lora, packed, hidden, dy, got, compute):
    dx, d_a, d_b = got
    t = dy.dtype
    w = nv.weight_materialize(weight).double()
    x = nv.act_unpack(packed, torch.float32).double()
    d, h, a, b = dy.double(), hidden.double(), lora.a.double(), lora.b.double()
    s = lora.alpha / lora.rank
    m = d.shape[0]
    tiny = 2.0 ** -24 if t == torch.float16 else 0.0

    def chain(n):
        return (n / 32 + 64) * S

    # (alpha / rank is a fp32 number that multiplies a fp32 sum: two roundings, in the chains' slack)
    want = s * (d.t() @ h)
    tol = s * chain(m) * (d.abs().t() @ h.abs())
    tol = tol * 1.01 + half(t) * (want.abs() + tol) + tiny
    assert bool(((d_b.double() - want).abs() <= tol).all())
    # dH may be rounded to the storage type (bf16, many rows)
    dh = d @ b
    eh = chain(weight.out_dim) * (d.abs() @ b.abs())
    eh = eh + half(t) * (dh.abs() + eh)
    want = s * (dh.t() @ x)
    tol = s * (eh.t() @ x.abs() + chain(m) * (dh.abs() + eh).t() @ x.abs())
    tol = tol * 1.01 + half(t) * (want.abs() + tol) + tiny
    assert bool(((d_a.double() - want).abs() <= tol).all())
    # dx: the scaled dH rounded once more; the frozen product; three roundings of the result
    want = d @ w + s * (dh @ a)
    part = (s * (eh + half(t) * (dh.abs() + eh))) @ a.abs() + chain(lora.rank) * s * (dh.abs() @ a.abs())
    once = (half(torch.bfloat16) * 1.01 if compute == nv.BF16 else 2.0 ** -16) if weight.storage == nv.I4 else 0.0
    if compute == nv.F16:
        once = 2 * half(torch.float16) * 1.01
    terms = d.abs() @ w.abs()
    tol = part * 1.01 + (once + chain(weight.out_dim) + S) * terms
    tol = tol + half(t) * ((d @ w).abs() + s * (dh @ a).abs() + want.abs() + 3 * tol) + tiny
    assert bool(((dx.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("storage,dtype,compute", [(orc.I8, torch.bfloat16, nv.F32), (orc.I8, torch.bfloat16, nv.BF16),
                                                   (orc.I4, torch.bfloat16, nv.BF16), (orc.I4, torch.bfloat16, nv.F32),
                                                   (orc.I8, torch.float32, nv.F32), (orc.I4, torch.float32, nv.F32)])
@pytest.mark.parametrize("in_dim,out_dim,m,rank", [(256, 384, 1, 16), (256, 384, 31, 16), (256, 384, 32, 16), (384, 256, 333, 8),
                                                   (512, 128, 1000, 64), (128, 1024, 130, 32), (1024, 1024, 700, 16)])
def test_backward_on_packed_rows(storage, dtype, compute, in_dim, out_dim, m, rank):
    case = make_case(m + rank, storage, dtype, in_dim, out_dim, m, rank)
    check_grads(*case, nv.lora_linear_bwd_packed(case[0], case[1], case[4], case[2], case[3], compute), compute)


@pytest.mark.parametrize("dtype,compute", [(torch.bfloat16, nv.F32), (torch.float32, nv.F32), (torch.float16, nv.F32)])
@pytest.mark.parametrize("in_dim,out_dim,m,rank", [(100, 36, 7, 3), (96, 130, 65, 5), (33, 64, 40, 16), (257, 129, 200, 12)])
def test_backward_on_packed_rows_of_any_width(dtype, compute, in_dim, out_dim, m, rank):
    case = make_case(in_dim, orc.I8, dtype, in_dim, out_dim, m, rank)
    check_grads(*case, nv.lora_linear_bwd_packed(case[0], case[1], case[4], case[2], case[3], compute), compute)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("in_dim,out_dim,m,rank", [(700, 130, 500, 5), (300, 600, 301, 40), (64, 100, 260, 300), (65, 63, 64, 33), (64, 64, 65, 1),
                                                   (2048, 1024, 150, 12), (512, 1030, 30, 64)])
def test_backward_in_general_of_more_rows(dtype, in_dim, out_dim, m, rank):
    case = make_case(in_dim + m, orc.I8, dtype, in_dim, out_dim, m, rank)
    got = nv.lora_linear_bwd_packed(case[0], case[1], case[4], case[2], case[3], nv.F32)
    check_grads(*case, got, nv.F32)
    for a, b in zip(nv.lora_linear_bwd_packed(case[0], case[1], case[4], case[2], case[3], nv.F32), got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("storage,compute", [(orc.I8, nv.F32), (orc.I4, nv.BF16)])
@pytest.mark.parametrize("in_dim,out_dim,m,rank", [(256, 1024, 1024, 16), (128, 1152, 1100, 8), (384, 1280, 2049, 32), (128, 2048, 2048, 8),
                                                   (256, 1024, 4097, 32), (128, 1024, 4095, 16), (128, 1408, 8300, 16), (256, 896, 3000, 16),
                                                   (256, 1024, 2500, 64)])
def test_backward_of_many_rows(storage, compute, in_dim, out_dim, m, rank):
    case = make_case(m + rank, storage, torch.bfloat16, in_dim, out_dim, m, rank)
    ws = torch.full((nv.lora_bwd_packed_workspace_bytes(case[0], case[1], m, compute),), 255, dtype=torch.uint8, device="cuda")
    got = nv.lora_linear_bwd_packed(case[0], case[1], case[4], case[2], case[3], compute, workspace=ws)
    check_grads(*case, got, compute)
    for a, b in zip(nv.lora_linear_bwd_packed(case[0], case[1], case[4], case[2], case[3], compute), got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("m", [32, 100, 127, 128, 300])
def test_backward_rounds_an_expanded_int4_weight_once(m):
    """Rows of one 1 pick rows of the weight: code times scale as bf16."""
    in_dim, out_dim = 1024, 2048
    weight, _, _ = make_weight(np.random.default_rng(m), out_dim, in_dim, orc.I4)
    zero = nv.Lora(torch.zeros(16, in_dim, dtype=torch.bfloat16, device="cuda"),
                   torch.zeros(out_dim, 16, dtype=torch.bfloat16, device="cuda"), 16.0)
    g = torch.Generator(device="cuda").manual_seed(m)
    pick = torch.randint(0, out_dim, (m,), generator=g, device="cuda")
    dy = torch.zeros(m, out_dim, dtype=torch.bfloat16, device="cuda")
    dy[torch.arange(m, device="cuda"), pick] = 1.0
    x = nv.act_pack(torch.randn(m, in_dim, generator=g, device="cuda").bfloat16())
    hidden = torch.zeros(m, 16, dtype=torch.bfloat16, device="cuda")
    dx, _, _ = nv.lora_linear_bwd_packed(weight, zero, dy, x, hidden, nv.BF16)
    assert torch.equal(dx, nv.weight_materialize(weight).float()[pick].bfloat16())


@pytest.mark.parametrize("m", [40, 333, 2500])
@pytest.mark.parametrize("what", ["hidden", "codes", "dy"])
def test_backward_off_a_16_byte_boundary(m, what):
    weight, lora, packed, hidden, dy = make_case(m, orc.I8, torch.bfloat16, 256, 384, m, 16)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    if what == "hidden":
        hidden = shifted(hidden)
    elif what == "codes":
        packed = nv.PackedRows(shifted(packed.codes), shifted(packed.scales))
    else:
        dy = shifted(dy)
    case = (weight, lora, packed, hidden, dy)
    check_grads(*case, nv.lora_linear_bwd_packed(weight, lora, dy, packed, hidden, nv.F32), nv.F32)


def test_backward_beside_the_one_on_full_rows():
    """On rows that eight bits hold, lora_linear_bwd gives the same gradients: dx bit for bit where alpha / rank is a power of
    two, dA and dB to the rounding of sums in another order."""
    weight, lora, packed, hidden, dy = make_case(4, orc.I8, torch.bfloat16, 512, 640, 500, 16, alpha=32.0)
    x = nv.act_unpack(packed)
    got = nv.lora_linear_bwd_packed(weight, lora, dy, packed, hidden)
    want = nv.lora_linear_bwd(weight, lora, dy, x, hidden, expanded=True)
    assert torch.equal(got[0], want[0])
    for g, w in zip(got[1:], want[1:]):
        assert float((g.double() - w.double()).norm()) <= 2 * half(torch.bfloat16) * float(w.double().norm())


def test_backward_repeats_bit_for_bit_and_takes_given_tensors():
    weight, lora, packed, hidden, dy = make_case(5, orc.I4, torch.bfloat16, 512, 640, 900, 16)
    first = nv.lora_linear_bwd_packed(weight, lora, dy, packed, hidden, nv.BF16)
    for _ in range(3):
        again = nv.lora_linear_bwd_packed(weight, lora, dy, packed, hidden, nv.BF16)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
    given = [torch.full_like(t, 9.0) for t in first]
    ws = torch.empty(nv.lora_bwd_packed_workspace_bytes(weight, lora, 900, nv.BF16), dtype=torch.uint8, device="cuda")
    ws.fill_(255)      # scratch holds anything
    got = nv.lora_linear_bwd_packed(weight, lora, dy, packed, hidden, nv.BF16, *given, workspace=ws)
    assert all(g.data_ptr() == t.data_ptr() and torch.equal(g, f) for g, t, f in zip(got, given, first))


def test_backward_no_rows():
    weight, lora, packed, hidden, dy = make_case(6, orc.I8, torch.bfloat16, 128, 256, 4, 16)
    dx, d_a, d_b = nv.lora_linear_bwd_packed(weight, lora, dy[:0], nv.act_pack(torch.empty(0, 128, dtype=torch.bfloat16, device="cuda")),
                                             hidden[:0])
    assert dx.shape == (0, 128) and not bool(d_a.any()) and not bool(d_b.any())


@pytest.mark.parametrize("m", [20, 200])
def test_backward_bad_blocks_stay_with_their_columns(m):
    weight, lora, packed, hidden, dy = make_case(7, orc.I8, torch.bfloat16, 256, 256, m, 16)
    clean = nv.lora_linear_bwd_packed(weight, lora, dy, packed, hidden)
    packed.scales[m // 2, 3] = 255
    packed.codes[m // 2, 96:128] = 0
    got = nv.lora_linear_bwd_packed(weight, lora, dy, packed, hidden)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    assert bool(torch.isnan(got[1][:, 96:128]).all())
    keep = [c for c in range(256) if not 96 <= c < 128]
    assert torch.equal(got[1][:, keep], clean[1][:, keep])


def test_backward_against_differences():
    """<dA, V> against central differences of <dy, x A^T B^T s> along V, which is linear in A, in 64 bits; within the bounds of
    check_grads, summed."""
    weight, lora, packed, hidden, dy = make_case(8, orc.I8, torch.float32, 96, 64, 30, 8)
    dx, d_a, d_b = nv.lora_linear_bwd_packed(weight, lora, dy, packed, hidden)
    g = torch.Generator(device="cuda").manual_seed(8)
    v = torch.randn(lora.a.shape, generator=g, device="cuda").double()
    vx = torch.randn(30, 96, generator=g, device="cuda").double()
    x, b, d = nv.act_unpack(packed, torch.float32).double(), lora.b.double(), dy.double()
    w = nv.weight_materialize(weight).double()
    s = lora.alpha / lora.rank

    def loss(ha, hx):
        z = x + hx * vx
        return float((d * (z @ w.t() + s * (z @ (lora.a.double() + ha * v).t()) @ b.t())).sum())

    h = 1e-3
    size_a = float((s * (d.abs() @ b.abs()).t() @ x.abs() * v.abs()).sum())
    assert abs(float((d_a.double() * v).sum()) - (loss(h, 0) - loss(-h, 0)) / (2 * h)) <= 200 * S * size_a
    size_x = float(((d.abs() @ w.abs() + s * d.abs() @ b.abs() @ lora.a.double().abs()) * vx.abs()).sum())
    assert abs(float((dx.double() * vx).sum()) - (loss(0, h) - loss(0, -h)) / (2 * h)) <= 200 * S * size_x


def test_captured_step():
    weight, lora, packed, hidden, dy = make_case(9, orc.I8, torch.bfloat16, 256, 384, 200, 16)
    x = nv.act_unpack(packed)
    want = nv.lora_linear_bwd_packed(weight, lora, dy, nv.act_pack(x), hidden)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = nv.lora_linear_bwd_packed(weight, lora, dy, nv.act_pack(x), hidden)
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    dy.mul_(-0.5)
    x.mul_(2.0)
    graph.replay()
    want = nv.lora_linear_bwd_packed(weight, lora, dy, nv.act_pack(x), hidden)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_refusals():
    weight, lora, packed, hidden, dy = make_case(10, orc.I8, torch.bfloat16, 128, 128, 40, 16)
    call = nv.lora_linear_bwd_packed
    with pytest.raises(nv.CaifqError, match="hidden has"):
        call(weight, lora, dy, packed, hidden[:39])
    with pytest.raises(nv.CaifqError, match="must be"):
        call(weight, lora, dy.float(), packed, hidden)
    with pytest.raises(nv.CaifqError, match="packed rows"):
        call(weight, lora, dy, nv.act_pack(torch.zeros(39, 128, device="cuda")), hidden)
    with pytest.raises(nv.CaifqError, match="packed rows"):
        call(weight, lora, dy, nv.act_pack(torch.zeros(80, 64, device="cuda")), hidden)
    with pytest.raises(nv.CaifqError, match="overlap"):
        call(weight, lora, dy, packed, hidden, dx=dy)
    with pytest.raises(nv.CaifqError, match="workspace"):
        call(weight, lora, dy, packed, hidden, workspace=torch.empty(100, dtype=torch.uint8, device="cuda"))
    with pytest.raises(nv.CaifqError, match="d_a has"):
        call(weight, lora, dy, packed, hidden, d_a=torch.empty(8, 128, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(nv.CaifqError, match="do not go with"):
        nv.PackedRows(packed.codes, packed.scales[:, :3].contiguous())
    with pytest.raises(nv.CaifqError, match="int8 codes"):
        nv.PackedRows(packed.codes.float(), packed.scales)
    with pytest.raises(nv.CaifqError, match="contiguous"):
        nv.act_pack(torch.zeros(64, 64, device="cuda").t())
    with pytest.raises(nv.CaifqError, match="no CPU fallback"):
        nv.act_pack(torch.zeros(4, 64))
    with pytest.raises(KeyError):
        nv.act_pack(torch.zeros(4, 64, dtype=torch.float64, device="cuda"))
