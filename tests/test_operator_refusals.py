"""Refusals of the C entry points that need no GPU: a bad call is answered before anything is launched."""
import ctypes

import pytest

from caif_b200 import native as nv

P = ctypes.c_void_p(4096)      # never read: every call here is refused before it touches memory


def refused(rc, text, code=1):
    assert rc == code
    assert text in nv.lib().caifq_last_error().decode()


@pytest.mark.parametrize("rows,dim,dtype,text", [(-1, 8, nv.F32, "bad shape"), (4, 0, nv.F32, "bad shape"),
                                                 (4, 8, nv.I8, "dtype"), (4, 8, nv.F32, "null pointer")])
def test_layernorm(rows, dim, dtype, text):
    lib = nv.lib()
    refused(lib.caifq_layernorm_fwd(None, None, None, None, None, None, 1e-5, dtype, rows, dim, None), text)
    refused(lib.caifq_layernorm_bwd(None, None, None, None, None, None, None, None, 0, None, dtype, rows, dim, None), text)


def test_layernorm_workspace():
    lib = nv.lib()
    refused(lib.caifq_layernorm_bwd(P, P, None, P, P, P, P, None, 0, None, nv.F32, 4, 8, None), "workspace")
    refused(lib.caifq_layernorm_bwd(P, P, None, P, P, P, None, P, 0, ctypes.c_void_p(4100), nv.F32, 4, 8, None), "workspace")
    assert lib.caifq_layernorm_bwd_workspace_bytes(0, 8) == 0
    assert lib.caifq_layernorm_bwd_workspace_bytes(4, 8) >= 4 * 2 * 8 * 4


def lora(a=P, b=P, dtype=nv.BF16, rank=16, alpha=32.0):
    return nv.CLora(a, b, dtype, rank, alpha)


def bank_of(loras, in_dim=128, out_dim=256):
    bank, image = nv.CLoraBank(), (nv.CLoraEntry * max(1, len(loras)))()
    rc = nv.lib().caifq_lora_bank_entries((nv.CLora * max(1, len(loras)))(*loras), len(loras), in_dim, out_dim, image,
                                          ctypes.byref(bank))
    return rc, bank, image


def test_bank_entries():
    rc, bank, image = bank_of([lora(), lora(rank=64, alpha=16.0), lora(rank=8)])
    assert rc == 0 and (bank.count, bank.max_rank, bank.vectors) == (3, 64, 1)
    assert (bank.dtype, bank.in_dim, bank.out_dim) == (nv.BF16, 128, 256)
    assert [(e.rank, e.scale) for e in image] == [(16, 2.0), (64, 0.25), (8, 4.0)] and image[0].a == P.value
    # what 16-byte loads cannot read is marked, not refused
    for other in (lora(rank=12), lora(rank=72), lora(a=4098), lora(b=4104)):
        rc, bank, _ = bank_of([lora(), other])
        assert rc == 0 and bank.vectors == 0
    rc, bank, _ = bank_of([lora(dtype=nv.F32), lora(dtype=nv.F32, rank=1024)])
    assert rc == 0 and bank.vectors == 0 and bank.max_rank == 1024


@pytest.mark.parametrize("loras,text", [([], "no adapters"), ([lora(a=None)], "null"), ([lora(), lora(b=None)], "adapter 1"),
                                        ([lora(rank=0)], "rank 0"), ([lora(rank=1025)], "rank 1025"),
                                        ([lora(dtype=nv.I8)], "dtype"), ([lora(), lora(dtype=nv.F16)], "adapter 1")])
def test_bank_entries_refused(loras, text):
    refused(bank_of(loras)[0], text)


def test_bank_linear():
    lib = nv.lib()
    w = nv.CWeight(P, P, nv.I8, 0, 128, 128, 256)
    _, bank, _ = bank_of([lora()])
    assert lib.caifq_lora_bank_workspace_bytes(w, bank, 0, nv.F32) == 0
    need = lib.caifq_lora_bank_workspace_bytes(w, bank, 20, nv.F32)
    assert need >= 20 * 16 * 4

    def call(w=w, bank=bank, rows=P, x=P, m=20, y=ctypes.c_void_p(1 << 20), ws=ctypes.c_void_p(1 << 21), size=need, compute=nv.F32):
        return lib.caifq_lora_bank_linear_fwd(w, bank, rows, x, m, y, ws, size, compute, None)

    refused(call(), "empty")       # the table is not on a device yet
    bank.entries = 8192
    refused(call(m=-1), "rows")
    refused(call(m=1 << 31), "rows")
    refused(call(compute=nv.I8), "compute dtype")
    refused(call(rows=None), "null")
    refused(call(size=need - 1), "workspace")
    refused(call(ws=ctypes.c_void_p((1 << 21) + 16)), "workspace")
    refused(call(y=P), "overlap")
    refused(call(w=nv.CWeight(P, P, nv.I8, 0, 128, 256, 256)), "the weight has")
    refused(call(w=nv.CWeight(None, P, nv.I8, 0, 128, 128, 256)), "not loaded")
    assert call(m=0) == 0
    bank.out_dim = w.out_dim = 65535 * 64 + 1
    refused(call(), "output features")
    bank.out_dim = w.out_dim = 256
    bank.count = (1 << 24) + 1
    refused(call(), "adapters")
    refused(lib.caifq_lora_bank_entries((nv.CLora * 1)(lora()), (1 << 24) + 1, 128, 256, (nv.CLoraEntry * 1)(), ctypes.byref(bank)),
            "adapters")


@pytest.mark.parametrize("rows,dim,dtype,text", [(-1, 8, nv.F32, "bad shape"), (4, 0, nv.F32, "bad shape"),
                                                 (4, 8, nv.I4, "dtype"), (4, 8, nv.F32, "null pointer")])
def test_pack(rows, dim, dtype, text):
    refused(nv.lib().caifq_act_pack(None, dtype, None, None, rows, dim, None), text)
    refused(nv.lib().caifq_act_unpack(None, None, None, dtype, rows, dim, None), text)


def test_backward_on_packed_rows():
    lib = nv.lib()
    w = nv.CWeight(P, P, nv.I8, 0, 128, 128, 256)
    l = lora()
    need = lib.caifq_lora_bwd_packed_workspace_bytes(w, l, 40, nv.F32)
    sizes = [lib.caifq_lora_bwd_packed_workspace_bytes(w, l, m, nv.F32) for m in (1, 31, 40, 127, 128, 700, 8192)]
    assert sizes == sorted(sizes) and need == sizes[2]
    assert lib.caifq_lora_bwd_packed_workspace_bytes(w, l, 0, nv.F32) == 0

    def call(l=l, dy=P, hidden=P, m=40, dx=ctypes.c_void_p(1 << 20), da=P, ws=ctypes.c_void_p(1 << 21), size=need, compute=nv.F32):
        return lib.caifq_lora_linear_bwd_packed(w, l, dy, P, P, hidden, m, dx, da, P, ws, size, compute, None)

    refused(call(m=-1), "negative")
    refused(call(da=None), "null")
    refused(call(hidden=None), "null")
    refused(call(compute=nv.I4), "compute dtype")
    refused(call(size=need - 1), "workspace")
    refused(call(ws=ctypes.c_void_p((1 << 21) + 8)), "workspace")
    refused(call(dx=P), "overlap")
    refused(call(l=lora(rank=0)), "rank")
