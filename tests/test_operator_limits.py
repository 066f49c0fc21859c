"""Sizes that the operators around an adapted projection refuse before anything is launched: no GPU needed."""
import ctypes

import pytest

from caif_b200 import native as nv

P = ctypes.c_void_p(4096)      # never read


def refused(rc, text):
    assert rc == 1
    assert text in nv.lib().caifq_last_error().decode()


@pytest.mark.parametrize("in_dim", [2 ** 31 - 1, 2 ** 31 - 512, 2 ** 29 + 1])
def test_bank_of_the_widest_rows(in_dim):
    """A warp steps over a row by up to 512 columns: near 2^31 the step would pass 32 bits and the loop would not end."""
    lib = nv.lib()
    w = nv.CWeight(P, P, nv.I8, 0, 128, in_dim, 64)
    bank, image = nv.CLoraBank(), (nv.CLoraEntry * 1)()
    assert lib.caifq_lora_bank_entries((nv.CLora * 1)(nv.CLora(P, P, nv.F32, 4, 4.0)), 1, in_dim, 64, image, ctypes.byref(bank)) == 0
    bank.entries = 8192
    refused(lib.caifq_lora_bank_linear_fwd(w, bank, P, P, 1, ctypes.c_void_p(1 << 50), ctypes.c_void_p(1 << 51), 1 << 40, nv.F32, None), "features")


@pytest.mark.parametrize("in_dim,out_dim", [(2 ** 31 - 1, 64), (64, 2 ** 31 - 64), (2 ** 29 + 1, 2 ** 29 + 1)])
def test_backward_of_the_widest_rows(in_dim, out_dim):
    lib = nv.lib()
    w = nv.CWeight(P, P, nv.I8, 0, 128, in_dim, out_dim)
    l = nv.CLora(P, P, nv.F32, 4, 4.0)
    refused(lib.caifq_lora_linear_bwd_packed(w, l, P, P, P, P, 1, ctypes.c_void_p(1 << 50), P, P, ctypes.c_void_p(1 << 51), 1 << 40, nv.F32, None), "features")
    # no rows: nothing is summed, but the shape is looked at all the same
    refused(lib.caifq_lora_linear_bwd_packed(w, l, P, P, P, P, 0, P, P, P, P, 0, nv.F32, None), "features")


@pytest.mark.parametrize("rank,dtype,m", [(16, nv.BF16, 16), (64, nv.F32, 300), (24, nv.BF16, 1000), (5, nv.F16, 40)])
def test_workspace_of_the_general_backward(rank, dtype, m):
    """Multiply-adds need dH and the sums over tokens, of as many slices as there are 32 tokens at most, and nothing besides."""
    lib, in_dim, out_dim = nv.lib(), 4096, 14336
    w = nv.CWeight(P, P, nv.I8, 0, 128, in_dim, out_dim)
    got = lib.caifq_lora_bwd_packed_workspace_bytes(w, nv.CLora(P, P, dtype, rank, 4.0), m, nv.F32)
    slices = max(1, min((m + 31) // 32, 888 // ((14336 // 64 + 4096 // 64) * ((rank + 31) // 32))))
    tensor = min((m + 63) // 64, 148 * (4 if rank <= 16 else 2) // ((in_dim + out_dim) // 128))
    assert got <= m * rank * 4 + max(slices, tensor, 1) * (in_dim + out_dim) * rank * 4 + 512
