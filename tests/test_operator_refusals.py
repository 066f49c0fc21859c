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
