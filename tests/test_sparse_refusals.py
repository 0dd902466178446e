"""More refusals of the sparse-layer entry points that need no GPU: each comes before any CUDA call."""
import ctypes

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import distspmm_b200 as d
from distspmm_b200._lib import P, c_f32, c_i64, c_vp, dsp_csr


def test_forward_mode_is_refused():
    """A dual tensor has no requires_grad: it would pass as a constant."""
    x = torch.ones(2, 1, 8)
    lists = torch.zeros(3, dtype=torch.int64), torch.zeros(0, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        flat = forward_ad.make_dual(x[:, 0].contiguous(), x[:, 0].contiguous())
        for call in (lambda: d.spmm_act("A", flat), lambda: d.spmm_act("A", x[:, 0], bias=flat), lambda: d.sparse_attention("A", dual, x, x),
                     lambda: d.sparse_attention("A", x, x, dual), lambda: d.sparse_attention_decode(x, dual, x, *lists)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="SparsePattern"):  # plain tensors inside the level are no concern
            d.spmm_act("A", x[:, 0])
    with pytest.raises(ValueError, match="SparsePattern"):
        d.sparse_attention("A", x, x, x)
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(lambda y: d.sparse_attention("A", y, x, x), (x,), (x,))


@pytest.mark.parametrize("nnz,code", [(2 ** 31 - 64, -6), (2 ** 31 - 40, -6), (2 ** 31 - 2, -6), (2 ** 31 - 65, -3), (5, -3)])
def test_entries_near_the_32_bit_limit(nnz, code):
    """A matrix that claims nnz entries: refused for its size where a step from the last ones would pass 2^31, else by validation
    (its row pointer says 0; nothing behind it is read)."""
    ptr, ids, val = np.zeros(1, np.int64), np.zeros(1, np.int64), np.zeros(1, np.float32)
    c = dsp_csr()
    c.num_rows, c.num_cols, c.nnz = 0, 1, nnz
    c.indptr, c.indices, c.values = ptr.ctypes.data_as(P(c_i64)), ids.ctypes.data_as(P(c_i64)), val.ctypes.data_as(P(c_f32))
    h = c_vp()
    assert d.lib().dsp_pattern_create(0, ctypes.byref(c), 0, ctypes.byref(h)) == code


@pytest.mark.parametrize("heads,kv,code", [(65535, 65535, -6), (4096, 1, -6), (1024, 1024, -1)])
def test_more_warps_than_a_grid_has(heads, kv, code):
    """2^21 chunks of 1024 entries for 4096 heads are 2^33 warps: refused, where the count would have been cut to 32 bits. (The last one
    fits, and is refused for its missing workspace.)"""
    from test_sparse_layers import decode_desc, status
    g = decode_desc(heads=heads, kv_heads=kv, nnz=2 ** 31 - 2, keys=5)
    assert status("dsp_attn_decode", ctypes.byref(g), None, 0, None) == code
