"""More refusals of the sparse-layer entry points that need no GPU: each comes before any CUDA call."""
import pytest
import torch
from torch.autograd import forward_ad

import distspmm_b200 as d


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
